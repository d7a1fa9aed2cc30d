// The loop of every bounded wait that a whole warp makes: all lanes leave it together and with one answer.  A lane that
// gave up alone would go on to the block's barrier while the others stand in the next shuffle, vote or __syncwarp, and the
// error would end in a hang.  Success asks for all lanes too, so each of them has seen the phase end (its writes with it).
#pragma once

#include <cstdint>

namespace b200 {

constexpr uint64_t kWaitLimitNs = 2000000000ull;  // 2 s

// arrived(): one look at the barrier.  The clock and the block's abort flag are looked at on every kEvery-th failure (a
// power of two).
template <uint32_t kEvery, typename Arrived>
__device__ __forceinline__ bool wait_together(Arrived&& arrived, volatile int* abort_flag, unsigned* status,
                                              unsigned role_bit) {
  if (__all_sync(0xFFFFFFFFu, arrived())) return true;
  const uint64_t t0 = global_timer_ns();
  uint32_t spins = 0;
  while (!__all_sync(0xFFFFFFFFu, arrived())) {
    if ((++spins & (kEvery - 1)) != 0u) continue;
    const bool told = *abort_flag != 0;
    const bool late = !told && global_timer_ns() - t0 > kWaitLimitNs;
    if (late) {
      *abort_flag = 1;
      if (status) atomicOr(status, role_bit);
    }
    if (__any_sync(0xFFFFFFFFu, told || late)) return false;
  }
  return true;
}

}  // namespace b200
