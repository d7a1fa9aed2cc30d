// The 16-bit code in which layers of fp16 keep a gate or up product for the gradient: sign and 15 bits for a magnitude
// relative to the largest of its block, more of them mantissa the nearer it is to that.  Integer arithmetic on the bits
// of a non-negative fp32 number f that is scaled so that the block's largest has exponent field 13:
//
//   exponent field of f    below the largest    mantissa bits    codes
//   9 .. 13                2^0  .. 2^-4         12               0x2C00 .. 0x7BFF (0x7C00: rounded up to field 14)
//   7, 8                   2^-5, 2^-6           11               0x1C00 .. 0x2BFF
//   0 .. 6                 2^-7 and less        10               0x0000 .. 0x1BFF, field 0 being fp32's denormals
//
// So a value is off by at most 2^-13 of itself near the largest, by 2^-11 (as plain fp16) down to 2^-12 of the largest's
// power of two, and by 2^-23 of that power below.  The code is a rising, convex function of f's bits made of three straight
// lines, so it is the largest of the three.  The way back rises by 4, 2 and 1 steps of f >> 11 per code, which fit into 16
// bits: two codes are taken back at once.  0x7FFF: f was not finite.
#pragma once

#include <cstdint>

namespace b200 {

constexpr int kKeptTop = 13;                                   // exponent field of a block's largest
constexpr uint32_t kKeptMidCode = 7u << 10;                    // first code of 11 and of 12 mantissa bits
constexpr uint32_t kKeptHighCode = 11u << 10;
constexpr uint32_t kKeptMid = 7u << 10;                        // code = f >> 13, (f >> 12) - kKeptMid,
constexpr uint32_t kKeptHigh = (9u << 12) - kKeptHighCode;     // (f >> 11) - kKeptHigh

__host__ __device__ __forceinline__ uint32_t kept_code(uint32_t f) {
  // half a step added (ties away from zero), the offset taken off before the shift; what wraps or is below its line is
  // negative and loses
  const int low = static_cast<int>(f + (1u << 12)) >> 13;
  const int mid = static_cast<int>(f + (1u << 11) - (kKeptMid << 12)) >> 12;
  const int high = static_cast<int>(f + (1u << 10) - (kKeptHigh << 11)) >> 11;
  const int most = low > mid ? low : mid;
  const int code = most > high ? most : high;
  return static_cast<uint32_t>(code < 0x7FFF ? code : 0x7FFF);
}

// both halves' f >> 11 from two codes below 0x7FFF; min2: the smaller of each half
template <typename Min2>
__host__ __device__ __forceinline__ uint32_t kept_bits2(uint32_t codes, Min2&& min2) {
  return codes + min2(codes, kKeptHighCode * 0x10001u) + 2u * min2(codes, kKeptMidCode * 0x10001u);
}

}  // namespace b200
