"""A warp's bounded wait, compiled for the host with 32 threads for its lanes: whichever lanes see the barrier, the abort
flag or the clock first, all of them return, with one answer."""

import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "triton_grouped_gemm_b200" / "csrc"

PROGRAM = r"""
#include <barrier>
#include <cstdint>
#include <cstdio>
#include <functional>
#include <thread>
#include <vector>
#define __device__
#define __forceinline__ inline
static std::barrier<> meet(32);
static thread_local int lane;
static thread_local int looks;                 // at the barrier, so far
static bool vote(bool v, bool any) {
  static int yes[32];
  yes[lane] = v;
  meet.arrive_and_wait();
  int sum = 0;
  for (int i = 0; i < 32; ++i) sum += yes[i];
  meet.arrive_and_wait();
  return any ? sum > 0 : sum == 32;
}
static bool __all_sync(unsigned, bool v) { return vote(v, false); }
static bool __any_sync(unsigned, bool v) { return vote(v, true); }
static std::function<uint64_t()> timer;
static uint64_t global_timer_ns() { return timer(); }
static unsigned atomicOr(unsigned* p, unsigned v) { return __atomic_fetch_or(p, v, __ATOMIC_RELAXED); }
#include "bounded_wait.cuh"

struct Result { int yes = 0, no = 0, flag = 0; unsigned status = 0; };
static Result warp(std::function<bool()> arrived, std::function<uint64_t()> clock, std::function<void(volatile int*)> other = nullptr) {
  timer = clock;
  volatile int flag = 0;
  unsigned status = 0;
  bool got[32];
  std::vector<std::thread> lanes;
  for (int i = 0; i < 32; ++i)
    lanes.emplace_back([&, i] {
      lane = i;
      looks = 0;
      got[i] = b200::wait_together<4>([&] { ++looks; if (other) other(&flag); return arrived(); }, &flag, &status, 2u);
    });
  for (auto& t : lanes) t.join();
  Result r;
  for (bool g : got) g ? ++r.yes : ++r.no;
  r.flag = flag;
  r.status = status;
  return r;
}
static void show(const Result& r) { std::printf("%d %d %d %u\n", r.yes, r.no, r.flag, r.status); }

int main() {
  const uint64_t late = b200::kWaitLimitNs + 1;
  auto still = [] { return uint64_t{0}; };
  show(warp([] { return true; }, still));                                        // there at once
  show(warp([] { return looks > 3 + lane; }, still));                            // seen by one lane after another
  show(warp([] { return false; }, [&] { return looks > 9 ? late : 0; }));        // never: all run out
  show(warp([] { return lane < 16 && looks > 3; }, [&] { return looks > 9 && lane >= 16 ? late : 0; }));  // half arrive, half run out
  show(warp([] { return false; }, [&] { return looks > 9 && lane == 5 ? late : 0; }));                    // one clock ahead
  show(warp([] { return lane != 7; }, still, [](volatile int* f) { if (lane == 7 && looks > 6) *f = 1; }));  // told by another role
}
"""


def test_all_lanes_leave_together(tmp_path):
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", "-I", str(CSRC), str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")],
                   check=True)
    out = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True, check=True, timeout=120).stdout
    rows = [tuple(map(int, line.split())) for line in out.splitlines()]
    assert rows == [(32, 0, 0, 0), (32, 0, 0, 0), (0, 32, 1, 2), (0, 32, 1, 2), (0, 32, 1, 2), (0, 32, 1, 0)]
