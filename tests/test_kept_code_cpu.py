"""The code of fp16 layers' kept gate and up products, compiled for the host: every code, and every rounding border."""

import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "triton_grouped_gemm_b200" / "csrc"

# `bad` counts what is not as it should be.  P = 2^-114 is the power of two of the block's largest; allowed errors: half a
# step of 12 mantissa bits above P / 16, of 11 above P / 64, of 10 down to P / 4096, and half that last step below it.
PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <cstring>
#include <initializer_list>
#define __host__
#define __device__
#define __forceinline__ inline
#include "kept_code.cuh"
static uint32_t kept_bits(uint32_t code, uint32_t beside = 0) {   // alone and beside any other code
  auto min2 = [](uint32_t a, uint32_t b) {
    const uint32_t l = (a & 0xFFFF) < (b & 0xFFFF) ? a & 0xFFFF : b & 0xFFFF, h = (a >> 16) < (b >> 16) ? a >> 16 : b >> 16;
    return l | h << 16;
  };
  const uint32_t lo = b200::kept_bits2(code | beside << 16, min2) & 0xFFFF, hi = b200::kept_bits2(beside | code << 16, min2) >> 16;
  return (lo == hi ? lo : 0xFFFFF) << 11;
}
static double value(uint32_t bits) { float f; std::memcpy(&f, &bits, 4); return f; }
static double allowed(double v) {
  const double p = std::ldexp(1.0, -114);
  if (v < p / 4096) v = p / 4096;
  int e;
  std::frexp(v, &e);                               // v in [2^(e-1), 2^e)
  return std::ldexp(1.0, e - 1 - (v >= p / 16 ? 13 : v >= p / 64 ? 12 : 11));
}
int main() {
  long long bad = 0;
  for (uint32_t c = 0; c <= 0x7C00; ++c) {         // every code stands for one value, in rising order
    if (b200::kept_code(kept_bits(c)) != c || kept_bits(c, 0x7FFF) != kept_bits(c) || kept_bits(c, 0x7C00) != kept_bits(c)) ++bad;
    if (c && value(kept_bits(c)) <= value(kept_bits(c - 1))) ++bad;
    if (!c) continue;
    // around the middle between two codes: the nearer one
    const uint32_t lo = kept_bits(c - 1), hi = kept_bits(c), mid = lo + (hi - lo) / 2;
    for (int d = -2; d <= 2; ++d) {
      const uint32_t want = mid + d < lo + (hi - lo + 1) / 2 ? c - 1 : c;
      if (hi - lo > 4 && b200::kept_code(mid + d) != want) ++bad;
    }
  }
  uint32_t last = 0;
  for (uint32_t f = 0; f < (14u << 23); f += 37) {  // errors, over everything a block can hold
    const uint32_t c = b200::kept_code(f);
    const double v = value(f), off = std::fabs(value(kept_bits(c)) - v);
    if (c < last || c > 0x7C00 || off > allowed(v)) ++bad;
    if (off > std::ldexp(v, -13) + std::ldexp(1.0, -114 - 18)) ++bad;   // and the former format's floor
    last = c;
  }
  for (uint32_t f : {0x7F800000u, 0x7F800001u, 0x7FC00000u, 0x7FFFFFFFu})
    if (b200::kept_code(f) != 0x7FFF) ++bad;
  std::printf("%lld\n", bad);
}
"""


def test_every_code_and_border(tmp_path):
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", str(CSRC), str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")], check=True)
    out = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True, check=True).stdout
    assert int(out) == 0
