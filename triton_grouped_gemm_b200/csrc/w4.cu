// M-grouped products with 4-bit weights and group scales, for few rows per expert (decoding):
//
//   c[r, n] = sum_grp scale[g, n, grp] * sum_{k in grp} (q[g, n, k] - zero[g, n, grp]) * a[r, k]
//
// and the gated form act(c_gate) * c_up of a weight tensor that holds gate rows, then up rows.  The work is the
// weights' bytes, N * K / 2 per expert that has a row; the arithmetic only has to keep up with them:
//
//   * a 4-bit value becomes a 16-bit one by OR-ing it into the mantissa of a power of two (128 + q in bf16,
//     1024 + q in fp16) and subtracting 128 + zero (1024 + zero): exact, 1.4 instructions per value.
//   * products run on mma.sync m16n8k16 with the WEIGHTS as the 16-row operand and up to 8 rows of `a` as the
//     8 columns.  tcgen05 has no use here: its smallest tile is 64 rows of `a` or of weights staged through
//     shared memory in 16 bits, four times the bytes that bound this kernel.
//   * q - zero is a whole number, so the products of a group are summed unscaled (fp32) and the scale enters once
//     per group and output: the only rounding is that of the result.
//   * eight neighbouring k of a row are one 32-bit word; the pairs that mask and shift take out of it are (0,4)
//     (1,5) (2,6) (3,7).  The order of k inside a product is free, so `a` is paired the same way (4 byte permutes
//     per 8 values) and the weights stay in their natural order in memory.
//
// A block takes a tile of kWN * 32 weight rows of one expert (gated: half gate, half up rows) and up to kNT * 8 rows
// of `a`.  kWK warps split each 256-wide stage of k; their partial sums are joined in shared memory in a fixed order,
// so results do not depend on timing.  Stages are fetched with 16-byte cp.async, kStages of them in flight.  Blocks
// are persistent over the (expert with rows, row chunk, tile) items; an expert's row chunks are neighbours, so the
// second one finds the weights in L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/b200gemm.h"
#include "activation.cuh"
#include "common.cuh"

namespace b200 {

constexpr int kW4Threads = 256;
constexpr int kW4StageK = 256;        // k per stage: 128 bytes of a weight row
constexpr int kW4RowBytes = 128 + 16; // stage pitch of a weight row: an odd number of 16-byte units, conflict-free
constexpr int kW4ABytes = 512 + 64;   // stage pitch of a row of `a`: 64 modulo 128, conflict-free 16-byte loads
constexpr int kW4WindowGroups = 128;  // scales are staged for this many groups at a time
constexpr int kW4MaxGroups = 1024;    // experts

struct W4Args {
  const uint8_t* a;      // [m_rows, k] 16-bit
  const uint8_t* w;      // [G, weight rows, k / 2]
  const uint8_t* scale;  // [G, weight rows, k / group_size] 16-bit
  const uint8_t* zero;   // same, bytes, or null (zero = 8)
  uint16_t* out;         // [m_rows, n]
  const void* sizes;
  int sizes_i64;
  int num_groups;
  long long m_rows;
  int n, k;
  int log_gs32;          // log2(group_size / 32)
  int act;
  int tiles;             // tiles per expert
  int scale_pitch;       // bytes per row of the staged scales / zeros
  int zero_pitch;
  int list_capacity;     // entries of the list of experts with rows
  unsigned* status;
};

struct W4Expert {
  int g, row0, rows, item0;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

template <bool kFp16>
__device__ __forceinline__ float to_float(uint32_t bits) {
  if constexpr (kFp16) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  return __uint_as_float(bits << 16);
}

// d = a * b + d, a: 16 weight rows x 16 k, b: 16 k x 8 rows of the activations
template <bool kFp16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kFp16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool kFp16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  if constexpr (kFp16) {
    const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  } else {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
}

// magic + zero in both halves: 0x43zz is 128 + zz in bf16 (zz < 128), 0x64zz is 1024 + zz in fp16
template <bool kFp16>
__device__ __forceinline__ uint32_t zero_pair(uint32_t zero) {
  return ((kFp16 ? 0x6400u : 0x4300u) + zero) * 0x10001u;
}

// the four pairs (0,4) (1,5) (2,6) (3,7) of a word of eight 4-bit values, minus their zero
template <bool kFp16>
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t zp, uint32_t (&p)[4]) {
  constexpr uint32_t kMagic = kFp16 ? 0x64006400u : 0x43004300u;
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = sub2<kFp16>(((w >> (4 * i)) & 0x000F000Fu) | kMagic, zp);
}

template <int kWN, int kWK, int kNT, int kStages>
struct W4Smem {
  static constexpr int kRows = kWN * 32;
  static constexpr int kWBytes = kRows * kW4RowBytes;
  static constexpr int kStageBytes = kWBytes + kNT * 8 * kW4ABytes;
  static constexpr int kRedPitch = kNT * 8 + 1;  // floats
  static constexpr int kRedBytes = kWK * kRows * kRedPitch * 4;
  static constexpr int kRing = kStages * kStageBytes > kRedBytes ? kStages * kStageBytes : kRedBytes;
  static_assert(kWN * kWK * 32 == kW4Threads);
  static_assert(kW4StageK / 32 % kWK == 0);
};

template <int kWN, int kWK, int kNT, int kStages, bool kGated, bool kFp16>
__global__ void __launch_bounds__(kW4Threads, 2) w4_m_grouped_kernel(const W4Args p) {
  using L = W4Smem<kWN, kWK, kNT, kStages>;
  constexpr int kBlocks = kW4StageK / 32 / kWK;   // 32-wide k blocks of a stage that one warp multiplies
  constexpr int kOutCols = kGated ? L::kRows / 2 : L::kRows;
  extern __shared__ __align__(128) uint8_t w4_smem[];
  const uint32_t ring = smem_u32(w4_smem);
  const uint32_t scales = ring + L::kRing;
  const uint32_t zeros = scales + L::kRows * p.scale_pitch;
  W4Expert* list = reinterpret_cast<W4Expert*>(w4_smem + L::kRing + L::kRows * (p.scale_pitch + p.zero_pitch));
  __shared__ int s_active, s_items;

  const int tid = threadIdx.x;
  const int warp = tid >> 5, lane = tid & 31;
  const int wn = warp % kWN, wk = warp / kWN;
  const int weight_rows = kGated ? 2 * p.n : p.n;
  const int groups = p.k >> (5 + p.log_gs32);
  const int nblk = p.k >> 5;
  const int stages = (nblk + 7) >> 3;

  // ---- the experts that have rows, in order, by one warp: lane i looks at expert 32 c + i
  if (warp == 0) {
    long long row = 0;   // rows before this chunk of experts
    int active = 0, items = 0;
    bool overflow = false;
    for (int g0 = 0; g0 < p.num_groups; g0 += 32) {
      const int g = g0 + lane;
      long long v = 0;
      if (g < p.num_groups)
        v = p.sizes_i64 ? static_cast<const long long*>(p.sizes)[g]
                        : static_cast<long long>(static_cast<const int*>(p.sizes)[g]);
      if (v < 0) v = 0;
      if (v > p.m_rows) {   // cut off below, like every M-grouped entry point; keeps the sums in range
        v = p.m_rows;
        overflow = true;
      }
      long long end = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xFFFFFFFFu, end, o);
        if (lane >= o) end += up;
      }
      end += row;
      long long begin = end - v;
      if (end > p.m_rows) {
        overflow |= v > 0;
        end = p.m_rows;
        if (begin > p.m_rows) begin = p.m_rows;
      }
      row = __shfl_sync(0xFFFFFFFFu, end, 31);
      const int rows = static_cast<int>(end - begin);
      const unsigned has = __ballot_sync(0xFFFFFFFFu, rows > 0);
      const int mine = rows > 0 ? (rows + kNT * 8 - 1) / (kNT * 8) * p.tiles : 0;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += up;
      }
      if (rows > 0) {
        const int at = active + __popc(has & ((1u << lane) - 1));
        if (at < p.list_capacity) list[at] = {g, static_cast<int>(begin), rows, items + upto - mine};
      }
      active += __popc(has);
      items += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
    if (lane == 0) {
      s_active = active < p.list_capacity ? active : p.list_capacity;
      s_items = items;
    }
    if (__any_sync(0xFFFFFFFFu, overflow) && lane == 0 && blockIdx.x == 0 && p.status) atomicOr(p.status, kDevBadGroupSize);
  }
  __syncthreads();
  const int active = s_active, items = s_items;

  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    int lo = 0, hi = active - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (list[mid].item0 <= item) lo = mid;
      else hi = mid - 1;
    }
    const W4Expert e = list[lo];
    const int chunks = (e.rows + kNT * 8 - 1) / (kNT * 8);
    const int tile = (item - e.item0) / chunks;
    const int chunk = (item - e.item0) - tile * chunks;
    const int row0 = e.row0 + chunk * kNT * 8;
    const int rows = min(kNT * 8, e.rows - chunk * kNT * 8);
    const int nt_used = (rows + 7) >> 3;
    const int n0 = tile * kOutCols;
    // weight row of tile row i: warps own 32 tile rows each; gated: 16 gate rows, then the 16 up rows of the same
    // outputs.  Rows past the end are read from the last one and their results dropped.
    auto weight_row = [&](int i) -> long long {
      long long r;
      if constexpr (kGated) {
        const int col = min(n0 + (i >> 5) * 16 + (i & 15), p.n - 1);
        r = (i & 16) ? p.n + col : col;
      } else {
        r = min(n0 + i, p.n - 1);
      }
      return static_cast<long long>(e.g) * weight_rows + r;
    };

    // this thread's pieces of a stage: weight rows (tid / 8) + 32 i, 16-byte column tid % 8; rows of `a` likewise
    const int w_col = tid & 7;
    const uint8_t* w_src[L::kRows / 32];
#pragma unroll
    for (int i = 0; i < L::kRows / 32; ++i)
      w_src[i] = p.w + weight_row((tid >> 3) + 32 * i) * (p.k >> 1) + w_col * 16;
    const uint8_t* a_src = p.a + static_cast<long long>(row0) * p.k * 2;

    auto fetch = [&](int st) {
      const uint32_t base = ring + (st % kStages) * L::kStageBytes;
      if (st * 8 + w_col < nblk) {
#pragma unroll
        for (int i = 0; i < L::kRows / 32; ++i)
          cp_async16(base + ((tid >> 3) + 32 * i) * kW4RowBytes + w_col * 16, w_src[i] + static_cast<long long>(st) * 128);
      }
      // `a`: 32 16-byte columns per row and stage, a warp per row
      const int col = st * 32 + lane;
      if (col * 8 < p.k) {
        for (int r = warp; r < rows; r += kW4Threads / 32)
          cp_async16(base + L::kWBytes + r * kW4ABytes + lane * 16, a_src + static_cast<long long>(r) * p.k * 2 + col * 16);
      }
    };
    // scales and zeros of the groups [first, first + count) of the tile's rows
    auto fetch_scales = [&](int first) {
      const int count = min(kW4WindowGroups, groups - first);
      for (int r = warp; r < L::kRows; r += kW4Threads / 32) {
        const long long at = weight_row(r) * groups + first;
        const uint8_t* s = p.scale + at * 2;
        const uint32_t d = scales + r * p.scale_pitch;
        if (((reinterpret_cast<uintptr_t>(s) | (count * 2)) & 15) == 0) {
          for (int c = lane; c < count / 8; c += 32) cp_async16(d + c * 16, s + c * 16);
        } else {
          for (int c = lane; c < count; c += 32)
            asm volatile("st.shared.b16 [%0], %1;" ::"r"(d + c * 2), "h"(reinterpret_cast<const uint16_t*>(s)[c]) : "memory");
        }
        if (p.zero) {
          const uint8_t* z = p.zero + at;
          const uint32_t dz = zeros + r * p.zero_pitch;
          if (((reinterpret_cast<uintptr_t>(z) | count) & 15) == 0) {
            for (int c = lane; c < count / 16; c += 32) cp_async16(dz + c * 16, z + c * 16);
          } else {
            for (int c = lane; c < count; c += 32)
              asm volatile("st.shared.u8 [%0], %1;" ::"r"(dz + c), "r"(static_cast<uint32_t>(z[c])) : "memory");
          }
        }
      }
    };

    float acc[2][kNT][4], part[2][kNT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[i][j][v] = part[i][j][v] = 0.f;

#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      if (s < stages) fetch(s);
      if (s == 0) fetch_scales(0);
      cp_async_commit();
    }

    const int lr = lane >> 2, lt = lane & 3;
    int window = 0;  // first group of the staged scales
    uint32_t zp[2][2] = {{zero_pair<kFp16>(8), zero_pair<kFp16>(8)}, {zero_pair<kFp16>(8), zero_pair<kFp16>(8)}};
    for (int st = 0; st < stages; ++st) {
      cp_async_wait<kStages - 2>();
      __syncthreads();   // stage st has landed for everybody, and everybody is done with stage st - 1
      if (const int g = (st * 8) >> p.log_gs32; g - window >= kW4WindowGroups) {
        window = g;
        fetch_scales(g);
        cp_async_commit();
        cp_async_wait<0>();
        __syncthreads();
      }
      if (st + kStages - 1 < stages) fetch(st + kStages - 1);
      cp_async_commit();

      const uint32_t base = ring + (st % kStages) * L::kStageBytes;
      const uint32_t w_row = base + (wn * 32 + lr) * kW4RowBytes + lt * 4;
      const uint32_t a_row = base + L::kWBytes + lr * kW4ABytes + lt * 16;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int in_stage = wk * kBlocks + b;
        const int blk = st * 8 + in_stage;
        if (blk >= nblk) break;
        const int grp = (blk >> p.log_gs32) - window;
        if (p.zero && (b == 0 || (blk & ((1 << p.log_gs32) - 1)) == 0)) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              zp[i][h] = zero_pair<kFp16>(lds8(zeros + (wn * 32 + i * 16 + h * 8 + lr) * p.zero_pitch + grp));
        }
        uint32_t wv[2][2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            unpack_word<kFp16>(lds32(w_row + (i * 16 + h * 8) * kW4RowBytes + in_stage * 16), zp[i][h], wv[i][h]);
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          if (kNT > 1 && j >= nt_used) break;
          const uint4 q = lds128(a_row + j * 8 * kW4ABytes + in_stage * 64);
          const uint32_t x04 = __byte_perm(q.x, q.z, 0x5410), x15 = __byte_perm(q.x, q.z, 0x7632);
          const uint32_t x26 = __byte_perm(q.y, q.w, 0x5410), x37 = __byte_perm(q.y, q.w, 0x7632);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t f0[4] = {wv[i][0][0], wv[i][1][0], wv[i][0][1], wv[i][1][1]};
            const uint32_t f1[4] = {wv[i][0][2], wv[i][1][2], wv[i][0][3], wv[i][1][3]};
            mma_16816<kFp16>(part[i][j], f0, x04, x15);
            mma_16816<kFp16>(part[i][j], f1, x26, x37);
          }
        }
        // the last block of a group, or of what this warp has of it: the scale enters
        if (b == kBlocks - 1 || blk + 1 == nblk || ((blk + 1) & ((1 << p.log_gs32) - 1)) == 0) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t sa = scales + (wn * 32 + i * 16 + lr) * p.scale_pitch + grp * 2;
            const float s0 = to_float<kFp16>(lds16(sa)), s1 = to_float<kFp16>(lds16(sa + 8 * p.scale_pitch));
#pragma unroll
            for (int j = 0; j < kNT; ++j) {
              if (kNT > 1 && j >= nt_used) break;
              acc[i][j][0] = fmaf(s0, part[i][j][0], acc[i][j][0]);
              acc[i][j][1] = fmaf(s0, part[i][j][1], acc[i][j][1]);
              acc[i][j][2] = fmaf(s1, part[i][j][2], acc[i][j][2]);
              acc[i][j][3] = fmaf(s1, part[i][j][3], acc[i][j][3]);
#pragma unroll
              for (int v = 0; v < 4; ++v) part[i][j][v] = 0.f;
            }
          }
        }
      }
    }

    // ---- join the kWK partial sums (in order) and store
    cp_async_wait<0>();
    __syncthreads();
    float* red = reinterpret_cast<float*>(w4_smem);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        if (kNT > 1 && j >= nt_used) break;
        float* d = red + ((wk * kWN + wn) * 32 + i * 16 + lr) * L::kRedPitch + j * 8 + lt * 2;
        d[0] = acc[i][j][0];
        d[1] = acc[i][j][1];
        d[8 * L::kRedPitch] = acc[i][j][2];
        d[8 * L::kRedPitch + 1] = acc[i][j][3];
      }
    __syncthreads();
    for (int o = tid; o < kOutCols * rows; o += kW4Threads) {
      const int r = o / kOutCols;          // a power of two: a shift
      const int c = o - r * kOutCols;
      if (n0 + c >= p.n) continue;
      auto joined = [&](int tile_row) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kWK; ++i) s += red[(i * L::kRows + tile_row) * L::kRedPitch + r];
        return s;
      };
      float v;
      if constexpr (kGated) {
        const int tr = (c >> 4) * 32 + (c & 15);
        v = gate_value(joined(tr), p.act) * joined(tr + 16);
      } else {
        v = joined(c);
      }
      uint16_t bits;
      if constexpr (kFp16) bits = __half_as_ushort(__float2half_rn(v));
      else bits = __bfloat16_as_ushort(__float2bfloat16_rn(v));
      p.out[static_cast<long long>(row0 + r) * p.n + n0 + c] = bits;
    }
    __syncthreads();  // the ring and the staged scales are free again
  }
}

// ------------------------------------------------------------------ quantiser
// One warp per 32 * kPer-element group: min / max by shuffles, then every lane packs kPer values.  Symmetric:
// scale = max|w| / 7, q = clamp(round(w / scale) + 8).  Asymmetric: scale = (max(w,0) - min(w,0)) / 15,
// zero = round(-min / scale), q = clamp(round(w / scale) + zero).  Scales are rounded to the weights' type first and
// that rounded scale is what the values are divided by; a group of zeros has scale 0.  Bound by HBM bytes; run once.
template <int kPer, bool kFp16>
__global__ void __launch_bounds__(256)
w4_quant_kernel(const uint16_t* __restrict__ w, uint8_t* __restrict__ q, uint16_t* __restrict__ scale,
                uint8_t* __restrict__ zero, long long num_groups) {
  constexpr int kLanes = 16;             // lanes per group: 2 values per lane at group size 32
  constexpr int kVals = kPer;            // values per lane, a multiple of 2
  const int lane = threadIdx.x & 31;
  const int sub = lane & (kLanes - 1);
  const long long stride = static_cast<long long>(gridDim.x) * (256 / kLanes);
  for (long long g0 = static_cast<long long>(blockIdx.x) * (256 / kLanes); g0 < num_groups; g0 += stride) {
    const long long g = g0 + threadIdx.x / kLanes;
    const bool ok = g < num_groups;      // every lane stays for the shuffles
    float v[kVals];
    const uint16_t* src = w + g * (kLanes * kVals) + sub * kVals;
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int i = 0; i < kVals; ++i) {
      v[i] = ok ? to_float<kFp16>(src[i]) : 0.f;
      lo = fminf(lo, v[i]);
      hi = fmaxf(hi, v[i]);
    }
#pragma unroll
    for (int o = kLanes / 2; o >= 1; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
    if (!ok) continue;
    const float exact = zero ? __fdiv_rn(hi - lo, 15.f) : __fdiv_rn(fmaxf(hi, -lo), 7.f);
    uint16_t sbits;
    if constexpr (kFp16) sbits = __half_as_ushort(__float2half_rn(exact));
    else sbits = __bfloat16_as_ushort(__float2bfloat16_rn(exact));
    const float s = to_float<kFp16>(sbits);
    float z = 8.f;
    if (zero) z = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.f), 15.f) : 0.f;
#pragma unroll
    for (int i = 0; i < kVals; i += 2) {
      unsigned byte = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float t = s > 0.f ? rintf(__fdiv_rn(v[i + h], s)) + z : z;
        byte |= static_cast<unsigned>(fminf(fmaxf(t, 0.f), 15.f)) << (4 * h);
      }
      q[(g * (kLanes * kVals) + sub * kVals + i) >> 1] = static_cast<uint8_t>(byte);
    }
    if (sub == 0) {
      scale[g] = sbits;
      if (zero) zero[g] = static_cast<uint8_t>(z);
    }
  }
}

// ------------------------------------------------------------------ host side
template <int kWN, int kWK, int kNT, int kStages, bool kGated, bool kFp16>
static int launch_w4(W4Args p, int want_sms, cudaStream_t stream) {
  using L = W4Smem<kWN, kWK, kNT, kStages>;
  auto kern = w4_m_grouped_kernel<kWN, kWK, kNT, kStages, kGated, kFp16>;
  constexpr int kOutCols = kGated ? L::kRows / 2 : L::kRows;
  p.tiles = (p.n + kOutCols - 1) / kOutCols;
  const int smem = L::kRing + L::kRows * (p.scale_pitch + p.zero_pitch) +
                   p.list_capacity * static_cast<int>(sizeof(W4Expert));
  B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int per_sm = 2 * (smem + 2048) <= 228 * 1024 ? 2 : 1;  // the registers allow two
  // at most this many items: every expert with rows has one partial chunk at most
  const long long chunks = p.m_rows / (kNT * 8) + (p.m_rows < p.num_groups ? p.m_rows : p.num_groups);
  const long long items = chunks * p.tiles;
  B200_REQUIRE(items < (1ll << 31), "b200gemm_w4_m_grouped: too many rows and columns for one call");
  const long long resident = static_cast<long long>(per_sm) * want_sms;
  kern<<<static_cast<unsigned>(items < resident ? items : resident), kW4Threads, smem, stream>>>(p);
  B200_CUDA(cudaGetLastError());
  return 0;
}

static int w4_m_grouped(const void* a, const void* w4, const void* scale, const void* zero, void* out, const void* sizes,
                        int sizes_is_i64, int num_groups, int64_t m_rows, int n, int k, int group_size, int gated,
                        int act, int dtype, int num_sms, cudaStream_t stream) {
  const char* who = "b200gemm_w4_m_grouped";
  B200_REQUIRE(dtype == 0 || dtype == 1, "%s: dtype must be 0 (bf16) or 1 (fp16), got %d", who, dtype);
  B200_REQUIRE(num_groups >= 0 && m_rows >= 0 && n >= 0 && k >= 0, "%s: negative dimension", who);
  B200_REQUIRE(group_size == 32 || group_size == 64 || group_size == 128, "%s: group_size must be 32, 64 or 128, got %d",
               who, group_size);
  B200_REQUIRE(k % group_size == 0, "%s: k must be a multiple of the group size (k=%d, group_size=%d)", who, k, group_size);
  B200_REQUIRE(!gated || (act >= 0 && act < kNumActivations), "%s: unknown activation %d", who, act);
  B200_REQUIRE(num_groups <= kW4MaxGroups, "%s: at most %d groups, got %d", who, kW4MaxGroups, num_groups);
  if (num_groups == 0 || m_rows == 0 || n == 0) return 0;
  B200_REQUIRE(k > 0, "%s: k must be positive", who);
  B200_REQUIRE(a && w4 && scale && out && sizes, "%s: null pointer", who);
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w4)) & 15) == 0,
               "%s: a and w4 must be 16-byte aligned", who);
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(scale) | reinterpret_cast<uintptr_t>(out)) & 1) == 0,
               "%s: scale and out must be 2-byte aligned", who);
  B200_REQUIRE(m_rows < (1ll << 31) && n < (1 << 30), "%s: m_rows and n must fit in int32", who);
  const int sms = sm_count();
  B200_REQUIRE(sms > 0, "%s: no CUDA device", who);
  W4Args p = {};
  p.a = static_cast<const uint8_t*>(a);
  p.w = static_cast<const uint8_t*>(w4);
  p.scale = static_cast<const uint8_t*>(scale);
  p.zero = static_cast<const uint8_t*>(zero);
  p.out = static_cast<uint16_t*>(out);
  p.sizes = sizes;
  p.sizes_i64 = sizes_is_i64;
  p.num_groups = num_groups;
  p.m_rows = m_rows;
  p.n = n;
  p.k = k;
  p.log_gs32 = group_size == 32 ? 0 : group_size == 64 ? 1 : 2;
  p.act = act;
  const int groups = k / group_size;
  const int window = groups < kW4WindowGroups ? groups : kW4WindowGroups;
  p.scale_pitch = ((window * 2 + 15) / 16 | 1) * 16;   // an odd number of 16-byte units: 8 rows, 8 different banks
  p.zero_pitch = zero ? ((window + 15) / 16 | 1) * 16 : 0;
  p.list_capacity = static_cast<int>(m_rows < num_groups ? m_rows : num_groups);
  p.status = device_status_ptr();
  const int want = num_sms > 0 && num_sms < sms ? num_sms : sms;
#define B200_W4(WN, WK, NT, ST)                                                          \
  (gated ? (dtype ? launch_w4<WN, WK, NT, ST, true, true>(p, want, stream)               \
                  : launch_w4<WN, WK, NT, ST, true, false>(p, want, stream))             \
         : (dtype ? launch_w4<WN, WK, NT, ST, false, true>(p, want, stream)              \
                  : launch_w4<WN, WK, NT, ST, false, false>(p, want, stream)))
  if (m_rows <= 8) return B200_W4(2, 4, 1, 4);
  return B200_W4(4, 2, 4, 3);
#undef B200_W4
}

static int w4_quant(const void* w, void* q, void* scale, void* zero, int64_t rows, int k, int group_size, int dtype,
                    cudaStream_t stream) {
  const char* who = "b200quant_w4_group";
  B200_REQUIRE(dtype == 0 || dtype == 1, "%s: dtype must be 0 (bf16) or 1 (fp16), got %d", who, dtype);
  B200_REQUIRE(rows >= 0 && k >= 0, "%s: negative dimension", who);
  B200_REQUIRE(group_size == 32 || group_size == 64 || group_size == 128, "%s: group_size must be 32, 64 or 128, got %d",
               who, group_size);
  B200_REQUIRE(k % group_size == 0, "%s: k must be a multiple of the group size (k=%d, group_size=%d)", who, k, group_size);
  if (rows == 0 || k == 0) return 0;
  B200_REQUIRE(w && q && scale, "%s: null pointer", who);
  const int sms = sm_count();
  B200_REQUIRE(sms > 0, "%s: no CUDA device", who);
  const long long groups = rows * (k / group_size);
  const long long blocks = (groups + 15) / 16;
  const unsigned grid = static_cast<unsigned>(blocks < 32ll * sms ? blocks : 32ll * sms);
  auto kern = dtype ? (group_size == 32 ? w4_quant_kernel<2, true> : group_size == 64 ? w4_quant_kernel<4, true> : w4_quant_kernel<8, true>)
                    : (group_size == 32 ? w4_quant_kernel<2, false> : group_size == 64 ? w4_quant_kernel<4, false> : w4_quant_kernel<8, false>);
  kern<<<grid, 256, 0, stream>>>(static_cast<const uint16_t*>(w), static_cast<uint8_t*>(q), static_cast<uint16_t*>(scale),
                                 static_cast<uint8_t*>(zero), groups);
  B200_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace b200

extern "C" {

int b200gemm_w4_m_grouped(const void* a, const void* w4, const void* scale, const void* zero, void* out,
                          const void* sizes, int sizes_is_i64, int num_groups, int64_t m_rows, int n, int k,
                          int group_size, int gated, int act, int dtype, int num_sms, void* stream) {
  return b200::w4_m_grouped(a, w4, scale, zero, out, sizes, sizes_is_i64, num_groups, m_rows, n, k, group_size, gated, act,
                            dtype, num_sms, static_cast<cudaStream_t>(stream));
}

int b200quant_w4_group(const void* w, void* q, void* scale, void* zero, int64_t rows, int k, int group_size, int dtype,
                       void* stream) {
  return b200::w4_quant(w, q, scale, zero, rows, k, group_size, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
