// M-grouped products with 4-bit weights and group scales, for few rows per expert (decoding):
//
//   c[r, n] = sum_grp scale[g, n, grp] * sum_{k in grp} (q[g, n, k] - zero[g, n, grp]) * a[r, k]
//
// and the gated form act(c_gate) * c_up of a weight tensor that holds gate rows, then up rows.  The work is the
// weights' bytes, N * K / 2 per expert that has a row; the arithmetic only has to keep up with them:
//
//   * a 4-bit value becomes a 16-bit one by OR-ing it into the mantissa of a power of two (128 + q in bf16,
//     1024 + q in fp16) and subtracting 128 + zero (1024 + zero): exact, 1.4 instructions per value (fp16: 1.1).  The
//     method is published: Kim, Henry, Fahim, Awadalla, "Who Says Elephants Can't Run: Bringing Large Scale MoE Models into
//     Cloud Scale Production", 2022; the constants follow from the two number formats.
//   * products run on mma.sync m16n8k16 with the WEIGHTS as the 16-row operand and up to 8 rows of `a` as the
//     8 columns.  tcgen05 wants the weights in 16 bits in shared memory (four times the bytes that bound this kernel)
//     or in tensor memory.  The latter was built - 128 weight rows unpacked into tensor memory by two warpgroups,
//     16 or 48 rows of `a`, a group's sums read back, scaled and added up by a third - and was slower: the three
//     hand-overs per 128 k take 0.8 us where this takes 0.3 (first case below 172 us against 113; 36 rows per expert,
//     groups of 32: 82 against 84).
//   * q - zero is a whole number, so the products of a group are summed unscaled (fp32) and the scale enters once
//     per group and output: the only rounding is that of the result.
//   * eight neighbouring k of a row are one 32-bit word; the pairs that mask and shift take out of it are (0,4)
//     (1,5) (2,6) (3,7).  The order of k inside a product is free, so `a` is paired the same way (4 byte permutes
//     per 8 values) and the weights stay in their natural order in memory.
//
// A block takes a tile of kWN * 32 weight rows of one expert (gated: half gate, half up rows) and up to kNT * 8 rows
// of `a`.  kWK warps split each stage of kSB * 32 k; their partial sums are joined in a fixed order, so results do not
// depend on timing.  Blocks are persistent over the (expert with rows, tile, row chunk) items; an expert's row chunks
// are neighbours, so the second one finds the weights in L2.  Of four further warps one fetches the stages by TMA and
// three the scales, all running ahead across the items' borders, so a block never drains, and the multiplying warps
// meet only to join their sums.  The 128-byte swizzle makes both operands' fragment loads free of bank conflicts (rows
// of `a` are taken in the order 0 4 1 5 2 6 3 7 for that).
//
// What bounds it now is issue: per 32 x 32 weights some 24 (bf16: 32) instructions of the half-rate logic pipe, 20 of
// the others, and as many again around them.  Measured (time, share of the floor of the weights' bytes at the copy
// bandwidth): 256 rows over 112 of 128 experts, gated, K 4096, 1024 + 1024 columns, fp16 with zeros 109 us, 0.69; the
// same in bf16 116 us, with zeros 121 us, 0.62; 256 rows, K 768, 2048 columns, groups of 64 with zeros 38 us, 0.39; one token's eight
// experts, K 2048, 768 + 768 columns 10 us a launch, of which 1 us is the walk over the sizes, 1-2 the first bytes'
// way, 3 the products and the rest the launch.  Each stage and warp has a fixed cost of about two blocks of 32 x 32, so
// a warp gets 8 (kNT = 2: 4) of a stage: the first case took 174 us at 2 of them, 115 at 4; 16 warps in one block
// per SM took 121, 64 rows per warp spilled.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/b200gemm.h"
#include "activation.cuh"
#include "common.cuh"

namespace b200 {

constexpr int kW4WindowGroups = 16;   // scales are staged for this many groups at a time
constexpr int kW4ScalePitch = 48;     // bytes per row of the staged scales / zeros: odd numbers of 16-byte units,
constexpr int kW4ZeroPitch = 16;      // so that 8 rows lie in 8 different banks
constexpr int kW4MaxGroups = 1024;    // experts

struct W4Args {
  const uint8_t* scale;  // [G, weight rows, k / group_size] 16-bit
  const uint8_t* zero;   // same, bytes, or null (zero = 8)
  uint16_t* out;         // [m_rows, n]
  const void* sizes;
  int sizes_i64;
  int num_groups;
  long long m_rows;
  int n, k;
  int act;
  int a_boxes;           // TMA boxes of `a` per stage: 1 where k is a multiple of 64, else one per 64 k
  int tiles;             // tiles per expert
  int log_scale_piece;   // log2 bytes of the pieces that scales / zeros are copied in: 16 where every row's begin is
  int log_zero_piece;    // aligned to that, down to one element
  int log_scale_pieces;  // log2 of the pieces per staged row, rounded up to a power of two
  int log_zero_pieces;
  int list_capacity;     // entries of the list of experts with rows
  unsigned* status;
};

struct W4Expert {
  int g, row0, rows, item0;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// this thread's arrival on `bar` once its copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <bool kFp16>
__device__ __forceinline__ float to_float(uint32_t bits) {
  if constexpr (kFp16) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  return __uint_as_float(bits << 16);
}

// d = a * b + c, a: 16 weight rows x 16 k, b: 16 k x 8 rows of the activations; kFirst: c = 0
template <bool kFp16, bool kFirst>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  const float c0 = kFirst ? 0.f : d[0], c1 = kFirst ? 0.f : d[1], c2 = kFirst ? 0.f : d[2], c3 = kFirst ? 0.f : d[3];
  if constexpr (kFp16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// (w & mask) | magic in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}

// magic + zero in both halves: 0x43zz is 128 + zz in bf16 (zz < 128), 0x64zz is 1024 + zz in fp16.  Zeros are 0 .. 15 by
// contract; beyond 127 the bf16 sum would need a ninth bit.
template <bool kFp16>
__device__ __forceinline__ uint32_t zero_pair(uint32_t zero) {
  return ((kFp16 ? 0x6400u : 0x4300u) + zero) * 0x10001u;
}

// the four pairs (0,4) (1,5) (2,6) (3,7) of a word of eight 4-bit values, minus their zero.  In fp16 the values at
// bits 4..7 need no shift: 1024 + 16 q, times 1/16, minus 64 + zero, in one exact multiply-add (bf16's 7 mantissa bits
// end below bit 7).
template <bool kFp16>
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t zp, uint32_t (&p)[4]) {
  if constexpr (kFp16) {
    const __half2 z = *reinterpret_cast<__half2*>(&zp);
    const __half2 z16 = __hsub2(__half2half2(__float2half_rn(960.f)), z);  // -(64 + zero) = 960 - (1024 + zero)
    const uint32_t w8 = w >> 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = and_or(i ? w8 : w, 0x000F000Fu, 0x64006400u), hi = and_or(i ? w8 : w, 0x00F000F0u, 0x64006400u);
      const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), z);
      const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), __half2half2(__float2half_rn(0.0625f)), z16);
      p[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
      p[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t q = and_or(w >> (4 * i), 0x000F000Fu, 0x43004300u);
      const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&q), *reinterpret_cast<__nv_bfloat162*>(&zp));
      p[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
}

template <int kWN, int kWK, int kNT, int kStages, int kSB>
struct W4Smem {
  static constexpr int kWarps = kWN * kWK;         // that multiply; one more fetches stages, three fetch scales
  static constexpr int kScaleWarps = 3;
  static constexpr int kThreads = (kWarps + 1 + kScaleWarps) * 32;
  // Registers of the forms with two blocks per SM: a launch of 384 threads has 80 each; the fetching warpgroup hands
  // some of its share to the two that multiply.  setmaxnreg.inc waits for registers that must exist in the block's own
  // allocation, so the shares may not add up to more than the launch's.
  static constexpr bool kRebalance = kWN > 1;
  static constexpr int kRegs = 80, kRegsFetch = 48, kRegsMultiply = 96;
  static_assert(kWarps == 8 && kThreads == 384 && 128 * kRegsFetch + 256 * kRegsMultiply <= 384 * kRegs);
  static constexpr int kRows = kWN * 32;
  static constexpr int kScaleBytes = kRows * kW4ScalePitch;
  static constexpr int kStagedBytes = kRows * (kW4ScalePitch + kW4ZeroPitch);
  static constexpr int kWBytes = kRows * kSB * 16;
  static constexpr int kStageBytes = kWBytes + kNT * 8 * kSB * 64;
  static constexpr int kRedFloats = (kWK - 1) * kWN * 32 * 2 * kNT * 4;   // two buffers of them
  static constexpr int kBarOffset = kStages * kStageBytes + 2 * kRedFloats * 4;
  static constexpr int kBars = 2 * kStages + 4;
  static constexpr int kScaleOffset = kBarOffset + (kBars * 8 + 15) / 16 * 16;
  static_assert(kSB % 8 == 0 && kSB % (2 * kWK) == 0 && kStageBytes % 1024 == 0);
};

template <int kWN, int kWK, int kNT, int kStages, int kSB, int kLogGs, bool kGated, bool kFp16, bool kZero>
__global__ void __launch_bounds__(kWN * kWK * 32 + 128, kNT > 1 || kWN > 1 ? 2 : 3)
w4_m_grouped_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const W4Args p) {
  using L = W4Smem<kWN, kWK, kNT, kStages, kSB>;
  constexpr int kBlocks = kSB / kWK;                // 32-wide k blocks of a stage that one warp multiplies
  constexpr int kPer = (1 << kLogGs) < kBlocks ? (1 << kLogGs) : kBlocks;   // of them under one scale
  constexpr int kOutCols = kGated ? L::kRows / 2 : L::kRows;
  constexpr int kWindowStages = kW4WindowGroups * (1 << kLogGs) / kSB;      // stages that share a window of scales
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem_base = smem_u32(smem);
  auto full_bar = [&](int s) { return smem_base + L::kBarOffset + 8u * s; };
  auto empty_bar = [&](int s) { return smem_base + L::kBarOffset + 8u * (kStages + s); };
  auto scale_full_bar = [&](int b) { return smem_base + L::kBarOffset + 8u * (2 * kStages + b); };
  auto scale_empty_bar = [&](int b) { return smem_base + L::kBarOffset + 8u * (2 * kStages + 2 + b); };
  uint8_t* const staged = smem + L::kScaleOffset;   // two buffers of scales and zeros
  W4Expert* const list = reinterpret_cast<W4Expert*>(staged + 2 * L::kStagedBytes);
  __shared__ int s_active, s_items, s_abort;

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
  const int weight_rows = kGated ? 2 * p.n : p.n;
  const int groups = p.k >> (5 + kLogGs);
  const int nblk = p.k >> 5;
  const int stages = (nblk + kSB - 1) / kSB;

  if (tid == 32) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), L::kWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(scale_full_bar(b), 32 * L::kScaleWarps);
      mbar_init(scale_empty_bar(b), L::kWarps);
    }
    s_abort = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_a);
  }

  chain_wait();
  // ---- the experts that have rows, in order, by one warp: lane i looks at experts 128 c + 4 i .. + 3
  if (warp == 0) {
    long long row = 0;   // rows before this chunk of experts
    int active = 0, items = 0;
    bool overflow = false;
    for (int g0 = 0; g0 < p.num_groups; g0 += 128) {
      long long end[4];    // after each of the lane's experts, counted from the lane's first
      long long sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int g = g0 + lane * 4 + i;
        long long v = 0;
        if (g < p.num_groups)
          v = p.sizes_i64 ? static_cast<const long long*>(p.sizes)[g]
                          : static_cast<long long>(static_cast<const int*>(p.sizes)[g]);
        end[i] = v;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (end[i] < 0) end[i] = 0;
        if (end[i] > p.m_rows) {   // cut off below, like every M-grouped entry point; keeps the sums in range
          end[i] = p.m_rows;
          overflow = true;
        }
        end[i] = sum += end[i];
      }
      long long before = sum;      // becomes the rows up to and including this lane's experts
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xFFFFFFFFu, before, o);
        if (lane >= o) before += up;
      }
      before += row - sum;
      int begin[4], rows[4], work[4], mine_active = 0, mine_items = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long lo = before + (i ? end[i - 1] : 0), hi = before + end[i];
        overflow |= hi > p.m_rows && hi > lo;
        begin[i] = static_cast<int>(lo < p.m_rows ? lo : p.m_rows);
        rows[i] = static_cast<int>(hi < p.m_rows ? hi : p.m_rows) - begin[i];
        work[i] = (rows[i] + kNT * 8 - 1) / (kNT * 8) * p.tiles;
        mine_active += rows[i] > 0;
        mine_items += work[i];
      }
      row = __shfl_sync(0xFFFFFFFFu, before + sum, 31);
      if (row > p.m_rows) row = p.m_rows;
      int upto_active = mine_active, upto_items = mine_items;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xFFFFFFFFu, upto_active, o), b = __shfl_up_sync(0xFFFFFFFFu, upto_items, o);
        if (lane >= o) {
          upto_active += a;
          upto_items += b;
        }
      }
      int at = active + upto_active - mine_active, item0 = items + upto_items - mine_items;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (rows[i] > 0) {
          if (at < p.list_capacity) list[at] = {g0 + lane * 4 + i, begin[i], rows[i], item0};
          ++at;
          item0 += work[i];
        }
      }
      active += __shfl_sync(0xFFFFFFFFu, upto_active, 31);
      items += __shfl_sync(0xFFFFFFFFu, upto_items, 31);
    }
    if (lane == 0) {
      s_active = active < p.list_capacity ? active : p.list_capacity;
      s_items = items;
    }
    if (__any_sync(0xFFFFFFFFu, overflow) && lane == 0 && blockIdx.x == 0 && p.status) atomicOr(p.status, kDevBadGroupSize);
  }
  __syncthreads();
  const int active = s_active, items = s_items;

  struct Item {
    int g, row0, rows, n0;
  };
  // Item by item, in rising order and by a whole warp: `at` is the list entry of the last one, and a vote finds how many
  // entries further the next one's is.
  auto item_at = [&](int item, int& at) {
    for (;;) {
      const int i = at + 1 + lane;
      const int step = __popc(__ballot_sync(0xFFFFFFFFu, i < active && list[i < active ? i : 0].item0 <= item));
      at += step;
      if (step < 32) break;
    }
    const W4Expert e = list[at];
    const int chunks = (e.rows + kNT * 8 - 1) / (kNT * 8);
    int tile = item - e.item0, chunk = 0;
    if (chunks > 1) {
      const int q = tile / chunks;
      chunk = tile - q * chunks;
      tile = q;
    }
    return Item{e.g, e.row0 + chunk * kNT * 8, min(kNT * 8, e.rows - chunk * kNT * 8), tile * kOutCols};
  };
  int at = 0;   // every warp walks the list on its own

  if constexpr (L::kRebalance) {
    if (warp >= L::kWarps) warpgroup_reg_dec<L::kRegsFetch>();
    else warpgroup_reg_inc<L::kRegsMultiply>();
  }
  if (warp == L::kWarps) {
    // ---- the stages of this block's items, by one thread
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const Item it = item_at(item, at);
      for (int st = 0; st < stages; ++st) {
        ok = __all_sync(0xFFFFFFFFu,
                        wait_bounded_parked(empty_bar(slot), phase ^ 1u, &s_abort, p.status, kDevTimeoutProducer));
        if (!ok) break;
        if (lane == 0) {
          const uint32_t bar = full_bar(slot), w_dst = smem_base + slot * L::kStageBytes, a_dst = w_dst + L::kWBytes;
          mbar_arrive_expect_tx(bar, L::kStageBytes);
#pragma unroll
          for (int i = 0; i < kSB / 8; ++i) {   // 128 bytes of every row; past the end of a dimension zeros come in
            const uint32_t d = w_dst + i * L::kRows * 128;
            const int x = st * (kSB * 16) + i * 128;
            tma_load_4d(d, &tm_w, bar, x, it.n0, 0, it.g);
            if constexpr (kGated) tma_load_4d(d + L::kRows * 64, &tm_w, bar, x, it.n0, 1, it.g);
          }
          if (p.a_boxes == 1) {
            tma_load_3d(a_dst, &tm_a, bar, 0, it.row0, st * (kSB / 2));
          } else {
#pragma unroll
            for (int i = 0; i < kSB / 2; ++i)
              tma_load_2d(a_dst + i * kNT * 1024, &tm_a, bar, st * (kSB * 32) + i * 64, it.row0);
          }
        }
        if (++slot == kStages) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp > L::kWarps) {
    // ---- the scales and zeros of this block's items, kW4WindowGroups groups at a time, by three warps.  Tile row r: gated:
    // gate rows, then the up rows of the same outputs; rows past the end are read from the last one.
    uint32_t use = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const Item it = item_at(item, at);
      // first rows of the tile's (gate) rows and of its up rows
      const long long row_a = (static_cast<long long>(it.g) * weight_rows + it.n0) * groups;
      const long long row_b = row_a + static_cast<long long>(p.n) * groups;
      const int last = p.n - 1 - it.n0;
      for (int first = 0; first < groups; first += kW4WindowGroups, ++use) {
        const int buf = use & 1u;
        ok = __all_sync(0xFFFFFFFFu, wait_bounded_parked(scale_empty_bar(buf), ((use >> 1) & 1u) ^ 1u, &s_abort, p.status,
                                                         kDevTimeoutProducer));
        if (!ok) break;
        const int count = min(kW4WindowGroups, groups - first);
        uint8_t* const base = staged + buf * L::kStagedBytes;
        auto row_at = [&](int r) {
          const bool up = kGated && r >= kOutCols;
          return (up ? row_b : row_a) + first + min(up ? r - kOutCols : r, last) * groups;
        };
        // `count` elements of `elem` bytes per row, in pieces of 1 << log_piece bytes, lane after lane
        auto stage = [&](const uint8_t* src, uint8_t* dst, int pitch, int elem, int log_piece, int log_pieces) {
          const int bytes = count * elem;
#pragma unroll 4
          for (int i = tid - (L::kWarps + 1) * 32; i < L::kRows << log_pieces; i += 32 * L::kScaleWarps) {
            const int r = i >> log_pieces, at = (i & ((1 << log_pieces) - 1)) << log_piece;
            if (at >= bytes) continue;
            const uint8_t* s = src + row_at(r) * elem + at;
            uint8_t* d = dst + r * pitch + at;
            if (log_piece == 4) cp_async16(smem_u32(d), s);
            else if (log_piece == 3) cp_async8(smem_u32(d), s);
            else if (log_piece == 2) cp_async4(smem_u32(d), s);
            else if (log_piece == 1) *reinterpret_cast<uint16_t*>(d) = *reinterpret_cast<const uint16_t*>(s);
            else *d = *s;
          }
        };
        stage(p.scale, base, kW4ScalePitch, 2, p.log_scale_piece, p.log_scale_pieces);
        if constexpr (kZero) stage(p.zero, base + L::kScaleBytes, kW4ZeroPitch, 1, p.log_zero_piece, p.log_zero_pieces);
        // every lane arrives for its own pieces; with copies alone the warp goes on to the next item meanwhile
        if (p.log_scale_piece >= 2 && (!kZero || p.log_zero_piece >= 2)) {
          cp_async_arrive(scale_full_bar(buf));
        } else {
          cp_async_wait_all();
          mbar_arrive(scale_full_bar(buf));
        }
      }
    }
  } else {
    // ---- multiplication
    const int wn = warp % kWN, wk = warp / kWN;
    const int lr = lane >> 2, lt = lane & 3;
    // fragment addresses inside a stage: weight row (its 8-row group's row lr), k block wk * kBlocks + b
    auto tile_row = [&](int i) { return kGated ? i * kOutCols + wn * 16 : wn * 32 + i * 16; };
    uint32_t w_off[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int c = wk * kBlocks + b;
      w_off[b] = (c >> 3) * (L::kRows * 128) + lr * 128 + (((c & 7) ^ lr) << 4) + lt * 4;
    }
    const int a_row = (lr >> 1) + 4 * (lr & 1);   // the row of `a` in column lr of a product
    uint32_t a_off[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      a_off[h] = L::kWBytes + wk * (kBlocks / 2) * kNT * 1024 + a_row * 128 + (((h * 4 + lt) ^ a_row) << 4);
    float* const red = reinterpret_cast<float*>(smem + kStages * L::kStageBytes);

    int slot = 0;
    uint32_t phase = 0, use = 0;
    int red_buf = 0;
    bool ok = true;   // false: a wait ran out; the rest is walked through without touching data
    for (int item = blockIdx.x; item < items; item += gridDim.x, red_buf ^= 1) {
      const Item it = item_at(item, at);
      const int nt_used = (it.rows + 7) >> 3;
      float acc[2][kNT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kNT; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[i][j][v] = 0.f;

      // `count` blocks of the stage in `slot` that share a scale, staged group `grp`; w_at(b), a_at(b): where block b's
      // fragments begin
      auto run = [&](auto columns, auto blocks, int grp, auto&& w_at, auto&& a_at) {
        constexpr int kJ = decltype(columns)::value;   // 8-row column tiles of `a` in use
        constexpr int kCount = decltype(blocks)::value;
        const uint8_t* const st = smem + slot * L::kStageBytes;
        const uint8_t* const s_frag = staged + (use & 1u) * L::kStagedBytes + lr * kW4ScalePitch;
        const uint8_t* const z_frag = staged + (use & 1u) * L::kStagedBytes + L::kScaleBytes + lr * kW4ZeroPitch;
        uint32_t zp[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            zp[i][h] = zero_pair<kFp16>(kZero ? z_frag[(tile_row(i) + h * 8) * kW4ZeroPitch + grp] : 8u);
        float part[2][kJ][4];
#pragma unroll
        for (int b = 0; b < kCount; ++b) {
          const uint8_t* const w_frag = st + w_at(b);
          const uint8_t* const a_frag = st + a_at(b);
          uint32_t wv[2][2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              unpack_word<kFp16>(*reinterpret_cast<const uint32_t*>(w_frag + (tile_row(i) + h * 8) * 128), zp[i][h], wv[i][h]);
#pragma unroll
          for (int j = 0; j < kJ; ++j) {
            const uint4 q = *reinterpret_cast<const uint4*>(a_frag + j * 1024);
            const uint32_t x04 = __byte_perm(q.x, q.z, 0x5410), x15 = __byte_perm(q.x, q.z, 0x7632);
            const uint32_t x26 = __byte_perm(q.y, q.w, 0x5410), x37 = __byte_perm(q.y, q.w, 0x7632);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t f0[4] = {wv[i][0][0], wv[i][1][0], wv[i][0][1], wv[i][1][1]};
              const uint32_t f1[4] = {wv[i][0][2], wv[i][1][2], wv[i][0][3], wv[i][1][3]};
              if (b == 0) mma_16816<kFp16, true>(part[i][j], f0, x04, x15);
              else mma_16816<kFp16, false>(part[i][j], f0, x04, x15);
              mma_16816<kFp16, false>(part[i][j], f1, x26, x37);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint8_t* sa = s_frag + tile_row(i) * kW4ScalePitch + grp * 2;
          const float s0 = to_float<kFp16>(*reinterpret_cast<const uint16_t*>(sa));
          const float s1 = to_float<kFp16>(*reinterpret_cast<const uint16_t*>(sa + 8 * kW4ScalePitch));
#pragma unroll
          for (int j = 0; j < kJ; ++j) {
            acc[i][j][0] = fmaf(s0, part[i][j][0], acc[i][j][0]);
            acc[i][j][1] = fmaf(s0, part[i][j][1], acc[i][j][1]);
            acc[i][j][2] = fmaf(s1, part[i][j][2], acc[i][j][2]);
            acc[i][j][3] = fmaf(s1, part[i][j][3], acc[i][j][3]);
          }
        }
      };
      // a stage whose first block is block0 of its window of scales and that holds `held` blocks
      auto multiply = [&](auto columns, int block0, int held) {
        if (held >= kSB) {   // a warp's kBlocks neighbours, kPer at a time
          const int grp = (block0 + wk * kBlocks) >> kLogGs;
#pragma unroll
          for (int b0 = 0; b0 < kBlocks; b0 += kPer)
            run(columns, std::integral_constant<int, kPer>{}, grp + (b0 >> kLogGs), [&](int b) { return w_off[b0 + b]; },
                [&](int b) { return a_off[(b0 + b) & 1] + ((b0 + b) >> 1) * kNT * 1024; });
        } else {             // the last stage of a k that is no multiple of it: block by block in turn
#pragma unroll 1
          for (int c = wk; c < held; c += kWK)
            run(columns, std::integral_constant<int, 1>{}, (block0 + c) >> kLogGs,
                [&](int) { return (c >> 3) * (L::kRows * 128) + lr * 128 + (((c & 7) ^ lr) << 4) + lt * 4; },
                [&](int) { return L::kWBytes + (c >> 1) * kNT * 1024 + a_row * 128 + ((((c & 1) * 4 + lt) ^ a_row) << 4); });
        }
      };

      for (int st0 = 0; st0 < stages; st0 += kWindowStages, ++use) {
        ok = __all_sync(0xFFFFFFFFu, ok && wait_bounded_parked(scale_full_bar(use & 1u), (use >> 1) & 1u, &s_abort, p.status,
                                                               kDevTimeoutMma));
        const int st_end = min(stages, st0 + kWindowStages);
        for (int st = st0; st < st_end; ++st) {
          ok = __all_sync(0xFFFFFFFFu, ok && wait_bounded_parked(full_bar(slot), phase, &s_abort, p.status, kDevTimeoutMma));
          if (!ok) continue;
          if (kNT > 1 && nt_used == 1) multiply(std::integral_constant<int, 1>{}, (st - st0) * kSB, nblk - st * kSB);
          else multiply(std::integral_constant<int, kNT>{}, (st - st0) * kSB, nblk - st * kSB);
          __syncwarp();
          if (lane == 0) mbar_arrive(empty_bar(slot));
          if (++slot == kStages) {
            slot = 0;
            phase ^= 1u;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(scale_empty_bar(use & 1u));
      }

      // ---- join the kWK partial sums (in order) and store.  Every warp holds its values in the same lanes; the two
      // buffers alternate, so one meeting per item is enough.
      float* const joined = red + red_buf * L::kRedFloats + wn * (2 * kNT * 4) * 32 + lane;
      constexpr int kWarpStep = kWN * (2 * kNT * 4) * 32;
      if (wk > 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < kNT; ++j) {
            if (kNT > 1 && j >= nt_used) break;
#pragma unroll
            for (int v = 0; v < 4; ++v) joined[(wk - 1) * kWarpStep + ((i * kNT + j) * 4 + v) * 32] = acc[i][j][v];
          }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(L::kWarps * 32) : "memory");
      if (wk == 0 && ok) {
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          if (kNT > 1 && j >= nt_used) break;
#pragma unroll
          for (int q = 1; q < kWK; ++q)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int v = 0; v < 4; ++v) acc[i][j][v] += joined[(q - 1) * kWarpStep + ((i * kNT + j) * 4 + v) * 32];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int r = j * 8 + lt + (v & 1) * 4;     // column 2 lt + (v & 1) of the product
            if (r >= it.rows) continue;
            uint16_t* out = p.out + static_cast<long long>(it.row0 + r) * p.n;
            auto store = [&](int col, float value) {
              if (col >= p.n) return;
              if constexpr (kFp16) out[col] = __half_as_ushort(__float2half_rn(value));
              else out[col] = __bfloat16_as_ushort(__float2bfloat16_rn(value));
            };
            const int c = lr + (v >> 1) * 8;            // row inside the warp's 16
            if constexpr (kGated) {
              const float g = acc[0][j][v];
              store(it.n0 + wn * 16 + c,
                    (p.act == kActSilu ? gate_value<kActSilu>(g) : gate_value<kActGeluTanh>(g)) * acc[1][j][v]);
            } else {
              store(it.n0 + wn * 32 + c, acc[0][j][v]);
              store(it.n0 + wn * 32 + 16 + c, acc[1][j][v]);
            }
          }
        }
      }
    }
  }
  chain_release();   // both products of a block, 128 rows, replayed: 61 -> 57 us; at the kernel's start 57 as well
  __syncthreads();
  if (*static_cast<volatile int*>(&s_abort))
    for (int i = 0; i < 64; ++i) __nanosleep(4000);   // copies still in flight land before the memory goes
}

// ------------------------------------------------------------------ quantiser
// 16 lanes per group of 16 * kPer elements: min / max by shuffles, then every lane packs kPer values.  Symmetric:
// scale = max|w| / 7, q = clamp(round(w / scale) + 8).  Asymmetric: scale = (max(w,0) - min(w,0)) / 15,
// zero = round(-min / scale), q = clamp(round(w / scale) + zero).  Scales are rounded to the weights' type first and
// that rounded scale is what the values are divided by; a group of zeros has scale 0.  Run once per weight tensor: 2-byte
// loads and a correctly rounded division per value bound it, far from the bytes (128 x 1536 x 2048 bf16, 1.0 GB: groups of
// 128 483 us, 2.1 TB/s; of 32 with zeros 889 us, 1.2 TB/s).
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
struct W4Operands {
  const void* a;
  const void* w;
};

template <int kWN, int kWK, int kNT, int kStages, int kSB, int kLogGs, bool kGated, bool kFp16, bool kZero>
static int launch_w4(const W4Operands& o, W4Args p, int want_sms, cudaStream_t stream) {
  using L = W4Smem<kWN, kWK, kNT, kStages, kSB>;
  static_assert((kW4WindowGroups << kLogGs) % kSB == 0, "a window ends with a stage");
  auto kern = w4_m_grouped_kernel<kWN, kWK, kNT, kStages, kSB, kLogGs, kGated, kFp16, kZero>;
  constexpr int kOutCols = kGated ? L::kRows / 2 : L::kRows;
  p.tiles = (p.n + kOutCols - 1) / kOutCols;
  const int smem = L::kScaleOffset + 2 * L::kStagedBytes +
                   p.list_capacity * static_cast<int>(sizeof(W4Expert)) + 1024;
  CUtensorMap tm_w, tm_a;
  {
    const uint64_t row = static_cast<uint64_t>(p.k) / 2, n = static_cast<uint64_t>(p.n), halves = kGated ? 2 : 1;
    const uint64_t dims[4] = {row, n, halves, static_cast<uint64_t>(p.num_groups)};
    const uint64_t strides[3] = {row, row * n, row * n * halves};
    const uint32_t box[4] = {128, static_cast<uint32_t>(kOutCols), 1, 1};
    if (int rc = encode_tmap(&tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, o.w, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                             "W4[G,N,K/2]"))
      return rc;
  }
  {
    // seen as [k / 64][m_rows][64] a whole stage of `a` is one box; as [m_rows][k] it takes one per 64 k (a small box
    // costs the TMA unit as much as a large one)
    const uint64_t k = static_cast<uint64_t>(p.k), rows = static_cast<uint64_t>(p.m_rows);
    p.a_boxes = p.k % 64 == 0 ? 1 : kSB / 2;
    const uint64_t dims[3] = {p.a_boxes == 1 ? 64 : k, rows, k / 64};
    const uint64_t strides[2] = {k * 2, 128};
    const uint32_t box[3] = {64, kNT * 8, kSB / 2};
    if (int rc = encode_tmap(&tm_a, CU_TENSOR_MAP_DATA_TYPE_UINT16, p.a_boxes == 1 ? 3 : 2, o.a, dims, strides, box,
                             CU_TENSOR_MAP_SWIZZLE_128B, "A"))
      return rc;
  }
  if constexpr (L::kRebalance) {   // the build must have given the launch the registers that the split counts on
    static int launch_regs = 0;
    if (!launch_regs) {
      cudaFuncAttributes attr;
      B200_CUDA(cudaFuncGetAttributes(&attr, kern));
      launch_regs = attr.numRegs;
    }
    if (launch_regs < L::kRegs)
      return set_error(kErrUnsupported, "b200gemm_w4_m_grouped: built with %d registers per thread, %d are needed", launch_regs,
                       L::kRegs);
  }
  B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  // what the registers (see __launch_bounds__) and the shared memory allow
  const int per_sm = min(kNT > 1 || kWN > 1 ? 2 : 3, 228 * 1024 / (smem + 2048));
  // at most this many items: every expert with rows has one partial chunk at most
  const long long chunks = p.m_rows / (kNT * 8) + (p.m_rows < p.num_groups ? p.m_rows : p.num_groups);
  const long long items = chunks * p.tiles;
  B200_REQUIRE(items < (1ll << 31) - 65536, "b200gemm_w4_m_grouped: too many rows and columns for one call");
  const long long resident = static_cast<long long>(per_sm) * want_sms;
  const unsigned grid = static_cast<unsigned>(items < resident ? items : resident);
  if constexpr (kWN > 1) {
    B200_CUDA(launch_chained(kern, grid, L::kThreads, smem, stream, tm_w, tm_a, p));
  } else {   // a launch of some 5 us: replayed from a graph, waiting costs it more than the early start gains (7.7, 7.4 us)
    kern<<<grid, L::kThreads, smem, stream>>>(tm_w, tm_a, p);
    B200_CUDA(cudaGetLastError());
  }
  return 0;
}

template <int kWN, int kWK, int kNT, int kStages, int kSB>
static int form_w4(const W4Operands& o, const W4Args& p, int log_gs, int gated, int dtype, int want_sms, cudaStream_t stream) {
#define B200_W4(GS, GATED, FP16)                                                                 \
  (p.zero ? launch_w4<kWN, kWK, kNT, kStages, kSB, GS, GATED, FP16, true>(o, p, want_sms, stream) \
          : launch_w4<kWN, kWK, kNT, kStages, kSB, GS, GATED, FP16, false>(o, p, want_sms, stream))
#define B200_W4_GS(GATED, FP16) \
  (log_gs == 0 ? B200_W4(0, GATED, FP16) : log_gs == 1 ? B200_W4(1, GATED, FP16) : B200_W4(2, GATED, FP16))
  return gated ? (dtype ? B200_W4_GS(true, true) : B200_W4_GS(true, false))
               : (dtype ? B200_W4_GS(false, true) : B200_W4_GS(false, false));
#undef B200_W4_GS
#undef B200_W4
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
  p.scale = static_cast<const uint8_t*>(scale);
  p.zero = static_cast<const uint8_t*>(zero);
  p.out = static_cast<uint16_t*>(out);
  p.sizes = sizes;
  p.sizes_i64 = sizes_is_i64;
  p.num_groups = num_groups;
  p.m_rows = m_rows;
  p.n = n;
  p.k = k;
  p.act = act;
  const int groups = k / group_size;
  const int window = groups < kW4WindowGroups ? groups : kW4WindowGroups;
  auto log_piece = [](const void* base, int row_bytes, int least) {
    int log = 4;
    while (log > least && ((reinterpret_cast<uintptr_t>(base) | static_cast<unsigned>(row_bytes)) & ((1u << log) - 1))) --log;
    return log;
  };
  auto log_pieces = [](int bytes, int piece) {
    int log = 0;
    while ((piece << log) < bytes) ++log;
    return log;
  };
  p.log_scale_piece = log_piece(scale, groups * 2, 1);
  p.log_scale_pieces = log_pieces(window * 2, 1 << p.log_scale_piece);
  if (zero) {
    p.log_zero_piece = log_piece(zero, groups, 0);
    p.log_zero_pieces = log_pieces(window, 1 << p.log_zero_piece);
  }
  p.list_capacity = static_cast<int>(m_rows < num_groups ? m_rows : num_groups);
  p.status = device_status_ptr();
  const int want = num_sms > 0 && num_sms < sms ? num_sms : sms;
  const int log_gs = group_size == 32 ? 0 : group_size == 64 ? 1 : 2;
  const W4Operands o = {a, w4};
  const long long rows_at_most = m_rows < num_groups ? m_rows : num_groups;
  if (m_rows <= 8ll * num_groups && rows_at_most * ((gated ? 2ll * n : n) / 64) <= 2ll * want)
    return form_w4<1, 8, 1, 3, 16>(o, p, log_gs, gated, dtype, want, stream);
  return m_rows <= 8ll * num_groups ? form_w4<4, 2, 1, 2, 16>(o, p, log_gs, gated, dtype, want, stream)
                                    : form_w4<4, 2, 2, 3, 8>(o, p, log_gs, gated, dtype, want, stream);
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
