// The experts' gated feed-forward block in 16 bits, the two products whose epilogue is the gate:
//
//   forward    [g | u] = x W13_e^T,  h = act(g) * u                  W13 [G, 2 I, K]: gate rows, then up rows
//   backward   dh = dy W2_e,  dg = dh * u * act'(g),  du = dh * act(g)       W2 [G, K, I]
//
// Both are bound by the tensor cores (K is the hidden size, thousands), so the epilogue's work must hide behind
// the next tile's products and its bytes must be few: the products g, u and dh never reach memory.
//
//   * A forward tile holds the gate and the up columns of the SAME kHalf outputs: two boxes of W13, one from each
//     half, side by side in one accumulator.  In the CTA-pair form (256 rows on two SMs) CTA 0 supplies the gate
//     box and CTA 1 the up box.  No interleaved copy of the weights is needed.
//   * For training the forward keeps g and u, which the backward epilogue reads back tile by tile into the buffers
//     it then overwrites with dg and du.  They are kept in 16 bits scaled by the largest of 32 neighbouring columns of
//     the row (see below).  That block is what a thread holds in registers, so its maximum costs no exchange, and what
//     the gradients lose is the rounding of dg and du alone, which the tensor cores ask for: error of dx in 2-norm,
//     4096 rows, K 2048, I 768: bf16 layers 2.4e-3, and 3.0e-3 with g and u in bf16 (1.7e-3 is the rounding of dx
//     itself); fp16 layers 3.0e-4 and 3.8e-4 (2.1e-4).  A column of fp16 layers far below its neighbours keeps the accuracy
//     that plain fp16 would give it down to 2^-12 of the largest of them, and loses a bit with every further factor of two.
//   * Everything else is the M-grouped kernel's: persistent CTAs, one walk over the group sizes, TMA ring, one MMA
//     issuer, two accumulators, epilogue warps that store through swizzled staging buffers.
//
// Measured with 655 360 rows over 128 groups, K 2048, I 768, beside the plain M-grouped product of the same shape on
// the same GPU: forward 2.78 ms (2.72), keeping g and u 3.26 ms, gradient
// 1.94 ms (1.66; it reads 2.0 GB and writes 2.0 GB where the plain product writes 1.0 GB).  With integer arithmetic for
// the codes and an exactly rounded reciprocal they took 3.96 and 3.54 ms: the epilogue, not the tensor cores, was the
// bound, and it still is in fp16 layers: keeping g and u 3.8-4.2 ms, gradient 2.2-2.5 ms (gelu 4.0 and 2.7; bf16 layers
// in the same runs 3.0 and 1.9, gelu 3.5 and 2.1).  With 128 rows over 80 of 128 groups the forward is bound by the weights: 503 MB in 89 us, 5.65 TB/s.
//
// Rows behind the last group have no product; the epilogue warps zero them in `tail` (the layer's output in the
// forward call, its input gradient in the backward call) once their tiles are done.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/b200gemm.h"
#include "activation.cuh"
#include "common.cuh"
#include "gemm_tile.cuh"
#include "kept_code.cuh"

namespace b200 {

enum class GatedMode { kForward, kForwardSave, kBackward };

// ------------------------------------------------------------------ block floating point
// A block of 32 values v is kept as 16-bit codes and the fp32 exponent field e of its largest finite magnitude.
//   bf16 layers   code = fp16(v * 2^(141 - e)): the largest lies in [2^14, 2^15), 10 mantissa bits down to 2^-28 of it.
//                 One multiplication and half a conversion per value, and fp16's own infinities and NaN.
//   fp16 layers   fp16 would add as much error as the output's rounding, so the values near the largest get two mantissa
//                 bits more, which are taken from the exponents far below it (kept_code.cuh).  Integer arithmetic, 1.5 and
//                 2 instructions per value more than with the same mantissa for all: 4 096 rows over 8 groups, K 2048,
//                 I 768, silu, keeping g and u 35.5 -> 36.3 us, gradient 29.8 -> 30.2 us.
constexpr uint32_t kBlockExpMin = 15;   // keeps 2^(141 - e) and its inverse normal numbers

__device__ __forceinline__ uint32_t block_exponent(const uint32_t (&v)[32]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = fmaxf(m, fabsf(__uint_as_float(v[i])));   // NaN is passed over
  if (m > 3.0e38f) {                                                         // rare: look again, without infinities
    m = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float a = fabsf(__uint_as_float(v[i]));
      if (a < __uint_as_float(0x7F800000u)) m = fmaxf(m, a);
    }
  }
  return max(__float_as_uint(m) >> 23, kBlockExpMin);
}

// 2^(141 - e), e in [15, 254]
__device__ __forceinline__ float block_down(uint32_t e) { return __uint_as_float((268u - e) << 23); }
// bf16 layers: its inverse; fp16 layers: 2^(e - 127), what is left after the code's own 2^121
template <bool kFp16>
__device__ __forceinline__ float block_up(uint32_t e) {
  return __uint_as_float((kFp16 ? e : e - 14u) << 23);
}

__device__ __forceinline__ uint32_t code16(uint32_t v, float down) {
  // times 2^-128 (a denormal): [2^14, 2^15) -> [2^-114, 2^-113), whose exponent field is kKeptTop
  const uint32_t f = __float_as_uint(__uint_as_float(v) * down * __uint_as_float(1u << 21));
  return kept_code(f & 0x7FFFFFFFu) | ((f >> 16) & 0x8000u);
}

template <bool kFp16>
__device__ __forceinline__ uint32_t encode2(uint32_t lo, uint32_t hi, float down) {
  if constexpr (!kFp16) return pack2_16bit(__uint_as_float(lo) * down, __uint_as_float(hi) * down, 1);
  return code16(lo, down) | code16(hi, down) << 16;
}

template <bool kFp16>
__device__ __forceinline__ float2 decode2(uint32_t codes, float up) {
  if constexpr (!kFp16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&codes));
    return make_float2(f.x * up, f.y * up);
  }
  const uint32_t mags = codes & 0x7FFF7FFFu;
  const uint32_t bits = kept_bits2(mags, [](uint32_t a, uint32_t b) { return __vminu2(a, b); });
  auto one = [&](uint32_t magnitude, uint32_t sign, bool finite) {
    const float f = __uint_as_float(magnitude | (sign & 0x80000000u)) * __uint_as_float((127u + 127u - kKeptTop) << 23) * up;
    return finite ? f : __uint_as_float(0x7FFFFFFFu);
  };
  return make_float2(one((bits << 11) & 0x07FFF800u, codes << 16, (mags & 0xFFFFu) != 0x7FFFu),
                     one((bits >> 5) & 0x07FFF800u, codes, mags < 0x7FFF0000u));
}

// runs f with the activation as a compile-time constant
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  if (act == kActSilu) f(std::integral_constant<int, kActSilu>{});
  else f(std::integral_constant<int, kActGeluTanh>{});
}

// ------------------------------------------------------------------ kernel
template <GatedMode kMode, bool kPair, int kHalf>
struct GatedSmem {
  static constexpr bool kBwd = kMode == GatedMode::kBackward;
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = (kPair ? 128 : 2 * kHalf) * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // 4 KB staging buffers of an epilogue warp: h alternates between two; h and the codes of g and u rotate over four;
  // the backward keeps two pairs (g, u)
  static constexpr int kEpiBuffers = kMode == GatedMode::kForward ? 2 : 4;
  static constexpr int kEpiBytes = 4 * kEpiBuffers * 4096;
  static constexpr int kBudget = 227 * 1024 - 1024 - 256;
  static constexpr int kFit = (kBudget - kEpiBytes) / kStageBytes;
  static constexpr int kStages = kFit < 6 ? kFit : 6;
  static constexpr int kEpiOffset = kStages * kStageBytes;
  static constexpr int kBarOffset = kEpiOffset + kEpiBytes;
  static constexpr int kNumBars = 2 * kStages + 4 + (kBwd ? 8 : 0);
  static constexpr int kDynamicBytes = kBarOffset + kNumBars * 8 + 16 + 1024;
  static_assert(kStages >= 3 && kDynamicBytes <= 227 * 1024);
};

struct GatedArgs {
  const void* sizes;
  int sizes_i64;
  int num_groups;
  int masked_stride;
  long long m_rows;
  int inter;          // I
  int k;
  int in_fmt;         // UMMA operand format: 0 = f16, 1 = bf16
  int act;
  uint16_t* h;        // forward: [m_rows, I]
  uint16_t* gu;       // forward with save: codes [m_rows, 2 I]; backward: unused (read through tm_gu)
  uint8_t* exps;      // block exponents [m_rows, 2, exp_pitch]
  int exp_pitch;
  uint16_t* dgu;      // backward: [m_rows, 2 I]
  uint4* tail;        // rows behind the last group are zeroed here (null: none)
  int tail_vecs;
  unsigned* status;
};

template <GatedMode kMode, bool kPair, int kHalf, bool kFp16>
__global__ void __launch_bounds__(kNumThreads, 1)
gated_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
             const __grid_constant__ CUtensorMap tm_h, const __grid_constant__ CUtensorMap tm_gu,
             const __grid_constant__ CUtensorMap tm_dgu, const GatedArgs p) {
  using L = GatedSmem<kMode, kPair, kHalf>;
  constexpr bool kBwd = L::kBwd;
  constexpr bool kSave = kMode == GatedMode::kForwardSave;
  constexpr int kStages = L::kStages;
  constexpr int kCols = 2 * kHalf;                   // accumulator columns
  constexpr int kOutCols = kBwd ? kCols : kHalf;     // columns of I that a tile covers
  constexpr int kTileRows = kPair ? 256 : 128;
  constexpr int kCtaGroup = kPair ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // still known to be shared memory
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_base + L::kBarOffset;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
  auto tmem_full_bar = [&](int a) { return bar_base + 8u * (2 * kStages + a); };
  auto tmem_empty_bar = [&](int a) { return bar_base + 8u * (2 * kStages + 2 + a); };
  auto load_bar = [&](int quarter, int b) { return bar_base + 8u * (2 * kStages + 4 + quarter * 2 + b); };
  volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(smem + L::kBarOffset + L::kNumBars * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kBarOffset + L::kNumBars * 8 + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? cluster_ctarank() : 0;  // 0 = leader
  const int worker = kPair ? blockIdx.x >> 1 : blockIdx.x;
  const int workers = kPair ? gridDim.x >> 1 : gridDim.x;
  const int n_tiles = (p.inter + kOutCols - 1) / kOutCols;
  const int num_kb = (p.k + kBlockK - 1) / kBlockK;
  constexpr uint32_t kTmemCols = 2 * kCols;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar(a), 1);
      mbar_init(tmem_empty_bar(a), kPair ? 8 : 4);
    }
    if constexpr (kBwd)
      for (int i = 0; i < 8; ++i) mbar_init(load_bar(i >> 1, i & 1), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    if constexpr (!kBwd) prefetch_tmap(&tm_h);
    if constexpr (kBwd || kSave) prefetch_tmap(&tm_gu);
    if constexpr (kBwd) prefetch_tmap(&tm_dgu);
  }
  if (warp == 1) {
    tmem_alloc<kCtaGroup>(smem_u32(const_cast<uint32_t*>(tmem_holder)), kTmemCols);
    tmem_relinquish<kCtaGroup>();
  }
  tc_fence_before_sync();
  if constexpr (kPair) cluster_sync_all();  // both CTAs' barriers exist before anyone signals across the pair
  else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  chain_wait();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    WarpGroupWalker w;
    w.init(p.sizes, p.sizes_i64, p.num_groups, p.masked_stride, kTileRows, p.m_rows);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = worker; ok; tile += workers) {
      const int mt = tile / n_tiles;
      const int nt = tile - mt * n_tiles;
      if (!w.seek(mt)) break;
      const int row0 = static_cast<int>(w.tile_row0(mt)) + static_cast<int>(rank) * 128;
      const int g = w.g;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, p.status, kDevTimeoutProducer)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          const uint32_t a_dst = smem_base + stage * L::kStageBytes;
          const uint32_t b_dst = a_dst + L::kABytes;
          if constexpr (kPair) {
            // one arrival per phase, by the leader, for the bytes of both CTAs
            const uint32_t leader_full = mapa_u32(full_bar(stage), 0);
            if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * L::kStageBytes);
            tma_load_2d_pair(a_dst, &tm_a, leader_full, kb * kBlockK, row0);
            if constexpr (!kBwd) {
              tma_load_4d_pair(b_dst, &tm_b, leader_full, kb * kBlockK, nt * kHalf, static_cast<int>(rank), g);
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j)
                tma_load_3d_pair(b_dst + j * (kBlockK * 128), &tm_b, leader_full,
                                 nt * kOutCols + static_cast<int>(rank) * 128 + j * 64, kb * kBlockK, g);
            }
          } else {
            mbar_arrive_expect_tx(full_bar(stage), L::kStageBytes);
            tma_load_2d(a_dst, &tm_a, full_bar(stage), kb * kBlockK, row0);
            if constexpr (!kBwd) {
              tma_load_4d(b_dst, &tm_b, full_bar(stage), kb * kBlockK, nt * kHalf, 0, g);
              tma_load_4d(b_dst + kHalf * 128, &tm_b, full_bar(stage), kb * kBlockK, nt * kHalf, 1, g);
            } else {
#pragma unroll
              for (int j = 0; j < kCols / 64; ++j)
                tma_load_3d(b_dst + j * (kBlockK * 128), &tm_b, full_bar(stage), nt * kOutCols + j * 64, kb * kBlockK, g);
            }
          }
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (pair: leader CTA only)
    if (rank == 0) {
      WarpGroupWalker w;
      w.init(p.sizes, p.sizes_i64, p.num_groups, p.masked_stride, kTileRows, p.m_rows);
      const uint32_t fmt = static_cast<uint32_t>(p.in_fmt);
      const uint32_t idesc = make_instr_desc(fmt, fmt, 0u, kBwd ? 1u : 0u, kTileRows, kCols);
      int stage = 0;
      uint32_t phase = 0;
      uint32_t tile_iter = 0;
      bool ok = true;
      for (int tile = worker; ok; tile += workers, ++tile_iter) {
        const int mt = tile / n_tiles;
        if (!w.seek(mt)) break;
        const uint32_t acc = tile_iter & 1u;
        const uint32_t acc_phase = (tile_iter >> 1) & 1u;
        if (!wait_bounded(tmem_empty_bar(acc), acc_phase ^ 1u, abort_flag, p.status, kDevTimeoutMma)) break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * kCols;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!wait_bounded(full_bar(stage), phase, abort_flag, p.status, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          if (lane == 0) {
            const uint32_t a_addr = smem_base + stage * L::kStageBytes;
            const uint32_t b_addr = a_addr + L::kABytes;
#pragma unroll
            for (int k16 = 0; k16 < kBlockK / kUmmaK; ++k16) {
              const uint64_t a_desc = make_smem_desc(a_addr + k16 * (kUmmaK * 2), 16, 1024, kSwizzle128);
              const uint64_t b_desc =
                  kBwd ? make_smem_desc(b_addr + k16 * (kUmmaK * 128), kBlockK * 128, 1024, kSwizzle128)
                       : make_smem_desc(b_addr + k16 * (kUmmaK * 2), 16, 1024, kSwizzle128);
              umma<kCtaGroup, false>(d_tmem, a_desc, b_desc, idesc, (kb | k16) != 0 ? 1u : 0u);
            }
            if constexpr (kPair) umma_commit_2cta(empty_bar(stage), 0x3);
            else umma_commit_1cta(empty_bar(stage));
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok && lane == 0) {
          if constexpr (kPair) umma_commit_2cta(tmem_full_bar(acc), 0x3);
          else umma_commit_1cta(tmem_full_bar(acc));
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (warps 2..5)
    WarpGroupWalker w;
    w.init(p.sizes, p.sizes_i64, p.num_groups, p.masked_stride, kTileRows, p.m_rows);
    const int quarter = warp & 3;
    uint8_t* epi = smem + L::kEpiOffset + quarter * (L::kEpiBuffers * 4096);
    const uint32_t row_off = lane * 128;       // this thread's row of a staging buffer
    const uint32_t swz = lane & 7;
    int sel = 0;                               // forward: next staging buffer
    uint32_t loads = 0;                        // backward: (g, u) chunks asked for so far
    uint32_t tile_iter = 0;
    bool ok = true;
    bool done = false;
    for (int tile = worker; ok; tile += workers, ++tile_iter) {
      const int mt = tile / n_tiles;
      const int nt = tile - mt * n_tiles;
      if (!w.seek(mt)) {
        done = true;
        break;
      }
      const long long row_w0 = w.tile_row0(mt) + static_cast<long long>(rank) * 128 + quarter * 32;
      const long long row_end = w.group_row_end();
      const long long row = row_w0 + lane;
      const bool row_ok = row < row_end;
      const bool some = row_w0 < row_end;                 // this warp has rows of the group
      const bool full = row_w0 + 32 <= row_end;           // all of its rows: staged TMA stores
      const uint32_t acc = tile_iter & 1u;
      const uint32_t acc_phase = (tile_iter >> 1) & 1u;
      const int col_tile = nt * kOutCols;

      // backward: bring chunk c's codes of g and u into the next buffer pair, whose stores have been read by then
      auto ask = [&](int c) {
        if (lane == 0) {
          tma_store_wait_read<0>();
          const uint32_t bar = load_bar(quarter, loads & 1u);
          const uint32_t dst = smem_u32(epi) + (loads & 1u) * 8192;
          mbar_arrive_expect_tx(bar, 8192);
          tma_load_3d(dst, &tm_gu, bar, col_tile + c * 64, 0, static_cast<int>(row_w0));
          tma_load_3d(dst + 4096, &tm_gu, bar, col_tile + c * 64, 1, static_cast<int>(row_w0));
        }
        ++loads;
      };
      uint32_t exp_g[kCols / 128 ? kCols / 128 : 1], exp_u[kCols / 128 ? kCols / 128 : 1];
      if constexpr (kBwd) {
        if (some) {
          ask(0);
          const uint8_t* e = p.exps + row * (2ll * p.exp_pitch) + col_tile / 32;
#pragma unroll
          for (int i = 0; i < kCols / 128; ++i) {
            exp_g[i] = row_ok ? *reinterpret_cast<const uint32_t*>(e + 4 * i) : 0x01010101u;
            exp_u[i] = row_ok ? *reinterpret_cast<const uint32_t*>(e + p.exp_pitch + 4 * i) : 0x01010101u;
          }
        }
      }

      if (!wait_bounded(tmem_full_bar(acc), acc_phase, abort_flag, p.status, kDevTimeoutEpilogue)) break;
      tc_fence_after_sync();
      const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kCols;

      if (some) {
        if constexpr (!kBwd) {
          uint32_t exps_g = 0, exps_u = 0;
#pragma unroll 1
          for (int c = 0; c < kHalf / 64; ++c) {
            const int col0 = col_tile + c * 64;
            if (col0 >= p.inter) break;
            // the buffers written next have left: one store may be on its way (see kEpiBuffers)
            if (lane == 0) tma_store_wait_read<1>();
            __syncwarp();
            uint8_t* buf_h = epi + (sel & (L::kEpiBuffers - 1)) * 4096;
            uint8_t* buf_g = epi + ((sel + 1) & (L::kEpiBuffers - 1)) * 4096;
            uint8_t* buf_u = epi + ((sel + 2) & (L::kEpiBuffers - 1)) * 4096;
            if (full) sel += kSave ? 3 : 1;   // only with a store: the wait above counts stores
#pragma unroll 1
            for (int s = 0; s < 2; ++s) {
              uint32_t g[32], u[32];
              tmem_ld_32x32b_x32(t_addr + c * 64 + s * 32, g);
              tmem_ld_32x32b_x32(t_addr + kHalf + c * 64 + s * 32, u);
              tmem_ld_wait();
              auto put = [&](uint8_t* buf, uint16_t* global, int v, const uint32_t (&q)[4]) {
                const uint4 vec = make_uint4(q[0], q[1], q[2], q[3]);
                if (full) *reinterpret_cast<uint4*>(buf + row_off + ((static_cast<uint32_t>(s * 4 + v) ^ swz) << 4)) = vec;
                else if (row_ok && col0 + s * 32 + v * 8 < p.inter) *reinterpret_cast<uint4*>(global + s * 32 + v * 8) = vec;
              };
              with_activation(p.act, [&](auto act) {
                constexpr int kAct = decltype(act)::value;
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                uint32_t q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int i = v * 8 + e * 2;
                  q[e] = pack2_16bit(gate_value<kAct>(__uint_as_float(g[i])) * __uint_as_float(u[i]),
                                     gate_value<kAct>(__uint_as_float(g[i + 1])) * __uint_as_float(u[i + 1]), kFp16);
                }
                put(buf_h, p.h + row * p.inter + col0, v, q);
              }
              });
              if constexpr (kSave) {
                const uint32_t eg = block_exponent(g), eu = block_exponent(u);
                const float down_g = block_down(eg), down_u = block_down(eu);
                exps_g |= eg << (8 * (c * 2 + s));
                exps_u |= eu << (8 * (c * 2 + s));
                uint16_t* gu_row = p.gu + row * (2ll * p.inter) + col0;
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  uint32_t qg[4], qu[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const int i = v * 8 + e * 2;
                    qg[e] = encode2<kFp16>(g[i], g[i + 1], down_g);
                    qu[e] = encode2<kFp16>(u[i], u[i + 1], down_u);
                  }
                  put(buf_g, gu_row, v, qg);
                  put(buf_u, gu_row + p.inter, v, qu);
                }
              }
            }
            if (full) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&tm_h, smem_u32(buf_h), col0, static_cast<int>(row_w0));
                tma_store_commit();
                if constexpr (kSave) {
                  tma_store_3d(&tm_gu, smem_u32(buf_g), col0, 0, static_cast<int>(row_w0));
                  tma_store_commit();
                  tma_store_3d(&tm_gu, smem_u32(buf_u), col0, 1, static_cast<int>(row_w0));
                  tma_store_commit();
                }
              }
            }
          }
          if constexpr (kSave) {
            if (row_ok) {
              uint8_t* e = p.exps + row * (2ll * p.exp_pitch) + col_tile / 32;
              if constexpr (kHalf == 128) {
                *reinterpret_cast<uint32_t*>(e) = exps_g;
                *reinterpret_cast<uint32_t*>(e + p.exp_pitch) = exps_u;
              } else {
                *reinterpret_cast<uint16_t*>(e) = static_cast<uint16_t>(exps_g);
                *reinterpret_cast<uint16_t*>(e + p.exp_pitch) = static_cast<uint16_t>(exps_u);
              }
            }
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < kCols / 64; ++c) {
            const int col0 = col_tile + c * 64;
            if (col0 >= p.inter) break;
            const uint32_t use = loads - 1;    // the chunk asked for last
            if (!wait_bounded(load_bar(quarter, use & 1u), (use >> 1) & 1u, abort_flag, p.status, kDevTimeoutEpilogue)) {
              ok = false;
              break;
            }
            uint8_t* buf = epi + (use & 1u) * 8192;
            uint32_t word_g = exp_g[0], word_u = exp_u[0];
            if constexpr (kCols == 256) {
              if (c >= 2) {
                word_g = exp_g[1];
                word_u = exp_u[1];
              }
            }
#pragma unroll 1
            for (int s = 0; s < 2; ++s) {
              uint32_t dh[32];
              tmem_ld_32x32b_x32(t_addr + c * 64 + s * 32, dh);
              const int shift = 8 * ((c & 1) * 2 + s);
              const float up_g = block_up<kFp16>((word_g >> shift) & 0xFFu);
              const float up_u = block_up<kFp16>((word_u >> shift) & 0xFFu);
              tmem_ld_wait();
              with_activation(p.act, [&](auto act) {
              constexpr int kAct = decltype(act)::value;
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                uint4* at_g = reinterpret_cast<uint4*>(buf + row_off + ((static_cast<uint32_t>(s * 4 + v) ^ swz) << 4));
                uint4* at_u = at_g + 4096 / 16;
                const uint4 cg = *at_g, cu = *at_u;
                const uint32_t wg[4] = {cg.x, cg.y, cg.z, cg.w}, wu[4] = {cu.x, cu.y, cu.z, cu.w};
                uint32_t qg[4], qu[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 g = decode2<kFp16>(wg[e], up_g), u = decode2<kFp16>(wu[e], up_u);
                  const float d0 = __uint_as_float(dh[v * 8 + e * 2]), d1 = __uint_as_float(dh[v * 8 + e * 2 + 1]);
                  float value0, value1, slope0, slope1;
                  gate_value_slope<kAct>(g.x, value0, slope0);
                  gate_value_slope<kAct>(g.y, value1, slope1);
                  qg[e] = pack2_16bit(d0 * u.x * slope0, d1 * u.y * slope1, kFp16);
                  qu[e] = pack2_16bit(d0 * value0, d1 * value1, kFp16);
                }
                const uint4 og = make_uint4(qg[0], qg[1], qg[2], qg[3]), ou = make_uint4(qu[0], qu[1], qu[2], qu[3]);
                if (full) {
                  *at_g = og;
                  *at_u = ou;
                } else if (row_ok && col0 + s * 32 + v * 8 < p.inter) {
                  uint16_t* d = p.dgu + row * (2ll * p.inter) + col0 + s * 32 + v * 8;
                  *reinterpret_cast<uint4*>(d) = og;
                  *reinterpret_cast<uint4*>(d + p.inter) = ou;
                }
              }
              });
              // the next chunk's codes travel while the second half of this one is worked on
              if (s == 0 && c + 1 < kCols / 64 && col0 + 64 < p.inter) ask(c + 1);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (full && lane == 0) {
              tma_store_3d(&tm_dgu, smem_u32(buf), col0, 0, static_cast<int>(row_w0));
              tma_store_3d(&tm_dgu, smem_u32(buf) + 4096, col0, 1, static_cast<int>(row_w0));
              tma_store_commit();
            }
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair) mbar_arrive_cluster(tmem_empty_bar(acc), 0);
        else mbar_arrive(tmem_empty_bar(acc));
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
    if (w.overflow && rank == 0 && quarter == 0 && lane == 0 && p.status) atomicOr(p.status, kDevBadGroupSize);
    // the walk has ended, so row_begin is the number of rows that belong to a group
    if (done && p.tail && p.masked_stride == 0) {
      const long long total = (p.m_rows - w.row_begin) * p.tail_vecs;
      uint4* t = p.tail + w.row_begin * p.tail_vecs;
      const long long step = static_cast<long long>(gridDim.x) * 128;
      for (long long i = static_cast<long long>(blockIdx.x) * 128 + quarter * 32 + lane; i < total; i += step)
        t[i] = make_uint4(0, 0, 0, 0);
    }
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    // a role gave up: give copies / MMAs still in flight time to land before the shared memory and TMEM go
    for (int i = 0; i < 64; ++i) __nanosleep(4000);
    __syncthreads();
  }
  if constexpr (kPair) cluster_sync_all();  // neither CTA leaves while the peer may still signal it or write its TMEM
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<kCtaGroup>(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------ host side
struct GatedMaps {
  CUtensorMap a, b, h, gu, dgu;
};

template <GatedMode kMode, bool kPair, int kHalf, bool kFp16>
static int launch_gated(const GatedMaps& t, const GatedArgs& p, int ctas, cudaStream_t stream) {
  using L = GatedSmem<kMode, kPair, kHalf>;
  auto kern = gated_kernel<kMode, kPair, kHalf, kFp16>;
  if constexpr (kPair) {   // no more CTAs than clusters of two can be resident
    static int resident[64] = {0};
    int dev = 0;
    B200_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return set_error(kErrUnsupported, "device index %d out of range", dev);
    if (!resident[dev]) resident[dev] = pair_kernel_grid();
    if (resident[dev] >= 2 && resident[dev] < ctas) ctas = resident[dev];
    ctas &= ~1;
  }
  B200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynamicBytes));
  B200_CUDA(launch_chained_clusters(kern, ctas, kNumThreads, L::kDynamicBytes, kPair ? 2 : 1, stream, t.a, t.b, t.h, t.gu,
                                    t.dgu, p));
  return 0;
}

static int rows_map(CUtensorMap* out, CUtensorMapDataType dt, const void* base, int64_t rows, int cols, int box_rows,
                    const char* what) {
  const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(cols) * 2};
  const uint32_t box[2] = {64, static_cast<uint32_t>(box_rows)};
  return encode_tmap(out, dt, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
}

// [rows, 2, cols]: the halves are a dimension of their own, so a box clips at the end of its half
static int halves_map(CUtensorMap* out, CUtensorMapDataType dt, const void* base, int64_t rows, int cols, const char* what) {
  const uint64_t dims[3] = {static_cast<uint64_t>(cols), 2, static_cast<uint64_t>(rows)};
  const uint64_t strides[2] = {static_cast<uint64_t>(cols) * 2, static_cast<uint64_t>(cols) * 4};
  const uint32_t box[3] = {64, 1, 32};
  return encode_tmap(out, dt, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, what);
}

// Which form runs.  CTA pairs when groups average `pair_tiles` 256-row tiles and every pair of SMs gets one; else 128-row
// tiles, `half` = 128 columns of each half wide unless that leaves SMs idle.  The pair form wastes more of a group's
// last tile but keeps more of its ring beside the larger staging buffers: with 128 groups, K 2048, 768 + 768 columns
// the plain forward is even at 1024 rows per group (818 us single, 789 pair), the saving forward and the gradient at
// 256 (333 against 322 us, 198 against 188) and the gradient 7 % faster at 1024.
static void gated_form(int64_t m_rows, int num_groups, int masked_stride, int inter, int out_cols_wide, int pair_tiles,
                       int sms, bool* pair, int* half) {
  const long long tiles_wide = (inter + out_cols_wide - 1) / out_cols_wide;
  *pair = false;
  if (sms >= 2 && masked_stride <= 0) {
    if (g_cta_pair_mode == 1) *pair = true;
    else if (g_cta_pair_mode != 0)
      *pair = m_rows / 256 * tiles_wide >= sms / 2 && m_rows / 256 >= static_cast<long long>(pair_tiles) * num_groups &&
              inter > out_cols_wide / 2;
  }
  *half = *pair ? 128 : (inter <= out_cols_wide / 2 || m_rows / 128 * tiles_wide < 2ll * sms) ? 64 : 128;
}

static int check_operands(const char* who, const void* a, const void* b, const void* sizes, int64_t m_rows, int inter,
                          int k) {
  B200_REQUIRE(a && b && sizes, "%s: null pointer", who);
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0,
               "%s: base pointers must be 16-byte aligned", who);
  B200_REQUIRE(k % 8 == 0, "%s: TMA required 16-byte alignment: k*2 bytes (k=%d)", who, k);
  B200_REQUIRE(inter % 8 == 0, "%s: TMA required 16-byte alignment: inter*2 bytes (inter=%d)", who, inter);
  B200_REQUIRE(m_rows < (1ll << 31), "%s: m_rows must fit in int32", who);
  return 0;
}

template <GatedMode kMode>
static int dispatch_gated(const GatedMaps& t, const GatedArgs& p, bool pair, int half, int dtype, int ctas,
                          cudaStream_t stream) {
  if (pair)
    return dtype ? launch_gated<kMode, true, 128, true>(t, p, ctas, stream)
                 : launch_gated<kMode, true, 128, false>(t, p, ctas, stream);
  if (half == 128)
    return dtype ? launch_gated<kMode, false, 128, true>(t, p, ctas, stream)
                 : launch_gated<kMode, false, 128, false>(t, p, ctas, stream);
  return dtype ? launch_gated<kMode, false, 64, true>(t, p, ctas, stream)
               : launch_gated<kMode, false, 64, false>(t, p, ctas, stream);
}

static int exp_pitch_of(int inter) { return (inter + 255) / 256 * 8; }

static int check_numbers(const char* who, int num_groups, int64_t m_rows, int inter, int k, int act, int dtype) {
  B200_REQUIRE(dtype == 0 || dtype == 1, "%s: dtype must be 0 (bf16) or 1 (fp16), got %d", who, dtype);
  B200_REQUIRE(act >= 0 && act < kNumActivations, "%s: unknown activation %d", who, act);
  B200_REQUIRE(num_groups >= 0 && m_rows >= 0 && inter >= 0 && k >= 0, "%s: negative dimension", who);
  return 0;
}

static int gated_forward(const void* a, const void* w13, void* h, void* gu, void* exps, const void* sizes,
                         int sizes_is_i64, int num_groups, int64_t m_rows, int masked_stride, int inter, int k, int act,
                         int dtype, void* tail, int tail_cols, int num_sms, cudaStream_t stream) {
  const char* who = "b200gemm_m_grouped_gated";
  if (int rc = check_numbers(who, num_groups, m_rows, inter, k, act, dtype)) return rc;
  if (m_rows == 0 || inter == 0) return 0;
  if (num_groups == 0) {   // every row lies behind the last group
    if (tail) B200_CUDA(cudaMemsetAsync(tail, 0, static_cast<size_t>(m_rows) * tail_cols * 2, stream));
    return 0;
  }
  B200_REQUIRE(k > 0, "%s: k must be positive", who);
  if (int rc = check_operands(who, a, w13, sizes, m_rows, inter, k)) return rc;
  B200_REQUIRE(h && (gu == nullptr) == (exps == nullptr), "%s: null pointer", who);
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(gu) | reinterpret_cast<uintptr_t>(exps) |
                 reinterpret_cast<uintptr_t>(tail)) & 15) == 0, "%s: base pointers must be 16-byte aligned", who);
  B200_REQUIRE(!tail || tail_cols % 8 == 0, "%s: tail_cols must be a multiple of 8", who);
  B200_REQUIRE(masked_stride >= 0, "%s: masked_stride must not be negative", who);
  const int sms = sm_count();
  B200_REQUIRE(sms > 0, "%s: no CUDA device", who);
  const int ctas = num_sms > 0 && num_sms < sms ? num_sms : sms;
  bool pair;
  int half;
  gated_form(m_rows, num_groups, masked_stride, inter, 128, gu ? 1 : 4, ctas, &pair, &half);
  const CUtensorMapDataType dt = dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  GatedMaps t = {};
  if (int rc = rows_map(&t.a, dt, a, m_rows, k, 128, "A")) return rc;
  {
    const uint64_t ku = static_cast<uint64_t>(k), iu = static_cast<uint64_t>(inter);
    const uint64_t dims[4] = {ku, iu, 2, static_cast<uint64_t>(num_groups)};
    const uint64_t strides[3] = {ku * 2, ku * iu * 2, ku * iu * 4};
    const uint32_t box[4] = {kBlockK, static_cast<uint32_t>(half), 1, 1};
    if (int rc = encode_tmap(&t.b, dt, 4, w13, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "W13[G,2I,K]")) return rc;
  }
  if (int rc = rows_map(&t.h, dt, h, m_rows, inter, 32, "H")) return rc;
  if (gu)
    if (int rc = halves_map(&t.gu, CU_TENSOR_MAP_DATA_TYPE_UINT16, gu, m_rows, inter, "saved gate / up")) return rc;
  GatedArgs p = {};
  p.sizes = sizes;
  p.sizes_i64 = sizes_is_i64;
  p.num_groups = num_groups;
  p.masked_stride = masked_stride;
  p.m_rows = m_rows;
  p.inter = inter;
  p.k = k;
  p.in_fmt = dtype == 1 ? 0 : 1;
  p.act = act;
  p.h = static_cast<uint16_t*>(h);
  p.gu = static_cast<uint16_t*>(gu);
  p.exps = static_cast<uint8_t*>(exps);
  p.exp_pitch = exp_pitch_of(inter);
  p.tail = static_cast<uint4*>(tail);
  p.tail_vecs = tail_cols / 8;
  p.status = device_status_ptr();
  return gu ? dispatch_gated<GatedMode::kForwardSave>(t, p, pair, half, dtype, ctas, stream)
            : dispatch_gated<GatedMode::kForward>(t, p, pair, half, dtype, ctas, stream);
}

static int gated_backward(const void* dy, const void* w2, const void* gu, const void* exps, void* dgu, const void* sizes,
                          int sizes_is_i64, int num_groups, int64_t m_rows, int inter, int k, int act, int dtype,
                          void* tail, int tail_cols, int num_sms, cudaStream_t stream) {
  const char* who = "b200gemm_m_grouped_gated_grad";
  if (int rc = check_numbers(who, num_groups, m_rows, inter, k, act, dtype)) return rc;
  if (m_rows == 0 || inter == 0) return 0;
  if (num_groups == 0) {   // every row lies behind the last group
    if (tail) B200_CUDA(cudaMemsetAsync(tail, 0, static_cast<size_t>(m_rows) * tail_cols * 2, stream));
    return 0;
  }
  B200_REQUIRE(k > 0, "%s: k must be positive", who);
  if (int rc = check_operands(who, dy, w2, sizes, m_rows, inter, k)) return rc;
  B200_REQUIRE(gu && exps && dgu, "%s: null pointer", who);
  B200_REQUIRE(((reinterpret_cast<uintptr_t>(gu) | reinterpret_cast<uintptr_t>(exps) | reinterpret_cast<uintptr_t>(dgu) |
                 reinterpret_cast<uintptr_t>(tail)) & 15) == 0, "%s: base pointers must be 16-byte aligned", who);
  B200_REQUIRE(!tail || tail_cols % 8 == 0, "%s: tail_cols must be a multiple of 8", who);
  const int sms = sm_count();
  B200_REQUIRE(sms > 0, "%s: no CUDA device", who);
  const int ctas = num_sms > 0 && num_sms < sms ? num_sms : sms;
  bool pair;
  int half;
  gated_form(m_rows, num_groups, 0, inter, 256, 1, ctas, &pair, &half);
  const CUtensorMapDataType dt = dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  GatedMaps t = {};
  if (int rc = rows_map(&t.a, dt, dy, m_rows, k, 128, "dY")) return rc;
  {
    const uint64_t ku = static_cast<uint64_t>(k), iu = static_cast<uint64_t>(inter);
    const uint64_t dims[3] = {iu, ku, static_cast<uint64_t>(num_groups)};
    const uint64_t strides[2] = {iu * 2, ku * iu * 2};
    const uint32_t box[3] = {64, kBlockK, 1};
    if (int rc = encode_tmap(&t.b, dt, 3, w2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "W2[G,K,I]")) return rc;
  }
  if (int rc = halves_map(&t.gu, CU_TENSOR_MAP_DATA_TYPE_UINT16, gu, m_rows, inter, "saved gate / up")) return rc;
  if (int rc = halves_map(&t.dgu, dt, dgu, m_rows, inter, "dGU")) return rc;
  GatedArgs p = {};
  p.sizes = sizes;
  p.sizes_i64 = sizes_is_i64;
  p.num_groups = num_groups;
  p.m_rows = m_rows;
  p.inter = inter;
  p.k = k;
  p.in_fmt = dtype == 1 ? 0 : 1;
  p.act = act;
  p.exps = const_cast<uint8_t*>(static_cast<const uint8_t*>(exps));
  p.exp_pitch = exp_pitch_of(inter);
  p.dgu = static_cast<uint16_t*>(dgu);
  p.tail = static_cast<uint4*>(tail);
  p.tail_vecs = tail_cols / 8;
  p.status = device_status_ptr();
  return dispatch_gated<GatedMode::kBackward>(t, p, pair, half, dtype, ctas, stream);
}

}  // namespace b200

extern "C" {

long long b200gemm_gated_exponent_bytes(int64_t m_rows, int inter) {
  if (m_rows < 0 || inter < 0) return 0;
  return 2ll * m_rows * b200::exp_pitch_of(inter);
}

int b200gemm_m_grouped_gated(const void* a, const void* w13, void* h, void* saved, void* saved_exps, const void* sizes,
                             int sizes_is_i64, int num_groups, int64_t m_rows, int masked_stride, int inter, int k, int act,
                             int dtype, void* tail, int tail_cols, int num_sms, void* stream) {
  return b200::gated_forward(a, w13, h, saved, saved_exps, sizes, sizes_is_i64, num_groups, m_rows, masked_stride, inter, k,
                             act, dtype, tail, tail_cols, num_sms, static_cast<cudaStream_t>(stream));
}

int b200gemm_m_grouped_gated_grad(const void* dy, const void* w2, const void* saved, const void* saved_exps, void* dgu,
                                  const void* sizes, int sizes_is_i64, int num_groups, int64_t m_rows, int inter, int k,
                                  int act, int dtype, void* tail, int tail_cols, int num_sms, void* stream) {
  return b200::gated_backward(dy, w2, saved, saved_exps, dgu, sizes, sizes_is_i64, num_groups, m_rows, inter, k, act, dtype,
                              tail, tail_cols, num_sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
