// Row movement between tokens and expert-major rows in 16 bits, with its gradients (training):
//
//   permute   rows[pos[t,j], :] = x[t, :]                     gradient  dx[t]    = sum_j drows[pos[t,j]]
//   combine   out[t] = sum_j w[t,j] * rows[pos[t,j]]          gradients drows[r] = w[t,j] * dout[t]
//                                                                       dw[t,j]  = <dout[t], rows[r]>
//
// pos (row of pair p = t * top_k + j) and order (pair of row r) are the two halves of the routing plan.
// Pair p owns row r = pos[p] if 0 <= r < num_rows and order[r] == p; any other pair (the -1 of a rejected
// routing entry, an index given twice) takes no part, and a row nobody owns reads as zeros.  Every row
// therefore has one writer, and the results do not depend on the order in which blocks run.
//
// All three kernels are bound by HBM bytes: a token's vector is read once, whatever its top_k, and a row is
// read or written once.  One warp (few tokens: one block) takes a token and walks its columns in 16-byte vectors
// with the loads of its top_k rows in flight together.  Sums and dot products are fp32, rounded once.  Measured, 81 920
// tokens, top-8, hidden 2048 (share of the measured copy bandwidth, 6569 GB/s): permute 504 us (0.91), combine and the
// gradient of permute 455 us (1.01; 868 us with the rows' addresses shuffled anew for every vector), the gradients of
// combine 909 us (0.95).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/b200gemm.h"
#include "common.cuh"
#include "gemm_tile.cuh"

namespace b200 {

constexpr int kRowsThreads = 128;
constexpr int kRowsMaxTopK = 32;  // a lane of the warp holds one pair's row

template <bool kFp16>
__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const uint32_t p[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (kFp16) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&p[e]));
      f[2 * e] = v.x;
      f[2 * e + 1] = v.y;
    } else {
      f[2 * e] = __uint_as_float(p[e] << 16);
      f[2 * e + 1] = __uint_as_float(p[e] & 0xFFFF0000u);
    }
  }
}

template <bool kFp16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2_16bit(f[0], f[1], kFp16), pack2_16bit(f[2], f[3], kFp16), pack2_16bit(f[4], f[5], kFp16),
                    pack2_16bit(f[6], f[7], kFp16));
}

// lane j < top_k: the row pair (t, j) owns, or -1 (and the status bit)
__device__ __forceinline__ long long owned_row(const long long* pos, const long long* order, long long t,
                                               int top_k, long long num_rows, int lane, unsigned* status) {
  long long r = -1;
  if (lane < top_k) {
    const long long p = t * top_k + lane;
    r = pos[p];
    if (r < 0 || r >= num_rows || order[r] != p) {
      r = -1;
      if (status) atomicOr(status, kDevBadRowIndex);
    }
  }
  return r;
}

// Zeros the rows of [first, first + count) that no pair owns (count <= 32).  vb0 / kStep: the warp's first vector
// and its stride.
template <int kStep>
__device__ __forceinline__ void zero_unowned(uint4* __restrict__ dst, const long long* pos, const long long* order,
                                             long long first, int count, long long pairs, int row_vecs, int lane, int vb0) {
  bool unowned = false;
  if (lane < count) {
    const long long p = order[first + lane];
    unowned = p < 0 || p >= pairs || pos[p] != first + lane;
  }
  unsigned todo = __ballot_sync(0xFFFFFFFFu, unowned);
  while (todo) {
    const int j = __ffs(todo) - 1;
    todo &= todo - 1;
    uint4* d = dst + (first + j) * row_vecs;
    for (int v = vb0 + lane; v < row_vecs; v += kStep) d[v] = make_uint4(0, 0, 0, 0);
  }
}

// The walk all three kernels share.  A unit u is token u (u < tokens) together with the rows [u * top_k,
// (u + 1) * top_k), whose ownership it checks where the kernel writes rows; units past the tokens only check rows.
// kSpread: one unit per block, its warps share the columns (few tokens); otherwise one unit per warp.
template <bool kSpread>
struct UnitWalk {
  static constexpr int kWarps = kRowsThreads / 32;
  static constexpr int kStep = kSpread ? kRowsThreads : 32;
  int lane, vb0;
  long long first, stride;
  __device__ __forceinline__ UnitWalk() {
    lane = threadIdx.x & 31;
    vb0 = kSpread ? static_cast<int>(threadIdx.x & ~31u) : 0;
    first = kSpread ? blockIdx.x : static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    stride = kSpread ? gridDim.x : static_cast<long long>(gridDim.x) * kWarps;
  }
};

template <bool kSpread>
__global__ void __launch_bounds__(kRowsThreads)
permute_rows_kernel(const uint4* x, const long long* pos, const long long* order, uint4* __restrict__ out, long long tokens,
                    int top_k, int row_vecs, long long num_rows, long long units, unsigned* status) {
  constexpr int kStep = UnitWalk<kSpread>::kStep;
  const UnitWalk<kSpread> w;
  chain_wait();
  for (long long u = w.first; u < units; u += w.stride) {
    if (u < tokens) {
      const long long mine = owned_row(pos, order, u, top_k, num_rows, w.lane, status);
      const uint4* s = x + u * row_vecs;
      for (int vb = w.vb0; vb < row_vecs; vb += 4 * kStep) {  // the same trip count in every lane: shuffles below
        const int v = vb + w.lane;
        uint4 q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v + e * kStep < row_vecs) q[e] = s[v + e * kStep];
        for (int j = 0; j < top_k; ++j) {
          const long long r = __shfl_sync(0xFFFFFFFFu, mine, j);
          if (r < 0) continue;
          uint4* d = out + r * row_vecs;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (v + e * kStep < row_vecs) d[v + e * kStep] = q[e];
        }
      }
    }
    const long long row0 = u * top_k;
    if (row0 < num_rows)
      zero_unowned<kStep>(out, pos, order, row0, num_rows - row0 < top_k ? static_cast<int>(num_rows - row0) : top_k,
                          tokens * top_k, row_vecs, w.lane, w.vb0);
  }
}

// out[t] = sum_j w[t,j] * rows[pos[t,j]] in the order of j; weights == nullptr: all ones (the gradient of permute).
// kK rows' loads of kU vectors are issued together; top_k > kK takes further rounds (kRounds), with the rows' addresses
// fetched anew from the lanes that hold them.
template <bool kSpread, int kK, int kU, bool kRounds, bool kFp16>
__global__ void __launch_bounds__(kRowsThreads)
combine_rows_kernel(const uint4* rows, const long long* pos, const long long* order, const float* weights,
                    uint4* __restrict__ out, long long tokens, int top_k, int row_vecs, long long num_rows,
                    unsigned* status) {
  constexpr int kStep = UnitWalk<kSpread>::kStep;
  const UnitWalk<kSpread> w;
  chain_wait();
  for (long long t = w.first; t < tokens; t += w.stride) {
    const long long mine = owned_row(pos, order, t, top_k, num_rows, w.lane, status);
    const float my_weight = w.lane < top_k ? (weights ? weights[t * top_k + w.lane] : 1.f) : 0.f;
    const uint4* src[kK];   // nullptr: no row
    float wk[kK];
    auto fetch = [&](int j0) {
#pragma unroll
      for (int j = 0; j < kK; ++j) {
        const long long r = __shfl_sync(0xFFFFFFFFu, mine, (j0 + j) & 31);
        wk[j] = __shfl_sync(0xFFFFFFFFu, my_weight, (j0 + j) & 31);
        src[j] = j0 + j < top_k && r >= 0 ? rows + r * row_vecs : nullptr;
      }
    };
    if constexpr (!kRounds) fetch(0);
    for (int vb = w.vb0; vb < row_vecs; vb += kU * kStep) {
      const int v = vb + w.lane;
      float acc[kU][8];
#pragma unroll
      for (int i = 0; i < kU; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[i][e] = 0.f;
      for (int j0 = 0; j0 < (kRounds ? top_k : 1); j0 += kK) {
        if constexpr (kRounds) fetch(j0);
        uint4 q[kU][kK];
#pragma unroll
        for (int i = 0; i < kU; ++i)
#pragma unroll
          for (int j = 0; j < kK; ++j)
            if (src[j] && v + i * kStep < row_vecs) q[i][j] = src[j][v + i * kStep];
#pragma unroll
        for (int i = 0; i < kU; ++i)
#pragma unroll
          for (int j = 0; j < kK; ++j) {
            if (!src[j]) continue;
            float f[8];
            unpack8<kFp16>(q[i][j], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[i][e] = fmaf(wk[j], f[e], acc[i][e]);
          }
      }
#pragma unroll
      for (int i = 0; i < kU; ++i)
        if (v + i * kStep < row_vecs) out[t * row_vecs + v + i * kStep] = pack8<kFp16>(acc[i]);
    }
  }
}

// drows[pos[t,j]] = w[t,j] * dout[t] and dw[t,j] = <dout[t], rows[pos[t,j]]> in one pass over the rows; drows or dw
// may be nullptr (that gradient is not wanted).  A pair without a row has dw = 0.  Five blocks per SM: left alone the
// compiler takes 145 registers, three blocks and 1000 us for the case above; 4, 5 and 6 blocks 926, 909 and 952 us.
template <bool kSpread, int kK, bool kFp16>
__global__ void __launch_bounds__(kRowsThreads, 5)
combine_rows_grad_kernel(const uint4* dout, const uint4* rows, const long long* pos, const long long* order,
                         const float* weights, uint4* __restrict__ drows, float* __restrict__ dweights,
                         long long tokens, int top_k, int row_vecs, long long num_rows, long long units,
                         unsigned* status) {
  constexpr int kStep = UnitWalk<kSpread>::kStep;
  constexpr int kWarps = kRowsThreads / 32;
  __shared__ float part[kWarps][kK];
  const UnitWalk<kSpread> w;
  chain_wait();
  for (long long u = w.first; u < units; u += w.stride) {
    if (u < tokens) {
      const long long mine = owned_row(pos, order, u, top_k, num_rows, w.lane, status);
      const float my_weight = w.lane < top_k ? weights[u * top_k + w.lane] : 0.f;
      for (int j0 = 0; j0 < top_k; j0 += kK) {
        long long r[kK];
        float wk[kK], dot[kK];
#pragma unroll
        for (int j = 0; j < kK; ++j) {
          r[j] = __shfl_sync(0xFFFFFFFFu, mine, (j0 + j) & 31);
          if (j0 + j >= top_k) r[j] = -1;
          wk[j] = __shfl_sync(0xFFFFFFFFu, my_weight, (j0 + j) & 31);
          dot[j] = 0.f;
        }
        for (int v = w.vb0 + w.lane; v < row_vecs; v += kStep) {
          const uint4 qd = dout[u * row_vecs + v];
          uint4 q[kK];
          if (dweights) {
#pragma unroll
            for (int j = 0; j < kK; ++j)
              if (r[j] >= 0) q[j] = rows[r[j] * row_vecs + v];
          }
          float d[8];
          unpack8<kFp16>(qd, d);
          if (drows) {
#pragma unroll
            for (int j = 0; j < kK; ++j) {
              if (r[j] < 0) continue;
              float g[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) g[e] = wk[j] * d[e];
              drows[r[j] * row_vecs + v] = pack8<kFp16>(g);
            }
          }
          if (dweights) {
#pragma unroll
            for (int j = 0; j < kK; ++j) {
              if (r[j] < 0) continue;
              float f[8];
              unpack8<kFp16>(q[j], f);
#pragma unroll
              for (int e = 0; e < 8; ++e) dot[j] = fmaf(d[e], f[e], dot[j]);
            }
          }
        }
        if (dweights) {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < kK; ++j) {
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], o);
          }
          if constexpr (kSpread) {  // u, and with it every branch on the way here, is the same in the whole block
            if (w.lane == 0) {
#pragma unroll
              for (int j = 0; j < kK; ++j) part[threadIdx.x >> 5][j] = dot[j];
            }
            __syncthreads();
            if (threadIdx.x < kK && j0 + static_cast<int>(threadIdx.x) < top_k) {
              float sum = 0.f;
#pragma unroll
              for (int i = 0; i < kWarps; ++i) sum += part[i][threadIdx.x];
              dweights[u * top_k + j0 + threadIdx.x] = sum;
            }
            __syncthreads();
          } else if (w.lane == 0) {
#pragma unroll
            for (int j = 0; j < kK; ++j)
              if (j0 + j < top_k) dweights[u * top_k + j0 + j] = dot[j];
          }
        }
      }
    }
    const long long row0 = u * top_k;
    if (drows && row0 < num_rows)
      zero_unowned<kStep>(drows, pos, order, row0, num_rows - row0 < top_k ? static_cast<int>(num_rows - row0) : top_k,
                          tokens * top_k, row_vecs, w.lane, w.vb0);
  }
}

// ------------------------------------------------------------------ host side
struct RowsLaunch {
  bool spread;
  unsigned grid;
};

// Units spread over a block when there are fewer of them than warps the GPU holds at a quarter of its occupancy
// (16 warps per SM).
static RowsLaunch rows_launch(long long units, int sms) {
  const bool spread = units < 16ll * sms;
  const long long blocks = spread ? units : (units + kRowsThreads / 32 - 1) / (kRowsThreads / 32);
  const long long most = 64ll * sms;
  return {spread, static_cast<unsigned>(blocks < most ? blocks : most)};
}

static int check_rows(const char* who, int64_t tokens, int top_k, int hidden, int64_t num_rows, int dtype) {
  B200_REQUIRE(dtype == 0 || dtype == 1, "%s: dtype must be 0 (bf16) or 1 (fp16), got %d", who, dtype);
  B200_REQUIRE(tokens >= 0 && hidden >= 0 && num_rows >= 0, "%s: negative dimension", who);
  B200_REQUIRE(top_k >= 1 && top_k <= kRowsMaxTopK, "%s: top_k must be in [1, %d], got %d", who, kRowsMaxTopK, top_k);
  B200_REQUIRE(hidden % 8 == 0, "%s: hidden must be a multiple of 8 (16-byte vectors), got %d", who, hidden);
  return 0;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int permute_rows(const void* x, const int64_t* pos, const int64_t* order, void* out, int64_t tokens, int top_k,
                        int hidden, int64_t num_rows, cudaStream_t stream) {
  const char* who = "b200moe_permute_rows";
  if (int rc = check_rows(who, tokens, top_k, hidden, num_rows, 0)) return rc;
  if (num_rows == 0 || hidden == 0) return 0;
  B200_REQUIRE((x || tokens == 0) && (pos || tokens == 0) && order && out, "%s: null pointer", who);
  B200_REQUIRE(aligned16(x) && aligned16(out), "%s: x and out must be 16-byte aligned", who);
  const int sms = sm_count();
  B200_REQUIRE(sms > 0, "%s: no CUDA device", who);
  const long long row_units = (num_rows + top_k - 1) / top_k;
  const long long units = tokens > row_units ? tokens : row_units;
  const RowsLaunch l = rows_launch(units, sms);
  auto kern = l.spread ? permute_rows_kernel<true> : permute_rows_kernel<false>;
  B200_CUDA(launch_chained(kern, l.grid, kRowsThreads, 0, stream, static_cast<const uint4*>(x),
                           reinterpret_cast<const long long*>(pos), reinterpret_cast<const long long*>(order),
                           static_cast<uint4*>(out), tokens, top_k, hidden / 8, num_rows, units, device_status_ptr()));
  return 0;
}

template <bool kSpread, bool kFp16>
static cudaError_t launch_combine(int top_k, unsigned grid, cudaStream_t stream, const uint4* rows, const long long* pos,
                           const long long* order, const float* weights, uint4* out, long long tokens, int row_vecs,
                           long long num_rows) {
  auto kern = top_k == 1   ? combine_rows_kernel<kSpread, 1, 4, false, kFp16>
              : top_k == 2 ? combine_rows_kernel<kSpread, 2, 4, false, kFp16>
              : top_k <= 4 ? combine_rows_kernel<kSpread, 4, 2, false, kFp16>
              : top_k <= 8 ? combine_rows_kernel<kSpread, 8, 1, false, kFp16>
                           : combine_rows_kernel<kSpread, 8, 1, true, kFp16>;
  return launch_chained(kern, grid, kRowsThreads, 0, stream, rows, pos, order, weights, out, tokens, top_k, row_vecs,
                        num_rows, device_status_ptr());
}

static int combine_rows(const void* rows, const int64_t* pos, const int64_t* order, const float* weights, void* out,
                        int64_t tokens, int top_k, int hidden, int64_t num_rows, int dtype, cudaStream_t stream) {
  const char* who = "b200moe_combine_rows";
  if (int rc = check_rows(who, tokens, top_k, hidden, num_rows, dtype)) return rc;
  if (tokens == 0 || hidden == 0) return 0;
  B200_REQUIRE((rows || num_rows == 0) && pos && (order || num_rows == 0) && out, "%s: null pointer", who);
  B200_REQUIRE(aligned16(rows) && aligned16(out), "%s: rows and out must be 16-byte aligned", who);
  const int sms = sm_count();
  B200_REQUIRE(sms > 0, "%s: no CUDA device", who);
  const RowsLaunch l = rows_launch(tokens, sms);
  auto go = l.spread ? (dtype ? launch_combine<true, true> : launch_combine<true, false>)
                     : (dtype ? launch_combine<false, true> : launch_combine<false, false>);
  B200_CUDA(go(top_k, l.grid, stream, static_cast<const uint4*>(rows), reinterpret_cast<const long long*>(pos),
               reinterpret_cast<const long long*>(order), weights, static_cast<uint4*>(out), tokens, hidden / 8, num_rows));
  return 0;
}

template <bool kSpread, bool kFp16>
static cudaError_t launch_combine_grad(int top_k, unsigned grid, cudaStream_t stream, const uint4* dout, const uint4* rows,
                                const long long* pos, const long long* order, const float* weights, uint4* drows,
                                float* dweights, long long tokens, int row_vecs, long long num_rows, long long units) {
  auto kern = top_k == 1   ? combine_rows_grad_kernel<kSpread, 1, kFp16>
              : top_k == 2 ? combine_rows_grad_kernel<kSpread, 2, kFp16>
              : top_k <= 4 ? combine_rows_grad_kernel<kSpread, 4, kFp16>
                           : combine_rows_grad_kernel<kSpread, 8, kFp16>;
  return launch_chained(kern, grid, kRowsThreads, 0, stream, dout, rows, pos, order, weights, drows, dweights, tokens,
                        top_k, row_vecs, num_rows, units, device_status_ptr());
}

static int combine_rows_grad(const void* dout, const void* rows, const int64_t* pos, const int64_t* order,
                             const float* weights, void* drows, float* dweights, int64_t tokens, int top_k, int hidden,
                             int64_t num_rows, int dtype, cudaStream_t stream) {
  const char* who = "b200moe_combine_rows_grad";
  if (int rc = check_rows(who, tokens, top_k, hidden, num_rows, dtype)) return rc;
  if (!drows && !dweights) return 0;
  if (tokens == 0 && (num_rows == 0 || !drows)) return 0;
  B200_REQUIRE((dout && pos && weights) || tokens == 0, "%s: null pointer", who);
  B200_REQUIRE((order && (rows || !dweights)) || num_rows == 0, "%s: null pointer", who);
  B200_REQUIRE(aligned16(dout) && aligned16(rows) && aligned16(drows), "%s: dout, rows and drows must be 16-byte aligned", who);
  const int sms = sm_count();
  B200_REQUIRE(sms > 0, "%s: no CUDA device", who);
  const long long row_units = drows ? (num_rows + top_k - 1) / top_k : 0;
  const long long units = tokens > row_units ? tokens : row_units;
  const RowsLaunch l = rows_launch(units, sms);
  auto go = l.spread ? (dtype ? launch_combine_grad<true, true> : launch_combine_grad<true, false>)
                     : (dtype ? launch_combine_grad<false, true> : launch_combine_grad<false, false>);
  B200_CUDA(go(top_k, l.grid, stream, static_cast<const uint4*>(dout), static_cast<const uint4*>(rows),
               reinterpret_cast<const long long*>(pos), reinterpret_cast<const long long*>(order), weights,
               static_cast<uint4*>(drows), dweights, tokens, hidden / 8, num_rows, units));
  return 0;
}

}  // namespace b200

extern "C" {

int b200moe_permute_rows(const void* x, const int64_t* pos, const int64_t* order, void* out, int64_t tokens, int top_k,
                         int hidden, int64_t num_rows, void* stream) {
  return b200::permute_rows(x, pos, order, out, tokens, top_k, hidden, num_rows, static_cast<cudaStream_t>(stream));
}

int b200moe_combine_rows(const void* rows, const int64_t* pos, const int64_t* order, const float* weights, void* out,
                         int64_t tokens, int top_k, int hidden, int64_t num_rows, int dtype, void* stream) {
  return b200::combine_rows(rows, pos, order, weights, out, tokens, top_k, hidden, num_rows, dtype,
                            static_cast<cudaStream_t>(stream));
}

int b200moe_combine_rows_grad(const void* dout, const void* rows, const int64_t* pos, const int64_t* order,
                              const float* weights, void* drows, float* dweights, int64_t tokens, int top_k, int hidden,
                              int64_t num_rows, int dtype, void* stream) {
  return b200::combine_rows_grad(dout, rows, pos, order, weights, drows, dweights, tokens, top_k, hidden, num_rows, dtype,
                                 static_cast<cudaStream_t>(stream));
}

}  // extern "C"
