// The kernels of paged_attention for one head_dim and their launches; see paged_attn.hip for the call.
//
// Requests of at most 16 rows (tokens x heads of a group) take the decode form (paged_decode.hpp, bound by
// HBM), the others the chunk form (paged_chunk.hpp, bound by the matrix cores).  A call with both runs them in
// one launch, the decode shares first, one per compute unit, so that they and the first chunk shares overlap.
// Against a launch of each, 46 single tokens and two chunks (14/2 heads, d 64, F32) took 71 instead of 83 us;
// with the care for values outside F16's range that was added since, 74 us.
// Dividing the resident workgroups between the two by their estimated times, and workgroups of the two in
// turn, won as much where the estimate was right and lost up to twice that elsewhere.
#pragma once

#include "paged_chunk.hpp"
#include "paged_decode.hpp"

#include <algorithm>
#include <type_traits>

namespace argus_paged {

namespace {

template <int D, typename T, bool CAP>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_decode_kernel(const PagedParams p) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int w = blockIdx.x / p.heads_kv;
  decode_share<D, T, CAP, 0>(p, PagedShare(p.sched, p.cu_new, p.kv_len, w), w, blockIdx.x % p.heads_kv, (float *)lds);
}

template <int D, typename T, bool CAP>
__global__ __launch_bounds__(256, (ChunkTile<D, std::is_same<T, float>::value>::WAVES_PER_SIMD)) void paged_chunk_kernel(const PagedParams p) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int w = blockIdx.x / p.heads_kv;
  chunk_share<D, T, CAP, 0>(p, PagedShare(p.sched, p.cu_new, p.kv_len, w), w, blockIdx.x % p.heads_kv, (_Float16 *)lds);
}

// Both forms: the decode shares first, then the chunk shares as compute units get free.
template <int D, typename T, bool CAP>
__global__ __launch_bounds__(256, (ChunkTile<D, std::is_same<T, float>::value>::WAVES_PER_SIMD)) void paged_mixed_kernel(const PagedParams dp, const PagedParams cp) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int g = blockIdx.x / dp.heads_kv, kvh = blockIdx.x % dp.heads_kv, w = g - dp.items;
  if (w < 0) decode_share<D, T, CAP, 0>(dp, PagedShare(dp.sched, dp.cu_new, dp.kv_len, g), g, kvh, (float *)lds);
  else chunk_share<D, T, CAP, 1>(cp, PagedShare(cp.sched, cp.cu_new, cp.kv_len, w), w, kvh, (_Float16 *)lds);
}

// Four channels of an output row; a row that saw nothing is zeros.
template <typename T>
__device__ __forceinline__ void store_row(T *out, const float4_t &o, float l) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (T)(l == 0.0f ? 0.0f : o[e] / l);
  *(T4 *)out = y;
}

// Merge of the parts of cut tiles: row m of a tile is sum_i o_i 2^(m_i - m) / sum_i l_i 2^(m_i - m).  One
// share begins a cut tile at most, its last one.  D / 4 threads share a row's channels.  Decode tiles have few
// rows and up to hundreds of parts: a workgroup takes one row, its thread groups every PG-th part, and the
// groups are added in LDS.  Chunk tiles have many rows of two or three parts: two rows per thread.  Bound by
// the latency of its loads: the descriptor, then everything else at once.
template <int D, typename T, bool DECODE>
__device__ __forceinline__ void combine_cut(const PagedParams &p, int block) {
  constexpr int TPR = D / 4, PG = 256 / TPR;
  constexpr int R = DECODE ? kDecodeRows : kChunkRows, RPB = DECODE ? 1 : 2 * PG;
  constexpr int blocks = R / RPB;
  static_assert(R % RPB == 0, "whole workgroups per tile");
  typedef float float2_t __attribute__((ext_vector_type(2)));
  const int w = block / (blocks * p.heads_kv), kvh = block / blocks % p.heads_kv;
  const PagedCut cut = p.cuts[w];
  const int first = block % blocks * RPB, group = threadIdx.x / TPR, ch = threadIdx.x % TPR * 4;
  if (cut.parts == 0 || first >= cut.rows) return;  // the whole workgroup
  const int G = p.sched.group, n = cut.parts;
  // parts: slot 2 w + 1, then 2 (w + 1), 2 (w + 2), ..
  const int64_t step = (int64_t)p.heads_kv * R;
  auto part = [&](int i, int row) { return (int64_t)(2 * (w + i) + (i == 0)) * step + (int64_t)kvh * R + row; };
  auto out = [&](int row) { return (T *)p.out + (int64_t)(cut.q_begin + row / G) * p.out_stride + (int64_t)(kvh * G + row % G) * D + ch; };
  if constexpr (DECODE) {
    constexpr int AHEAD = 4;
    const int lane = threadIdx.x & 63;
    float4_t x[AHEAD];  // this group's first parts (behind the last one: that again)
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (u * PG < n) x[u] = *(const float4_t *)(p.ws_o + part(min(u * PG + group, n - 1), first) * D + ch);
    float2_t ml = {kNegInf, 0.0f};  // of part `lane`, every wave for itself
    if (lane < n) ml = *(const float2_t *)(p.ws_ml + part(lane, first) * 2);
    float m = ml[0];
    for (int i = lane + 64; i < n; i += 64) m = fmaxf(m, p.ws_ml[part(i, first) * 2]);
    m = wave_allreduce_max(m);
    const float m_ref = m == kNegInf ? 0.0f : m;
    const float f64 = __builtin_amdgcn_exp2f(ml[0] - m_ref);  // factors of the first 64 parts
    float l = ml[1] * f64;
    for (int i = lane + 64; i < n; i += 64) l += p.ws_ml[part(i, first) * 2 + 1] * __builtin_amdgcn_exp2f(p.ws_ml[part(i, first) * 2] - m_ref);
    l = wave_allreduce_sum(l);
    float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (u * PG < n) {  // AHEAD * PG <= 64
        const int i = u * PG + group;
        const float f = __shfl(f64, i, 64);
        if (i < n) o += x[u] * f;
      }
#pragma unroll 4
    for (int i = AHEAD * PG + group; i < n; i += PG) {
      const int64_t at = part(i, first);
      o += *(const float4_t *)(p.ws_o + at * D + ch) * __builtin_amdgcn_exp2f(p.ws_ml[at * 2] - m_ref);
    }
    __shared__ float4_t sum[256];
    sum[threadIdx.x] = o;
    __syncthreads();
    if (threadIdx.x >= TPR) return;
#pragma unroll
    for (int g = 1; g < PG; ++g) o += sum[g * TPR + threadIdx.x];
    store_row(out(cut.row0 + first), o, l);
  } else {
    float4_t x[2][2];
    float2_t ml[2][2];
    int row[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      row[k] = first + k * PG + group;
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // a cut tile has two parts at least
        const int64_t at = part(i, min(row[k], cut.rows - 1));
        x[k][i] = *(const float4_t *)(p.ws_o + at * D + ch);
        ml[k][i] = *(const float2_t *)(p.ws_ml + at * 2);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float m = kNegInf, l = 0.0f;
      float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
      auto add = [&](const float4_t &xi, const float2_t &mli) {
        const float m_new = fmaxf(m, mli[0]), m_ref = m_new == kNegInf ? 0.0f : m_new;
        const float old = __builtin_amdgcn_exp2f(m - m_ref), f = __builtin_amdgcn_exp2f(mli[0] - m_ref);
        m = m_new;
        l = l * old + mli[1] * f;
        o = o * old + xi * f;
      };
      add(x[k][0], ml[k][0]);
      add(x[k][1], ml[k][1]);
      for (int i = 2; i < n; ++i) {
        const int64_t at = part(i, min(row[k], cut.rows - 1));
        add(*(const float4_t *)(p.ws_o + at * D + ch), *(const float2_t *)(p.ws_ml + at * 2));
      }
      if (row[k] < cut.rows) store_row(out(cut.row0 + row[k]), o, l);
    }
  }
}

template <int D, bool DECODE>
constexpr int kCutBlocks = DECODE ? kDecodeRows : kChunkRows / (2 * (256 / (D / 4)));  // workgroups per cut and KV head

template <int D, typename T, bool DECODE>
__global__ __launch_bounds__(256) void paged_combine_kernel(const PagedParams p) {
  combine_cut<D, T, DECODE>(p, blockIdx.x);
}
template <int D, typename T>
__global__ __launch_bounds__(256) void paged_combine_both_kernel(const PagedParams dp, const PagedParams cp) {
  const int chunk_blocks = (cp.sched.target - 1) * cp.heads_kv * kCutBlocks<D, false>;
  if ((int)blockIdx.x < chunk_blocks) combine_cut<D, T, false>(cp, blockIdx.x);
  else combine_cut<D, T, true>(dp, blockIdx.x - chunk_blocks);
}

// dp, cp: the two forms' parameters; items 0: the form is not there
template <int D, typename T, bool CAP>
int launch_call(argus_hip_ctx *ctx, const PagedParams &dp, const PagedParams &cp, KernelTimer &timer, hipStream_t stream) {
  constexpr int chunk_lds = ChunkTile<D, std::is_same<T, float>::value>::LDS_BYTES, decode_lds = kDecodeLds<D>;
  const bool dcut = dp.items && dp.cuts, ccut = cp.items && cp.cuts;
  const unsigned dgrid = (unsigned)(dp.items * dp.heads_kv), cgrid = (unsigned)(cp.items * cp.heads_kv);
  if (dp.items && cp.items) {
    constexpr int lds = chunk_lds > decode_lds ? chunk_lds : decode_lds;
    auto kern = paged_mixed_kernel<D, T, CAP>;
    ARGUS_HIP_CHECK(ctx, argus_raise_lds_limit(ctx, kern, lds));
    hipLaunchKernelGGL(kern, dim3(dgrid + cgrid), dim3(256), lds, stream, dp, cp);
  } else if (dp.items) {
    auto kern = paged_decode_kernel<D, T, CAP>;
    ARGUS_HIP_CHECK(ctx, argus_raise_lds_limit(ctx, kern, decode_lds));
    hipLaunchKernelGGL(kern, dim3(dgrid), dim3(256), decode_lds, stream, dp);
  } else {
    auto kern = paged_chunk_kernel<D, T, CAP>;
    ARGUS_HIP_CHECK(ctx, argus_raise_lds_limit(ctx, kern, chunk_lds));
    hipLaunchKernelGGL(kern, dim3(cgrid), dim3(256), chunk_lds, stream, cp);
  }
  ARGUS_HIP_CHECK(ctx, hipGetLastError());
  timer.mark();
  const unsigned dcuts = dcut ? (dp.sched.target - 1) * dp.heads_kv * kCutBlocks<D, true> : 0;
  const unsigned ccuts = ccut ? (cp.sched.target - 1) * cp.heads_kv * kCutBlocks<D, false> : 0;
  if (dcuts && ccuts) hipLaunchKernelGGL((paged_combine_both_kernel<D, T>), dim3(dcuts + ccuts), dim3(256), 0, stream, dp, cp);
  else if (dcuts) hipLaunchKernelGGL((paged_combine_kernel<D, T, true>), dim3(dcuts), dim3(256), 0, stream, dp);
  else if (ccuts) hipLaunchKernelGGL((paged_combine_kernel<D, T, false>), dim3(ccuts), dim3(256), 0, stream, cp);
  ARGUS_HIP_CHECK(ctx, hipGetLastError());
  return ARGUS_HIP_OK;
}

template <int D>
int launch_call(argus_hip_ctx *ctx, const PagedParams &dp, const PagedParams &cp, bool f32, bool cap, hipStream_t stream) {
  KernelTimer timer(ctx, stream);
  if (f32) return cap ? launch_call<D, float, true>(ctx, dp, cp, timer, stream) : launch_call<D, float, false>(ctx, dp, cp, timer, stream);
  return cap ? launch_call<D, _Float16, true>(ctx, dp, cp, timer, stream) : launch_call<D, _Float16, false>(ctx, dp, cp, timer, stream);
}

}  // namespace

}  // namespace argus_paged
