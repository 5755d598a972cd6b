// Norm of every query and key head, rotation by position, and the write of K and V into their page
// slots, in one pass over the new tokens (include/argus_hip.h, argus_hip_qk_norm_rope).
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + b);   (a, b) -> (a cos - b sin, b cos + a sin)
//
// D / 8 lanes share a head; a lane holds the two groups of four channels that rotate into each other
// (4i .. 4i+3 and rot/2 + 4i .., or 8i .. 8i+7 with adjacent pairs), so the rotation needs no exchange
// and the norm one reduction over the head's lanes.  Bound by HBM for many tokens, by the launch for few.
#include "paged_common.hpp"

#include <type_traits>

namespace {

struct QkNormRopeParams {
  const void *q, *k, *v;
  const float *q_weight, *k_weight, *cos_sin;
  const int32_t *positions, *slots;
  void *q_out, *k_cache, *v_cache;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  PoolStrides pool;
  int32_t heads_q, heads_kv, rot_dim, interleaved, n_positions, n_slots, page_shift;
  int32_t chunks;  // workgroups per token
  float eps, weight_bias;
};

__device__ __forceinline__ void load4(const float *p, float (&x)[4]) {
  const float4_t v = *(const float4_t *)p;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = v[e];
}
__device__ __forceinline__ void load4(const _Float16 *p, float (&x)[4]) {
  const half4_t v = *(const half4_t *)p;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (float)v[e];
}
__device__ __forceinline__ void store4(float *p, const float (&x)[4]) { *(float4_t *)p = float4_t{x[0], x[1], x[2], x[3]}; }
__device__ __forceinline__ void store4(_Float16 *p, const float (&x)[4]) {
  *(half4_t *)p = half4_t{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}

template <int D, typename IN, typename OUT>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const QkNormRopeParams p) {
  constexpr int LPH = D / 8;            // lanes per head
  constexpr int HPB = 256 / LPH;        // heads per workgroup
  const int token = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int u = chunk * HPB + threadIdx.x / LPH;  // query heads, key heads, value heads
  const int i = threadIdx.x % LPH;
  const int pos = p.positions ? p.positions[token] : 0;
  if (pos < 0 || (p.rot_dim > 0 && pos >= p.n_positions)) return;  // padding
  if (u >= p.heads_q + 2 * p.heads_kv) return;                     // whole heads: no lane of a head's reduction is missing
  const bool is_q = u < p.heads_q, is_v = u >= p.heads_q + p.heads_kv;
  const int h = is_q ? u : is_v ? u - p.heads_q - p.heads_kv : u - p.heads_q;

  // channels of this lane
  const int half = p.rot_dim / 2;
  int c0, c1;
  bool turn;
  if (p.interleaved) {
    c0 = 8 * i, c1 = c0 + 4;
    turn = c0 < p.rot_dim;
  } else {
    turn = 4 * i < half;
    c0 = turn ? 4 * i : 8 * i;  // lanes past half / 4: the channels behind rot_dim, eight in a row
    c1 = turn ? c0 + half : c0 + 4;
  }
  const IN *src = is_q ? (const IN *)p.q + token * p.q_stride : is_v ? (const IN *)p.v + token * p.v_stride : (const IN *)p.k + token * p.k_stride;
  src += (int64_t)h * D;
  float a[4], b[4];
  load4(src + c0, a);
  load4(src + c1, b);

  if (!is_v) {
    const float *w = is_q ? p.q_weight : p.k_weight;
    if (w) {
      float sq = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) sq += a[e] * a[e] + b[e] * b[e];
      sq = group_allreduce_sum<LPH>(sq);
      const float inv = 1.0f / sqrtf(sq * (1.0f / D) + p.eps);
      float wa[4], wb[4];
      load4(w + c0, wa);
      load4(w + c1, wb);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = a[e] * inv * (wa[e] + p.weight_bias);
        b[e] = b[e] * inv * (wb[e] + p.weight_bias);
      }
    }
    if (turn) {
      const float *row = p.cos_sin + (int64_t)pos * p.rot_dim;
      const int j = 4 * i;  // first of this lane's four angles
      float cs[4], sn[4];
      load4(row + j, cs);
      load4(row + half + j, sn);
      if (p.interleaved) {
        float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float r = x[2 * e] * cs[e] - x[2 * e + 1] * sn[e], s = x[2 * e + 1] * cs[e] + x[2 * e] * sn[e];
          x[2 * e] = r;
          x[2 * e + 1] = s;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = x[e], b[e] = x[4 + e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float r = a[e] * cs[e] - b[e] * sn[e], s = b[e] * cs[e] + a[e] * sn[e];
          a[e] = r;
          b[e] = s;
        }
      }
    }
  }
  if (is_q) {
    OUT *dst = (OUT *)p.q_out + token * p.q_out_stride + (int64_t)h * D;
    store4(dst + c0, a);
    store4(dst + c1, b);
  } else {
    const int slot = p.slots[token];
    if ((uint32_t)slot >= (uint32_t)p.n_slots) return;
    const int page = slot >> p.page_shift, row = slot & ((1 << p.page_shift) - 1);
    _Float16 *dst = (_Float16 *)(is_v ? p.v_cache : p.k_cache) + page * p.pool.page + h * p.pool.head + row * p.pool.row;
    store4(dst + c0, a);
    store4(dst + c1, b);
  }
}

template <int D, typename IN>
int launch(argus_hip_ctx *ctx, QkNormRopeParams &p, int tokens, bool out_f16, hipStream_t stream) {
  constexpr int HPB = 256 / (D / 8);
  p.chunks = (p.heads_q + 2 * p.heads_kv + HPB - 1) / HPB;
  const int64_t grid = (int64_t)tokens * p.chunks;
  if (grid > 0x7fffffff) return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "qk_norm_rope: too many tokens");
  if (out_f16) hipLaunchKernelGGL((qk_norm_rope_kernel<D, IN, _Float16>), dim3((unsigned)grid), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<D, IN, float>), dim3((unsigned)grid), dim3(256), 0, stream, p);
  ARGUS_HIP_CHECK(ctx, hipGetLastError());
  return ARGUS_HIP_OK;
}

template <int D>
int launch(argus_hip_ctx *ctx, QkNormRopeParams &p, int tokens, bool in_f16, bool out_f16, hipStream_t stream) {
  return in_f16 ? launch<D, _Float16>(ctx, p, tokens, out_f16, stream) : launch<D, float>(ctx, p, tokens, out_f16, stream);
}

}  // namespace

ARGUS_API int argus_hip_qk_norm_rope(argus_hip_ctx *ctx, const argus_hip_qk_norm_rope_args *a) {
  if (!ctx || !a) return ARGUS_HIP_ERR_INVALID;
  if (a->tokens < 0 || a->heads_q <= 0 || a->heads_kv <= 0 || a->n_pages <= 0 || a->n_positions < 0)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: tokens %d heads %d / %d n_pages %d n_positions %d", a->tokens, a->heads_q,
                      a->heads_kv, a->n_pages, a->n_positions);
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "qk_norm_rope: head_dim %d is not 64, 128 or 256", a->head_dim);
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 8)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: rot_dim %d is not a multiple of 8 up to head_dim %d", a->rot_dim, a->head_dim);
  if (!argus_page_size_ok(a->page_size))
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "qk_norm_rope: page_size %d is not a power of two from 16 to %d", a->page_size,
                      ARGUS_HIP_MAX_PAGE_SIZE);
  if ((int64_t)a->n_pages * a->page_size > 0x7fffffff)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: %d pages of %d tokens are more than 2^31 - 1 slots", a->n_pages, a->page_size);
  if (a->layout != ARGUS_HIP_HEAD_MAJOR && a->layout != ARGUS_HIP_SEQ_MAJOR)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: layout %d", a->layout);
  const auto float_type = [](int t) { return t == ARGUS_HIP_F32 || t == ARGUS_HIP_F16; };
  if (!float_type(a->in_dtype) || !float_type(a->out_dtype))
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "qk_norm_rope: dtypes %d -> %d", a->in_dtype, a->out_dtype);
  if (a->tokens == 0) return ARGUS_HIP_OK;
  if (!a->q || !a->k || !a->v || !a->q_out || !a->k_cache || !a->v_cache || !a->slots || (a->rot_dim && (!a->cos_sin || !a->positions)))
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: null pointer");
  const int d = a->head_dim;
  QkNormRopeParams p{};
  p.q_stride = a->q_stride ? a->q_stride : (int64_t)a->heads_q * d;
  p.k_stride = a->k_stride ? a->k_stride : (int64_t)a->heads_kv * d;
  p.v_stride = a->v_stride ? a->v_stride : (int64_t)a->heads_kv * d;
  p.q_out_stride = a->q_out_stride ? a->q_out_stride : (int64_t)a->heads_q * d;
  if ((p.q_stride | p.k_stride | p.v_stride | p.q_out_stride) % 4 || p.q_stride < 0 || p.k_stride < 0 || p.v_stride < 0 || p.q_out_stride < 0)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: row strides are non-negative multiples of 4 elements");
  const uintptr_t in_mask = a->in_dtype == ARGUS_HIP_F16 ? 7 : 15, out_mask = a->out_dtype == ARGUS_HIP_F16 ? 7 : 15;
  if ((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v) & in_mask) || ((uintptr_t)a->q_out & out_mask) ||
      (((uintptr_t)a->k_cache | (uintptr_t)a->v_cache) & 15) ||
      (((uintptr_t)a->q_weight | (uintptr_t)a->k_weight | (uintptr_t)a->cos_sin) & 15))
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: a pointer is not aligned to four elements (pools, weights, cos_sin: 16 bytes)");
  const DeviceGuard guard(ctx);
  p.q = a->q, p.k = a->k, p.v = a->v, p.q_weight = a->q_weight, p.k_weight = a->k_weight, p.cos_sin = a->cos_sin;
  p.positions = a->positions, p.slots = a->slots, p.q_out = a->q_out, p.k_cache = a->k_cache, p.v_cache = a->v_cache;
  p.pool = argus_pool_strides(a->layout, a->heads_kv, a->page_size, d);
  p.heads_q = a->heads_q, p.heads_kv = a->heads_kv, p.rot_dim = a->rot_dim, p.interleaved = a->interleaved != 0;
  p.n_positions = a->n_positions, p.n_slots = a->n_pages * a->page_size, p.page_shift = argus_log2(a->page_size);
  p.eps = a->eps, p.weight_bias = a->weight_bias;
  const bool in_f16 = a->in_dtype == ARGUS_HIP_F16, out_f16 = a->out_dtype == ARGUS_HIP_F16;
  const hipStream_t stream = (hipStream_t)a->stream;
  switch (d) {
    case 64: return launch<64>(ctx, p, a->tokens, in_f16, out_f16, stream);
    case 128: return launch<128>(ctx, p, a->tokens, in_f16, out_f16, stream);
    default: return launch<256>(ctx, p, a->tokens, in_f16, out_f16, stream);
  }
}
