// Norm of every query and key head, rotation by position, and the write of K and V into their page
// slots, in one pass over the new tokens (include/argus_hip.h, argus_hip_qk_norm_rope).
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + b);   (a, b) -> (a cos - b sin, b cos + a sin)
//
// A lane holds the two groups of W channels that rotate into each other (W i .. and rot/2 + W i .., or
// 2 W i .. 2 W i + 2 W - 1 with adjacent pairs), so the rotation needs no exchange and the norm one
// reduction over the head's lanes; W = 8, or 4 where alignment or rot_dim asks for it.  Bound by HBM for many tokens (8192 of 32/8 heads, d 128,
// F16: 40.3 us, 5.1 TB/s), by the launch for few (16 in F32: 3.5 us).
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

// W consecutive channels (4, or 8 from two loads of a 4-byte type) as F32
template <int W>
__device__ __forceinline__ void load(const float *p, float (&x)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const float4_t v = *(const float4_t *)(p + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i + e] = v[e];
  }
}
template <int W>
__device__ __forceinline__ void load(const _Float16 *p, float (&x)[W]) {
  typedef _Float16 half_w __attribute__((ext_vector_type(W)));
  const half_w v = *(const half_w *)p;
#pragma unroll
  for (int e = 0; e < W; ++e) x[e] = (float)v[e];
}
template <int W>
__device__ __forceinline__ void store(float *p, const float (&x)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 4) *(float4_t *)(p + i) = float4_t{x[i], x[i + 1], x[i + 2], x[i + 3]};
}
template <int W>
__device__ __forceinline__ void store(_Float16 *p, const float (&x)[W]) {
  typedef _Float16 half_w __attribute__((ext_vector_type(W)));
  half_w v;
#pragma unroll
  for (int e = 0; e < W; ++e) v[e] = (_Float16)x[e];
  *(half_w *)p = v;
}

// W: channels per group; a lane holds two groups, D / (2 W) lanes a head.
template <int D, int W, typename IN, typename OUT>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const QkNormRopeParams p) {
  constexpr int LPH = D / (2 * W);      // lanes per head
  constexpr int HPB = 256 / LPH;        // heads per workgroup and turn
  const int token = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int i = threadIdx.x % LPH;
  const int pos = p.positions ? p.positions[token] : 0;
  if (pos < 0 || (p.rot_dim > 0 && pos >= p.n_positions)) return;  // padding

  // channels of this lane
  const int half = p.rot_dim / 2;
  int c0, c1;
  bool turn;
  if (p.interleaved) {
    c0 = 2 * W * i, c1 = c0 + W;
    turn = c0 < p.rot_dim;
  } else {
    turn = W * i < half;
    c0 = turn ? W * i : 2 * W * i;  // lanes past half / W: the channels behind rot_dim, 2 W in a row
    c1 = turn ? c0 + half : c0 + W;
  }
  float cs[W], sn[W];
  if (turn) {
    const float *row = p.cos_sin + (int64_t)pos * p.rot_dim + W * i;
    load<W>(row, cs);
    load<W>(row + half, sn);
  }
  const int units = p.heads_q + 2 * p.heads_kv;  // query heads, key heads, value heads
  for (int u = chunk * HPB + threadIdx.x / LPH; u < units; u += p.chunks * HPB) {  // whole heads: no lane of a head's sum is missing
    const bool is_q = u < p.heads_q, is_v = u >= p.heads_q + p.heads_kv;
    const int h = is_q ? u : is_v ? u - p.heads_q - p.heads_kv : u - p.heads_q;
    const IN *src = is_q ? (const IN *)p.q + token * p.q_stride : is_v ? (const IN *)p.v + token * p.v_stride : (const IN *)p.k + token * p.k_stride;
    src += (int64_t)h * D;
    float a[W], b[W];
    load<W>(src + c0, a);
    load<W>(src + c1, b);
    if (!is_v) {
      const float *w = is_q ? p.q_weight : p.k_weight;
      if (w) {
        float sq = 0.0f;
#pragma unroll
        for (int e = 0; e < W; ++e) sq += a[e] * a[e] + b[e] * b[e];
        sq = group_allreduce_sum<LPH>(sq);
        const float inv = 1.0f / sqrtf(sq * (1.0f / D) + p.eps);
        float wa[W], wb[W];
        load<W>(w + c0, wa);
        load<W>(w + c1, wb);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          a[e] = a[e] * inv * (wa[e] + p.weight_bias);
          b[e] = b[e] * inv * (wb[e] + p.weight_bias);
        }
      }
      if (turn) {
        if (p.interleaved) {
          float x[2 * W];
#pragma unroll
          for (int e = 0; e < W; ++e) x[e] = a[e], x[W + e] = b[e];
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const float r = x[2 * e] * cs[e] - x[2 * e + 1] * sn[e], s = x[2 * e + 1] * cs[e] + x[2 * e] * sn[e];
            x[2 * e] = r;
            x[2 * e + 1] = s;
          }
#pragma unroll
          for (int e = 0; e < W; ++e) a[e] = x[e], b[e] = x[W + e];
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const float r = a[e] * cs[e] - b[e] * sn[e], s = b[e] * cs[e] + a[e] * sn[e];
            a[e] = r;
            b[e] = s;
          }
        }
      }
    }
    if (is_q) {
      OUT *dst = (OUT *)p.q_out + token * p.q_out_stride + (int64_t)h * D;
      store<W>(dst + c0, a);
      store<W>(dst + c1, b);
    } else {
      const int slot = p.slots[token];
      if ((uint32_t)slot >= (uint32_t)p.n_slots) continue;
      const int page = slot >> p.page_shift, row = slot & ((1 << p.page_shift) - 1);
      _Float16 *dst = (_Float16 *)(is_v ? p.v_cache : p.k_cache) + page * p.pool.page + h * p.pool.head + row * p.pool.row;
      store<W>(dst + c0, a);
      store<W>(dst + c1, b);
    }
  }
}

template <int D, int W, typename IN, typename OUT>
int launch(argus_hip_ctx *ctx, QkNormRopeParams &p, int tokens, hipStream_t stream) {
  constexpr int HPB = 256 / (D / (2 * W));
  // few tokens: a token's heads over several workgroups, for shorter chains; many: one, which loads the angles once
  const int chunks = (p.heads_q + 2 * p.heads_kv + HPB - 1) / HPB;
  p.chunks = (int64_t)tokens * chunks <= (int64_t)ctx->compute_units * 8 ? chunks : 1;
  const int64_t grid = (int64_t)tokens * p.chunks;
  if (grid > 0x7fffffff) return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "qk_norm_rope: too many tokens");
  hipLaunchKernelGGL((qk_norm_rope_kernel<D, W, IN, OUT>), dim3((unsigned)grid), dim3(256), 0, stream, p);
  ARGUS_HIP_CHECK(ctx, hipGetLastError());
  return ARGUS_HIP_OK;
}

template <int D, typename IN>
int launch(argus_hip_ctx *ctx, QkNormRopeParams &p, int tokens, bool wide, bool out_f16, hipStream_t stream) {
  if (wide) return out_f16 ? launch<D, 8, IN, _Float16>(ctx, p, tokens, stream) : launch<D, 8, IN, float>(ctx, p, tokens, stream);
  return out_f16 ? launch<D, 4, IN, _Float16>(ctx, p, tokens, stream) : launch<D, 4, IN, float>(ctx, p, tokens, stream);
}

template <int D>
int launch(argus_hip_ctx *ctx, QkNormRopeParams &p, int tokens, bool wide, bool in_f16, bool out_f16, hipStream_t stream) {
  return in_f16 ? launch<D, _Float16>(ctx, p, tokens, wide, out_f16, stream) : launch<D, float>(ctx, p, tokens, wide, out_f16, stream);
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
  if (a->tokens > 1 && p.q_out_stride < (int64_t)a->heads_q * d)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: rows of q_out overlap (q_out_stride %lld)", (long long)p.q_out_stride);
  if (a->q_out == a->q && (a->in_dtype != a->out_dtype || (a->tokens > 1 && p.q_stride != p.q_out_stride)))
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "qk_norm_rope: q in place takes one type and one stride");
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
  // groups of eight channels (16-byte accesses of F16) where the rotation's halves and every row allow it
  const bool wide = a->rot_dim % 16 == 0 && (p.q_stride | p.k_stride | p.v_stride | p.q_out_stride) % 8 == 0 &&
                    (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out) & 15) == 0;
  switch (d) {
    case 64: return launch<64>(ctx, p, a->tokens, wide, in_f16, out_f16, stream);
    case 128: return launch<128>(ctx, p, a->tokens, wide, in_f16, out_f16, stream);
    default: return launch<256>(ctx, p, a->tokens, wide, in_f16, out_f16, stream);
  }
}
