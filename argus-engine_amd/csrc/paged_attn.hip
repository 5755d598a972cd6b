// Causal GQA attention of the new tokens of many requests over their pages (include/argus_hip.h,
// argus_hip_paged_attention).
//
//   s_c = cap((q . k_c) * scale) for the visible keys c of a row;  out = sum_c softmax(s)_c v_c
//
// One wave per (token, query head): 64 keys per step, one lane per key for the logits, one lane per
// D / 64 channels for the weighted sum, running maximum and sum in F32.
#include "paged_common.hpp"

#include <algorithm>
#include <type_traits>

namespace {

struct PagedParams {
  const void *q;
  const _Float16 *k, *v;
  const int32_t *page_table, *cu_new, *kv_len;
  void *out;
  int64_t q_stride, out_stride;
  PoolStrides pool;
  int32_t n_seqs, n_tokens, heads_q, heads_kv, group, n_pages, page_shift, table_stride, window;
  float softcap, scale;
};

template <int D, typename T>
__global__ __launch_bounds__(64) void paged_row_kernel(const PagedParams p) {
  const int h = blockIdx.x % p.heads_q, token = blockIdx.x / p.heads_q, lane = threadIdx.x;
  if (token >= p.cu_new[p.n_seqs]) return;
  int lo = 0, hi = p.n_seqs;  // the request with cu_new[lo] <= token < cu_new[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_new[mid] <= token) lo = mid;
    else hi = mid;
  }
  const int len = min(max(p.kv_len[lo], 0), (int)min((int64_t)p.table_stride << p.page_shift, (int64_t)0x7fffffff));
  const int pos = p.kv_len[lo] - (p.cu_new[lo + 1] - token);
  const int end = min(pos + 1, len);
  const int begin = p.window > 0 ? max(0, pos - p.window + 1) : 0;

  __shared__ float q_lds[D];
  __shared__ float p_lds[64];
  const T *q = (const T *)p.q + token * p.q_stride + (int64_t)h * D;
  for (int c = lane; c < D; c += 64) q_lds[c] = (float)q[c];
  __syncthreads();
  const int64_t head_off = (int64_t)(h / p.group) * p.pool.head;
  const int32_t *table = p.page_table + (int64_t)lo * p.table_stride;
  auto row_of = [&](int key) -> int64_t {  // element offset of a key's row, -1: not in the pool
    const int page = table[key >> p.page_shift];
    if ((uint32_t)page >= (uint32_t)p.n_pages) return -1;
    return page * p.pool.page + head_off + (key & ((1 << p.page_shift) - 1)) * p.pool.row;
  };
  float m = kNegInf, l = 0.0f, o[D / 64];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) o[c] = 0.0f;
  for (int base = begin; base < end; base += 64) {
    float s = kNegInf;
    if (base + lane < end) {
      const int64_t off = row_of(base + lane);
      s = 0.0f;
      if (off >= 0)
        for (int c = 0; c < D; c += 8) {
          const half8_t kv = *(const half8_t *)(p.k + off + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) s += q_lds[c + e] * (float)kv[e];
        }
      s *= p.scale;
      if (p.softcap > 0.0f) s = p.softcap * tanhf(s / p.softcap);
    }
    const float m_new = fmaxf(m, wave_allreduce_max(s));
    const float m_ref = m_new == kNegInf ? 0.0f : m_new;
    const float w = expf(s - m_ref), alpha = expf(m - m_ref);
    l = l * alpha + wave_allreduce_sum(w);
    m = m_new;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) o[c] *= alpha;
    p_lds[lane] = w;
    __syncthreads();
    const int n = min(64, end - base);
    for (int t = 0; t < n; ++t) {
      const int64_t off = row_of(base + t);
      if (off < 0) continue;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) o[c] += p_lds[t] * (float)p.v[off + c * 64 + lane];
    }
    __syncthreads();
  }
  T *out = (T *)p.out + token * p.out_stride + (int64_t)h * D;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) out[c * 64 + lane] = (T)(l == 0.0f ? 0.0f : o[c] / l);
}

int check(argus_hip_ctx *ctx, const argus_hip_paged_attention_args *a) {
  if (a->n_seqs < 0 || a->n_tokens < 0 || a->heads_q <= 0 || a->heads_kv <= 0 || a->heads_q % a->heads_kv || a->n_pages <= 0 ||
      a->table_stride <= 0)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: n_seqs %d n_tokens %d heads %d / %d n_pages %d table_stride %d", a->n_seqs,
                      a->n_tokens, a->heads_q, a->heads_kv, a->n_pages, a->table_stride);
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: head_dim %d is not 64, 128 or 256", a->head_dim);
  if (!argus_page_size_ok(a->page_size))
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: page_size %d is not a power of two from 16 to %d", a->page_size,
                      ARGUS_HIP_MAX_PAGE_SIZE);
  if (a->layout != ARGUS_HIP_HEAD_MAJOR && a->layout != ARGUS_HIP_SEQ_MAJOR)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: layout %d", a->layout);
  if (a->dtype != ARGUS_HIP_F32 && a->dtype != ARGUS_HIP_F16)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: dtype %d", a->dtype);
  if (a->window < 0 || a->min_new < 0 || a->max_new < 0 || a->max_kv < 0 || !(a->softcap >= 0.0f) || !(a->softcap < __builtin_huge_valf()) ||
      !(a->scale > -__builtin_huge_valf() && a->scale < __builtin_huge_valf()))
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: window %d min_new %d max_new %d max_kv %d softcap %g scale %g", a->window,
                      a->min_new, a->max_new, a->max_kv, a->softcap, a->scale);
  if (a->q_stride < 0 || a->out_stride < 0 || (a->q_stride | a->out_stride) % 8)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: row strides are non-negative multiples of 8 elements");
  return ARGUS_HIP_OK;
}

}  // namespace

ARGUS_API int64_t argus_hip_paged_attention_workspace(const argus_hip_ctx *ctx, const argus_hip_paged_attention_args *a) {
  if (!a) return ARGUS_HIP_ERR_INVALID;
  const int rc = check(const_cast<argus_hip_ctx *>(ctx), a);
  return rc != ARGUS_HIP_OK ? rc : 0;
}

ARGUS_API int argus_hip_paged_attention(argus_hip_ctx *ctx, const argus_hip_paged_attention_args *a) {
  if (!ctx || !a) return ARGUS_HIP_ERR_INVALID;
  const int rc = check(ctx, a);
  if (rc != ARGUS_HIP_OK) return rc;
  if (a->n_seqs == 0 || a->n_tokens == 0) return ARGUS_HIP_OK;
  if (!a->q || !a->k_cache || !a->v_cache || !a->page_table || !a->cu_new || !a->kv_len || !a->out)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: null pointer");
  if (((uintptr_t)a->q | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache | (uintptr_t)a->out) & 15)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: q, out and the pools are 16-byte aligned");
  const int d = a->head_dim;
  const int64_t grid = (int64_t)a->n_tokens * a->heads_q;
  if (grid > 0x7fffffff) return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: too many rows");
  const DeviceGuard guard(ctx);
  PagedParams p{a->q, (const _Float16 *)a->k_cache, (const _Float16 *)a->v_cache, a->page_table, a->cu_new, a->kv_len, a->out,
                a->q_stride ? a->q_stride : (int64_t)a->heads_q * d, a->out_stride ? a->out_stride : (int64_t)a->heads_q * d,
                argus_pool_strides(a->layout, a->heads_kv, a->page_size, d), a->n_seqs, a->n_tokens, a->heads_q, a->heads_kv,
                a->heads_q / a->heads_kv, a->n_pages, argus_log2(a->page_size), a->table_stride, a->window, a->softcap,
                a->scale != 0.0f ? a->scale : 1.0f / sqrtf((float)d)};
  const hipStream_t stream = (hipStream_t)a->stream;
  const bool f16 = a->dtype == ARGUS_HIP_F16;
  auto kern = d == 64 ? (f16 ? paged_row_kernel<64, _Float16> : paged_row_kernel<64, float>)
              : d == 128 ? (f16 ? paged_row_kernel<128, _Float16> : paged_row_kernel<128, float>)
                         : (f16 ? paged_row_kernel<256, _Float16> : paged_row_kernel<256, float>);
  KernelTimer timer(ctx, stream);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64), 0, stream, p);
  ARGUS_HIP_CHECK(ctx, hipGetLastError());
  return ARGUS_HIP_OK;
}
