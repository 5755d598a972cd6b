// One scheduler step over paged caches: prefix sums of the new lengths, pages from the free list,
// positions and write slots of every new token (include/argus_hip.h, argus_hip_page_plan).
//
//   need_s = pages(past_s + new_s) - pages(past_s),  base_s = sum_{r<s} need_r,  cu_s = sum_{r<s} new_r
//   page of (s, i) = i < pages(past_s) ? table[s][i] : free[base_s + i - pages(past_s)]
//
// Bound by latency (a few hundred KB at most): one launch, and no workgroup waits for another.  Every
// workgroup scans all lengths for itself -- 2048 requests are two loads of four per thread and one
// block scan -- and keeps both prefix sums in LDS, where the tokens and the new pages it owns find their
// request by binary search.  A new page is read from the free list, never from the table entry another
// workgroup writes.
#include "paged_common.hpp"

#include <algorithm>

namespace {

constexpr int kThreads = 512;
constexpr int kPerThread = 4;                         // requests per thread and scan round
constexpr int kRound = kThreads * kPerThread;
constexpr int kMaxSeqs = 16384;                       // two prefix sums of 4 bytes each in 160 KB of LDS

struct PagePlanParams {
  const int32_t *past_len, *new_len, *free_pages;
  int32_t *page_table, *cu_new, *kv_len, *positions, *slots, *counts;
  int32_t n_seqs, n_free, n_pages, page_shift, table_stride, token_capacity;
};

// Sums of lengths saturate: min(a + b, 2^31 - 1) is associative on non-negative numbers.
__device__ __forceinline__ int sat_add(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7fffffffu); }

__device__ __forceinline__ int pages_of(const PagePlanParams &p, int tokens) {
  const uint32_t n = ((uint32_t)tokens + ((1u << p.page_shift) - 1)) >> p.page_shift;
  return (int)min(n, (uint32_t)p.table_stride);
}

// Index s with sum[s] <= x < sum[s + 1]; sum[n] > x.
__device__ __forceinline__ int find_seq(const int *sum, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int new_page(const PagePlanParams &p, int at) {
  const int page = at < p.n_free ? p.free_pages[at] : -1;
  return (uint32_t)page < (uint32_t)p.n_pages ? page : -1;
}

__global__ __launch_bounds__(kThreads) void page_plan_kernel(const PagePlanParams p) {
  extern __shared__ int lds[];
  int *cu = lds, *base = lds + p.n_seqs + 1;  // exclusive sums of new tokens and of needed pages
  __shared__ int wave_sum[2][2][kThreads / 64];
  __shared__ int n_short;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool first = blockIdx.x == 0;
  if (tid == 0) n_short = 0;

  int carry_t = 0, carry_p = 0;
  for (int r0 = 0, round = 0; r0 < p.n_seqs; r0 += kRound, ++round) {
    int past[kPerThread], fresh[kPerThread], need[kPerThread];
    int sum_t = 0, sum_p = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int s = r0 + tid * kPerThread + i;
      past[i] = s < p.n_seqs ? max(p.past_len[s], 0) : 0;
      fresh[i] = s < p.n_seqs ? max(p.new_len[s], 0) : 0;
    }
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      need[i] = fresh[i] > 0 ? pages_of(p, sat_add(past[i], fresh[i])) - pages_of(p, past[i]) : 0;
      sum_t = sat_add(sum_t, fresh[i]);
      sum_p = sat_add(sum_p, need[i]);
    }
    int inc_t = sum_t, inc_p = sum_p;  // inclusive over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int a = __shfl_up(inc_t, d, 64), b = __shfl_up(inc_p, d, 64);
      if (lane >= d) {
        inc_t = sat_add(inc_t, a);
        inc_p = sat_add(inc_p, b);
      }
    }
    if (lane == 63) {
      wave_sum[round & 1][0][wave] = inc_t;
      wave_sum[round & 1][1][wave] = inc_p;
    }
    __syncthreads();
    // exclusive value of this thread: carry of the rounds before, the waves before, the lanes before
    int at_t = carry_t, at_p = carry_p;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      const int a = wave_sum[round & 1][0][w], b = wave_sum[round & 1][1][w];
      if (w < wave) {
        at_t = sat_add(at_t, a);
        at_p = sat_add(at_p, b);
      }
      carry_t = sat_add(carry_t, a);
      carry_p = sat_add(carry_p, b);
    }
    const int lanes_t = __shfl_up(inc_t, 1, 64), lanes_p = __shfl_up(inc_p, 1, 64);
    if (lane > 0) {
      at_t = sat_add(at_t, lanes_t);
      at_p = sat_add(at_p, lanes_p);
    }
    int shorts = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int s = r0 + tid * kPerThread + i;
      if (s < p.n_seqs) {
        cu[s] = at_t;
        base[s] = at_p;
        if (first) {
          const int len = sat_add(past[i], fresh[i]);
          p.cu_new[s] = at_t;
          p.kv_len[s] = len;
          const int64_t room = (int64_t)p.table_stride << p.page_shift;
          shorts += fresh[i] > 0 && (len > room || (need[i] > 0 && new_page(p, sat_add(at_p, need[i]) - 1) < 0));
        }
      }
      at_t = sat_add(at_t, fresh[i]);
      at_p = sat_add(at_p, need[i]);
    }
    if (first && shorts) atomicAdd(&n_short, shorts);  // LDS, whole numbers: any order gives the same sum
  }
  if (tid == 0) {
    cu[p.n_seqs] = carry_t;
    base[p.n_seqs] = carry_p;
  }
  __syncthreads();
  if (first && tid == 0) {
    p.cu_new[p.n_seqs] = carry_t;
    p.counts[0] = carry_t;
    p.counts[1] = carry_p;
    p.counts[2] = n_short;
  }

  // new pages into their table entries
  const int64_t step = (int64_t)gridDim.x * kThreads;
  for (int64_t j = (int64_t)blockIdx.x * kThreads + tid; j < carry_p; j += step) {
    const int s = find_seq(base, p.n_seqs, (int)j);
    const int had = pages_of(p, max(p.past_len[s], 0));
    p.page_table[(int64_t)s * p.table_stride + had + ((int)j - base[s])] = new_page(p, (int)j);
  }
  // tokens
  for (int64_t j = (int64_t)blockIdx.x * kThreads + tid; j < p.token_capacity; j += step) {
    int pos = -1, slot = -1;
    if (j < carry_t) {
      const int s = find_seq(cu, p.n_seqs, (int)j);
      const int past = max(p.past_len[s], 0);
      pos = sat_add(past, (int)j - cu[s]);
      const int col = pos >> p.page_shift, had = pages_of(p, past);
      if (col < p.table_stride) {
        int page = col < had ? p.page_table[(int64_t)s * p.table_stride + col] : new_page(p, sat_add(base[s], col - had));
        if ((uint32_t)page < (uint32_t)p.n_pages) slot = (page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
      }
    }
    p.positions[j] = pos;
    p.slots[j] = slot;
  }
}

}  // namespace

ARGUS_API int argus_hip_page_plan(argus_hip_ctx *ctx, const argus_hip_page_plan_args *a) {
  if (!ctx || !a) return ARGUS_HIP_ERR_INVALID;
  if (a->n_seqs < 0 || a->n_free < 0 || a->token_capacity < 0 || a->table_stride <= 0 || a->n_pages <= 0)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "page_plan: n_seqs %d n_free %d n_pages %d table_stride %d token_capacity %d",
                      a->n_seqs, a->n_free, a->n_pages, a->table_stride, a->token_capacity);
  if (!argus_page_size_ok(a->page_size))
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "page_plan: page_size %d is not a power of two from 16 to %d", a->page_size,
                      ARGUS_HIP_MAX_PAGE_SIZE);
  if ((int64_t)a->n_pages * a->page_size > 0x7fffffff)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "page_plan: %d pages of %d tokens are more than 2^31 - 1 slots", a->n_pages, a->page_size);
  if (a->n_seqs > kMaxSeqs)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "page_plan: %d requests, at most %d", a->n_seqs, kMaxSeqs);
  if (!a->cu_new || !a->counts || (a->n_seqs && (!a->past_len || !a->new_len || !a->page_table || !a->kv_len)) ||
      (a->token_capacity && (!a->positions || !a->slots)) || (a->n_free && !a->free_pages))
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "page_plan: null pointer");
  // every workgroup reads the lengths, in its own time
  const auto meet = [&](const int32_t *in, const int32_t *out, int n_out) {
    return (uintptr_t)in < (uintptr_t)(out + n_out) && (uintptr_t)out < (uintptr_t)(in + a->n_seqs);
  };
  for (const int32_t *in : {a->past_len, a->new_len})
    if (a->n_seqs && (meet(in, a->kv_len, a->n_seqs) || meet(in, a->cu_new, a->n_seqs + 1)))
      return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "page_plan: kv_len and cu_new lie in the lengths they are computed from");
  const DeviceGuard guard(ctx);
  PagePlanParams p{a->past_len, a->new_len, a->free_pages, a->page_table, a->cu_new, a->kv_len, a->positions, a->slots, a->counts,
                   a->n_seqs, a->n_free, a->n_pages, argus_log2(a->page_size), a->table_stride, a->token_capacity};
  const size_t lds = (size_t)2 * (a->n_seqs + 1) * sizeof(int32_t);
  ARGUS_HIP_CHECK(ctx, argus_raise_lds_limit(ctx, page_plan_kernel, 2 * (kMaxSeqs + 1) * (int)sizeof(int32_t)));
  // 2016 single tokens and 32 chunks 7.1 us, 64 single tokens 4.7 us.  One token per thread; beyond two workgroups per CU the scan of every further one costs more than it takes over
  const int64_t want = ((int64_t)a->token_capacity + kThreads - 1) / kThreads;
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(want, (int64_t)ctx->compute_units * 2));
  hipLaunchKernelGGL(page_plan_kernel, dim3(grid), dim3(kThreads), lds, (hipStream_t)a->stream, p);
  ARGUS_HIP_CHECK(ctx, hipGetLastError());
  return ARGUS_HIP_OK;
}
