// Pieces shared by the paged-cache operators: geometry of a page pool and its checks, and the guard
// that issues a call on the context's device.
#pragma once

#include "argus_hip_internal.hpp"
#include "paged_sched.hpp"

// Issues a call on the context's device whatever device is current in the calling thread, and puts
// that one back.
struct DeviceGuard {
  int before = -1;
  explicit DeviceGuard(const argus_hip_ctx *ctx) {
    int now = -1;
    if (hipGetDevice(&now) == hipSuccess && now != ctx->device && hipSetDevice(ctx->device) == hipSuccess) before = now;
  }
  ~DeviceGuard() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

inline bool argus_page_size_ok(int page_size) {
  return page_size >= 16 && page_size <= ARGUS_HIP_MAX_PAGE_SIZE && (page_size & (page_size - 1)) == 0;
}
inline int argus_log2(int x) { return 31 - __builtin_clz((unsigned)x); }

// Strides of a pool in elements: row `r` of page `g`, KV head `h` starts at g * page + h * head + r * row.
struct PoolStrides {
  int64_t page, head, row;
};
inline PoolStrides argus_pool_strides(int layout, int heads_kv, int page_size, int head_dim) {
  const int64_t page = (int64_t)heads_kv * page_size * head_dim;
  if (layout == ARGUS_HIP_HEAD_MAJOR) return {page, (int64_t)page_size * head_dim, head_dim};
  return {page, head_dim, (int64_t)heads_kv * head_dim};
}

namespace argus_paged {

struct PagedParams {
  const void *q;
  const _Float16 *k, *v;
  const int32_t *page_table, *cu_new, *kv_len;
  void *out;
  // Partial results of tiles that are cut: slot 2 w for the end of a tile begun before share w, 2 w + 1 for
  // the begin of one that ends behind it.
  float *ws_ml;  // [slots, Hkv, tile_rows, 2]: running maximum (log2 units) and sum of a part's rows
  float *ws_o;   // [slots, Hkv, tile_rows, D]: un-normalised output rows
  PagedCut *cuts;  // [shares]
  int64_t q_stride, out_stride;
  PoolStrides pool;  // elements
  PagedSched sched;
  int32_t items;  // workgroups per KV head
  int32_t heads_kv, n_pages, page_shift, table_stride;
  float scale, softcap;
};

// rows of a request's tile and their positions
constexpr int kDecodeRows = 16;  // requests of at most this many rows (tokens x heads of a group) take the decode kernel
constexpr int kChunkRows = 128;  // rows per workgroup of the chunk kernel

// dp, cp: parameters of the decode and the chunk form (items 0: not in this call)
int launch_paged_64(argus_hip_ctx *ctx, const PagedParams &dp, const PagedParams &cp, bool f32, bool cap, hipStream_t stream);
int launch_paged_128(argus_hip_ctx *ctx, const PagedParams &dp, const PagedParams &cp, bool f32, bool cap, hipStream_t stream);
int launch_paged_256(argus_hip_ctx *ctx, const PagedParams &dp, const PagedParams &cp, bool f32, bool cap, hipStream_t stream);
constexpr int decode_align(int D) { return D <= 128 ? 32 : 16; }   // keys per wave step of the decode kernel
constexpr int chunk_align(int D) { return D <= 64 ? 64 : 32; }     // keys per tile of the chunk kernel

#if defined(__HIPCC__)
// dword 3 of a raw (untyped, unstrided) buffer descriptor on this target
constexpr int kRawBuffer = 0x00020000;

// One head's rows of the pages of a pool.
struct PagePool {
  const char *base;  // the head's first row in page 0
  uint32_t bytes;    // from there to the end of the head's last row in a page
  __device__ __forceinline__ PagePool(const _Float16 *pool, const PagedParams &p, int kvh, int D)
      : base((const char *)(pool + kvh * p.pool.head)), bytes((uint32_t)(((1 << p.page_shift) - 1) * p.pool.row + D) * 2) {}
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(uint64_t page_off) const {
    return __builtin_amdgcn_make_buffer_rsrc((void *)(base + page_off), 0, bytes, kRawBuffer);
  }
};

// Byte offsets of a request's consecutive pages, 64 per register pair: where a page lies is two lane reads,
// not a memory access in the way of its rows.  Pages are asked for in ascending order.  A number outside the
// pool, or a page behind the table, stands for page 0: what is read then is not specified, but is inside.
struct PageWindow {
  const int32_t *row;  // the request's row of the page table
  int stride, first, next;
  uint32_t n_pages, page_bytes, lo, hi;
  __device__ __forceinline__ int load(int at) const {
    const int i = at + (int)(threadIdx.x & 63);
    const int number = i < stride ? row[i] : 0;
    return (uint32_t)number < n_pages ? number : 0;
  }
  __device__ __forceinline__ void take(int numbers) {
    const uint64_t off = (uint64_t)(uint32_t)numbers * page_bytes;
    lo = (uint32_t)off;
    hi = (uint32_t)(off >> 32);
  }
  template <int SPAN>
  __device__ __forceinline__ void start(const PagedParams &p, int seq, int page) {
    row = p.page_table + (int64_t)seq * p.table_stride;
    stride = p.table_stride;
    n_pages = (uint32_t)p.n_pages;
    page_bytes = (uint32_t)p.pool.page * 2;
    first = page;
    take(load(first));
    next = load(first + 64 - SPAN);
  }
  // makes pages page .. page + SPAN - 1 available; page at most 32 ahead of the last one
  template <int SPAN>
  __device__ __forceinline__ void advance(int page) {
    if (page + SPAN > first + 64) {
      first += 64 - SPAN;
      take(next);
      next = load(first + 64 - SPAN);
    }
  }
  __device__ __forceinline__ uint64_t offset(int page) const {
    const int l = page - first;
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)lo, l);
  }
};

// The kernel's arguments read again from where they came: what is needed only after a long loop does not
// stay in scalar registers through it.
template <int ARG>  // the kernel's arguments are PagedParams only: which of them
__device__ __forceinline__ const PagedParams &params_again() {
  typedef const __attribute__((address_space(4))) PagedParams *const_ptr;
  const_ptr a = (const_ptr)__builtin_amdgcn_kernarg_segment_ptr() + ARG;
  asm volatile("" : "+s"(a));
  return *(const PagedParams *)a;
}

// cap * tanh(s / cap) from y = s / cap: 1 - 2 / (exp(2 y) + 1), whose error is that of the 1 it is taken
// from (2^-23, times the cap).  EXACT, for results that keep F32's error: the series of tanh where |y| is
// small, which is where logits mostly are (the first term left out is 1382 y^11 / 155925: below 2^-24 of y
// up to |y| = 1/4).
template <bool EXACT>
__device__ __forceinline__ float soft_cap(float s, float cap, float inv_cap) {
  const float y = s * inv_cap;
  const float e = __builtin_amdgcn_exp2f(y * 2.885390081777927f);  // infinite, or zero, where tanh is 1 or -1
  float t = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  if constexpr (EXACT) {
    const float z = y * y;
    const float series = y + y * z * __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f);
    t = z < 0.0625f ? series : t;
  }
  return cap * t;
}

// F32 queries enter the products as F16 pairs, hi + lo.  A row is brought to 2^14 .. 2^15 by a power of two
// first, which the factor of its logits takes back: so the pair holds 22 bits of it whatever its size is.
// (An infinite element of the row stays one, and is left out of what is taken for the largest.)
__device__ __forceinline__ float larger_finite(float largest, float x) {
  x = __builtin_fabsf(x);
  return x < __builtin_huge_valf() ? fmaxf(largest, x) : largest;
}
__device__ __forceinline__ int row_shift(float largest) {
  const int shift = 15 - __builtin_amdgcn_frexp_expf(largest);
  return shift < 100 ? shift : 100;  // the factor stays a normal number
}

// A factor of logits: where it overflows, the products it meets do so as well, but for zero, which stays zero.
__device__ __forceinline__ float factor(float x) { return fminf(fmaxf(x, -__FLT_MAX__), __FLT_MAX__); }

__device__ __forceinline__ bool not_finite(_Float16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7c00) == 0x7c00; }
#endif

}  // namespace argus_paged
