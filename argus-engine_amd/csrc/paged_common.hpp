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
  int64_t q_stride, out_stride;
  PoolStrides pool;  // elements
  PagedSched sched;
  int32_t heads_kv, n_pages, page_shift, table_stride;
  float scale, softcap;
};

// rows of a request's tile and their positions
constexpr int kDecodeRows = 16;  // requests of at most this many rows (tokens x heads of a group) take the decode kernel
constexpr int kChunkRows = 128;  // rows per workgroup of the chunk kernel

int launch_paged_decode(argus_hip_ctx *ctx, const PagedParams &p, int D, bool f32, int items, hipStream_t stream);
int launch_paged_chunk(argus_hip_ctx *ctx, const PagedParams &p, int D, bool f32, int items, hipStream_t stream);
int launch_paged_combine(argus_hip_ctx *ctx, const PagedParams &p, int D, bool f32, hipStream_t stream);
constexpr int decode_align(int D) { return D <= 128 ? 32 : 16; }   // keys per wave step of the decode kernel
constexpr int chunk_align(int D) { return D <= 64 ? 64 : 32; }     // keys per tile of the chunk kernel

#if defined(__HIPCC__)
// dword 3 of a raw (untyped, unstrided) buffer descriptor on this target
constexpr int kRawBuffer = 0x00020000;

// Page numbers of a request's consecutive pages, 64 per register: the number of a page is a lane read,
// not a memory access in the way of the page's rows.  `first` only moves up.
struct PageWindow {
  const int32_t *row;  // the request's row of the page table
  int stride, first, now, next;
  __device__ __forceinline__ int load(int at, int lane) const { return at + lane < stride ? row[at + lane] : -1; }
  __device__ __forceinline__ PageWindow(const PagedParams &p, int seq, int page, int lane)
      : row(p.page_table + (int64_t)seq * p.table_stride), stride(p.table_stride), first(page) {
    now = load(first, lane);
    next = load(first + 64, lane);
  }
  __device__ __forceinline__ void advance(int page, int lane) {  // wave-uniform; pages below `page` are not asked for again
    if (page >= first + 64) {
      first += 64;
      now = next;
      next = load(first + 64, lane);
    }
  }
  __device__ __forceinline__ int number(int page) const {  // first <= page < first + 128
    const int rel = page - first;
    return __builtin_amdgcn_readlane(rel < 64 ? now : next, rel & 63);
  }
};

// Descriptor of one head's rows of a page that ends behind row `rows` - 1: rows past it, and every row
// of a page whose number is none, read as zeros without touching memory.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rows(const _Float16 *pool, const PagedParams &p, int number, int kvh, int rows, int D) {
  const bool ok = (uint32_t)number < (uint32_t)p.n_pages && rows > 0;
  const _Float16 *base = pool + (ok ? (int64_t)number * p.pool.page : 0) + (int64_t)kvh * p.pool.head;
  const uint32_t bytes = ok ? (uint32_t)((rows - 1) * p.pool.row + D) * 2 : 0;
  return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes, kRawBuffer);
}

// cap * tanh(s / cap), tanh(x) = 1 - 2 / (exp(2x) + 1); the argument is clamped where tanh is 1 in F32
__device__ __forceinline__ float soft_cap(float s, float cap, float inv_cap) {
  const float x = fminf(fmaxf(s * inv_cap, -15.0f), 15.0f);
  const float e = __expf(2.0f * x);
  const float t = cap * (1.0f - 2.0f * __frcp_rn(e + 1.0f));
  return s != s ? s : t;
}

__device__ __forceinline__ bool not_finite(_Float16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7c00) == 0x7c00; }
#endif

}  // namespace argus_paged
