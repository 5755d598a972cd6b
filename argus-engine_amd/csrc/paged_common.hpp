// Pieces shared by the paged-cache operators: geometry of a page pool and its checks, and the guard
// that issues a call on the context's device.
#pragma once

#include "argus_hip_internal.hpp"

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
