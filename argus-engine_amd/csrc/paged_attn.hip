// Causal GQA attention of the new tokens of many requests over their pages (include/argus_hip.h,
// argus_hip_paged_attention): checks, the plan of a call, and the entry points.  Kernels: paged_launch.hpp.
//
//   s_c = cap((q . k_c) * scale) for the visible keys c of a row;  out = sum_c softmax(s)_c v_c
#include "paged_common.hpp"

#include <algorithm>
#include <cmath>

namespace argus_paged {

namespace {

// How a call is cut: which kernels run, with how many workgroups, and where their partial results lie.
struct CallPlan {
  bool decode, chunk;
  PagedSched ds, cs;
  int64_t d_items, c_items, d_slots, c_slots;
  int64_t ws_floats;  // decode, chunk: [output rows][cuts][maxima and sums]
};

int make_plan(argus_hip_ctx *ctx, int compute_units, const argus_hip_paged_attention_args *a, CallPlan &pl) {
  const int G = a->heads_q / a->heads_kv, d = a->head_dim;
  const int64_t room = std::min<int64_t>((int64_t)a->table_stride * a->page_size, 0x7fffffff - 4096);
  const int64_t longest = a->max_kv > 0 ? std::min<int64_t>(a->max_kv, room) : room;
  PagedSched s{};
  s.n_seqs = a->n_seqs;
  s.n_tokens = a->n_tokens;
  s.group = G;
  s.window = a->window;
  s.max_len = (int)room;
  pl = CallPlan{};
  pl.decode = G <= kDecodeRows && (int64_t)a->min_new * G <= kDecodeRows;
  pl.chunk = !pl.decode || a->max_new == 0 || (int64_t)a->max_new * G > kDecodeRows;
  // A call that is nearly all chunks gives its few short requests to the chunk form too: each costs it at most
  // one tile more, and the decode form's workgroups begin ahead of the chunk shares and merge, whether there is
  // a request for them or not.  Measured both ways over 33 calls (prompts of 300 to 4096, 1 to 3 chunks behind
  // up to 12000, 0 to 4 single tokens beside them, d 64 / 128 / 256, F16 and F32): 1 to 9 % less time in 31 of them
  // (700 new tokens and one single token at d 128 97.8 against 103.7 us), 4 % more in two (4 single tokens beside
  // 2 x 2000 at d 128).
  if (pl.decode && pl.chunk && (int64_t)a->n_seqs * kChunkRows * 8 <= (int64_t)a->n_tokens * G) pl.decode = false;
  if (pl.decode) {
    PagedSched &c = pl.ds = s;
    c.rows_upto = c.tile_rows = kDecodeRows;
    c.align = decode_align(d);
    c.unit = 4 * c.align;
    c.min_share = 2;
    c.cut_cost = 2;  // 10 us; a unit of 128 keys is 5 us at d 128 with the device full
    // Resident workgroups (beside the chunk form half of them, so that chunk shares begin at once: 60 single
    // tokens and a chunk of 64 at d 128 124 -> 115 us), and no more shares than the longest lengths make.
    const int64_t tiles = sched_tiles_bound(c, a->min_new);
    const int64_t most = tiles * std::max<int64_t>(1, (longest + 2 * c.align) / c.unit + 1);
    c.target = (int)std::min<int64_t>(std::max(1, compute_units * (pl.chunk ? 1 : 2) / a->heads_kv), std::max<int64_t>(1, most / c.min_share));
    if (c.target == 1) c.cut_cost = -1;
    pl.d_items = c.cut_cost < 0 ? tiles : c.target;  // more requests than shares: a share takes several
    c.rooms = (int)pl.d_items;
    pl.d_slots = c.cut_cost >= 0 ? sched_slots_bound(c) : 0;
  }
  if (pl.chunk) {
    PagedSched &c = pl.cs = s;
    c.rows_over = pl.decode ? kDecodeRows : 0;
    c.rows_upto = 0x7fffffff;
    c.tile_rows = kChunkRows;
    c.align = chunk_align(d);
    c.min_share = 512;
    const int64_t tiles = sched_tiles_bound(c, a->min_new);
    const int resident = d <= 128 ? 2 : 1;               // workgroups per compute unit
    c.target = std::max(1, compute_units * resident / a->heads_kv);
    c.alone = resident == 2 ? compute_units / a->heads_kv : 0;
    // in keys a workgroup gets through meanwhile.  Measured over prompts of 512 to 8192 tokens and chunks of
    // 64 to 700 behind up to 8192: half or twice as much lose up to 30 % somewhere (700 tokens behind 2300 at
    // d 64 37 -> 49 us with 1800, 2048 tokens at d 128 66 -> 77 us with 500, at d 256 64 -> 100 us with 1600).
    c.cut_cost = d == 64 ? 1300 : d == 128 ? 1100 : 700;
    if (longest + 96 <= c.min_share) c.cut_cost = -1;    // tiles too short to be cut
    if (tiles == 0) pl.chunk = false;                    // too few rows for any request of this class
    pl.c_items = c.cut_cost < 0 ? tiles : std::max<int64_t>(tiles, c.target);
    if (!pl.chunk) pl.c_items = 0;
    c.rooms = (int)std::min<int64_t>(pl.c_items, 0x7fffffff);
    pl.c_slots = c.cut_cost >= 0 && pl.chunk ? sched_slots_bound(c) : 0;
  }
  constexpr int64_t kGrid = 0x7fffffff;
  if ((pl.d_items + pl.c_items) * a->heads_kv > kGrid)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: %d rows are too many for one call", a->n_tokens);
  pl.ws_floats = (pl.d_slots * kDecodeRows + pl.c_slots * kChunkRows) * a->heads_kv * (d + 2) +
                 ((pl.d_slots ? pl.ds.target : 0) + (pl.c_slots ? pl.cs.target : 0)) * (int64_t)(sizeof(PagedCut) / sizeof(float));
  return ARGUS_HIP_OK;
}

int check(argus_hip_ctx *ctx, const argus_hip_paged_attention_args *a) {
  if (a->n_seqs < 0 || a->n_tokens < 0 || a->heads_q <= 0 || a->heads_kv <= 0 || a->heads_q % a->heads_kv || a->n_pages <= 0 ||
      a->table_stride <= 0)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: n_seqs %d n_tokens %d heads %d / %d n_pages %d table_stride %d", a->n_seqs,
                      a->n_tokens, a->heads_q, a->heads_kv, a->n_pages, a->table_stride);
  if ((int64_t)a->n_tokens * (a->heads_q / a->heads_kv) > 0x7fffffff)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: %d tokens of %d heads per KV head are more than 2^31 - 1 rows", a->n_tokens,
                      a->heads_q / a->heads_kv);
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: head_dim %d is not 64, 128 or 256", a->head_dim);
  if (!argus_page_size_ok(a->page_size))
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: page_size %d is not a power of two from 16 to %d", a->page_size,
                      ARGUS_HIP_MAX_PAGE_SIZE);
  if ((int64_t)a->heads_kv * a->page_size * a->head_dim * 2 > 0x7fffffff)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: a page of %d heads x %d tokens is larger than 2 GiB", a->heads_kv, a->page_size);
  if (a->layout != ARGUS_HIP_HEAD_MAJOR && a->layout != ARGUS_HIP_SEQ_MAJOR)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: layout %d", a->layout);
  if (a->dtype != ARGUS_HIP_F32 && a->dtype != ARGUS_HIP_F16)
    return argus_fail(ctx, ARGUS_HIP_ERR_UNSUPPORTED, "paged_attention: dtype %d", a->dtype);
  if (a->window < 0 || a->min_new < 0 || a->max_new < 0 || a->max_kv < 0 ||
      !(a->softcap == 0.0f || a->softcap >= __FLT_MIN__) || !(a->softcap < __builtin_huge_valf()) ||
      !(a->scale > -__builtin_huge_valf() && a->scale < __builtin_huge_valf()))
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: window %d min_new %d max_new %d max_kv %d softcap %g scale %g", a->window,
                      a->min_new, a->max_new, a->max_kv, a->softcap, a->scale);
  if (a->q_stride < 0 || a->out_stride < 0 || (a->q_stride | a->out_stride) % 8)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: row strides are non-negative multiples of 8 elements");
  if (a->n_tokens > 1 && a->out_stride && a->out_stride < (int64_t)a->heads_q * a->head_dim)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: rows of out overlap (out_stride %lld)", (long long)a->out_stride);
  return ARGUS_HIP_OK;
}

}  // namespace

}  // namespace argus_paged

using namespace argus_paged;

ARGUS_API int64_t argus_hip_paged_attention_workspace(const argus_hip_ctx *ctx, const argus_hip_paged_attention_args *a) {
  if (!a) return ARGUS_HIP_ERR_INVALID;
  argus_hip_ctx *c = const_cast<argus_hip_ctx *>(ctx);  // for the error text
  int rc = check(c, a);
  CallPlan pl;
  if (rc == ARGUS_HIP_OK) rc = make_plan(c, ctx ? ctx->compute_units : 256, a, pl);
  return rc != ARGUS_HIP_OK ? rc : pl.ws_floats * (int64_t)sizeof(float);
}

ARGUS_API int argus_hip_paged_attention(argus_hip_ctx *ctx, const argus_hip_paged_attention_args *a) {
  if (!ctx || !a) return ARGUS_HIP_ERR_INVALID;
  int rc = check(ctx, a);
  CallPlan pl;
  if (rc == ARGUS_HIP_OK) rc = make_plan(ctx, ctx->compute_units, a, pl);
  if (rc != ARGUS_HIP_OK) return rc;
  if (a->n_seqs == 0 || a->n_tokens == 0 || pl.d_items + pl.c_items == 0) return ARGUS_HIP_OK;  // no request can have a token
  if (!a->q || !a->k_cache || !a->v_cache || !a->page_table || !a->cu_new || !a->kv_len || !a->out)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: null pointer");
  if (((uintptr_t)a->q | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache | (uintptr_t)a->out) & 15)
    return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: q, out and the pools are 16-byte aligned");
  const DeviceGuard guard(ctx);
  const hipStream_t stream = (hipStream_t)a->stream;
  const size_t need = (size_t)pl.ws_floats * sizeof(float);
  float *ws = (float *)a->workspace;
  if (ws) {
    if ((uintptr_t)ws & 255) return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: the workspace is not 256-byte aligned");
    if (a->workspace_bytes < need)
      return argus_fail(ctx, ARGUS_HIP_ERR_NOMEM, "paged_attention: the workspace holds %zu bytes, the call needs %zu", a->workspace_bytes, need);
  } else if (need) {
    // A captured call keeps the workspace's address: the context's may be replaced by a larger one.
    hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
    ARGUS_HIP_CHECK(ctx, hipStreamIsCapturing(stream, &capturing));
    if (capturing != hipStreamCaptureStatusNone)
      return argus_fail(ctx, ARGUS_HIP_ERR_INVALID, "paged_attention: a call under stream capture brings its own workspace (%zu bytes)", need);
    rc = argus_ws_reserve(ctx, need);
    if (rc != ARGUS_HIP_OK) return rc;
    ws = argus_ws(ctx);
  }
  const int d = a->head_dim;
  const bool f32 = a->dtype == ARGUS_HIP_F32;
  PagedParams p{};
  p.q = a->q, p.k = (const _Float16 *)a->k_cache, p.v = (const _Float16 *)a->v_cache, p.out = a->out;
  p.page_table = a->page_table, p.cu_new = a->cu_new, p.kv_len = a->kv_len;
  p.q_stride = a->q_stride ? a->q_stride : (int64_t)a->heads_q * d;
  p.out_stride = a->out_stride ? a->out_stride : (int64_t)a->heads_q * d;
  p.pool = argus_pool_strides(a->layout, a->heads_kv, a->page_size, d);
  p.heads_kv = a->heads_kv, p.n_pages = a->n_pages, p.page_shift = argus_log2(a->page_size), p.table_stride = a->table_stride;
  p.softcap = a->softcap, p.scale = a->scale != 0.0f ? a->scale : 1.0f / std::sqrt((float)d);
  // a form's part of the workspace: output rows (read and written 16 bytes at a time), cuts, maxima and sums
  auto form = [&](const PagedSched &sched, int64_t items, int64_t slots) {
    PagedParams f = p;
    f.sched = sched;
    f.items = (int)items;
    if (slots) {
      f.ws_o = ws;
      f.cuts = (PagedCut *)(ws + slots * sched.tile_rows * a->heads_kv * d);
      f.ws_ml = (float *)(f.cuts + sched.target);
      ws = f.ws_ml + slots * sched.tile_rows * a->heads_kv * 2;
    }
    return f;
  };
  const PagedParams dp = form(pl.ds, pl.decode ? pl.d_items : 0, pl.d_slots), cp = form(pl.cs, pl.chunk ? pl.c_items : 0, pl.c_slots);
  const bool cap = a->softcap > 0.0f;
  switch (d) {
    case 64: return launch_paged_64(ctx, dp, cp, f32, cap, stream);
    case 128: return launch_paged_128(ctx, dp, cp, f32, cap, stream);
    default: return launch_paged_256(ctx, dp, cp, f32, cap, stream);
  }
}
