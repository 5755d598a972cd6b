// How a paged_attention call is cut into workgroups.  Lengths live on the device, so every workgroup
// works this out for itself from the same numbers; the host only knows bounds of the counts, for the
// grid and the workspace.  Plain functions, compiled for both sides (and testable without a device).
//
// A request's rows (new tokens x heads of a GQA group) form tiles of `tile_rows`; a tile's keys are cut
// into `splits` parts of about `chunk` units of `unit` keys where the call has too few tiles to fill the
// device, or one request is much longer than the average.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define ARGUS_HD __host__ __device__ __forceinline__
#else
#define ARGUS_HD inline
#endif

struct PagedSched {
  int32_t n_seqs, n_tokens, group;
  int32_t rows_over, rows_upto;  // takes the requests with rows_over < rows <= rows_upto
  int32_t tile_rows, unit;       // rows per tile; keys per unit
  int32_t min_units;             // a part is not shorter than this many units
  int32_t target;                // parts wanted per KV head
  int32_t max_splits;            // 1: no request is cut
  int32_t window, max_len;       // max_len: keys the page table has room for
};

ARGUS_HD int sched_min(int a, int b) { return a < b ? a : b; }
ARGUS_HD int sched_max(int a, int b) { return a > b ? a : b; }
ARGUS_HD int sched_add(int a, int b) { return (int)((uint32_t)a + (uint32_t)b); }  // device lengths may be anything: no undefined overflow

// A request as the device arrays give it, clipped to what the buffers hold.
struct PagedSeq {
  int32_t q_begin, q_end;   // rows of q
  int32_t pos0;             // position of row q_begin
  int32_t len;              // keys
  int32_t key_begin, key_end;  // keys any of its rows sees; key_begin a multiple of `align`
};
ARGUS_HD PagedSeq sched_seq(const PagedSched &c, int cu0, int cu1, int kv, int align) {
  PagedSeq s;
  s.q_begin = sched_min(sched_max(cu0, 0), c.n_tokens);
  s.q_end = sched_min(sched_max(cu1, s.q_begin), c.n_tokens);
  s.pos0 = sched_add(sched_add(kv, s.q_begin), -cu1);
  s.len = sched_min(sched_max(kv, 0), c.max_len);
  const int last = sched_add(s.pos0, s.q_end - s.q_begin - 1);
  s.key_end = last < 0 ? 0 : sched_min(s.len, last == 0x7fffffff ? last : last + 1);
  s.key_begin = c.window > 0 && s.pos0 >= c.window ? (s.pos0 - c.window + 1) / align * align : 0;
  s.key_begin = sched_min(s.key_begin, s.key_end / align * align);
  return s;
}
ARGUS_HD int sched_rows(const PagedSched &c, const PagedSeq &s) {
  const int64_t rows = (int64_t)(s.q_end - s.q_begin) * c.group;
  return rows > 0x7fffffff ? 0x7fffffff : (int)rows;
}
// tiles of a request in this class (0: not in it) and the units of keys a tile has at most
ARGUS_HD int sched_tiles(const PagedSched &c, const PagedSeq &s) {
  const int rows = sched_rows(c, s);
  if (rows <= c.rows_over || rows > c.rows_upto) return 0;
  return (int)(((int64_t)rows + c.tile_rows - 1) / c.tile_rows);
}
ARGUS_HD int sched_units(const PagedSched &c, const PagedSeq &s) { return (int)(((int64_t)s.key_end - s.key_begin + c.unit - 1) / c.unit); }

// units per part, from the sums of tiles and of tiles x units over the class: at most `target` parts
// where the tiles leave room for that, and parts of the average length of a round otherwise
ARGUS_HD int64_t sched_chunk(const PagedSched &c, int64_t tiles, int64_t work) {
  int64_t parts = (int64_t)c.target - tiles;
  if (parts < (c.target + 1) / 2) parts = (c.target + 1) / 2;
  int64_t chunk = (work + parts - 1) / parts;
  return chunk < c.min_units ? c.min_units : chunk;
}
ARGUS_HD int sched_splits(const PagedSched &c, int units, int64_t chunk) {
  const int64_t n = (units + chunk - 1) / chunk;
  return (int)(n < 1 ? 1 : n > c.max_splits ? c.max_splits : n);
}

// Bounds the host can give.  With parts = target - tiles or target / 2 as above, work / chunk <= target:
// the parts of a call are at most tiles + target, and those of requests that are cut at all (more units
// than a chunk, so ceil(u / chunk) < 2 u / chunk) at most 2 target.
inline int64_t sched_tiles_bound(const PagedSched &c, int min_new) {
  const int64_t seqs = c.n_seqs < c.n_tokens ? c.n_seqs : c.n_tokens;
  int64_t in_class = seqs;  // a request in the class has more than rows_over rows
  const int64_t rows = (int64_t)c.n_tokens * c.group;
  if (c.rows_over > 0 && rows / (c.rows_over + 1) < in_class) in_class = rows / (c.rows_over + 1);
  if (min_new > 0 && c.n_tokens / min_new < in_class) in_class = c.n_tokens / min_new;
  return rows / c.tile_rows + in_class;
}
inline int64_t sched_items_bound(const PagedSched &c, int64_t tiles) { return c.max_splits > 1 ? tiles + c.target : tiles; }
inline int64_t sched_slots_bound(const PagedSched &c, int64_t tiles) {
  if (c.max_splits <= 1) return 0;
  const int64_t cut = tiles * c.max_splits;
  return cut < 2 * (int64_t)c.target ? cut : 2 * (int64_t)c.target;
}
inline int64_t sched_cut_tiles_bound(const PagedSched &c, int64_t tiles) {  // tiles of requests that are cut
  if (c.max_splits <= 1) return 0;
  return tiles < c.target ? tiles : c.target;  // each has two parts at least
}

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

// One part of the call: split `split` of `nsplit` of tile `tile` of a request; its partial results (where
// nsplit > 1) go to slot + split.
struct PagedItem {
  PagedSeq s;
  int32_t seq, tile, split, nsplit, slot;
  int64_t chunk;
};

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}
__device__ __forceinline__ int wave_scan_add(int x, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(x, d, 64);
    if (lane >= d) x += a;
  }
  return x;
}

// The request, tile and split of part `item` (CUT false), or the request and tile of cut tile `item`
// (CUT true: split 0, for the merge).  Every wave of the workgroup calls it with the same item and gets
// the same answer; false: the call has fewer.
template <bool CUT>
__device__ bool sched_find(const PagedSched &c, const int32_t *cu, const int32_t *kv, int align, int item, PagedItem &out) {
  const int lane = threadIdx.x & 63;
  // sums over the class; a lone block of 64 requests stays in registers for the search
  int64_t tiles_sum = 0, work_sum = 0;
  PagedSeq s{};
  int tiles = 0, units = 0;
  for (int b = 0; b < c.n_seqs; b += 64) {
    tiles = units = 0;
    if (b + lane < c.n_seqs) {
      s = sched_seq(c, cu[b + lane], cu[b + lane + 1], kv[b + lane], align);
      tiles = sched_tiles(c, s);
      units = sched_units(c, s);
    }
    tiles_sum += tiles;
    work_sum += (int64_t)tiles * units;
  }
  tiles_sum = wave_sum64(tiles_sum);
  work_sum = wave_sum64(work_sum);
  const int64_t chunk = sched_chunk(c, tiles_sum, work_sum);
  int at = 0, slot_at = 0;  // parts and slots of the requests before block b
  for (int b = 0; b < c.n_seqs; b += 64) {
    if (c.n_seqs > 64) {
      tiles = units = 0;
      if (b + lane < c.n_seqs) {
        s = sched_seq(c, cu[b + lane], cu[b + lane + 1], kv[b + lane], align);
        tiles = sched_tiles(c, s);
        units = sched_units(c, s);
      }
    }
    const int splits = sched_splits(c, units, chunk);
    const int slots = splits > 1 ? tiles * splits : 0;
    const int items = CUT ? (splits > 1 ? tiles : 0) : tiles * splits;
    const int inc = wave_scan_add(items, lane), slot_inc = wave_scan_add(slots, lane);
    const uint64_t past = __builtin_amdgcn_ballot_w64(at + inc > item);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int before = at + __shfl(inc, l, 64) - __shfl(items, l, 64);
      const int nsplit = __shfl(splits, l, 64);
      const int k = item - before;
      out.s.q_begin = __shfl(s.q_begin, l, 64);
      out.s.q_end = __shfl(s.q_end, l, 64);
      out.s.pos0 = __shfl(s.pos0, l, 64);
      out.s.len = __shfl(s.len, l, 64);
      out.s.key_begin = __shfl(s.key_begin, l, 64);
      out.s.key_end = __shfl(s.key_end, l, 64);
      // the last tiles of a request see the most keys: they come first
      const int n_tiles = __shfl(tiles, l, 64);
      if (k < 0 || (CUT ? k : k / nsplit) >= n_tiles) return false;  // sums that wrapped: lengths that are none
      out.seq = __builtin_amdgcn_readfirstlane(b + l);
      out.nsplit = __builtin_amdgcn_readfirstlane(nsplit);
      const int tile = CUT ? k : k / nsplit;
      out.tile = __builtin_amdgcn_readfirstlane(n_tiles - 1 - tile);
      out.split = CUT ? 0 : __builtin_amdgcn_readfirstlane(k % nsplit);
      out.slot = __builtin_amdgcn_readfirstlane(slot_at + __shfl(slot_inc, l, 64) - __shfl(slots, l, 64) + tile * nsplit);
      out.s.q_begin = __builtin_amdgcn_readfirstlane(out.s.q_begin);
      out.s.q_end = __builtin_amdgcn_readfirstlane(out.s.q_end);
      out.s.pos0 = __builtin_amdgcn_readfirstlane(out.s.pos0);
      out.s.len = __builtin_amdgcn_readfirstlane(out.s.len);
      out.s.key_begin = __builtin_amdgcn_readfirstlane(out.s.key_begin);
      out.s.key_end = __builtin_amdgcn_readfirstlane(out.s.key_end);
      out.chunk = chunk;
      return true;
    }
    at += __shfl(inc, 63, 64);
    slot_at += __shfl(slot_inc, 63, 64);
  }
  return false;
}
#endif
