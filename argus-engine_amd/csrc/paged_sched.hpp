// How a paged_attention call is cut into workgroups.  Lengths live on the device, so every workgroup
// works this out for itself from the same numbers; the host only knows bounds, for the grid and the
// workspace.  Plain functions, compiled for both sides (and testable without a device).
//
// A request's rows (new tokens x heads of a GQA group) form tiles of `tile_rows`, and a tile costs about
// as many units as it sees keys.  The tiles of all requests, laid end to end, are one line of work that
// is cut into equal shares, one per workgroup and KV head: a share ends in the middle of a tile where it
// falls there, and the tile's parts are merged afterwards.  So a call fills the device whatever its
// lengths are, and no workgroup carries more than another.  A call of very many tiles is not cut: every
// workgroup takes one tile, the tiles of a request that see most keys first.
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
  int32_t tile_rows;
  int32_t unit;                  // keys per unit of cost, and what a cut falls on; 0: costs are in keys (see sched_cost)
  int32_t align;                 // key ranges start on a multiple of this
  int32_t min_share;             // a share is not smaller than this
  int32_t target;                // shares per KV head
  int32_t whole_from;            // from this many tiles per KV head on every tile is a share
  int32_t window, max_len;       // max_len: keys the page table has room for
};

ARGUS_HD int sched_min(int a, int b) { return a < b ? a : b; }
ARGUS_HD int sched_max(int a, int b) { return a > b ? a : b; }
ARGUS_HD int sched_add(int a, int b) { return (int)((uint32_t)a + (uint32_t)b); }  // device lengths may be anything: no undefined overflow

// A request as the device arrays give it, clipped to what the buffers hold.
struct PagedSeq {
  int32_t q_begin, q_end;      // rows of q
  int32_t pos0;                // position of row q_begin
  int32_t len;                 // keys
  int32_t key_begin, key_end;  // keys any of its rows sees; key_begin a multiple of `align`
};
ARGUS_HD PagedSeq sched_seq(const PagedSched &c, int cu0, int cu1, int kv) {
  PagedSeq s;
  s.q_begin = sched_min(sched_max(cu0, 0), c.n_tokens);
  s.q_end = sched_min(sched_max(cu1, s.q_begin), c.n_tokens);
  s.pos0 = sched_add(sched_add(kv, s.q_begin), -cu1);
  s.len = sched_min(sched_max(kv, 0), c.max_len);
  const int last = sched_add(s.pos0, s.q_end - s.q_begin - 1);
  s.key_end = last < 0 ? 0 : sched_min(s.len, last == 0x7fffffff ? last : last + 1);
  s.key_begin = c.window > 0 && s.pos0 >= c.window ? (s.pos0 - c.window + 1) / c.align * c.align : 0;
  s.key_begin = sched_min(s.key_begin, s.key_end / c.align * c.align);
  return s;
}

// Tiles of a request in this class (0: not in it) and their cost: tile t costs base + slope * t.
struct PagedCost {
  int32_t tiles;
  int64_t base, slope;
};
ARGUS_HD PagedCost sched_cost(const PagedSched &c, const PagedSeq &s) {
  PagedCost k{0, 0, 0};
  const int64_t rows = (int64_t)(s.q_end - s.q_begin) * c.group;
  if (rows <= c.rows_over || rows > c.rows_upto) return k;
  k.tiles = (int)((rows + c.tile_rows - 1) / c.tile_rows);
  if (c.unit) {  // one tile: whole units, at least one (rows that see nothing are written too)
    const int64_t units = ((int64_t)s.key_end - s.key_begin + c.unit - 1) / c.unit;
    k.base = units < 1 ? 1 : units;
    return k;
  }
  // keys the first tile sees, and how many more each further one does: exact enough to share work by
  const int per = sched_max(1, c.tile_rows / c.group);
  int64_t first = (int64_t)s.pos0 + sched_min(per, s.q_end - s.q_begin);
  if (first > s.key_end) first = s.key_end;
  first -= s.key_begin;
  if (first < 0) first = 0;
  k.slope = c.window > 0 ? 0 : per;
  if (c.window > 0 && k.tiles > 1) {  // between the first tile and a full window
    const int64_t full = (int64_t)c.window + per < s.key_end ? (int64_t)c.window + per : s.key_end;
    first = (first + full) / 2;
  }
  k.base = first + 96;  // what a tile costs beside its keys: its queries, the first round trip, its output
  return k;
}
ARGUS_HD int64_t sched_before(const PagedCost &k, int t) { return k.base * t + k.slope * ((int64_t)t * (t - 1) / 2); }  // of tiles 0 .. t - 1

ARGUS_HD int64_t sched_share(const PagedSched &c, int64_t work) {
  const int64_t share = (int64_t)((double)work / c.target) + 1;  // target shares hold at least the work
  return share < c.min_share ? c.min_share : share;
}

// Bounds the host can give: tiles of a class, workgroups per KV head, and partial results (two per share:
// the end of a tile begun before it and the begin of one that ends behind it).
inline int64_t sched_tiles_bound(const PagedSched &c, int min_new) {
  const int64_t rows = (int64_t)c.n_tokens * c.group;
  int64_t seqs = c.n_seqs < c.n_tokens ? c.n_seqs : c.n_tokens;
  if (c.rows_over > 0 && rows / (c.rows_over + 1) < seqs) seqs = rows / (c.rows_over + 1);
  if (min_new > 0 && c.n_tokens / min_new < seqs) seqs = c.n_tokens / min_new;
  if (c.rows_upto <= c.tile_rows) return seqs;
  return seqs ? rows / c.tile_rows + seqs : 0;
}
inline int64_t sched_items_bound(const PagedSched &c, int64_t tiles) {
  return tiles >= c.whole_from ? tiles : (int64_t)c.target < (int64_t)c.whole_from ? c.target : c.whole_from;
}
inline int64_t sched_slots_bound(const PagedSched &c) { return 2 * (int64_t)c.target; }

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

__device__ __forceinline__ int64_t wave_add64(int64_t x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}
__device__ __forceinline__ int64_t wave_scan64(int64_t x, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t a = __shfl_up(x, d, 64);
    if (lane >= d) x += a;
  }
  return x;
}
__device__ __forceinline__ int wave_same(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t wave_same(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

// A tile on the line of work.
struct PagedPlace {
  PagedSeq s;
  int32_t seq, tile;
  int64_t start, cost;  // of the tile, on the line
};

// The line of work of one class.  Every wave of a workgroup gets the same answers; lane l looks after
// requests l, 64 + l, ...  Nothing but the sums stays in registers: a search looks the lengths up again.
struct PagedLine {
  int64_t work, tiles, share;

  static __device__ __forceinline__ void look(const PagedSched &c, const int32_t *cu, const int32_t *kv, int i, PagedSeq &s, PagedCost &k) {
    k = PagedCost{0, 0, 0};
    s = PagedSeq{};
    if (i < c.n_seqs) {
      s = sched_seq(c, cu[i], cu[i + 1], kv[i]);
      k = sched_cost(c, s);
    }
  }
  __device__ __forceinline__ PagedLine(const PagedSched &c, const int32_t *cu, const int32_t *kv) {
    const int lane = threadIdx.x & 63;
    int64_t w = 0, t = 0;
    for (int b = 0; b < c.n_seqs; b += 64) {
      PagedSeq s;
      PagedCost k;
      look(c, cu, kv, b + lane, s, k);
      w += sched_before(k, k.tiles);
      t += k.tiles;
    }
    work = wave_same(wave_add64(w));
    tiles = wave_same(wave_add64(t));
    share = sched_share(c, work);
  }
  __device__ __forceinline__ bool whole(const PagedSched &c) const { return tiles >= c.whole_from; }
};

// The tile that holds position x of the line (by_tile: tile number x, the last tiles of a request first).
__device__ __forceinline__ bool sched_find(const PagedSched &c, const int32_t *cu, const int32_t *kv, bool by_tile, int64_t x, PagedPlace &out) {
  const int lane = threadIdx.x & 63;
  int64_t at = 0;
  for (int b = 0; b < c.n_seqs; b += 64) {
    PagedSeq s;
    PagedCost k;
    PagedLine::look(c, cu, kv, b + lane, s, k);
    const int64_t mine = by_tile ? (int64_t)k.tiles : sched_before(k, k.tiles);
    const int64_t inc = wave_scan64(mine, lane);
    const uint64_t past = __builtin_amdgcn_ballot_w64(at + inc > x);
    if (past) {
      const int l = __builtin_ctzll(past);
      PagedCost cost;
      cost.tiles = wave_same(__shfl(k.tiles, l, 64));
      cost.base = wave_same(__shfl(k.base, l, 64));
      cost.slope = wave_same(__shfl(k.slope, l, 64));
      const int64_t before = at + wave_same(__shfl(inc - mine, l, 64));
      int tile = 0;
      if (by_tile) {
        tile = cost.tiles - 1 - (int)(x - before);
      } else if (cost.tiles > 1) {
        int hi = cost.tiles;  // the last tile with sched_before <= x - before
        while (hi - tile > 1) {
          const int mid = (tile + hi) >> 1;
          if (sched_before(cost, mid) <= x - before) tile = mid;
          else hi = mid;
        }
      }
      if (tile < 0 || tile >= cost.tiles) return false;  // lengths that are none: sums that wrapped
      out.tile = wave_same(tile);
      out.seq = wave_same(b + l);
      out.start = before + sched_before(cost, tile);
      out.cost = cost.base + cost.slope * tile;
      out.s.q_begin = wave_same(__shfl(s.q_begin, l, 64));
      out.s.q_end = wave_same(__shfl(s.q_end, l, 64));
      out.s.pos0 = wave_same(__shfl(s.pos0, l, 64));
      out.s.len = wave_same(__shfl(s.len, l, 64));
      out.s.key_begin = wave_same(__shfl(s.key_begin, l, 64));
      out.s.key_end = wave_same(__shfl(s.key_end, l, 64));
      return true;
    }
    at += wave_same(__shfl(inc, 63, 64));
  }
  return false;
}
#endif
