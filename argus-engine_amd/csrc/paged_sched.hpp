// How a paged_attention call is cut into workgroups.  Lengths live on the device, so every workgroup
// works this out for itself from the same numbers; the host only knows bounds, for the grid and the
// workspace.  Plain functions, compiled for both sides (and testable without a device).
//
// A request's rows (new tokens x heads of a GQA group) form tiles of `tile_rows`, and a tile costs about
// as many units as it sees keys.  The tiles of all requests, laid end to end, are one line of work that
// is cut into equal shares, one per workgroup and KV head: a share ends in the middle of a tile where it
// falls there, and the tile's parts are merged afterwards.  So a call fills the device whatever its
// lengths are, and no workgroup carries more than another.  Where whole tiles fill it as well -- what the
// rounds of workgroups take, or the longest tile, is not more than the shares and what the cutting costs --
// every workgroup takes one tile, the tiles of a request that see most keys first.
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
  int32_t alone;                 // up to this many shares per KV head run without another on their compute unit: ~0.6 of the time
  int32_t rooms;                 // workgroups per KV head there are: no more tiles than that are taken whole
  int32_t cut_cost;              // what cutting costs a call: further starts, partial results, the merge; < 0: no tile is cut
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
  int64_t share = (int64_t)((double)work / c.target);
  if (share * c.target < work) ++share;  // target shares hold the work
  return share < c.min_share ? c.min_share : share;
}

// Are the tiles taken whole?  tiles, work, longest: over the class.
ARGUS_HD bool sched_whole(const PagedSched &c, int64_t tiles, int64_t work, int64_t longest) {
  if (c.cut_cost < 0 || tiles == 0) return true;
  if (tiles > c.rooms) return false;
  const double rounds = (double)((tiles + c.target - 1) / c.target) * ((double)work / (double)tiles);
  double whole = rounds > (double)longest ? rounds : (double)longest;
  if (tiles <= c.alone) whole *= 0.6;
  return whole <= (double)work / c.target + c.cut_cost;
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
inline int64_t sched_slots_bound(const PagedSched &c) { return 2 * (int64_t)c.target; }

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

// Inclusive sum over the wave's lanes, in the vector ALU: within rows of 16 lanes, then the rows' ends
// broadcast to the rows behind them.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp_add64(int64_t x) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return x + (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}
__device__ __forceinline__ int64_t wave_scan64(int64_t x) {
  x = dpp_add64<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add64<0x112, 0xf>(x);
  x = dpp_add64<0x114, 0xf>(x);
  x = dpp_add64<0x118, 0xf>(x);
  x = dpp_add64<0x142, 0xa>(x);  // row_bcast 15 into rows 1 and 3
  x = dpp_add64<0x143, 0xc>(x);  // row_bcast 31 into rows 2 and 3
  return x;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_max(int x) {
  const int y = __builtin_amdgcn_update_dpp(x, x, CTRL, ROWS, 0xf, false);
  return y > x ? y : x;
}
__device__ __forceinline__ int wave_max(int x) {  // in lane 63
  x = dpp_max<0x111, 0xf>(x);
  x = dpp_max<0x112, 0xf>(x);
  x = dpp_max<0x114, 0xf>(x);
  x = dpp_max<0x118, 0xf>(x);
  x = dpp_max<0x142, 0xa>(x);
  return dpp_max<0x143, 0xc>(x);
}
__device__ __forceinline__ int lane_value(int x, int l) { return __builtin_amdgcn_readlane(x, l); }
__device__ __forceinline__ int64_t lane_value(int64_t x, int l) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)x, l));
}
// A tile on the line of work.
struct PagedPlace {
  PagedSeq s;
  int32_t seq, tile, left;  // left: further tiles of the request
  int64_t block;            // where the requests' block of 64 begins
  int64_t start, cost;      // of the tile, on the line
  int64_t slope;            // cost of the request's next tile above this one's
};

// A block of 64 requests, one per lane.
struct PagedBlock {
  PagedSeq s;
  PagedCost k;
  int64_t total, inc;  // cost of this lane's request, and of the block's requests up to it

  __device__ __forceinline__ PagedBlock(const PagedSched &c, const int32_t *cu, const int32_t *kv, int b) : s{}, k{0, 0, 0} {
    const int i = b + (threadIdx.x & 63);
    if (i < c.n_seqs) {
      s = sched_seq(c, cu[i], cu[i + 1], kv[i]);
      k = sched_cost(c, s);
    }
    total = sched_before(k, k.tiles);
    inc = wave_scan64(total);
  }
  __device__ __forceinline__ int longest() const {
    const int64_t last = k.tiles > 0 ? k.base + k.slope * (k.tiles - 1) : 0;
    return lane_value(wave_max(last > 0x7fffffff ? 0x7fffffff : (int)last), 63);
  }
  // the tile that holds position x of the line; `at`: where the block begins.  False: behind the block
  __device__ __forceinline__ bool find(int b, int64_t at, int64_t x, PagedPlace &out) const {
    const uint64_t past = __builtin_amdgcn_ballot_w64(at + inc > x);
    if (!past) return false;
    const int l = __builtin_ctzll(past);
    PagedCost cost;
    cost.tiles = lane_value(k.tiles, l);
    cost.base = lane_value(k.base, l);
    cost.slope = lane_value(k.slope, l);
    const int64_t before = at + lane_value(inc - total, l);
    int tile = 0, hi = cost.tiles;  // the last tile with sched_before <= x - before
    while (hi - tile > 1) {
      const int mid = (tile + hi) >> 1;
      if (sched_before(cost, mid) <= x - before) tile = mid;
      else hi = mid;
    }
    place(b, l, cost, tile, before, out);
    out.block = at;
    return true;
  }
  // tile number x of the line, the last tiles of a request first
  __device__ __forceinline__ bool find_tile(int b, int64_t at, int64_t inc_tiles, int64_t x, PagedPlace &out) const {
    const uint64_t past = __builtin_amdgcn_ballot_w64(at + inc_tiles > x);
    if (!past) return false;
    const int l = __builtin_ctzll(past);
    PagedCost cost;
    cost.tiles = lane_value(k.tiles, l);
    cost.base = lane_value(k.base, l);
    cost.slope = lane_value(k.slope, l);
    place(b, l, cost, (int)(at + lane_value(inc_tiles, l) - 1 - x), 0, out);
    out.block = 0;  // not used: a share is one tile then
    return true;
  }
  __device__ __forceinline__ void place(int b, int l, const PagedCost &cost, int tile, int64_t before, PagedPlace &out) const {
    out.tile = tile;
    out.seq = b + l;
    out.left = cost.tiles - 1 - tile;
    out.slope = cost.slope;
    out.start = before + sched_before(cost, tile);
    out.cost = cost.base + cost.slope * tile;
    out.s.q_begin = lane_value(s.q_begin, l);
    out.s.q_end = lane_value(s.q_end, l);
    out.s.pos0 = lane_value(s.pos0, l);
    out.s.len = lane_value(s.len, l);
    out.s.key_begin = lane_value(s.key_begin, l);
    out.s.key_end = lane_value(s.key_end, l);
  }
};

// Share `w` of the line of work of a class, tile by tile.  Every wave of a workgroup gets the same
// answers.  The lengths are looked up again for each further request: nothing but a few sums stays in
// registers beside a tile's work.
struct PagedShare {
  int64_t x, end;    // what is left of the share
  int64_t share;     // of every workgroup
  bool whole;        // tiles are not cut
  bool found;        // a tile is there
  PagedPlace at;

  __device__ __forceinline__ PagedShare(const PagedSched &c, const int32_t *cu, const int32_t *kv, int64_t w) {
    int64_t work = 0, tiles = 0;
    PagedBlock first(c, cu, kv, 0);
    const int64_t first_tiles = wave_scan64(first.k.tiles);
    work = lane_value(first.inc, 63);
    tiles = lane_value(first_tiles, 63);
    int longest = first.longest();
#pragma unroll 4
    for (int b = 64; b < c.n_seqs; b += 64) {
      const PagedBlock block(c, cu, kv, b);
      work += lane_value(block.inc, 63);
      tiles += lane_value(wave_scan64(block.k.tiles), 63);
      const int l = block.longest();
      longest = l > longest ? l : longest;
    }
    share = sched_share(c, work);
    whole = sched_whole(c, tiles, work, longest);
    x = whole ? w : w * share;
    end = whole ? tiles : work;
    if (x + (whole ? 1 : share) < end) end = x + (whole ? 1 : share);
    found = x < end && (whole ? first.find_tile(0, 0, first_tiles, x, at) : first.find(0, 0, x, at));
    if (x < end && !found) search(c, cu, kv, lane_value(whole ? first_tiles : first.inc, 63), 64);
  }
  __device__ __forceinline__ void search(const PagedSched &c, const int32_t *cu, const int32_t *kv, int64_t before, int b) {
    found = false;
    for (; b < c.n_seqs && !found; b += 64) {
      const PagedBlock block(c, cu, kv, b);
      const int64_t inc = whole ? wave_scan64(block.k.tiles) : block.inc;
      found = whole ? block.find_tile(b, before, inc, x, at) : block.find(b, before, x, at);
      before += lane_value(inc, 63);
    }
  }
  // part of the tile that lies in the share
  __device__ __forceinline__ int64_t from() const { return whole ? 0 : x - at.start; }
  __device__ __forceinline__ int64_t upto() const { return whole ? at.cost : end - at.start < at.cost ? end - at.start : at.cost; }
  __device__ __forceinline__ void next(const PagedSched &c, const int32_t *cu, const int32_t *kv) {
    x = whole ? end : at.start + at.cost;
    if (x >= end) {
      found = false;
    } else if (at.left > 0) {
      ++at.tile;
      --at.left;
      at.start = x;
      at.cost += at.slope;
    } else {
      search(c, cu, kv, at.block, at.seq & ~63);
    }
  }
};

// What the merge has to know of a tile that is cut: left in the workspace by the share it begins in.
struct PagedCut {
  int32_t parts;    // 0: the share ends with a tile
  int32_t q_begin;  // row of q of its request
  int32_t row0;     // first of its rows in the request
  int32_t rows;
};
#endif
