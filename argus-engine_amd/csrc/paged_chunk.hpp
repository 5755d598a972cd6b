// The chunk kernel of paged_attention: requests of more rows (new tokens x heads of a GQA group) than the
// decode kernel takes.
//
// One workgroup = 128 rows of one KV head, four waves of 32.  A row is a (token, head of the group) pair, so
// the whole group shares each K / V tile and a short chunk fills its rows with heads.
// v_mfma_f32_32x32x16_f16 in the transposed form
//     S^T = K . Q^T  (A = K rows from LDS, B = Q rows in registers)
//     O^T = V^T . P^T (A = V^T through a transposing LDS read, B = the S^T accumulators' own layout)
// a lane owns one row: the softmax is in-lane plus one exchange between the wave's halves, the running
// maximum and sum are F32, and P never goes through LDS.  Bound by issue: at d 128 (8192 tokens, 32/8 heads,
// F16: 600 to 640 us from box to box, 860 to 915 TFLOP/s) the matrix cores are busy 45 % of the cycles and the vector ALU
// 35 %.  F32 queries take 1.5 to 1.75 times the time of F16 ones (prompts of 4096: 114 / 292 / 223 us at d 64 / 128 / 256).
#pragma once

#include "paged_common.hpp"

#include <algorithm>
#include <type_traits>

namespace argus_paged {

namespace {

typedef float float16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ half4_t lds_read_tr16(const _Float16 *p) {
  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t lds_short4_t;
  return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t *)p));
}

template <int D, bool F32>
struct ChunkTile {
  static constexpr int BN = chunk_align(D);            // keys per tile
  static constexpr int KP = D + 8, VP = D + 32;        // row pitches (halfs): no bank is hit twice by one read
  static constexpr int LDS_BYTES = 2 * BN * (KP + VP) * 2;  // two buffers each of K and V tiles
  static constexpr bool DEEP = !F32 && D <= 128;       // tiles are requested a step earlier (registers allow a second set)
  static constexpr int WAVES_PER_SIMD = D <= 128 ? 2 : 1;
};

// Software pipeline of a wave, as the logits of tile t + 1 are formed while tile t is exponentiated:
//   phase A   S(t+1) = K . Q^T on the matrix cores  beside  the second half of tile t's exponentials
//   phase B   O += V . P(t)                         beside  the first half of tile t + 1's
// K tiles are staged in LDS two steps ahead, V tiles one; one barrier per step.  Interior steps -- every row
// of the workgroup sees all of tiles t and t + 1 -- carry no masks and take no maximum: their exponents
// stand against a reference some earlier tile of the row set.  A weight only leaves F16's range where a logit
// exceeds it by 16 (log2; 6 in F32 rows), and the row sum tells: of F16 rows it adds the rounded weights, an infinity among
// them; of F32 rows the weights themselves, none of which is above the sum, so it is held below F16's largest
// number.  Then the tile is weighed again against its own maximum.
// Share `w` of KV head `kvh`; ARG: which of the kernel's PagedParams arguments `p` is.
template <int D, typename T, bool CAP, int ARG>
__device__ __forceinline__ void chunk_share(const PagedParams &p, PagedShare work, int w, int kvh, _Float16 *smem) {
  constexpr bool F32 = std::is_same<T, float>::value;
  using TL = ChunkTile<D, F32>;
  constexpr int BN = TL::BN, KP = TL::KP, VP = TL::VP;
  constexpr int KK = D / 16, KB = BN / 32, RB = D / 32, PS = BN / 16;  // logits MFMAs per 32 keys, row blocks of S^T and O^T, P^T slices
  constexpr int CH = BN * D / 8 / 256;  // 16-byte pieces of a K (or V) tile per thread
  constexpr int RPW = 64 / (D / 8);     // rows of a piece that one wave covers
  constexpr bool DEEP = TL::DEEP;
  constexpr int SETS = DEEP ? 2 : 1;
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int kSplit = PS / 2;        // slices of P^T formed in phase B of the step before
  constexpr float kMostSum = F32 ? 65504.0f : 1e30f;  // of a lane's weights in an interior step, as they are
  constexpr int kAhead = 4, kVAhead = D <= 64 ? 4 : 3;  // operand reads kept in flight
  
  _Float16 *const sK = smem, *const sV = smem + 2 * BN * KP;  // [2][BN][KP], [2][BN][VP]
  __shared__ int bad_tile[2];  // tile whose V held infinities or NaN under a mask
  __shared__ int unseen;       // a row's first tile had no logit above -inf
  __shared__ int not_a_number;  // a part's row

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, hl = lane >> 5;
  const int G = p.sched.group;
  const bool windowed = p.sched.window > 0;
  const int window = p.sched.window;
  const int page_mask = (1 << p.page_shift) - 1;
  const uint32_t row_bytes = (uint32_t)p.pool.row * 2;
  const int my_row = lane / (D / 8), my_col = lane % (D / 8);
  const uint32_t lane_off = my_row * row_bytes + 16 * my_col;
  const PagePool k_pool(p.k, p, kvh, D), v_pool(p.v, p, kvh, D);
  // exponents are logit * ce - m_ref (CAP: of the capped logit); a negative scale turns the queries round instead
  float ce = CAP ? kLog2e : factor(__builtin_fabsf(p.scale) * kLog2e);
  const float q_sign = p.scale < 0.0f ? -1.0f : 1.0f;
  const float cap = p.softcap;
  float cap_in = CAP ? factor(__builtin_fabsf(p.scale) / p.softcap) : 0.0f;  // cap * tanh(product * cap_in)
  // V^T operand: ds_read_b64_tr_b16 gives lane i of 16 channel ch0 + i of keys key0 .. key0 + 3 when lane s
  // addresses V[key0 + s / 4][ch0 + 4 (s % 4)]; P^T holds keys 4 hl + {0..3} and 8 + 4 hl + {0..3} of 16
  const int g16 = lane >> 4, s16 = lane & 15;
  const int vlane_off = (4 * (g16 >> 1) + (s16 >> 2)) * VP + 16 * (g16 & 1) + 4 * (s16 & 3);

  PagedCut cut{0, 0, 0, 0};
  // F32: rows that come out as NaN are formed once more, in masked steps only.  They tell an infinite logit from
  // the NaN that its two halves make of it, and add an infinite value by itself, which times the two halves of a
  // weight is NaN as well; the other steps take no such care.
  bool again = false;
  uint64_t again_rows = ~0ull;  // of this wave: the rows to store
  while (work.found) {  // the tiles this share touches
  const PagedPlace it = work.at;
  const int64_t from = work.from(), upto = work.upto();
  const bool entire = from == 0 && upto == it.cost;
  const int slot = 2 * w + (from == 0 ? 1 : 0);
  const int n_rows = (int)std::min<int64_t>((int64_t)(it.s.q_end - it.s.q_begin) * G, 0x7fffffff);
  const int row0 = it.tile * kChunkRows;
  const int row_last = min(n_rows, row0 + kChunkRows) - 1;
  if (!entire && from == 0) cut = PagedCut{(int)((it.start + it.cost - 1) / work.share) - w + 1, it.s.q_begin, row0, row_last + 1 - row0};

  const int row = row0 + 32 * wave + ln;
  const bool row_ok = row < n_rows && (again_rows >> lane & 1);
  const int rr = min(row, row_last);  // rows past the last one repeat it and are not stored
  const int tok = rr / G, head = kvh * G + rr % G;
  const int pos = it.s.pos0 + tok;
  const int wg_first = it.s.pos0 + row0 / G, wg_last = it.s.pos0 + row_last / G;  // positions of the workgroup's rows

  // keys the tile's rows see, and this part of them
  const int key_end = min(it.s.len, max(wg_last, -1) + 1);
  const int key_begin = windowed && wg_first >= window ? (wg_first - window + 1) / BN * BN : 0;
  const int n_tiles = key_end > key_begin ? (key_end - key_begin + BN - 1) / BN : 0;
  const int t0 = (int)((double)from * n_tiles / it.cost), n_it = (int)((double)upto * n_tiles / it.cost) - t0;
  const int base0 = key_begin + t0 * BN;
  const int part_end = min(key_end, base0 + n_it * BN);
  // key tiles that every row sees whole
  const int full_from = windowed && wg_last >= window ? max(0, (wg_last - window + BN - base0) / BN) : 0;
  const int full_upto = min(n_it, max(0, min(wg_first + 1, key_end) - base0) / BN);

  // ---- tiles: a wave fetches BN / 4 consecutive rows, which lie in one page, in CH pieces of 16 bytes per lane
  constexpr int SPAN = BN / 16;  // pages a tile touches at most
  static_assert(BN / 4 <= 16, "a wave's rows of a tile lie in one page");
  PageWindow pages;
  pages.start<SPAN>(p, it.seq, base0 >> p.page_shift);
  half8_t kpre[SETS][CH], vpre[SETS][CH];
  uint64_t page_off = 0;  // of the K tile requested last; its V tile follows a step later
  uint32_t row_off = 0;
  auto fetch_k = [&](int t, half8_t(&pre)[CH]) __attribute__((always_inline)) {  // behind the part: its last page again
    const int base = base0 + t * BN, key = base + wave * (BN / 4);
    pages.advance<SPAN>(min(base, part_end - 1) >> p.page_shift);
    page_off = pages.offset(min(key, part_end - 1) >> p.page_shift);
    row_off = (uint32_t)(key & page_mask) * row_bytes;
    const __amdgpu_buffer_rsrc_t rows = k_pool.rows(page_off);
#pragma unroll
    for (int i = 0; i < CH; ++i)
      pre[i] = __builtin_bit_cast(half8_t, __builtin_amdgcn_raw_buffer_load_b128(rows, lane_off, row_off + i * (RPW * row_bytes), 0));
  };
  auto fetch_v = [&](half8_t(&pre)[CH]) __attribute__((always_inline)) {  // of the K tile requested last
    const __amdgpu_buffer_rsrc_t rows = v_pool.rows(page_off);
#pragma unroll
    for (int i = 0; i < CH; ++i)
      pre[i] = __builtin_bit_cast(half8_t, __builtin_amdgcn_raw_buffer_load_b128(rows, lane_off, row_off + i * (RPW * row_bytes), 0));
  };
  const int stage_row = wave * (BN / 4) + my_row;
  auto stage_k = [&](auto buf_c, half8_t(&pre)[CH]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      *(half8_t *)(sK + stage_row * KP + 8 * my_col + (decltype(buf_c)::value * BN + RPW * i) * KP) = pre[i];
  };
  auto stage_v = [&](auto buf_c, int t, half8_t(&pre)[CH], bool seen_whole) __attribute__((always_inline)) {  // tile t into buffer t % 2
    if (!seen_whole) {
      // A weight of zero does not keep an infinity or a NaN out of the product: such values of V leave the
      // tile here and are added, by themselves, to the rows that see their key.
      bool bad = false;
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (not_finite(pre[i][e])) {
            bad = true;
            pre[i][e] = (_Float16)0.0f;
          }
      if (bad) bad_tile[decltype(buf_c)::value] = t;
    }
#pragma unroll
    for (int i = 0; i < CH; ++i)
      *(half8_t *)(sV + stage_row * VP + 8 * my_col + (decltype(buf_c)::value * BN + RPW * i) * VP) = pre[i];
  };
  auto seen_whole = [&](int t) __attribute__((always_inline)) { return !(F32 && again) && t >= full_from && t < full_upto; };

  // ---- Q as the B operand: lane (row ln, half hl) holds channels 16 kk + 8 hl .. + 7
  half8_t qh[KK], ql[F32 ? KK : 1];
  auto load_q = [&]() __attribute__((always_inline)) {
    const T *qp = (const T *)p.q + (int64_t)(it.s.q_begin + tok) * p.q_stride + (int64_t)head * D + 8 * hl;
    int shift = 0;
    if constexpr (F32) {
      float largest = 0.0f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const float4_t a = *(const float4_t *)(qp + 16 * kk), b = *(const float4_t *)(qp + 16 * kk + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) largest = larger_finite(largest, e < 4 ? a[e] : b[e - 4]);
      }
      shift = row_shift(xor32_combine(largest, [](float a, float b) { return fmaxf(a, b); }));
      if constexpr (CAP) cap_in = factor(__builtin_ldexpf(factor(__builtin_fabsf(p.scale) / cap), -shift));
      else ce = factor(__builtin_ldexpf(factor(__builtin_fabsf(p.scale) * kLog2e), -shift));
      asm volatile("" : "+v"(qp));  // read again rather than held
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if constexpr (F32) {
        const float4_t a = *(const float4_t *)(qp + 16 * kk), b = *(const float4_t *)(qp + 16 * kk + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          _Float16 hi, lo;
          split_f16(__builtin_ldexpf((e < 4 ? a[e] : b[e - 4]) * q_sign, shift), hi, lo);
          qh[kk][e] = hi;
          ql[kk][e] = lo;
        }
      } else {
        qh[kk] = *(const half8_t *)(qp + 16 * kk);
        if (q_sign < 0.0f) qh[kk] = -qh[kk];
      }
    }
  };

  float16_t o_acc[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int i = 0; i < 16; ++i) o_acc[r][i] = 0.0f;
  float m_run = kNegInf, m_ref = 0.0f, l_run = 0.0f;  // m_ref: what exponents stand against; m_run the same, -inf while no key was seen

  typedef float16_t STile[KB];
  typedef half8_t PTile[PS];
  auto qk_tile = [&](auto buf_c, STile &s) __attribute__((always_inline)) {
    const _Float16 *kt = sK + ln * KP + 8 * hl + decltype(buf_c)::value * BN * KP;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const half8_t a = *(const half8_t *)(kt + 32 * kb * KP + 16 * kk);
        s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[kk], kk == 0 ? float16_t{0.0f} : s[kb], 0, 0, 0);
        if constexpr (F32) s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[kk], s[kb], 0, 0, 0);
      }
  };
  // Order of a phase, given once its code has been emitted: operand reads a few MFMAs ahead.  (Placing the
  // exponentials behind the MFMAs as well made no difference at d 128 and cost 4 % at d 256.)
  auto sched_qk = [&]() __attribute__((always_inline)) {
    constexpr int N = KK * KB, AH = kAhead < N ? kAhead : N;
    __builtin_amdgcn_sched_group_barrier(0x100, AH, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, F32 ? 2 : 1, 0);
      if (i < N - AH) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  };
  auto pv_tile = [&](auto buf_c, PTile &ph, PTile &pl) __attribute__((always_inline)) {
    const _Float16 *vt = sV + vlane_off + decltype(buf_c)::value * BN * VP;
#pragma unroll
    for (int jn = 0; jn < PS; ++jn)
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const _Float16 *vp = vt + 16 * jn * VP + 32 * r;
        const half4_t lo = lds_read_tr16(vp), hi = lds_read_tr16(vp + 8 * VP);
        const half8_t a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        o_acc[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[jn], o_acc[r], 0, 0, 0);
        if constexpr (F32) o_acc[r] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[jn], o_acc[r], 0, 0, 0);
      }
  };
  auto sched_pv = [&]() __attribute__((always_inline)) {
    constexpr int N = PS * RB, AH = kVAhead < N ? kVAhead : N;
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * AH, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, F32 ? 2 : 1, 0);
      if (i < N - AH) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  };
  auto row_max = [&](STile &s, auto raw_c) __attribute__((always_inline)) {  // raw: products of q and k, not capped yet
    float mt = kNegInf;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mt = fmaxf(mt, s[kb][i]);
    mt = xor32_combine(mt, [](float a, float b) { return fmaxf(a, b); });
    if constexpr (CAP && decltype(raw_c)::value) mt = soft_cap<F32>(mt, cap, cap_in);
    return mt * ce;
  };
  // Weights of F32 rows stand 2^10 higher, so that what a pair of F16 halves cannot hold is 2^-35 of the reference,
  // not 2^-25 (thousands of keys that far below the largest one add up): its weight is 2^10, and 2^15 where the
  // reference lags most, which leaves F16's range a factor of two.
  constexpr float kUp = F32 ? 10.0f : 0.0f;
  constexpr float kLazy = F32 ? 5.0f : 8.0f;
  // Cap, mask and maximum of tile t.  The reference moves where a row's maximum exceeds it by more than
  // kLazy (log2), or when the row sees its first key; the factor its sums take with it is returned.
  auto mask_max = [&](auto buf_c, int t, STile &s) __attribute__((always_inline)) -> float {
    const int base = base0 + t * BN;
    if constexpr (CAP) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = soft_cap<F32>(s[kb][i], cap, cap_in);
    }
    if (!seen_whole(t)) {
      const int hi = min(pos, key_end - 1), lo = windowed ? pos - window : -1;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = base + 32 * kb + 8 * (i / 4) + 4 * hl + (i % 4);
          s[kb][i] = key <= hi && key > lo ? s[kb][i] : kNegInf;
        }
    }
    if constexpr (F32) {
      // An infinite key times the two halves of a query is infinity minus infinity, or infinity times zero:
      // where a logit is NaN, the high half alone says whether it is infinite.
      float any = 0.0f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) any += s[kb][i];
      if (__builtin_amdgcn_ballot_w64(any != any) != 0) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          float16_t high = {0.0f};
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
            high = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                *(const half8_t *)(sK + ln * KP + 8 * hl + (decltype(buf_c)::value * BN + 32 * kb) * KP + 16 * kk), qh[kk], high, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x = high[i];
            if constexpr (CAP) x = soft_cap<F32>(x, cap, cap_in);
            if (s[kb][i] != s[kb][i] && __builtin_isinf(high[i])) s[kb][i] = x;
          }
        }
      }
    }
    const float mt = row_max(s, std::false_type{});
    const bool first = m_run == kNegInf;
    const float over = mt - m_ref;
    const float delta = first ? (mt == kNegInf ? 0.0f : over) : over > kLazy ? over : 0.0f;
    m_ref += delta;
    if (!first || mt != kNegInf) m_run = m_ref;
    return first ? 0.0f : __builtin_amdgcn_exp2f(-delta);
  };
  auto rescale = [&](float alpha) __attribute__((always_inline)) {
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) o_acc[r][i] *= alpha;
      l_run *= alpha;
    }
  };
  // probabilities of slices [J0, J1) of a tile; returns their row sum (this half's keys)
  auto exp_part = [&](STile &s, PTile &ph, PTile &pl, auto raw_c, auto j0_c, auto j1_c) __attribute__((always_inline)) -> float {
    float sum = 0.0f;
    const float off = F32 ? kUp - m_ref : -m_ref;
#pragma unroll
    for (int jn = decltype(j0_c)::value; jn < decltype(j1_c)::value; ++jn) {
      typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float x = s[jn / 2][8 * (jn % 2) + e];
        if constexpr (CAP && decltype(raw_c)::value) x = soft_cap<F32>(x, cap, cap_in);
        x = __builtin_amdgcn_exp2f(__builtin_fmaf(x, ce, off));
        if constexpr (F32) {
          _Float16 hi, lo;
          split_f16(x, hi, lo);
          ph[jn][e] = hi;
          pl[jn][e] = lo;
          sum += x;
        } else {
          ph[jn][e] = (_Float16)x;
        }
      }
      if constexpr (!F32) {
        // the sum takes the rounded weights the matrix cores consume
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const half2_t pr = {ph[jn][e], ph[jn][e + 1]}, one = {(_Float16)1.0f, (_Float16)1.0f};
          sum = __builtin_amdgcn_fdot2(pr, one, sum, false);
        }
      }
    }
    return sum;
  };
  typedef std::integral_constant<int, 0> J0;
  typedef std::integral_constant<int, kSplit> JS;
  typedef std::integral_constant<int, PS> JN;
  // the infinities and NaN that were taken out of V tile t, to the rows that see them
  auto add_bad = [&](int t) __attribute__((always_inline)) {
    for (int k = 0; k < BN; ++k) {
      const int key = base0 + t * BN + k;
      if (key >= part_end) break;
      const int number = pages.row[key >> p.page_shift];  // key < key_end <= the table's room
      if ((uint32_t)number >= pages.n_pages) continue;
      const _Float16 *vrow = (const _Float16 *)(v_pool.base + (uint64_t)(uint32_t)number * pages.page_bytes + (uint32_t)(key & page_mask) * row_bytes);
      const bool sees = key <= pos && !(windowed && key <= pos - window);
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const half4_t x = *(const half4_t *)(vrow + 32 * r + 8 * i4 + 4 * hl);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (sees && not_finite(x[e])) o_acc[r][4 * i4 + e] += (float)x[e];
          __builtin_amdgcn_sched_barrier(0);  // a few conditions at a time: this path is rare and must not cost the common one registers
        }
    }
  };

  auto row_is_nan = [&]() __attribute__((always_inline)) {  // this lane's part of the row, or its sum
    float x = l_run;
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) x = __builtin_fmaf(o_acc[r][i], 0.0f, x);
    return x != x;
  };

  PTile p_a, p_b, p_lo;
  float l_head = 0.0f;   // row sum of the slices formed early
  // One step: on entry s_cur holds the logits of tile t (edge steps: masked, their reference set, the sums'
  // factor in alpha; interior steps: the first slices of P formed).
  auto step = [&](int t, STile &s_cur, STile &s_next, PTile &p_cur, PTile &p_next, float &alpha, auto interior_c, auto parity_c) __attribute__((always_inline)) {
    constexpr bool INTERIOR = decltype(interior_c)::value;
    typedef std::integral_constant<int, decltype(parity_c)::value> Buf;         // t % 2
    typedef std::integral_constant<int, 1 - decltype(parity_c)::value> Other;
    constexpr int FETCH = DEEP ? Buf::value : 0, STAGE = DEEP ? Other::value : 0;
    constexpr int AHEAD = DEEP ? 1 : 0;
    if constexpr (!INTERIOR) rescale(alpha);
    fetch_v(vpre[FETCH]);                  // tile t + 1 + AHEAD
    fetch_k(t + 2 + AHEAD, kpre[FETCH]);
    qk_tile(Other{}, s_next);  // behind the last tile: of zeros, or of what is staged, and not used
    if constexpr (INTERIOR) {
      float sum = l_head + exp_part(s_cur, p_cur, p_lo, std::true_type{}, JS{}, JN{});
      sched_qk();
      if (__builtin_amdgcn_ballot_w64(!(sum < kMostSum)) != 0) {
        const float delta = fmaxf(row_max(s_cur, std::true_type{}) - m_ref, 0.0f);
        rescale(__builtin_amdgcn_exp2f(-delta));
        m_ref += delta;
        m_run = m_ref;
        sum = exp_part(s_cur, p_cur, p_lo, std::true_type{}, J0{}, JN{});
      }
      l_run += sum;
    } else {
      sched_qk();
      l_run += exp_part(s_cur, p_cur, p_lo, std::false_type{}, J0{}, JN{});
    }
    pv_tile(Buf{}, p_cur, p_lo);
    if constexpr (INTERIOR) {
      l_head = exp_part(s_next, p_next, p_lo, std::true_type{}, J0{}, JS{});
      // formed here, beside the MFMAs, and not where they are first used
#pragma unroll
      for (int jn = 0; jn < kSplit; ++jn) asm volatile("" : "+v"(p_next[jn]));
      asm volatile("" : "+v"(l_head));
      sched_pv();
    } else {
      sched_pv();
      if (!seen_whole(t) && bad_tile[Buf::value] == t) add_bad(t);
      if (t + 1 < n_it) alpha = mask_max(Other{}, t + 1, s_next);
      else if (F32 && row_is_nan()) not_a_number = 1;
    }
    stage_k(Buf{}, kpre[STAGE]);
    stage_v(Other{}, t + 1, vpre[STAGE], INTERIOR || seen_whole(t + 1));
    __syncthreads();  // fills are visible; every wave is done with the buffers the next step refills
  };

  STile s_a, s_b;
  if (threadIdx.x < 2) bad_tile[threadIdx.x] = -1;
  if (threadIdx.x == 2) unseen = 0;
  if (n_it > 0) {
    constexpr int S1 = DEEP ? 1 : 0;
    typedef std::integral_constant<int, 0> Even;
    typedef std::integral_constant<int, 1> Odd;
    fetch_k(0, kpre[0]);
    fetch_v(vpre[0]);
    if constexpr (DEEP) fetch_k(1, kpre[1]);
    __builtin_amdgcn_sched_barrier(0);
    load_q();
    __syncthreads();  // bad_tile, unseen
    if (threadIdx.x == 2) not_a_number = 0;  // everyone has read the last part's
    stage_k(Even{}, kpre[0]);
    stage_v(Even{}, 0, vpre[0], seen_whole(0));
    if constexpr (!DEEP) fetch_k(1, kpre[0]);
    stage_k(Odd{}, kpre[S1]);
    if constexpr (DEEP) {  // what step 0 stages at its end
      fetch_v(vpre[1]);
      fetch_k(2, kpre[1]);
    }
    __syncthreads();
    qk_tile(Even{}, s_a);
    sched_qk();
    float alpha = mask_max(Even{}, 0, s_a);
    if (m_run == kNegInf) unseen = 1;
    __syncthreads();  // sK[0] is refilled by the first step
    int t = 0;
    // Steps whose tile and the next are seen whole.  They need a reference: where a row has met no key yet (all
    // its logits are -inf), the masked steps, which set one at the first key, take all tiles.  So they do where a
    // window hides the first keys from some rows: the steps behind those would be interior ones, but are not taken.
    const int n_int = full_from == 0 && !unseen && !again ? max(0, full_upto - 1) & ~1 : 0;
    if (n_int > 0) {
      if constexpr (CAP) {  // an interior step starts from products
        qk_tile(Even{}, s_a);
        __syncthreads();
      }
      l_head = exp_part(s_a, p_a, p_lo, std::true_type{}, J0{}, JS{});
      for (; t < n_int; t += 2) {
        step(t, s_a, s_b, p_a, p_b, alpha, std::true_type{}, Even{});
        step(t + 1, s_b, s_a, p_b, p_a, alpha, std::true_type{}, Odd{});
      }
      // tile t has its logits but no maximum yet, and its early slices are formed again with the others
      alpha = mask_max(Even{}, t, s_a);
      if constexpr (F32) __syncthreads();  // it may have read K tile t again, which the next step refills
    }
    for (; t < n_it; t += 2) {
      step(t, s_a, s_b, p_a, p_a, alpha, std::false_type{}, Even{});
      if (t + 1 < n_it) step(t + 1, s_b, s_a, p_a, p_a, alpha, std::false_type{}, Odd{});
    }
  }

  l_run += __shfl_xor(l_run, 32, 64);
  {
  const PagedParams &p = params_again<ARG>();
  if (!entire) {
    if (row_ok) {
      const int64_t at = ((int64_t)slot * p.heads_kv + kvh) * kChunkRows + 32 * wave + ln;
      float *o = p.ws_o + at * D;
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          *(float4_t *)(o + 32 * r + 8 * i4 + 4 * hl) = float4_t{o_acc[r][4 * i4], o_acc[r][4 * i4 + 1], o_acc[r][4 * i4 + 2], o_acc[r][4 * i4 + 3]};
      if (hl == 0) {
        p.ws_ml[at * 2] = m_run;
        p.ws_ml[at * 2 + 1] = l_run;
      }
    }
  } else if (row_ok) {
    const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
    T *out = (T *)p.out + (int64_t)(it.s.q_begin + tok) * p.out_stride + (int64_t)head * D;
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)(l_run == 0.0f ? 0.0f : o_acc[r][4 * i4 + e] * inv);
        *(T4 *)(out + 32 * r + 8 * i4 + 4 * hl) = o;
      }
  }
  if constexpr (F32) {
    const bool first = !again;
    again = false;
    again_rows = ~0ull;
    if (first && n_it > 0 && __builtin_amdgcn_readfirstlane(not_a_number) != 0) {
      again = true;
      again_rows = __builtin_amdgcn_ballot_w64(row_is_nan());
      again_rows |= again_rows >> 32 | again_rows << 32;  // a row's two lanes
      continue;
    }
  }
  work.next(p.sched, p.cu_new, p.kv_len);
  }
  }
  if (p.cuts && w < p.sched.target && kvh == 0 && threadIdx.x == 0) p.cuts[w] = cut;
}

}  // namespace

}  // namespace argus_paged
