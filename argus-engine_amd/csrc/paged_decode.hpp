// paged_attention of requests with few rows (new tokens x heads of a GQA group, at most 16): decode
// steps and short drafts.  Split over the keys, both products on the matrix cores.
//
//   S^T[key][row] = K . Q^T   v_mfma_f32_16x16x32_f16: A lane (j, r) = chunk 4 kk + j of key r's row -- 16
//                             consecutive keys lie in one page, so this is one 16-byte load per lane with the
//                             page's descriptor in scalar registers; B = the same chunk of row r of Q
//   O[row][channel] = P . V   A = the lane's own probabilities (keys 4j .. 4j + 3 of each 16), B = V rows
//                             transposed 4 x 8 in registers
//
// Nothing goes through LDS in the key loop.  The scale is applied to the F32 logit, so F16 queries enter as
// they are and their products are exact; probabilities are rounded to F16, as the output will be.  F32
// queries and the probabilities of their rows are held as F16 pairs, hi + lo, in two MFMAs each, which
// leaves F32's error.  Bound by HBM: every key is read once per KV head for all rows.  Measured: 16 requests
// of up to 32768 tokens (32/8 heads, d 128, F32) 190 us, 6.4 TB/s; 32 requests of 4 tokens over 8192 (F16)
// 166 us, 6.5 TB/s; 64 windows of 2048 keys (8/4 heads, d 256, soft cap) 88 us, 5.9 TB/s.
#pragma once

#include "paged_common.hpp"

#include <algorithm>
#include <type_traits>

namespace argus_paged {

namespace {

template <int D>
struct DecodeShape {
  static constexpr int KK = D / 32;              // logits MFMAs per 16 keys
  static constexpr int VC = D >= 128 ? 8 : 4;    // channels of a V piece
  static constexpr int VSEG = D / (16 * VC);     // pieces per row and lane
  static constexpr int NACC = VC * VSEG;
  static constexpr int TW = D <= 128 ? 2 : 1;    // blocks of 16 keys per wave step
};
constexpr int kWaves = 4;  // of a workgroup, each taking every fourth step of the keys

template <typename T>
__device__ __forceinline__ T load_stream(__amdgpu_buffer_rsrc_t rsrc, uint32_t voff, uint32_t soff);
template <>
__device__ __forceinline__ half8_t load_stream<half8_t>(__amdgpu_buffer_rsrc_t rsrc, uint32_t voff, uint32_t soff) {
  return __builtin_bit_cast(half8_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, voff, soff, 2));
}
template <>
__device__ __forceinline__ half4_t load_stream<half4_t>(__amdgpu_buffer_rsrc_t rsrc, uint32_t voff, uint32_t soff) {
  return __builtin_bit_cast(half4_t, __builtin_amdgcn_raw_buffer_load_b64(rsrc, voff, soff, 2));
}

template <int D>
constexpr int kDecodeLds = kWaves * 16 * (D + 4) * (int)sizeof(float);  // merge of the waves

// Share `w` of KV head `kvh`; ARG: which of the kernel's PagedParams arguments `p` is.
template <int D, typename T, bool CAP, int ARG>
__device__ __forceinline__ void decode_share(const PagedParams &p, PagedShare work, int w, int kvh, float *lds_acc) {  // lds_acc: [kWaves][16][D + 4]
  using SH = DecodeShape<D>;
  constexpr int KK = SH::KK, VC = SH::VC, VSEG = SH::VSEG, NACC = SH::NACC, TW = SH::TW;
  constexpr int STEP = 16 * TW;
  static_assert(STEP == decode_align(D), "key ranges start on a step");
  constexpr bool F32 = std::is_same<T, float>::value;
  typedef typename std::conditional<VC == 8, half8_t, half4_t>::type vpiece_t;
  constexpr float kLog2e = 1.4426950408889634f;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane >> 4, r = lane & 15;
  const int G = p.sched.group;
  const int window = p.sched.window > 0 ? p.sched.window : 0x7fffffff;
  const int page_mask = (1 << p.page_shift) - 1;
  const uint32_t row_bytes = (uint32_t)p.pool.row * 2;
  const uint32_t k_lane = r * row_bytes + 16 * j, v_lane = 4 * j * row_bytes + 2 * VC * r;
  const PagePool k_pool(p.k, p, kvh, D), v_pool(p.v, p, kvh, D);
  const float inv_cap = CAP ? 1.0f / p.softcap : 0.0f;
  __shared__ float lds_m[kWaves][16], lds_l[kWaves][16];

  PagedCut cut{0, 0, 0, 0};
  // F32: an infinite V times the two halves of a weight is NaN.  A wave whose results hold one goes over its keys
  // again with the care that masked keys get, which adds such values by themselves.
  bool again = false;
  while (work.found) {  // the requests this share touches
  const PagedPlace it = work.at;
  const int rows = (it.s.q_end - it.s.q_begin) * G;  // at most 16: one tile
  const int64_t from = work.from(), upto = work.upto();
  const bool entire = from == 0 && upto == it.cost;
  const int slot = 2 * w + (from == 0 ? 1 : 0);
  if (!entire && from == 0) cut = PagedCut{(int)((it.start + it.cost - 1) / work.share) - w + 1, it.s.q_begin, 0, rows};
  const int begin = std::min<int64_t>(it.s.key_end, it.s.key_begin + from * p.sched.unit);
  const int end = std::min<int64_t>(it.s.key_end, it.s.key_begin + upto * p.sched.unit);

  // row r: token r / G, head r % G; columns past the last row repeat it and are never stored
  const int rr = min(r, rows - 1);
  const int pos = it.s.pos0 + rr / G;
  const int pos_last = it.s.pos0 + (rows - 1) / G;

  PageWindow pages;
  pages.start<TW>(p, it.seq, begin >> p.page_shift);
  half8_t kr[TW][KK];
  vpiece_t vr[TW][VSEG][4];
  // 16 consecutive keys lie in one page: where, of the K rows requested last (the V rows follow)
  uint64_t page_off[TW];
  uint32_t row_off[TW];
  auto load_k = [&](int base) {  // behind the part: its last page again
    pages.advance<TW>(max(min(base, end - 1), begin) >> p.page_shift);
#pragma unroll
    for (int tw = 0; tw < TW; ++tw) {
      page_off[tw] = pages.offset(max(min(base + 16 * tw, end - 1), begin) >> p.page_shift);
      row_off[tw] = (uint32_t)((base + 16 * tw) & page_mask) * row_bytes;
      const __amdgpu_buffer_rsrc_t rsrc = k_pool.rows(page_off[tw]);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) kr[tw][kk] = load_stream<half8_t>(rsrc, k_lane + 64 * kk, row_off[tw]);
    }
  };
  auto load_v = [&]() {
#pragma unroll
    for (int tw = 0; tw < TW; ++tw) {
      const __amdgpu_buffer_rsrc_t rsrc = v_pool.rows(page_off[tw]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int sg = 0; sg < VSEG; ++sg) vr[tw][sg][e] = load_stream<vpiece_t>(rsrc, v_lane + e * row_bytes + 32 * VC * sg, row_off[tw]);
    }
  };
  // Q: lane (j, r) holds chunk 4 kk + j of row r.  Requested ahead of the first keys and waited for ahead of
  // the loop: a wait for the query inside it would be one for everything requested since.
  half8_t qh[KK], ql[F32 ? KK : 1];
  const T *qp = (const T *)p.q + (int64_t)(it.s.q_begin + rr / G) * p.q_stride + (int64_t)(kvh * G + rr % G) * D + 8 * j;
  float qx[F32 ? KK : 1][8];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    if constexpr (F32) {
      const float4_t a = *(const float4_t *)(qp + 32 * kk), b = *(const float4_t *)(qp + 32 * kk + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) qx[kk][e] = e < 4 ? a[e] : b[e - 4];
    } else {
      qh[kk] = *(const half8_t *)(qp + 32 * kk);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  const int base0 = begin + wave * STEP;
  load_k(base0);
  load_v();
  __builtin_amdgcn_sched_barrier(0);
  int shift = 0;
  if constexpr (F32) {
    float largest = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e) largest = larger_finite(largest, qx[kk][e]);
    shift = row_shift(rows_allreduce_max(largest));
  }
  const float c = factor(__builtin_ldexpf(factor(CAP ? p.scale : p.scale * kLog2e), -shift));  // of row r: products to logits (CAP) or exponents
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        _Float16 hi, lo;
        split_f16(__builtin_ldexpf(qx[kk][e], shift), hi, lo);
        qh[kk][e] = hi;
        ql[kk][e] = lo;
      }
    } else {
      asm volatile("" : "+v"(qh[kk]));
    }
  }


  float4_t o_acc[NACC];
#pragma unroll
  for (int a = 0; a < NACC; ++a) o_acc[a] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m_run = kNegInf, l_run = 0.0f;  // of row r; l: this lane group's keys

  for (int base = base0; base < end; base += kWaves * STEP) {
    float4_t s[TW];
#pragma unroll
    for (int tw = 0; tw < TW; ++tw) {
      s[tw] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      float4_t low = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        s[tw] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr[tw][kk], qh[kk], s[tw], 0, 0, 0);
        if constexpr (F32) low = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr[tw][kk], ql[kk], low, 0, 0, 0);
      }
      if constexpr (F32) {  // an infinite logit is the high half's: the low one would add the other sign, or zero times it
#pragma unroll
        for (int i = 0; i < 4; ++i) s[tw][i] += __builtin_isinf(s[tw][i]) ? 0.0f : low[i];
      }
    }
    load_k(base + kWaves * STEP);
    // keys some row does not see: past the first token's position, in front of the last one's window, past the part
    const bool edge = (F32 && again) || base + STEP - 1 > it.s.pos0 || base + STEP > end || (window != 0x7fffffff && base <= pos_last - window);
#pragma unroll
    for (int tw = 0; tw < TW; ++tw)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (CAP) s[tw][i] = soft_cap<F32>(s[tw][i] * c, p.softcap, inv_cap) * kLog2e;
        else s[tw][i] *= c;
      }
    if (edge) {
      const int hi = min(pos, end - 1), lo = window != 0x7fffffff ? pos - window : -1;
#pragma unroll
      for (int tw = 0; tw < TW; ++tw)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = base + 16 * tw + 4 * j + i;
          s[tw][i] = key <= hi && key > lo ? s[tw][i] : kNegInf;
        }
    }
    float mt = kNegInf;
#pragma unroll
    for (int tw = 0; tw < TW; ++tw)
#pragma unroll
      for (int i = 0; i < 4; ++i) mt = fmaxf(mt, s[tw][i]);
    mt = rows_allreduce_max(mt);
    const float m_new = fmaxf(m_run, mt);
    const float m_ref = m_new == kNegInf ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_ref);
    m_run = m_new;
    half4_t pa[TW], pl[F32 ? TW : 1];
    float lsum = 0.0f;
    // Weights of F32 rows stand 2^14 higher: what a pair of F16 halves cannot hold is then 2^-39 of the largest
    const float off = F32 ? m_ref - 14.0f : m_ref;
#pragma unroll
    for (int tw = 0; tw < TW; ++tw)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = __builtin_amdgcn_exp2f(s[tw][i] - off);
        lsum += w;
        if constexpr (F32) {
          _Float16 hi, lo;
          split_f16(w, hi, lo);
          pa[tw][i] = hi;
          pl[tw][i] = lo;
        } else {
          pa[tw][i] = (_Float16)w;
        }
      }
    l_run = l_run * alpha + lsum;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
      float al[4];  // accumulator register i of lane group j belongs to row 4j + i
#pragma unroll
      for (int i = 0; i < 4; ++i) al[i] = __shfl(alpha, 4 * j + i, 64);
#pragma unroll
      for (int a = 0; a < NACC; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) o_acc[a][i] *= al[i];
    }
    if (edge) {
      // A weight of zero does not keep an infinity or a NaN out of the product.  Such values of V leave
      // the operands here and are added, by themselves, to the rows that see their key.
      bool any = false;
#pragma unroll
      for (int tw = 0; tw < TW; ++tw)
#pragma unroll
        for (int sg = 0; sg < VSEG; ++sg)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int ch = 0; ch < VC; ++ch) any |= not_finite(vr[tw][sg][e][ch]);
      if (__builtin_amdgcn_ballot_w64(any) != 0) {
#pragma unroll
        for (int tw = 0; tw < TW; ++tw)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            for (int jj = 0; jj < 4; ++jj) {
              const int key = base + 16 * tw + 4 * jj + e;
              bool sees[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int row_pos = it.s.pos0 + min(4 * j + i, rows - 1) / G;
                sees[i] = key <= row_pos && key < end && !(window != 0x7fffffff && key <= row_pos - window);
              }
#pragma unroll
              for (int sg = 0; sg < VSEG; ++sg)
#pragma unroll
                for (int ch = 0; ch < VC; ++ch) {
                  const float x = __shfl((float)vr[tw][sg][e][ch], 16 * jj + r, 64);
                  if (!(__builtin_fabsf(x) < __builtin_huge_valf()))
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                      if (sees[i]) o_acc[sg * VC + ch][i] += x;
                  __builtin_amdgcn_sched_barrier(0);  // one value at a time: this path is rare and must not cost the common one registers
                }
            }
#pragma unroll
        for (int tw = 0; tw < TW; ++tw)
#pragma unroll
          for (int sg = 0; sg < VSEG; ++sg)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int ch = 0; ch < VC; ++ch)
                if (not_finite(vr[tw][sg][e][ch])) vr[tw][sg][e][ch] = (_Float16)0.0f;
      }
    }
#pragma unroll
    for (int sg = 0; sg < VSEG; ++sg)
#pragma unroll
      for (int ch = 0; ch < VC; ++ch) {
        float4_t &o = o_acc[sg * VC + ch];
        if constexpr (TW == 2) {
          // contraction slots 8j + e hold keys 4j + e of the first block, 8j + 4 + e those of the second
          const half8_t bv = {vr[0][sg][0][ch], vr[0][sg][1][ch], vr[0][sg][2][ch], vr[0][sg][3][ch],
                              vr[1][sg][0][ch], vr[1][sg][1][ch], vr[1][sg][2][ch], vr[1][sg][3][ch]};
          const half8_t av = {pa[0][0], pa[0][1], pa[0][2], pa[0][3], pa[1][0], pa[1][1], pa[1][2], pa[1][3]};
          o = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, bv, o, 0, 0, 0);
          if constexpr (F32) {
            const half8_t lv = {pl[0][0], pl[0][1], pl[0][2], pl[0][3], pl[1][0], pl[1][1], pl[1][2], pl[1][3]};
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(lv, bv, o, 0, 0, 0);
          }
        } else {
          const half4_t bv = {vr[0][sg][0][ch], vr[0][sg][1][ch], vr[0][sg][2][ch], vr[0][sg][3][ch]};
          o = __builtin_amdgcn_mfma_f32_16x16x16f16(pa[0], bv, o, 0, 0, 0);
          if constexpr (F32) o = __builtin_amdgcn_mfma_f32_16x16x16f16(pl[0], bv, o, 0, 0, 0);
        }
      }
    load_v();
  }
  if constexpr (F32) {
    float x = 0.0f;
#pragma unroll
    for (int a = 0; a < NACC; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) x = __builtin_fmaf(o_acc[a][i], 0.0f, x);
    again = !again && __builtin_amdgcn_ballot_w64(x != x) != 0;
    if (again) continue;
  }

  // ---- merge: lane groups (row sum), then the waves through LDS -----------------------------------
  const PagedParams &p = params_again<ARG>();
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  if (j == 0) {
    lds_m[wave][r] = m_run;
    lds_l[wave][r] = l_run;
  }
#pragma unroll
  for (int sg = 0; sg < VSEG; ++sg)
#pragma unroll
    for (int ch = 0; ch < VC; ++ch)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * j + i < rows) lds_acc[(wave * 16 + 4 * j + i) * (D + 4) + 16 * VC * sg + VC * r + ch] = o_acc[sg * VC + ch][i];
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += 64 * kWaves) {
    const int row = i / D, ch = i % D;
    float mm = lds_m[0][row];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) mm = fmaxf(mm, lds_m[v][row]);
    const float m_ref = mm == kNegInf ? 0.0f : mm;
    float o = 0.0f, l = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float f = __builtin_amdgcn_exp2f(lds_m[v][row] - m_ref);
      o += lds_acc[(v * 16 + row) * (D + 4) + ch] * f;
      l += lds_l[v][row] * f;
    }
    if (entire) {
      T *out = (T *)p.out + (int64_t)(it.s.q_begin + row / G) * p.out_stride + (int64_t)(kvh * G + row % G) * D;
      out[ch] = (T)(l == 0.0f ? 0.0f : o / l);
    } else {
      const int64_t at = ((int64_t)slot * p.heads_kv + kvh) * kDecodeRows + row;
      p.ws_o[at * D + ch] = o;
      if (ch == 0) {
        p.ws_ml[at * 2] = mm;
        p.ws_ml[at * 2 + 1] = l;
      }
    }
  }
  __syncthreads();  // the merge area is free for the next request
  work.next(p.sched, p.cu_new, p.kv_len);
  }
  if (p.cuts && kvh == 0 && threadIdx.x == 0) p.cuts[w] = cut;
}

}  // namespace

}  // namespace argus_paged
