// Attention of few queries over the codes of an fp16 cache, with a sliding window
// and first tokens that stay visible (gfx950).
//
// A workgroup takes one kv head of one sequence, up to 16 rows (the kv head's
// query heads, of several queries where they fit) and a share of the blocks of
// 32 tokens that any of the rows sees; its eight waves take runs of blocks,
// coded or uncoded, each on its own until the end.
//
// A coded block: a pair of key codes is an entry of a table of levels as fp16 pairs
// (hi + lo: 2^-22; scaled single ones were 1 us of 33 faster, and the result's error
// a third larger), four of them an operand of K Q^T as they are; the group's scale
// goes into the query, a pair too (over a power of two where a product passes fp16),
// its mean into the scores afterwards.  A side-list
// entry, whose code is the zero level, adds q (val - mean): the block's entries
// stand in an otherwise zero LDS tile of the wave, the first halves of their fp16
// pairs, then the second ones, each a second operand of the same product, and are
// cleared one by one.  They go there before the block's lookups, whose time hides
// the trip.  A lane then holds one row's scores of 8 tokens, which are the operand
// of V^T P^T as they are.  Value codes become centroids by pairs through a table,
// the codebook scaled so that its fp16 roundings nearly vanish (best of 128 scales:
// 2^-12 of a centroid becomes about 2^-14 to 2^-15).  Weights times norms, and an
// uncoded block's weights, are rounded to fp16 as the matrix cores take them (at most
// 2^-11 of each; pairs would double the lookups' and values' products): 2.8e-4 to
// 3.0e-4 off 64 bits, where the output's rounding alone is 2.1e-4 off.  The coded part
// is rotated back once a workgroup, by the matrix cores in fp16 pairs.  Up to head_dim 128 a table entry has a row of 256
// bytes of copies, by lane: a lookup's bank is its lane's own, and its address one
// byte permutation; at head_dim 256 the waves' tiles leave room for four copies.
// Bound: few sequences, the chain of dependent loads (lengths, tables, codes) and
// the set-up; many, a wave's chain of LDS trips and products beside its codes from
// HBM: 16 sequences of 32768 tokens, 8 kv heads of 128, 37.6 us with a window of 4096,
// of which a one-block window takes 8; with every page and group the same one, in
// cache, no more than 3% less.
#include "tqk_attend_few.h"

namespace {

constexpr int kFewRows = 16;

struct FewArgs {
  tqk_cache_desc d;
  tqk_cache_ptrs p;
  const uint16_t* q;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  void* out;
  float* part_acc;  // [split][row][D]
  float* part_ml;   // [split][row][2]: running maximum (log2 units) and sum
  long long rows;   // rows of all sequences, heads and queries
  long long q_stride[3];
  long long o_stride[3];
  int q_len, max_len, window, sinks, out_type;
  int per_item;     // queries of a workgroup
  int q_items;      // workgroups a sequence's queries take
  int n_splits;
};

// KB: key code bits; PK: PolarQuant keys (KB == VB); TILED: value codes in units
// of 4 tokens x 8 channels.
template <int D, int VB, int KB, bool PK, bool TILED>
__global__ __launch_bounds__(kFewThreads, 2) void tqk_attend_codes(FewArgs a) {
  constexpr int CPL = D / 4;          // channels of a lane in a score product: CPL lg + 8 m + e
  constexpr int NM = D / 32;          // steps of a score product
  constexpr int KW = CPL * KB / 32 > 0 ? (CPL * KB + 31) / 32 : 1;  // words of a lane's key codes
  constexpr int NC = D >= 128 ? 8 : 4;          // channels of a lane's value piece
  constexpr int NS = D == 256 ? 2 : 1;          // value pieces a lane takes (128 channels apart)
  constexpr int NV = NC * NS;                   // 16-row accumulator tiles
  constexpr int VROW = D * VB / 8, KROW = D * KB / 8;
  const tqk_cache_desc& d = a.d;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int ln = lane & 15, lg = lane >> 4;
  const int G = d.group_tokens, P = d.page_tokens, Hkv = d.n_kv_heads, Hq = d.n_q_heads, gq = Hq / Hkv;
  int x = blockIdx.x;
  const int split = x % a.n_splits;
  x /= a.n_splits;
  const int h = x % Hkv;
  x /= Hkv;
  const int q0 = x % a.q_items * a.per_item, b = x / a.q_items;

  // a wave's side-list tile (32 x D fp16), later its accumulators
  __shared__ __align__(16) uint16_t stage_s[kFewWaves][2 * 16 * D + 8];
  __shared__ __align__(16) float stat_s[kFewWaves][2][D];    // the group's scale and mean
  // a pair of key codes -> its levels, {hi, hi} and {lo, lo}; a pair of value codes
  // -> its centroids; with 4-bit keys and values one row for both
  constexpr bool kRow = D <= 128, kShared = kRow && KB == 4 && VB == 4;
  constexpr int kKeyLog = kRow ? 8 : 5, kValLog = kRow ? 8 : 4;  // log2 of an entry's bytes
  constexpr int kKeyCopies = kShared ? 16 : (1 << kKeyLog) / 8, kValCopies = kShared ? 32 : (1 << kValLog) / 4;
  constexpr int kKeyEntries = 1 << (2 * KB), kValEntries = 1 << (2 * VB);
  __shared__ __align__(256) uint8_t key_s[kKeyEntries << kKeyLog];
  __shared__ __align__(256) uint8_t val_own[kShared ? 4 : kValEntries << kValLog];
  uint8_t* const val_s = kShared ? key_s : val_own;
  constexpr uint32_t kValOff = kShared ? 128 : 0;
  __shared__ __align__(16) float lev_s[16], cen_s[16];
  __shared__ float up_s[2][2];  // the best of the scales of a half: its loss, itself
  __shared__ float ml_s[2][kFewWaves][kFewRows];

  const int n = min(a.seq_lens[b], a.max_len);
  const int m = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
  if (tid < 16) lev_s[tid] = PK ? a.p.vcent[tid & ((1 << VB) - 1)] : key_level(d.key_grid, tid);
  if (tid < (1 << VB)) cen_s[tid] = a.p.vcent[tid];
  // the rows: query q0 + row / gq, head h gq + row % gq
  const int n_rows = min(a.per_item, m - q0) * gq;  // (negative: none)
  const int row = min(ln, max(n_rows, 1) - 1), t = q0 + row / gq, p = n - m + t;
  const int p_lo = n - m + q0, p_hi = n - m + min(q0 + a.per_item, m) - 1;
  const int ng = n_groups_of(n, d.hot_window, G), n_cold = ng * G;
  auto low = [&](int pos) { return a.window > 0 && a.window <= pos ? pos - a.window + 1 : 0; };
  const int lo = low(p), lo_first = low(p_lo), lo_last = low(p_hi);
  const int sinks = min(a.sinks, max(n, 0));
  auto sees = [&](int tok) { return (tok <= p) & ((tok >= lo) | (tok < sinks)); };
  auto all_see = [&](int tok, int cnt) { return tok + cnt - 1 <= p_lo && (tok >= lo_last || tok + cnt <= sinks); };
  // blocks of tokens [from, to) that any row sees, by block(token)
  auto runs = [&](int from, int to, auto block) {
    BlockRuns r{0, 0, 0};
    const int end = min(to, p_hi + 1), s_end = min(min(sinks, end), max(lo_first, from));
    if (n_rows <= 0 || end <= from) return r;
    if (s_end > from) r.n0 = block(s_end - 1) + 1;
    r.from = r.n0;
    r.n = r.n0;
    const int w = max(lo_first, from);
    if (w < end) {
      r.from = max(block(w), r.n0);
      r.n += max(block(end - 1) + 1 - r.from, 0);
    }
    return r;
  };
  const int nblk = (G + 31) / 32;  // blocks of a group
  const BlockRuns cold = runs(0, n_cold, [&](int tok) { return tok / G * nblk + tok % G / 32; });
  const BlockRuns hot = runs(n_cold, n, [&](int tok) { return (tok - n_cold) / 32; });
  // equal runs for the waves of all splits, coded ones first
  const int n_waves = a.n_splits * kFewWaves;
  int run = max((cold.n + hot.n + n_waves - 1) / n_waves, 1);
  while ((cold.n + run - 1) / run + (hot.n + run - 1) / run > n_waves) ++run;
  const int cold_waves = (cold.n + run - 1) / run;
  const int gw = split * kFewWaves + wave;
  const bool is_cold = gw < cold_waves;
  const int i0 = (is_cold ? gw : gw - cold_waves) * run;
  const int i1 = min(i0 + run, is_cold ? cold.n : hot.n);

  // Q: row ln, channels CPL lg + 8 m .. + 7 (rows past the last: a real one's, dropped later)
  h8_t qf[NM];
  const uint16_t* const qp = a.q + b * a.q_stride[0] + (h * gq + row % gq) * a.q_stride[1] +
                             (long long)min(max(t, 0), a.q_len - 1) * a.q_stride[2];
#pragma unroll
  for (int mm = 0; mm < NM; ++mm) qf[mm] = *reinterpret_cast<const h8_t*>(qp + CPL * lg + 8 * mm);
  // the coded keys' weights, an fp16 pair: q * scale group by group, or for
  // rotated keys q @ Pi^T; over a power of two, w_up, where they pass fp16
  h8_t wh[NM], wl[NM];
  float w_up = 1.f;
  // the wave's largest |q| (what is not finite: as the largest of fp16; its rows
  // are lost whatever the power)
  float q_top = 0.f;
  if constexpr (!PK) {
    typedef uint16_t us8_t __attribute__((ext_vector_type(8)));
    us8_t top = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int mm = 0; mm < NM; ++mm)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(us8_t, qf[mm]) & (uint16_t)0x7FFF);
    uint16_t one = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) one = top[e] > one ? top[e] : one;
    q_top = wave_reduce<true>(h2f(one < 0x7C00 ? one : (uint16_t)0x7BFF));
  }

  // ---- the coded blocks of this wave: state and loads
  uint16_t* const list_s = stage_s[wave];
  auto at = [](int tok, int ch) { return (tok * (D / 8) + (ch ^ (tok & 7))) * 8; };  // (turned by the row: bank conflicts)
  const size_t head = (size_t)h * d.n_pages * P;
  const int32_t* const bt = a.p.block_table + (size_t)b * d.max_pages_per_seq;
  const int32_t* const gt = a.p.group_table + (size_t)b * d.max_groups_per_seq;
  const bool listed = !PK && d.outliers_per_channel > 0;
  // (a valid pointer even without a side-list)
  const uint32_t* const oent = listed ? a.p.oent : reinterpret_cast<const uint32_t*>(a.p.ocount);
  const int cap = listed ? d.outlier_cap : 1;

  // Every load of the loop is issued, at an index inside its table, so that the
  // waits on them stay exact.  What the tables say of 64 blocks of the run at a
  // time, one a lane: their chain of loads is paid once.
  const float per_page = 1.0f / (float)P;
  const int group_pages = G / P;
  // the page row of token o of group g (pages inside a group by a product: fewer
  // than 256 tokens, exact)
  auto page_row = [&](int g, int o) {
    const int pg = (int)(((float)o + 0.5f) * per_page);
    return bt[g * group_pages + pg] * P + o - pg * P;
  };
  int meta_i = i0, meta_g = 0, meta_k = 0, meta_ob = 0, meta_lo = 0, meta_hi = 0, meta_row[2] = {0, 0};
  auto load_meta = [&](int i) {
    meta_i = i;
    const int blk = cold.at(min(i + lane, i1 - 1));
    meta_g = blk / nblk;
    meta_k = blk % nblk;
    meta_ob = gt[meta_g] * Hkv + h;
    if constexpr (TILED) {  // (16 tokens lie in one page)
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) meta_row[tile] = page_row(meta_g, 32 * meta_k + 16 * tile);
    }
    const int32_t* oc = a.p.ocount + (size_t)meta_ob * TQK_NOB;
    const int lo_ = oc[max(meta_k - 1, 0)], hi_ = oc[meta_k];
    meta_lo = listed && meta_k > 0 ? min(lo_, cap) : 0;
    meta_hi = listed ? min(hi_, cap) : 0;
  };
  auto of = [&](int x, int i) { return __builtin_amdgcn_readlane(x, i - meta_i); };  // block i's
  // rows of block i (past the run: of its last): TILED, of its tiles' first
  // tokens; else of token lane % 32 (past the block's: of the last)
  struct Rows {
    int r[2];
  };
  auto rows_of = [&](int i) {
    i = min(i, i1 - 1);
    if constexpr (TILED) return Rows{of(meta_row[0], i), of(meta_row[1], i)};
    else return Rows{page_row(of(meta_g, i), min(32 * of(meta_k, i) + (lane & 31), G - 1)), 0};
  };
  constexpr int SPL = D / 64;  // channels a lane brings of the next group's scale and mean
  uint32_t kw[2][KW], ent[2];
  float nsc[SPL], nmu[SPL];
  uint32_t vw[NS][8];
  float norm[8], kn[8];
  size_t ob = 0;
  int e_lo = 0, e_hi = 0;
  // the norms of a lane's 8 tokens of a block: 4 lg .. + 3 and 16 + 4 lg .. + 3
  auto load_norms = [&](float (&x)[8], const float* from, const Rows& rw) {
    if constexpr (TILED) {
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const f4_t y = *reinterpret_cast<const f4_t*>(from + (head + rw.r[tile]) + (uint32_t)(4 * lg));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * tile + e] = y[e];
      }
    } else {
      x[0] = from[head + rw.r[0]];  // (token lane % 32's: handed out when needed)
    }
  };
  auto norm_of = [&](const float (&x)[8], int e) {
    return TILED ? x[e] : __shfl(x[0], 16 * (e / 4) + 4 * lg + e % 4, 64);
  };
  auto load_keys = [&](int i, const Rows& rw) {
    ob = of(meta_ob, i);
    e_lo = of(meta_lo, i);
    e_hi = of(meta_hi, i);
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      const uint8_t* src;
      if constexpr (TILED) src = a.p.kcodes + (head + rw.r[tile]) * KROW + (uint32_t)(ln * KROW + lg * (CPL * KB / 8));
      else src = a.p.kcodes + (head + __shfl(rw.r[0], 16 * tile + ln, 64)) * KROW + lg * (CPL * KB / 8);
      if constexpr (CPL * KB % 32 == 0) {
#pragma unroll
        for (int e = 0; e < KW; ++e) kw[tile][e] = reinterpret_cast<const uint32_t*>(src)[e];
      } else {  // six bytes (3-bit keys at head_dim 64)
        const uint16_t* s2 = reinterpret_cast<const uint16_t*>(src);
        kw[tile][0] = (uint32_t)s2[0] | (uint32_t)s2[1] << 16;
        kw[tile][1] = s2[2];
      }
    }
    if constexpr (PK) {
      load_norms(kn, a.p.knorm, rw);
    } else {
#pragma unroll
      for (int e = 0; e < SPL; ++e) {
        nsc[e] = a.p.gscale[ob * D + SPL * lane + e];
        nmu[e] = a.p.gmean[ob * D + SPL * lane + e];
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) ent[s] = oent[ob * cap + min(e_lo + lane + 64 * s, cap - 1)];
    }
  };
  // a group's weights and the rest of its scores (q . mean)
  float bias = 0.f;
  auto begin_group = [&]() {
    // q * scale within fp16: a scale of keys near 65504 times a large query is not
    float s_top = 0.f;
#pragma unroll
    for (int e = 0; e < SPL; ++e) s_top = fmaxf(s_top, fabsf(nsc[e]));
    w_up = 1.f;
    if (__builtin_expect(__any(s_top * q_top > 65504.f), 0)) {
      s_top = wave_reduce<true>(s_top);
      // (s_top q_top < 2^e; an infinite scale's group is lost whatever the power)
      const int e = min(__builtin_amdgcn_frexp_expf(s_top) + __builtin_amdgcn_frexp_expf(q_top), 126);
      w_up = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, ldexpf(1.f, e - 15))));
#pragma unroll
      for (int i = 0; i < SPL; ++i) nsc[i] *= ldexpf(1.f, 15 - e);
    }
#pragma unroll
    for (int e = 0; e < SPL; ++e) {
      stat_s[wave][0][SPL * lane + e] = nsc[e];
      stat_s[wave][1][SPL * lane + e] = nmu[e];
    }
    wave_sync();
    float y = 0.f;
#pragma unroll
    for (int mm = 0; mm < NM; ++mm)
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const int ch = CPL * lg + 8 * mm + e;
        const f4_t s4 = *reinterpret_cast<const f4_t*>(&stat_s[wave][0][ch]);
        const f4_t m4 = *reinterpret_cast<const f4_t*>(&stat_s[wave][1][ch]);
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float q1 = (float)qf[mm][e + k];
          y = fmaf(q1, m4[k], y);
          x[k] = q1 * s4[k];
        }
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          // (towards zero: two in one instruction)
          const h2_t hh = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(x[k], x[k + 1]));
          const h2_t ll = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float)hh.x, -1.f, x[k]),
                                                                              fmaf((float)hh.y, -1.f, x[k + 1])));
          wh[mm][e + k] = hh.x;
          wh[mm][e + k + 1] = hh.y;
          wl[mm][e + k] = ll.x;
          wl[mm][e + k + 1] = ll.y;
        }
      }
    bias = colgroup_sum(y);
  };
  auto load_values = [&](const Rows& rw) {
    load_norms(norm, a.p.vnorm, rw);
    if constexpr (TILED) {
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(a.p.vcodes + (head + rw.r[tile]) * VROW +
                                                                (uint32_t)v_unit_offset(lg, ln, VROW));
#pragma unroll
        for (int e = 0; e < VB; ++e) vw[0][4 * tile + e] = src[e];
      }
    } else {
      // eight codes of each of the lane's tokens
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int rr = __shfl(rw.r[0], 16 * (e / 4) + 4 * lg + e % 4, 64);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const uint8_t* src = a.p.vcodes + (head + rr) * VROW + ((D == 64 ? ln / 2 : ln) + 16 * s) * VB;
          if constexpr (VB == 4)
            vw[s][e] = *reinterpret_cast<const uint32_t*>(src);
          else if constexpr (VB == 3)
            vw[s][e] = (uint32_t)src[0] | (uint32_t)src[1] << 8 | (uint32_t)src[2] << 16;
          else
            vw[s][e] = *reinterpret_cast<const uint16_t*>(src);
        }
      }
    }
  };
  Rows next_rows{0, 0};
  const bool has_codes = is_cold && i0 < i1;
  if (has_codes) {
    load_meta(i0);
    const Rows first = rows_of(i0);
    next_rows = rows_of(i0 + 1);
    load_keys(i0, first);
    load_values(first);
  }

  lds_barrier();

  // the scale of the value codebook: candidate 1 + i / 128 whose centroids lose
  // least to fp16, the first of equals; half of them by even waves, half by odd ones
  {
    const float g = 1.0f + (float)(2 * lane + wave % 2) * (1.0f / 128);
    float err = 0.f;
#pragma unroll
    for (int i = 0; i < (1 << VB); ++i) {
      const float y = cen_s[i] * g, r = y - (float)(_Float16)y;
      err = fmaf(r, r, err);
    }
    err *= __builtin_amdgcn_rcpf(g * g);
    const float best = -wave_reduce<true>(-err);
    const uint64_t first = __builtin_amdgcn_ballot_w64(err == best);
    if (wave < 2 && lane == 0) {
      up_s[wave][0] = best;
      up_s[wave][1] = 1.0f + (float)(first ? 2 * __builtin_ctzll(first) + wave : 0) * (1.0f / 128);
    }
  }
  for (int i = tid; i < kKeyEntries * kKeyCopies / 2; i += kFewThreads) {
    const int e = i / (kKeyCopies / 2);
    const uint2 y = split_pair(lev_s[k_code_even(e, KB)], lev_s[k_code_odd(e, KB)]);
    *reinterpret_cast<u32x4_t*>(key_s + (e << kKeyLog) + 16 * (i % (kKeyCopies / 2))) = u32x4_t{y.x, y.y, y.x, y.y};
  }
  lds_barrier();
  const float up = up_s[up_s[1][0] < up_s[0][0]][1];
  for (int i = tid; i < kValEntries * kValCopies / 4; i += kFewThreads) {
    const int e = i / (kValCopies / 4);
    const uint32_t y = pk_f16(cen_s[e & ((1 << VB) - 1)] * up, cen_s[e >> VB] * up);
    *reinterpret_cast<u32x4_t*>(val_s + (e << kValLog) + kValOff + 16 * (i % (kValCopies / 4))) = u32x4_t{y, y, y, y};
  }
  // a table read: the field of `bits` bits at bit `bit` of the word array w, as an
  // entry of 2^lg bytes and this lane's copy in it
  const uint32_t k_copy = 8 * (lane % kKeyCopies), v_copy = kValOff + 4 * (lane % kValCopies);
  auto place_in = [](const uint32_t* w, int bit, int bits, int lg, uint32_t copy) -> uint32_t {
    const int wd = bit / 32, sh = bit % 32;
    if (bits == 8 && lg == 8)  // byte sh / 8 above the copy's byte
      return __builtin_amdgcn_perm(w[wd], copy, 0x0C0C0000u | (4u + sh / 8) << 8);
    const uint32_t mask = ((1u << bits) - 1u) << lg;
    const uint32_t x = sh + bits > 32 ? __builtin_amdgcn_alignbit(w[wd + 1], w[wd], sh) << lg
                       : sh >= lg     ? w[wd] >> (sh - lg)
                                      : w[wd] << (lg - sh);
    return (x & mask) | copy;
  };
  auto levels = [&](const uint32_t* w, int bit) {
    return *reinterpret_cast<const uint2*>(key_s + place_in(w, bit, 2 * KB, kKeyLog, k_copy));
  };
  auto centroids = [&](const uint32_t* w, int bit) {
    return *reinterpret_cast<const uint32_t*>(val_s + place_in(w, bit, 2 * VB, kValLog, v_copy));
  };
  // (the side-list tile starts at zero)
#pragma unroll
  for (int i = 0; i < 4 * D / 64; ++i) reinterpret_cast<u32x4_t*>(stage_s[wave])[64 * i + lane] = u32x4_t{0u, 0u, 0u, 0u};

  if constexpr (PK) {
    __syncthreads();
    float* const q_s = reinterpret_cast<float*>(&stage_s[0][0]);  // [16][D]
    float* const r_s = reinterpret_cast<float*>(&stage_s[1][0]);  // [16][D]
    if (wave == 0) {
#pragma unroll
      for (int mm = 0; mm < NM; ++mm)
#pragma unroll
        for (int e = 0; e < 8; ++e) q_s[ln * D + CPL * lg + 8 * mm + e] = (float)qf[mm][e];
    }
    __syncthreads();
    for (int i = tid; i < kFewRows * D; i += kFewThreads) {
      const int r = i / D, j = i % D;
      float y = 0.f;
#pragma unroll 8
      for (int k = 0; k < D; ++k) y = fmaf(q_s[r * D + k], a.p.pi_t[k * D + j], y);
      r_s[i] = y;
    }
    __syncthreads();
    // (the rotation may gather a row's channels in one, sqrt(D) times as large: over a
    // power of two then, of every row here, so that every wave has the same)
    float y_top = 0.f;
#pragma unroll
    for (int mm = 0; mm < NM; ++mm)
#pragma unroll
      for (int e = 0; e < 8; ++e) y_top = fmaxf(y_top, fabsf(r_s[ln * D + CPL * lg + 8 * mm + e]));
    y_top = fminf(wave_reduce<true>(y_top), 16.f * 65504.f);  // (more: not of finite queries)
    float down = 1.f;
    if (y_top > 65504.f) {
      const int e = __builtin_amdgcn_frexp_expf(y_top);  // y_top < 2^e
      down = ldexpf(1.f, 15 - e);
      w_up = ldexpf(1.f, e - 15);
    }
#pragma unroll
    for (int mm = 0; mm < NM; ++mm)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = r_s[ln * D + CPL * lg + 8 * mm + e] * down;
        wh[mm][e] = (_Float16)y;
        wl[mm][e] = (_Float16)(y - (float)wh[mm][e]);
      }
  }
  lds_barrier();

  const float c = d.sm_scale * 1.4426950408889634f;
  float m_run = -INFINITY, l_run = 0.f;
  f4_t O[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) O[i] = f4_t{0.f, 0.f, 0.f, 0.f};

  // the 8 scores of row ln: tokens 4 lg + i, then 16 + 4 lg + i, of a block at
  // tok0; tokens from cnt on are none.  Returns the weights.
  auto weights = [&](f4_t (&S)[2], int tok0, int cnt, bool whole, float (&w)[8]) {
    S[0] *= c;
    S[1] *= c;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int o = 16 * (i / 4) + 4 * lg + i % 4;
        S[i / 4][i % 4] = (o < cnt) & sees(tok0 + o) ? S[i / 4][i % 4] : -INFINITY;
      }
      asm volatile("");  // (one branch for the eight)
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, S[i / 4][i % 4]);
    if (__any(mx > m_run + kFewLazy)) {
      mx = colgroup_max(mx);
      const float m_new = fmaxf(m_run, mx);
      const float f = m_new == -INFINITY ? 1.f : above_zero(__builtin_amdgcn_exp2f(m_run - m_new));
      m_run = m_new;
      l_run *= f;
#pragma unroll
      for (int i = 0; i < NV; ++i) O[i] *= f;
    }
    const float at = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = __builtin_amdgcn_exp2f(S[i / 4][i % 4] - at);
      l_run += w[i];
    }
  };

  if (has_codes) {
    for (int i = i0; i < i1; ++i) {
      const int k = of(meta_k, i), tok0 = of(meta_g, i) * G + 32 * k, cnt = min(32, G - 32 * k);
      if (i + 2 >= meta_i + 64 && i + 1 < i1) load_meta(i);
      const Rows after = rows_of(i + 2);
      if (!PK && (i == i0 || k == 0 || i == cold.n0)) begin_group();  // (the second run may start inside a group)
      // the block's side-list entries, 128 at a time: an entry's place in the sparse
      // tile (none: behind it) and its value over the mean, as a pair: its first
      // half there, then its second
      struct Spot {
        int o;
        uint16_t half[2];
      };
      auto spot_of = [&](uint32_t y, bool real) {
        const int tok = (int)((y & 0xFFFFu) / D) - 32 * k, ch = (int)(y & (D - 1));
        const float v = h2f((uint16_t)(y >> 16)) - stat_s[wave][1][ch];
        const h2_t hh = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(v, 0.f));
        return Spot{real & ((unsigned)tok < 32u) ? at(tok, ch / 8) + ch % 8 : 32 * D,
                    {__builtin_bit_cast(uint16_t, hh.x), f2h(v - (float)hh.x)}};
      };
      Spot spot[2];
      auto put = [&](int half) {  // (2: cleared)
#pragma unroll
        for (int s = 0; s < 2; ++s) list_s[spot[s].o] = half == 2 ? 0 : spot[s].half[half];
        wave_sync();
      };
      const bool lists = !PK && e_hi > e_lo;
      if (lists) {
#pragma unroll
        for (int s = 0; s < 2; ++s) spot[s] = spot_of(ent[s], e_lo + lane + 64 * s < e_hi);
        put(0);
      }
      f4_t S[2];
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        S[tile] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int mm = 0; mm < NM; ++mm) {
          union { h8_t h; uint32_t u[4]; } hi, lo16;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint2 y = levels(kw[tile], KB * (8 * mm + 2 * e));
            hi.u[e] = y.x;
            lo16.u[e] = y.y;
          }
          S[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo16.h, wh[mm], S[tile], 0, 0, 0);
          S[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi.h, wl[mm], S[tile], 0, 0, 0);
          S[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi.h, wh[mm], S[tile], 0, 0, 0);
        }
        if constexpr (!PK) {
#pragma unroll
          for (int e = 0; e < 4; ++e) S[tile][e] = fmaf(S[tile][e], w_up, bias);
        }
      }
      if (lists) {
        for (int e = e_lo;;) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (half) put(1);
#pragma unroll
            for (int mm = 0; mm < NM; ++mm)
#pragma unroll
              for (int tile = 0; tile < 2; ++tile)
                S[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    *reinterpret_cast<const h8_t*>(list_s + at(16 * tile + ln, (CPL / 8) * lg + mm)), qf[mm], S[tile], 0, 0, 0);
            wave_sync();
          }
          put(2);
          if ((e += 128) >= e_hi) break;
#pragma unroll
          for (int s = 0; s < 2; ++s) spot[s] = spot_of(oent[ob * cap + min(e + lane + 64 * s, cap - 1)], e + lane + 64 * s < e_hi);
          put(0);
        }
      }
      if constexpr (PK) {  // score = |k| (q_rot . centroids)
#pragma unroll
        for (int e = 0; e < 8; ++e) S[e / 4][e % 4] *= norm_of(kn, e) * w_up;
      }
      load_keys(min(i + 1, i1 - 1), next_rows);
      float w[8];
      const bool whole = cnt == 32 && all_see(tok0, 32);
      weights(S, tok0, cnt, whole, w);
      h8_t pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float nv = norm_of(norm, e);
        pf[e] = (_Float16)(w[e] == 0.f ? 0.f : w[e] * nv);  // (no weight: whatever norm stands there)
      }
      // V^T P^T: row ln of the first operand is channel NC ln + j of the piece
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        if constexpr (TILED) {
          // a channel's token pairs side by side in the unit's bits
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            union { h8_t h; uint32_t u[4]; } y;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              y.u[f] = centroids(vw[0] + 4 * (f / 2), (2 * j + f % 2) * 2 * VB);
            }
            O[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y.h, pf, O[j], 0, 0, 0);
          }
        } else {
          // by channel pairs, the tokens of a channel then brought together
#pragma unroll
          for (int j = 0; j < NC; j += 2) {
            uint32_t two[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t y = D == 64 ? vw[s][e] >> ((ln & 1) * 4 * VB) : vw[s][e];
              two[e] = centroids(&y, VB * j);
            }
            union { h8_t h; uint32_t u[4]; } y0, y1;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              y0.u[f] = __builtin_amdgcn_perm(two[2 * f + 1], two[2 * f], 0x05040100u);
              y1.u[f] = __builtin_amdgcn_perm(two[2 * f + 1], two[2 * f], 0x07060302u);
            }
            O[NC * s + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y0.h, pf, O[NC * s + j], 0, 0, 0);
            O[NC * s + j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y1.h, pf, O[NC * s + j + 1], 0, 0, 0);
          }
        }
      }
      load_values(next_rows);
      next_rows = after;
    }
  } else if (!is_cold) {
    // uncoded blocks, straight from the ring
    const size_t ring = ((size_t)b * Hkv + h) * d.hot_ring;
    const uint16_t* const hk = static_cast<const uint16_t*>(a.p.hot_k);
    const uint16_t* const hv = static_cast<const uint16_t*>(a.p.hot_v);
    // a block's place in the ring: token tok0 + o, o < cnt (cnt is at most the
    // ring's size)
    auto place = [&](int at0, int o) { return ring + (at0 + o >= d.hot_ring ? at0 + o - d.hot_ring : at0 + o); };
    // up to head_dim 128 the next block's rows are on their way meanwhile
    constexpr bool kAhead = D <= 128;
    h8_t kf[2][NM];
    u32x4_t vn[NS][8];
    auto load = [&](int i) {
      const int tok0 = n_cold + 32 * hot.at(i), cnt = min(32, n - tok0), at0 = tok0 % d.hot_ring;
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const uint16_t* kr = hk + place(at0, min(16 * tile + ln, cnt - 1)) * D + CPL * lg;
#pragma unroll
        for (int mm = 0; mm < NM; ++mm) kf[tile][mm] = *reinterpret_cast<const h8_t*>(kr + 8 * mm);
      }
      // values: token e of this lane, channels NC ln .. + NC - 1 of the piece
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t* vr = hv + place(at0, min(16 * (e / 4) + 4 * lg + e % 4, cnt - 1)) * D + NC * ln;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          if constexpr (NC == 8) {
            vn[s][e] = *reinterpret_cast<const u32x4_t*>(vr + 128 * s);
          } else {
            const u32x2_t y = *reinterpret_cast<const u32x2_t*>(vr);
            vn[s][e] = u32x4_t{y.x, y.y, 0u, 0u};
          }
        }
      }
    };
    if (kAhead && i0 < i1) load(i0);
    for (int i = i0; i < i1; ++i) {
      if constexpr (!kAhead) load(i);
      const int tok0 = n_cold + 32 * hot.at(i), cnt = min(32, n - tok0), at0 = tok0 % d.hot_ring;
      f4_t S[2];
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        S[tile] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int mm = 0; mm < NM; ++mm)
          S[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tile][mm], qf[mm], S[tile], 0, 0, 0);
      }
      // values of tokens that no row sees: zero, whatever stands there
      u32x4_t vv[NS][8];
      typedef uint16_t us2_t __attribute__((ext_vector_type(2)));
      us2_t top = {0, 0};  // the largest exponent fields
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int o = 16 * (e / 4) + 4 * lg + e % 4, tok = tok0 + o;
        const bool any = o < cnt && tok <= p_hi && (tok >= lo_first || tok < sinks);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          vv[s][e] = any ? vn[s][e] : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
          for (int f = 0; f < NC / 2; ++f)
            top = __builtin_elementwise_max(top, __builtin_bit_cast(us2_t, vv[s][e][f] & 0x7C007C00u));
        }
      }
      if (kAhead && i + 1 < i1) load(i + 1);
      float w[8];
      weights(S, tok0, cnt, cnt == 32 && all_see(tok0, 32), w);
      h8_t pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) pf[e] = (_Float16)w[e];
      // (infinities and NaN set aside: a row may not see them, and a weight that
      // fp16 rounds to zero would make a NaN of an infinity)
      const bool apart = __any(top.x == 0x7C00 || top.y == 0x7C00);
      if (__builtin_expect(apart, 0)) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int f = 0; f < NC / 2; ++f) {
              uint32_t y = vv[s][e][f];
              y &= (y & 0x7C00u) == 0x7C00u ? 0xFFFF0000u : ~0u;
              y &= (y & 0x7C000000u) == 0x7C000000u ? 0xFFFFu : ~0u;
              vv[s][e][f] = y;
            }
      }
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          union { h8_t h; uint32_t u[4]; } y;
#pragma unroll
          for (int f = 0; f < 4; ++f)
            y.u[f] = __builtin_amdgcn_perm(vv[s][2 * f + 1][j / 2], vv[s][2 * f][j / 2],
                                           (j & 1) ? 0x07060302u : 0x05040100u);
          O[NC * s + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y.h, pf, O[NC * s + j], 0, 0, 0);
        }
      if (__builtin_expect(apart, 0)) {
        // ... and added to the rows that see it (any positive weight gives the same)
#pragma unroll 1
        for (int o = 0; o < cnt; ++o) {
          const bool vis = sees(tok0 + o);
          const uint16_t* vr = hv + place(at0, o) * D;
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int j = 0; j < NC; ++j) {
                const float y = h2f(vr[128 * s + NC * (4 * lg + e) + j]);
                O[NC * s + j][e] += vis && !(fabsf(y) < INFINITY) ? y : 0.f;
              }
        }
      }
    }
  }

  // ---- the waves' states joined: coded ones, rotated back, and uncoded ones
  const int first_hot = min(max(cold_waves - split * kFewWaves, 0), kFewWaves);  // waves before it are coded
  // Pi^T's rows e = 16 (wave + 8 nt) + ln, channels 32 mm + 8 lg .. + 7: the
  // first of them asked for early
  constexpr int NTR = (D / 16 + kFewWaves - 1) / kFewWaves;
  f4_t pr[NM][2];
  auto load_pi = [&](int nt) {
#pragma unroll
    for (int mm = 0; mm < NM; ++mm)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        pr[mm][e] = *reinterpret_cast<const f4_t*>(
            a.p.pi_t + (size_t)(16 * ((wave + kFewWaves * nt) % (D / 16)) + ln) * D + 32 * mm + 8 * lg + 4 * e);
  };
  if (first_hot > 0) load_pi(0);
  {
    const float l = colgroup_sum(l_run);
    if (lg == 0) {
      ml_s[0][wave][ln] = m_run;
      ml_s[1][wave][ln] = l;
    }
    float* const o = reinterpret_cast<float*>(stage_s[wave]);  // [16][D]
    wave_sync();
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[ln * D + 128 * s + NC * (4 * lg + e) + j] = O[NC * s + j][e];
  }
  __syncthreads();
  constexpr int kRowGroups = kFewThreads / D;            // rows side by side
  constexpr int RPT = (kFewRows + kRowGroups - 1) / kRowGroups;  // rows a thread
  const int j = tid % D, r0 = tid / D;
  float cs[RPT], hs[RPT], ls[RPT], ms[RPT];
#pragma unroll
  for (int k = 0; k < RPT; ++k) {
    const int r = r0 + kRowGroups * k;
    cs[k] = hs[k] = ls[k] = 0.f;
    ms[k] = -INFINITY;
    if (r >= n_rows) continue;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) ms[k] = fmaxf(ms[k], ml_s[0][w][r]);
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      const float mw = ml_s[0][w][r], f = mw == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(mw - ms[k]));
      const float y = reinterpret_cast<const float*>(stage_s[w])[r * D + j];
      ls[k] = fmaf(ml_s[1][w][r], f, ls[k]);
      // (a state without a maximum holds zeros; a NaN among its scores leaves it one)
      if (w < first_hot) cs[k] += y * f; else hs[k] += y * f;
    }
  }
  if (first_hot > 0) {
    __syncthreads();
    // the coded sums over their weights' sum (within fp16's range then) as an
    // fp16 pair, times Pi's
    uint16_t* const c_s = &stage_s[0][0];                         // [2][16][D]
    float* const y_s = reinterpret_cast<float*>(&stage_s[1][0]);  // [16][D]
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const int r = r0 + kRowGroups * k;
      if (r < kFewRows) {
        const float y = ls[k] != 0.f ? cs[k] / (ls[k] * up) : 0.f;
        const _Float16 hi = (_Float16)y;
        c_s[r * D + j] = __builtin_bit_cast(uint16_t, hi);
        c_s[(kFewRows + r) * D + j] = f2h(y - (float)hi);
      }
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NTR; ++nt) {
      if (wave + kFewWaves * nt < D / 16) {
        f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int mm = 0; mm < NM; ++mm) {
          h8_t ph, pl;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = pr[mm][e / 4][e % 4];
            ph[e] = (_Float16)y;
            pl[e] = (_Float16)(y - (float)ph[e]);
          }
          const h8_t ch = *reinterpret_cast<const h8_t*>(c_s + ln * D + 32 * mm + 8 * lg);
          const h8_t cl = *reinterpret_cast<const h8_t*>(c_s + (kFewRows + ln) * D + 32 * mm + 8 * lg);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(cl, ph, acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch, pl, acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch, ph, acc, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y_s[(4 * lg + e) * D + 16 * (wave + kFewWaves * nt) + ln] = acc[e];
        if (nt + 1 < NTR) load_pi(nt + 1);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RPT; ++k)
      if (r0 + kRowGroups * k < kFewRows) hs[k] = fmaf(y_s[(r0 + kRowGroups * k) * D + j], ls[k], hs[k]);
  }
  // (rows past the queries of the sequence: zero)
  const int all_rows = min(a.per_item, a.q_len - q0) * gq;
#pragma unroll
  for (int k = 0; k < RPT; ++k) {
    const int r = r0 + kRowGroups * k;
    if (r >= all_rows) continue;
    const int tr = q0 + r / gq, hq = h * gq + r % gq;
    if (a.n_splits == 1) {
      const long long o = b * a.o_stride[0] + hq * a.o_stride[1] + tr * a.o_stride[2] + j;
      const float y = r < n_rows && n - m + tr >= 0 ? hs[k] / ls[k] : 0.f;
      if (a.out_type == 0) static_cast<float*>(a.out)[o] = y;
      else static_cast<_Float16*>(a.out)[o] = (_Float16)y;
    } else {
      const long long o = split * a.rows + ((long long)b * Hq + hq) * a.q_len + tr;
      a.part_acc[o * D + j] = hs[k];
      if (j == 0) {
        a.part_ml[2 * o] = ms[k];
        a.part_ml[2 * o + 1] = ls[k];
      }
    }
  }
}

// The splits of a row joined: one wave a row, D / 64 channels a lane.
template <int D>
__global__ __launch_bounds__(256) void tqk_attend_join(FewArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int t = (int)(row % a.q_len);
  const long long bh = row / a.q_len;
  const int hq = (int)(bh % a.d.n_q_heads), b = (int)(bh / a.d.n_q_heads);
  // every split's numbers by a lane of its own, then all accumulators in flight
  const bool in = lane < a.n_splits;
  const float ml = in ? a.part_ml[2 * (lane * a.rows + row)] : -INFINITY;
  const float ll = in ? a.part_ml[2 * (lane * a.rows + row) + 1] : 0.f;
  const float M = wave_reduce<true>(ml);
  const float f = ml == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(ml - M));
  const float l = wave_reduce<false>(ll * f);
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.n_splits; ++s) {
    const float g = __shfl(f, s, 64);
    const float* src = a.part_acc + (s * a.rows + row) * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(src[e], g, acc[e]);
  }
  const int n = min(a.seq_lens[b], a.max_len);
  const int m = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
  const bool any = t < m && n - m + t >= 0;
  const long long o = b * a.o_stride[0] + hq * a.o_stride[1] + t * a.o_stride[2] + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y = any ? acc[e] / l : 0.f;
    if (a.out_type == 0) static_cast<float*>(a.out)[o + e] = y;
    else static_cast<_Float16*>(a.out)[o + e] = (_Float16)y;
  }
}

struct FewPlan {
  int per_item, q_items, n_splits;
  long long rows, groups;  // rows of all, workgroups
  size_t ws_bytes;
};

constexpr long long kMostFewGroups = 1LL << 22;  // workgroups of a launch (512 threads each: fewer than 2^32)
FewPlan few_plan(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  FewPlan fp{};
  const int gq = d->n_q_heads / d->n_kv_heads;
  fp.per_item = kFewRows / gq < t->q_len ? kFewRows / gq : t->q_len;
  fp.q_items = (t->q_len + fp.per_item - 1) / fp.per_item;
  fp.rows = (long long)t->batch * d->n_q_heads * t->q_len;
  const long long pairs = (long long)t->batch * fp.q_items * d->n_kv_heads;
  // blocks of 32 tokens that a workgroup's rows see at most
  long long tokens = t->max_len;
  if (t->window > 0 && t->window < t->max_len) {
    const long long w = (long long)t->window + fp.per_item + t->sinks + 64;
    if (w < tokens) tokens = w;
  }
  fp.n_splits = few_splits(pairs, (tokens + 31) / 32 + 1, 2.0);
  fp.groups = pairs * fp.n_splits;
  fp.ws_bytes = fp.n_splits > 1 ? (size_t)fp.n_splits * fp.rows * (d->head_dim + 2) * sizeof(float) + 256 : 16;
  return fp;
}

template <int D, int VB, bool TILED>
void launch_keys(const FewArgs& a, dim3 grid, hipStream_t st) {
  if (a.d.key_grid == 2)
    hipLaunchKernelGGL((tqk_attend_codes<D, VB, VB, true, TILED>), grid, dim3(kFewThreads), 0, st, a);
  else if (a.d.key_bits == 4)
    hipLaunchKernelGGL((tqk_attend_codes<D, VB, 4, false, TILED>), grid, dim3(kFewThreads), 0, st, a);
  else if (a.d.key_bits == 3)
    hipLaunchKernelGGL((tqk_attend_codes<D, VB, 3, false, TILED>), grid, dim3(kFewThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tqk_attend_codes<D, VB, 2, false, TILED>), grid, dim3(kFewThreads), 0, st, a);
}
template <int D, bool TILED>
void launch_values(const FewArgs& a, dim3 grid, hipStream_t st) {
  if (a.d.value_bits == 2)
    launch_keys<D, 2, TILED>(a, grid, st);
  else if (a.d.value_bits == 3)
    launch_keys<D, 3, TILED>(a, grid, st);
  else
    launch_keys<D, 4, TILED>(a, grid, st);
}
template <int D>
void launch_few(const FewArgs& a, dim3 grid, hipStream_t st) {
  if constexpr (D == TQK_D) {
    if (v_tiled(a.d.group_tokens, a.d.page_tokens, D, 0))
      launch_values<D, true>(a, grid, st);
    else
      launch_values<D, false>(a, grid, st);
  } else {
    launch_values<D, false>(a, grid, st);
  }
  if (a.n_splits > 1)
    hipLaunchKernelGGL(tqk_attend_join<D>, dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a);
}

}  // namespace

size_t tqk_few_workspace_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t) { return few_plan(d, t).ws_bytes; }
bool tqk_few_fits(const tqk_cache_desc* d, const tqk_attend_desc* t) { return few_plan(d, t).groups <= kMostFewGroups; }

int tqk_run_few(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
                const int32_t* seq_lens, const int32_t* q_lens, void* out, void* workspace, size_t workspace_bytes,
                void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const FewPlan fp = few_plan(d, t);
  if (workspace_bytes < fp.ws_bytes) return TQK_EWORKSPACE;
  if (fp.groups > kMostFewGroups) return TQK_EINVAL;
  FewArgs a{};
  a.d = *d;
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.out = out;
  a.part_acc = static_cast<float*>(workspace);
  a.part_ml = a.part_acc + (size_t)fp.n_splits * fp.rows * d->head_dim;
  a.rows = fp.rows;
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = t->q_stride[i];
    a.o_stride[i] = t->o_stride[i];
  }
  a.q_len = t->q_len;
  a.max_len = t->max_len;
  a.window = t->window;
  a.sinks = t->sinks;
  a.out_type = t->out_type;
  a.per_item = fp.per_item;
  a.q_items = fp.q_items;
  a.n_splits = fp.n_splits;
  const dim3 grid((unsigned)fp.groups);
  if (d->head_dim == 64)
    launch_few<64>(a, grid, st);
  else if (d->head_dim == 128)
    launch_few<128>(a, grid, st);
  else
    launch_few<256>(a, grid, st);
  return hipGetLastError() == hipSuccess ? TQK_OK : TQK_EHIP;
}
