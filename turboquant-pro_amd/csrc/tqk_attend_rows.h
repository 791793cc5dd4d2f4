// Attention of up to eight rows over the codes of an fp16 cache (gfx950): the decode
// steps of tqk_attend_more.hip, over a window, listed groups, or what follows a prefix.
//
// A workgroup takes one kv head of one sequence and at most 8 rows (the kv head's query
// heads, of several queries where they fit); its eight waves take runs of blocks of 32
// tokens, coded or uncoded, each on its own until the end.
//
// The matrix instructions have 16 columns for 8 rows: columns c and c + 8 take one
// row's two fp16 halves, of the weights q * scale in K Q^T and of the probabilities
// times norms in V^T P^T, and the two results are added.  So both products keep 2^-22
// without a second pass (a single fp16 probability is 2.4e-4 of the result).  A key
// byte's table row {hi, hi, lo, lo} of its two levels is half of an operand as it is:
// k-slots hi, lo of a channel meet the same weight.
//
// The side-list: for each stretch of tokens (`kSeg`) the wave adds up q (val - mean) of
// the stretch's entries by token, a lane a run of the sorted list and a segmented scan
// over the lanes; a block's scores start from these sums (and q . mean).  Entries as a
// sparse tile of a second product cost a block 16 products, 22 LDS reads and six stores.
//
// The next block's scores are computed beside this block's exponentials and values.
//
// What bounds it: a block's chain (look-ups of levels -> products -> exponentials ->
// look-ups of centroids -> products) at two waves a SIMD, 256 registers each; three or
// four waves spill 190 to 320 registers (313 us for 190).  Measured, 32 / 8 heads of 128:
// 16 sequences of 32768 tokens, every group's weight kept, 175 us (3.2 TB/s; with the
// pages in cache some 20 less, without the blocks' sums 10 less): the waves wait 48 % of
// their cycles, vector issue half of the time, LDS 32 %, the matrix cores 14 %
// (tqk_decode_split_mfma over the same cache, one query: 135 us, a fifth fewer vector
// instructions, 33 % waiting); 16 groups of 127
// listed, ten blocks a wave, 34 us; 64 of 511 of one sequence, three blocks a wave, 20
// us; one block a wave 14.5.  Of a short run some 9 us are set-up (lengths -> list ->
// tables -> codes, one load after another; the tables and the group's weights meanwhile)
// and 3 the waves' joining and rotation.  head_dim 256: 60 to 90 registers spill, 42 us
// for 8 groups of 30, 8 sequences.
#pragma once

#include "tqk_attend_few.h"

namespace {

constexpr int kRows8 = 8;
constexpr int kPreEntries = 12;  // entries of a lane that are loaded ahead

template <int N>
__device__ __forceinline__ float row_ror(float x) {
  return bitsf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fbits(x), 0x120 + N, 0xF, 0xF, true));
}
// the value of the lane before / after (the first / last one's: 0)
__device__ __forceinline__ int lane_before(int x) { return __builtin_amdgcn_update_dpp(0, x, 0x138, 0xF, 0xF, true); }
__device__ __forceinline__ int lane_after(int x) { return __builtin_amdgcn_update_dpp(0, x, 0x130, 0xF, 0xF, true); }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t entries_of(const uint32_t* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(base), (short)0, (int)bytes, 0x00020000);
}

// KB: key code bits; PK: PolarQuant keys (KB == VB); TILED: value codes in units of 4
// tokens x 8 channels; NR: rows that the side-list's sums are kept for (4 or 8).
template <int D, int VB, int KB, bool PK, bool TILED, int NR>
__global__ __launch_bounds__(kFewThreads, 2) void tqk_attend_rows(MoreArgs a) {
  constexpr int CPL = D / 4;          // channels of a lane in a score product: CPL lg ..
  constexpr int NM = D / 32;
  constexpr int NSL = D / 16;         // steps of a score product: 4 channels of a lane, both halves
  constexpr int KW = (CPL * KB + 31) / 32;  // words of a lane's key codes
  constexpr int NC = D >= 128 ? 8 : 4;      // channels of a lane's value piece
  constexpr int NS = D == 256 ? 2 : 1;      // value pieces a lane takes (128 channels apart)
  constexpr int NV = NC * NS;               // 16-row accumulator tiles
  constexpr int VROW = D * VB / 8, KROW = D * KB / 8;
  constexpr int kSegMost = 32768 / D < TQK_MAX_G ? 32768 / D : TQK_MAX_G;
  constexpr int kSeg = 1024 / NR < kSegMost ? 1024 / NR : kSegMost;  // tokens of a stretch
  constexpr int SB = kSeg / 32, kCorr = kSeg + 4;
  const tqk_cache_desc& d = a.d;
  touch_args<MoreArgs>();
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int ln = lane & 15, lg = lane >> 4;
  const bool is_lo = (ln & 8) != 0;
  const float lo_sel = is_lo ? 1.f : 0.f;
  const int G = d.group_tokens, P = d.page_tokens, Hkv = d.n_kv_heads, Hq = d.n_q_heads, gq = a.by.heads_of.n;
  int x = blockIdx.x, y = a.by.splits(x);
  const int split = x - y * a.n_splits;
  x = y;
  y = a.by.heads(x);
  const int h = x - y * Hkv, b = a.by.items(y), q0 = a.t0 + (y - b * a.q_items) * a.per_item;

  // a pair of key codes -> its levels, {hi, hi} and {lo, lo}; a pair of value codes
  // -> its centroids; with 4-bit keys and values one row for both.  Copies by lane:
  // a lookup's bank is its lane's own.  The waves' accumulators take the keys' place.
  constexpr bool kShared = KB == 4 && VB == 4;
  constexpr int kKeyLog = 8, kValLog = D == 256 && VB == 4 && !kShared ? 7 : 8;  // log2 of an entry's bytes
  constexpr int kKeyCopies = kShared ? 16 : 32, kValCopies = kShared ? 32 : (1 << kValLog) / 4;
  constexpr int kKeyEntries = 1 << (2 * KB), kValEntries = 1 << (2 * VB);
  constexpr int OST = D + 4;  // floats of a row of the waves' accumulators
  constexpr int kOutBytes = kFewWaves * kRows8 * OST * 4, kKeyBytes = kKeyEntries << kKeyLog;
  // Both tables in one array, values from a multiple of their size on: a value's entry
  // and copy are joined by one and-or.
  constexpr int kValBytes = kShared ? 0 : kValEntries << kValLog;
  constexpr int kKeyRoom = kOutBytes > kKeyBytes ? kOutBytes : kKeyBytes;
  // (one struct: the tables first, no gap before them)
  struct Lds {
    uint8_t table[kValBytes + kKeyRoom];
    float stat[kFewWaves][2][D];       // the group's scale and mean
    float corr[kFewWaves][NR][kCorr];  // scores' first values of a stretch
    float zero[4];
    uint16_t qc[D][NR];                // queries by channel
    uint16_t qr[kRows8][D];            // and by row
    float ml[2][kFewWaves][kRows8];
  };
  __shared__ __align__(65536) Lds lds;
  uint8_t* const val_s = lds.table + (kShared ? 128 : 0);
  uint8_t* const key_s = lds.table + kValBytes;
  auto& stat_s = lds.stat;
  auto& corr_s = lds.corr;
  auto& zero_s = lds.zero;
  auto& qc_s = lds.qc;
  auto& qr_s = lds.qr;
  auto& ml_s = lds.ml;

  // What waits for nothing is asked for first: the queries, a table entry's levels and
  // centroids (a thread fills a part of one entry of each table).
  struct Part {
    int entry, first, pieces;  // entry -1: none
  };
  auto part_of = [&](int entries, int pieces) {  // of `pieces` 16-byte pieces an entry
    const int mine = max(entries * pieces / kFewThreads, 1), each = pieces / mine;
    return Part{tid < entries * each ? tid / each : -1, tid % each * mine, mine};
  };
  const Part kp = part_of(kKeyEntries, kKeyCopies / 2), vp = part_of(kValEntries, kValCopies / 4);
  const int ke = max(kp.entry, 0), ve = max(vp.entry, 0);
  auto level = [&](int i) { return PK ? a.p.vcent[i] : key_level(d.key_grid, i); };
  const float lev0 = level(k_code_even(ke, KB)), lev1 = level(k_code_odd(ke, KB));
  const float cen0 = a.p.vcent[ve & ((1 << VB) - 1)], cen1 = a.p.vcent[ve >> VB];
  float cen[1 << VB];
#pragma unroll
  for (int i = 0; i < (1 << VB); ++i) cen[i] = a.p.vcent[i];
  const int m = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
  // the rows: query q0 + row / gq, head h gq + row % gq
  const int n_rows = min(a.per_item, min(m, a.t0 + a.t_len) - q0) * gq;  // (negative: none)
  const int row = min(ln & 7, max(n_rows, 1) - 1), row_t = a.by.heads_of(row), row_h = row - row_t * gq, t = q0 + row_t;
  // Q: this column's row, channels CPL lg + 8 m .. + 7 (rows past the last: a real one's, dropped later)
  h8_t q8[NM];
  {
    const uint16_t* const qp = a.q + b * a.q_stride[0] + (h * gq + row_h) * a.q_stride[1] + min(max(t, 0), a.q_len - 1) * a.q_stride[2];
#pragma unroll
    for (int mm = 0; mm < NM; ++mm) q8[mm] = *reinterpret_cast<const h8_t*>(qp + CPL * lg + 8 * mm);
  }
  const int32_t* const list = a.groups ? a.groups + b * a.g_stride[0] + h * a.g_stride[1] + q0 * a.g_stride[2] : nullptr;
  const int listed0 = list && lane < a.n_list ? list[lane] : -1;
  const int n = min(a.seq_lens[b], a.max_len), p = n - m + t;
  if (tid < 4) zero_s[tid] = 0.f;
  const int p_lo = n - m + q0, p_hi = n - m + min(q0 + a.per_item, m) - 1;
  const int ng = n > d.hot_window ? a.by.group(n - d.hot_window - 1) + 1 : 0, n_cold = ng * G;
  auto low = [&](int pos) { return max(a.window > 0 && a.window <= pos ? pos - a.window + 1 : 0, a.skip); };
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
  const int nblk = a.by.blocks.n;  // blocks of a group
  BlockRuns cold{0, 0, 0};
  if (list) {  // block i: block i % nblk of group list[i / nblk], up to the last that there is
    int last = 0;
    for (int i = 0; i < a.n_list; i += 64) {
      const int g = i == 0 ? listed0 : i + lane < a.n_list ? list[i + lane] : -1;
      const uint64_t real = __builtin_amdgcn_ballot_w64((unsigned)g < (unsigned)ng);
      last = real ? i + 64 - __builtin_clzll(real) : last;
    }
    cold.n = n_rows > 0 ? last * nblk : 0;
  } else {
    cold = runs(0, n_cold, [&](int tok) {
      const int g = a.by.group(tok);
      return g * nblk + (tok - g * G) / 32;
    });
  }
  const BlockRuns hot = runs(n_cold, n, [&](int tok) { return (tok - n_cold) / 32; });
  // equal runs for the waves of all splits, coded ones first
  const int n_waves = a.n_splits * kFewWaves;
  int run = max(a.by.waves(cold.n + hot.n + n_waves - 1), 1), cold_waves;
  for (;; ++run) {
    cold_waves = few_quotient(cold.n + run - 1, run);
    if (cold_waves + few_quotient(hot.n + run - 1, run) <= n_waves) break;
  }
  const int gw = split * kFewWaves + wave;
  const bool is_cold = gw < cold_waves;
  const int i0 = (is_cold ? gw : gw - cold_waves) * run;
  const int i1 = min(i0 + run, is_cold ? cold.n : hot.n);

  // (the queries in LDS: the loop has no registers for them)
  float q_top = 0.f;  // the largest |q| (what is not finite: as the largest of fp16; its rows are lost whatever the power)
  {
    typedef uint16_t us2_t __attribute__((ext_vector_type(2)));
    us2_t two = {0, 0};
#pragma unroll
    for (int mm = 0; mm < NM; ++mm) {
      if (wave == mm && !is_lo) *reinterpret_cast<h8_t*>(&qr_s[ln][CPL * lg + 8 * mm]) = q8[mm];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const _Float16 y = q8[mm][e];
        if (wave == mm && ln < NR) qc_s[CPL * lg + 8 * mm + e][ln] = __builtin_bit_cast(uint16_t, y);
      }
      union { h8_t h; uint32_t u[4]; } bits;
      bits.h = q8[mm];
#pragma unroll
      for (int e = 0; e < 4; ++e) two = __builtin_elementwise_max(two, __builtin_bit_cast(us2_t, bits.u[e] & 0x7FFF7FFFu));
    }
    if constexpr (!PK) {
      const uint16_t one = max(two.x, two.y);
      q_top = wave_reduce<true>(h2f(one < 0x7C00 ? one : (uint16_t)0x7BFF));
    }
  }
  // the coded keys' weights, this column's half of an fp16 pair: q * scale group by
  // group, or for rotated keys q @ Pi^T; over a power of two, w_up, where they pass fp16
  union Half { h8_t h; uint32_t u[4]; };
  Half bw[NSL];
  float w_up = 1.f, w_down = 1.f;
  auto put_weights = [&](int s, float x0, float x1, float x2, float x3) {
    // (towards zero: two in one instruction)
    const h2_t y = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    const h2_t z = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(x2, x3));
    const uint32_t v01 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float)y.x, -lo_sel, x0), fmaf((float)y.y, -lo_sel, x1)));
    const uint32_t v23 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float)z.x, -lo_sel, x2), fmaf((float)z.y, -lo_sel, x3)));
    bw[s].u[0] = bw[s].u[1] = v01;
    bw[s].u[2] = bw[s].u[3] = v23;
  };

  // ---- the coded blocks of this wave: state and loads
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
  const float per_page = a.by.per_page;
  const int group_pages = a.by.group_pages;
  // the page row of token o of group g (pages inside a group by a product: fewer
  // than 256 tokens, exact)
  auto page_row = [&](int g, int o) {
    const int pg = (int)(((float)o + 0.5f) * per_page);
    return bt[g * group_pages + pg] * P + o - pg * P;
  };
  int meta_i = i0, meta_g = 0, meta_k = 0, meta_tok = 0, meta_ob = 0, meta_lo = 0, meta_n = 0, meta_row[2] = {0, 0};
  auto load_meta = [&](int i) {
    meta_i = i;
    const int blk = cold.at(min(i + lane, i1 - 1));
    meta_g = a.by.blocks(blk);
    meta_k = blk - meta_g * nblk;
    meta_tok = meta_g * G;
    if (list) {
      const int g = list[meta_g];
      const bool real = (unsigned)g < (unsigned)ng;
      meta_g = real ? g : 0;  // (a group that there is: nobody sees it here)
      meta_tok = real ? g * G : kNoToken;
    }
    meta_tok += 32 * meta_k;
    meta_ob = gt[meta_g] * Hkv + h;
    if constexpr (TILED) {  // (16 tokens lie in one page)
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) meta_row[tile] = page_row(meta_g, 32 * meta_k + 16 * tile);
    }
    // the entries of the blocks that the wave takes of a stretch from this one on
    const int32_t* oc = a.p.ocount + (size_t)meta_ob * TQK_NOB;
    const int end = min(min((meta_k / SB + 1) * SB, nblk), meta_k + i1 - min(i + lane, i1 - 1));
    const int lo_ = oc[max(meta_k - 1, 0)], hi_ = oc[end - 1];
    meta_lo = listed && meta_k > 0 ? min(max(lo_, 0), cap) : 0;
    meta_n = listed ? max(min(hi_, cap) - meta_lo, 0) : 0;
  };
  auto of = [&](int y, int i) { return __builtin_amdgcn_readlane(y, i - meta_i); };  // block i's
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
  uint32_t kw[2][KW], ent[kPreEntries];
  float nsc[SPL], nmu[SPL];
  uint32_t vw[NS][8];
  float norm[8], kn[8];
  int n_ob = 0, n_lo = 0, n_ent = 0;  // of the block whose keys are loaded
  // the norms of a lane's 8 tokens of a block: 4 lg .. + 3 and 16 + 4 lg .. + 3
  auto load_norms = [&](float (&y)[8], const float* from, const Rows& rw) {
    if constexpr (TILED) {
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        const f4_t z = *reinterpret_cast<const f4_t*>(from + (head + rw.r[tile]) + (uint32_t)(4 * lg));
#pragma unroll
        for (int e = 0; e < 4; ++e) y[4 * tile + e] = z[e];
      }
    } else {
      y[0] = from[head + rw.r[0]];  // (token lane % 32's: handed out when needed)
    }
  };
  auto norm_of = [&](const float (&y)[8], int e) {
    return TILED ? y[e] : __shfl(y[0], 16 * (e / 4) + 4 * lg + e % 4, 64);
  };
  // keys of block i (at rows rw), its group's statistics and its stretch's entries
  auto load_keys = [&](int i, const Rows& rw) {
    i = min(i, i1 - 1);
    n_ob = of(meta_ob, i);
    n_lo = of(meta_lo, i);
    n_ent = of(meta_n, i);
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
        nsc[e] = a.p.gscale[(size_t)n_ob * D + SPL * lane + e];
        nmu[e] = a.p.gmean[(size_t)n_ob * D + SPL * lane + e];
      }
      // lane's run of the stretch's entries: its first ones (a block inside a stretch:
      // of a list of no bytes, which reads nothing)
      const int each = (n_ent + 63) >> 6;
      const int first = (int)(of(meta_k, i) % SB == 0) | (int)(i == i0) | (int)(i == cold.n0);
      const __amdgpu_buffer_rsrc_t ro = entries_of(oent + (size_t)n_ob * cap, 4u * (uint32_t)(cap * first));
      const int off = 4 * (n_lo + lane * each);
#pragma unroll
      for (int e = 0; e < kPreEntries; e += 4) {
        const u32x4_t y = __builtin_amdgcn_raw_buffer_load_b128(ro, off + 4 * e, 0, 0);
        ent[e] = y.x;
        ent[e + 1] = y.y;
        ent[e + 2] = y.z;
        ent[e + 3] = y.w;
      }
    }
  };
  // a group's weights and the rest of its scores (q . mean, over w_up)
  float bias = 0.f;
  auto begin_group = [&]() {
    // q * scale within fp16: a scale of keys near 65504 times a large query is not
    float s_top = 0.f;
#pragma unroll
    for (int e = 0; e < SPL; ++e) s_top = fmaxf(s_top, fabsf(nsc[e]));
    w_up = w_down = 1.f;
    if (__builtin_expect(__any(s_top * q_top > 65504.f), 0)) {
      s_top = wave_reduce<true>(s_top);
      // (s_top q_top < 2^e; an infinite scale's group is lost whatever the power)
      const int e = __builtin_amdgcn_readfirstlane(min(__builtin_amdgcn_frexp_expf(s_top) + __builtin_amdgcn_frexp_expf(q_top), 126));
      w_up = ldexpf(1.f, e - 15);
      w_down = ldexpf(1.f, 15 - e);
#pragma unroll
      for (int i = 0; i < SPL; ++i) nsc[i] *= w_down;
    }
#pragma unroll
    for (int e = 0; e < SPL; ++e) {
      stat_s[wave][0][SPL * lane + e] = nsc[e];
      stat_s[wave][1][SPL * lane + e] = nmu[e];
    }
    wave_sync();
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < NSL; ++s) {
      const int ch = CPL * lg + 4 * s;
      const f4_t s4 = *reinterpret_cast<const f4_t*>(&stat_s[wave][0][ch]);
      const f4_t m4 = *reinterpret_cast<const f4_t*>(&stat_s[wave][1][ch]);
      typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
      const h4_t qh = *reinterpret_cast<const h4_t*>(&qr_s[ln & 7][ch]);
      float q4[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        q4[k] = (float)qh[k];
        y = fmaf(q4[k], m4[k], y);
      }
      put_weights(s, q4[0] * s4[0], q4[1] * s4[1], q4[2] * s4[2], q4[3] * s4[3]);
    }
    bias = colgroup_sum(y) * w_down;
  };
  // the scores' first values of stretch `sg`: q . mean, and the side-list's sums
  float* const corr = &corr_s[wave][0][0];
  auto begin_stretch = [&](int sg) {
    float br[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) br[i] = bitsf((uint32_t)__builtin_amdgcn_readlane((int)fbits(bias), i));
    {
      constexpr int kStep = 256 / NR;  // tokens that the lanes fill at a time: four each, row lane % NR
      const float y = __shfl(bias, lane % NR, 64);
      float* const to = corr + lane % NR * kCorr + lane / NR * 4;
      for (int i = 0; i < min(kSeg, G - kSeg * sg); i += kStep) *reinterpret_cast<f4_t*>(to + i) = f4_t{y, y, y, y};
    }
    wave_sync();
    if (PK || n_ent == 0) return;
    // Lane L takes `each` consecutive entries of the list, which is sorted by token: a
    // token's run that ends inside the lane is written; the first one may have begun in
    // the lanes before, the last one may go on in the next.
    const int each = (n_ent + 63) >> 6, mine = n_ent - lane * each, t0 = kSeg * sg;
    float acc[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) acc[i] = 0.f;
    int tcur = -1, tf = -1;
    struct Ops {
      float mean;
      uint32_t q[NR / 2];
    };
    auto gather = [&](uint32_t y, Ops& o) {
      const int ch = (int)(y & (uint32_t)(D - 1));
      o.mean = stat_s[wave][1][ch];
      if constexpr (NR == 4) {
        const u32x2_t z = *reinterpret_cast<const u32x2_t*>(&qc_s[ch][0]);
        o.q[0] = z.x;
        o.q[1] = z.y;
      } else {
        const u32x4_t z = *reinterpret_cast<const u32x4_t*>(&qc_s[ch][0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) o.q[i] = z[i];
      }
    };
    auto entry = [&](int k, uint32_t y, const Ops& o) {
      // (an entry outside the stretch is dropped, whatever the list holds: every
      // index below stays in corr_s)
      const int tx = (int)((y & 0xFFFFu) / D) - t0;
      const bool valid = k < mine && (unsigned)tx < (unsigned)kSeg;
      const int tk = valid ? tx : -1;
      const bool same = tk == tcur;
      if (!same && tcur >= 0) {
#pragma unroll
        for (int i = 0; i < NR; ++i) corr[i * kCorr + tcur] = acc[i] + br[i];
      }
      tf = tf < 0 ? tk : tf;
      tcur = tk;
      const float dv = valid ? (h2f((uint16_t)(y >> 16)) - o.mean) * w_down : 0.f;
#pragma unroll
      for (int i = 0; i < NR; ++i)
        acc[i] = fmaf(h2f((uint16_t)(o.q[i / 2] >> (16 * (i & 1)))), dv, same ? acc[i] : 0.f);
    };
#pragma unroll
    for (int k0 = 0; k0 < kPreEntries; k0 += 4) {
      if (k0 < each) {
        Ops o[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) gather(ent[k0 + u], o[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (k0 + u < each) entry(k0 + u, ent[k0 + u], o[u]);
      }
    }
    const uint32_t* const rest = oent + (size_t)n_ob * cap;
    for (int k = kPreEntries; k < each; ++k) {  // long lists only
      const uint32_t y = rest[min(n_lo + lane * each + k, cap - 1)];
      Ops o;
      gather(y, o);
      entry(k, y, o);
    }
    // The lanes' last runs summed along the lanes, by token: each lane has the sum of
    // its token's runs so far, a lane's first run takes its left neighbour's, and the
    // last lane of a token's chain writes it.  Only a token over three or more lanes
    // needs the scan.
    float sv[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) sv[i] = acc[i];
    const int tl = tcur;
    const int tl_up = lane_before(tl), tf_dn = lane_after(tf);
    const int tl_prev = lane > 0 ? tl_up : -1, tf_next = lane < 63 ? tf_dn : -1;
    int kd = tl_prev;  // the last run's token `o` lanes before
    for (int o = 1; o < 64 && __builtin_amdgcn_ballot_w64(tl >= 0 && kd == tl) != 0; o <<= 1) {
      const bool add = kd == tl && tl >= 0;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const float v = o == 1 ? bitsf((uint32_t)lane_before((int)fbits(sv[i]))) : __shfl_up(sv[i], o, 64);
        sv[i] += add ? v : 0.f;
      }
      kd = __shfl_up(tl, 2 * o, 64);
      kd = lane >= 2 * o ? kd : -1;
    }
    float sprev[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) sprev[i] = bitsf((uint32_t)lane_before((int)fbits(sv[i])));
    if (tf >= 0 && tf != tl && tl_prev == tf) {  // the first run ends inside this lane: and what came before
#pragma unroll
      for (int i = 0; i < NR; ++i) corr[i * kCorr + tf] += sprev[i];
    }
    if (tl >= 0 && tf_next != tl) {
#pragma unroll
      for (int i = 0; i < NR; ++i) corr[i * kCorr + tl] = sv[i] + br[i];
    }
    wave_sync();
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
          else if constexpr (VB == 3) {
            // (a dword of the row at any byte: from the byte before, of the first piece from itself)
            const int piece = (D == 64 ? ln / 2 : ln) + 16 * s;
            uint32_t y;
            __builtin_memcpy(&y, src - (piece > 0), 4);
            vw[s][e] = piece > 0 ? y >> 8 : y;
          } else
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

  // ---- the tables, while the first codes are on their way
  {
    const uint2 y = split_pair(lev0, lev1);
    if (kp.entry >= 0)
#pragma unroll
      for (int k = 0; k < kp.pieces; ++k)  // (entries apart by a table row: each begins at another piece)
        *reinterpret_cast<u32x4_t*>(key_s + (ke << kKeyLog) + 16 * (kp.first + (k + ke) % kp.pieces)) = u32x4_t{y.x, y.y, y.x, y.y};
  }
  // the scale of the value codebook: candidate 1 + i / 128 whose centroids lose least to
  // fp16
  float up;
  {
    float best = INFINITY, at = 1.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const float g = 1.0f + (float)(2 * lane + half) * (1.0f / 128);
      float err = 0.f;
#pragma unroll
      for (int i = 0; i < (1 << VB); ++i) {
        const float y = cen[i] * g, r = y - (float)(_Float16)y;
        err = fmaf(r, r, err);
      }
      err *= __builtin_amdgcn_rcpf(g * g);
      if (err < best) {
        best = err;
        at = g;
      }
    }
    const float least = -wave_reduce<true>(-best);
    const uint64_t first = __builtin_amdgcn_ballot_w64(best == least);
    up = bitsf((uint32_t)__builtin_amdgcn_readlane((int)fbits(at), first ? __builtin_ctzll(first) : 0));
  }
  {
    const uint32_t y = pk_f16(cen0 * up, cen1 * up);
    if (vp.entry >= 0)
#pragma unroll
      for (int k = 0; k < vp.pieces; ++k)
        *reinterpret_cast<u32x4_t*>(val_s + (ve << kValLog) + 16 * (vp.first + (k + ve) % vp.pieces)) = u32x4_t{y, y, y, y};
  }
  // a table read: the field of `bits` bits at bit `bit` of the word array w, as an
  // entry of 2^lg bytes and this lane's copy in it
  typedef __attribute__((address_space(3))) const uint32_t lds_t;
  const uint32_t k_copy = 8 * (lane % kKeyCopies);
  const uint32_t v_copy = (uint32_t)(uintptr_t)(lds_t*)reinterpret_cast<const uint32_t*>(val_s) + 4 * (lane % kValCopies);
  auto place_in = [](const uint32_t* w, int bit, int bits, int lg_, uint32_t copy, bool byte) -> uint32_t {
    const int wd = bit / 32, sh = bit % 32;
    if (byte)  // byte sh / 8 above the copy's byte
      return __builtin_amdgcn_perm(w[wd], copy, 0x0C0C0000u | (4u + sh / 8) << 8);
    const uint32_t mask = ((1u << bits) - 1u) << lg_;
    const uint32_t y = sh + bits > 32 ? __builtin_amdgcn_alignbit(w[wd + 1], w[wd], sh) << lg_
                       : sh >= lg_    ? w[wd] >> (sh - lg_)
                                      : w[wd] << (lg_ - sh);
    return (y & mask) | copy;
  };
  auto levels = [&](const uint32_t* w, int bit) {
    return *reinterpret_cast<const u32x2_t*>(key_s + place_in(w, bit, 2 * KB, kKeyLog, k_copy, KB == 4));
  };
  auto centroids = [&](const uint32_t* w, int bit) {
    return *(lds_t*)(uintptr_t)place_in(w, bit, 2 * VB, kValLog, v_copy, false);
  };

  if constexpr (PK) {
    // q @ Pi^T: rows in corr_s' place
    static_assert(kRows8 * D * 8 <= (int)sizeof(corr_s), "rotated queries fit");
    __syncthreads();
    float* const q_s = &corr_s[0][0][0];  // [8][D]
    float* const r_s = q_s + kRows8 * D;  // [8][D]
    for (int i = tid; i < kRows8 * D; i += kFewThreads) q_s[i] = h2f(qr_s[i / D][i % D]);
    __syncthreads();
    for (int i = tid; i < kRows8 * D; i += kFewThreads) {
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
    for (int e = 0; e < CPL; ++e) y_top = fmaxf(y_top, fabsf(r_s[(ln & 7) * D + CPL * lg + e]));
    y_top = fminf(wave_reduce<true>(y_top), 16.f * 65504.f);  // (more: not of finite queries)
    if (y_top > 65504.f) {
      const int e = __builtin_amdgcn_frexp_expf(y_top);  // y_top < 2^e
      w_down = ldexpf(1.f, 15 - e);
      w_up = ldexpf(1.f, e - 15);
    }
#pragma unroll
    for (int s = 0; s < NSL; ++s) {
      const float* y = r_s + (ln & 7) * D + CPL * lg + 4 * s;
      put_weights(s, y[0] * w_down, y[1] * w_down, y[2] * w_down, y[3] * w_down);
    }
    __syncthreads();  // (corr_s is the waves' own again)
  }
  lds_barrier();

  const float c = d.sm_scale * 1.4426950408889634f;
  float m_run = -INFINITY, l_run = 0.f;  // of the scores times c
  f4_t O[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) O[i] = f4_t{0.f, 0.f, 0.f, 0.f};

  // the 8 scores (over c) of this column's row: tokens 4 lg + i, then 16 + 4 lg + i, of
  // a block at tok0; tokens from cnt on are none.  The running maximum.
  auto mask_and_max = [&](f4_t (&S)[2], int tok0, int cnt, bool whole, auto hide) {
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int o = 16 * (i / 4) + 4 * lg + i % 4;
        const bool seen = (o < cnt) & sees(tok0 + o);
        S[i / 4][i % 4] = seen ? S[i / 4][i % 4] : -INFINITY;
        hide(i, seen);
      }
      asm volatile("");  // (one branch for the eight)
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, S[i / 4][i % 4]);
    mx *= c;
    if (__any(mx > m_run + kFewLazy)) {
      mx = colgroup_max(mx);
      const float m_new = fmaxf(m_run, mx);
      const float f = m_new == -INFINITY ? 1.f : above_zero(__builtin_amdgcn_exp2f(m_run - m_new));
      m_run = m_new;
      l_run *= f;
#pragma unroll
      for (int i = 0; i < NV; ++i) O[i] *= f;
    }
  };
  auto weights = [&](const f4_t (&S)[2], float (&w)[8]) {
    const float at = m_run == -INFINITY ? 0.f : m_run;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = __builtin_amdgcn_exp2f(fmaf(S[i / 4][i % 4], c, -at));
      sum += w[i];
    }
    l_run += sum;
    return sum;
  };
  // eight numbers as this column's half of their fp16 pairs
  auto halves = [&](const float (&y)[8]) {
    union { h8_t h; uint32_t u[4]; } z;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const h2_t hi = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(y[e], y[e + 1]));
      z.u[e / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float)hi.x, -lo_sel, y[e]), fmaf((float)hi.y, -lo_sel, y[e + 1])));
    }
    return z.h;
  };

  if (has_codes) {
    const float* const init = is_lo ? zero_s : corr + min(row, NR - 1) * kCorr + 4 * lg;
    const int init_step = is_lo ? 0 : 1;
    // scores of the loaded keys, block kb of its stretch: before the halves are added
    auto product = [&](f4_t (&S)[2], int kb) {
#pragma unroll
      for (int tile = 0; tile < 2; ++tile) {
        S[tile] = PK ? f4_t{0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const f4_t*>(init + init_step * (32 * kb + 16 * tile));
        // (at head_dim 256 half of the levels at a time: there are no registers for all)
        constexpr int kAtOnce = NSL < 8 ? NSL : 8;
#pragma unroll
        for (int s0 = 0; s0 < NSL; s0 += kAtOnce) {
          union { h8_t h; u32x2_t u[2]; } y[kAtOnce];
#pragma unroll
          for (int s = 0; s < kAtOnce; ++s) {
            y[s].u[0] = levels(kw[tile], KB * 4 * (s0 + s));
            y[s].u[1] = levels(kw[tile], KB * (4 * (s0 + s) + 2));
          }
#pragma unroll
          for (int s = 0; s < kAtOnce; ++s)
            S[tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y[s].h, bw[s0 + s].h, S[tile], 0, 0, 0);
          if constexpr (D == 256) __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    if constexpr (!PK) {
      begin_group();
      begin_stretch(of(meta_k, i0) / SB);
    }
    f4_t S[2];
    float kn_now[8];
    product(S, of(meta_k, i0) % SB);
    if constexpr (PK) {
#pragma unroll
      for (int e = 0; e < 8; ++e) kn_now[e] = kn[e];
    }
    float up_now = w_up;
    int k = of(meta_k, i0), tok0 = of(meta_tok, i0), g = of(meta_g, i0);
    Rows after = next_rows;
    load_keys(i0 + 1, next_rows);
    int i = i0;
    // The last block without a next one's scores beside it, in a copy of the loop's body
    // (the last one's again in their place: 2 us more of every run)
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const bool more = part == 0;
      while (!more || i + 1 < i1) {
        const int cnt = min(32, G - 32 * k);
        if (more) {
          if (i + 3 >= meta_i + 64) load_meta(i + 1);
          after = rows_of(i + 2);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = S[e / 4][e % 4], z = y + row_ror<8>(y);
          S[e / 4][e % 4] = PK ? z * norm_of(kn_now, e) : z;  // (PK: score = |k| (q_rot . centroids))
        }
        if (__builtin_expect(up_now != 1.f, 0)) {
          S[0] *= up_now;
          S[1] *= up_now;
        }
        const bool whole = cnt == 32 && all_see(tok0, 32);
        // (a hidden token's norm may be anything: its weight is zero)
        float nv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) nv[e] = norm_of(norm, e);
        mask_and_max(S, tok0, cnt, whole, [&](int e, bool seen) { nv[e] = seen ? nv[e] : 0.f; });
        int k_n = 0, tok_n = 0, g_n = 0;
        f4_t N[2];
        if (more) {
          k_n = of(meta_k, i + 1);
          tok_n = of(meta_tok, i + 1);
          g_n = of(meta_g, i + 1);
          if constexpr (!PK) {
            const bool apart = i + 1 == cold.n0;  // (the second run may start inside a group)
            if (k_n == 0 || apart) begin_group();
            if (k_n % SB == 0 || apart) begin_stretch(k_n / SB);
          }
          product(N, k_n % SB);
          if constexpr (PK) {
#pragma unroll
            for (int e = 0; e < 8; ++e) kn_now[e] = kn[e];
          }
          up_now = w_up;
          load_keys(i + 2, after);
        }
        float w[8];
        const float sum = weights(S, w);
        float pw[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pw[e] = w[e] * nv[e];
        }
        const h8_t pf = halves(pw);
        // V^T P^T: row ln of the first operand is channel NC ln + j of the piece
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          if constexpr (TILED) {
            // a channel's token pairs side by side in the unit's bits
#pragma unroll
            for (int j = 0; j < NC; ++j) {
              union { h8_t h; uint32_t u[4]; } y;
#pragma unroll
              for (int f = 0; f < 4; ++f) y.u[f] = centroids(vw[0] + 4 * (f / 2), (2 * j + f % 2) * 2 * VB);
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
        if (a.block_ml) {
          const float y = colgroup_sum(sum);
          if (lg == 0 && ln < n_rows && !is_lo) {
            const long long o = ((((long long)b * Hq + h * gq + row_h) * a.t_len + t - a.t0) * a.blocks + g * nblk + k) * 2;
            a.block_ml[o] = m_run;
            a.block_ml[o + 1] = y;
          }
        }
        if (!more) break;
        load_values(next_rows);
        next_rows = after;
        S[0] = N[0];
        S[1] = N[1];
        k = k_n;
        tok0 = tok_n;
        g = g_n;
        ++i;
      }
    }
  } else if (!is_cold) {
    // uncoded blocks, straight from the ring
    h8_t qf[NM];
#pragma unroll
    for (int mm = 0; mm < NM; ++mm) qf[mm] = *reinterpret_cast<const h8_t*>(&qr_s[ln & 7][CPL * lg + 8 * mm]);
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
      mask_and_max(S, tok0, cnt, cnt == 32 && all_see(tok0, 32), [](int, bool) {});
      float w[8];
      weights(S, w);
      const h8_t pf = halves(w);
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
        // ... and added to the rows that see it (any positive weight gives the same),
        // in their first column
#pragma unroll 1
        for (int o = 0; o < cnt; ++o) {
          const bool vis = sees(tok0 + o) && !is_lo;
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
  float* const out_s = reinterpret_cast<float*>(key_s);  // [wave][8][D]
  {
    const float l = colgroup_sum(l_run);
    if (lg == 0 && !is_lo) {
      ml_s[0][wave][ln] = m_run;
      ml_s[1][wave][ln] = l;
    }
    lds_barrier();  // (every wave has read its last levels)
    // (the two columns of a row write two of its four stretches of channels each)
    float* const to = out_s + (wave * kRows8 + (ln & 7)) * OST;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < NC; j += 4) {
        f4_t z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float y = O[NC * s + j + k][e];
            z[e][k] = y + row_ror<8>(y);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f4_t y;
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = is_lo ? z[2 + e][k] : z[e][k];
          *reinterpret_cast<f4_t*>(to + 128 * s + NC * (4 * lg + (is_lo ? 2 : 0) + e) + j) = y;
        }
      }
  }
  __syncthreads();
  constexpr int kRowGroups = kFewThreads / D;                 // rows side by side
  constexpr int RPT = (kRows8 + kRowGroups - 1) / kRowGroups;  // rows a thread
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
      const float y = out_s[(w * kRows8 + r) * OST + j];
      ls[k] = fmaf(ml_s[1][w][r], f, ls[k]);
      // (a state without a maximum holds zeros; a NaN among its scores leaves it one)
      if (w < first_hot) cs[k] += y * f; else hs[k] += y * f;
    }
  }
  if (first_hot > 0) {
    __syncthreads();
    // the coded sums over their weights' sum (within fp16's range then) as an
    // fp16 pair, times Pi's
    constexpr int CST = D + 8;
    uint16_t* const c_s = reinterpret_cast<uint16_t*>(key_s);           // [2][8][CST]
    float* const y_s = reinterpret_cast<float*>(key_s) + kRows8 * CST;  // [8][D]
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const int r = r0 + kRowGroups * k;
      if (r < kRows8) {
        const float y = ls[k] != 0.f ? cs[k] / (ls[k] * up) : 0.f;
        const _Float16 hi = (_Float16)y;
        c_s[r * CST + j] = __builtin_bit_cast(uint16_t, hi);
        c_s[(kRows8 + r) * CST + j] = f2h(y - (float)hi);
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
          // (rows 8 to 15 of the operand: the sums' second halves)
          const h8_t ch = *reinterpret_cast<const h8_t*>(c_s + ln * CST + 32 * mm + 8 * lg);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch, pl, acc, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch, ph, acc, 0, 0, 0);
        }
        // rows 4 lg + e: first halves in lanes of lg 0 and 1, second ones in 2 and 3
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float z = acc[e] + __shfl_xor(acc[e], 32, 64);
          if (lg < 2) y_s[(4 * lg + e) * D + 16 * (wave + kFewWaves * nt) + ln] = z;
        }
        if (nt + 1 < NTR) load_pi(nt + 1);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RPT; ++k)
      if (r0 + kRowGroups * k < kRows8) hs[k] = fmaf(y_s[(r0 + kRowGroups * k) * D + j], ls[k], hs[k]);
  }
  // (rows past the queries of the sequence: zero)
  const int all_rows = min(a.per_item, a.t0 + a.t_len - q0) * gq;
#pragma unroll
  for (int k = 0; k < RPT; ++k) {
    const int r = r0 + kRowGroups * k;
    if (r >= all_rows) continue;
    const int rt = a.by.heads_of(r), tr = q0 + rt, hq = h * gq + r - rt * gq;
    if (a.direct) {
      const long long o = b * a.o_stride[0] + hq * a.o_stride[1] + tr * a.o_stride[2] + j;
      // (a query in a coded group that is not listed may see nothing)
      const float y = r < n_rows && n - m + tr >= 0 && ls[k] != 0.f ? hs[k] / ls[k] : 0.f;
      if (a.out_type == 0) static_cast<float*>(a.out)[o] = y;
      else static_cast<_Float16*>(a.out)[o] = (_Float16)y;
    } else {
      const long long o = (a.split0 + split) * a.rows + ((long long)b * Hq + hq) * a.t_len + tr - a.t0;
      a.part_acc[o * D + j] = hs[k];
      if (j == 0) {
        a.part_ml[2 * o] = ms[k];
        a.part_ml[2 * o + 1] = ls[k];
      }
    }
  }
}

template <int D, int VB, bool TILED, int NR>
void launch_rows_keys(const MoreArgs& a, unsigned groups, hipStream_t st) {
  const dim3 grid(groups), block(kFewThreads);
  if (a.d.key_grid == 2)
    hipLaunchKernelGGL((tqk_attend_rows<D, VB, VB, true, TILED, NR>), grid, block, 0, st, a);
  else if (a.d.key_bits == 4)
    hipLaunchKernelGGL((tqk_attend_rows<D, VB, 4, false, TILED, NR>), grid, block, 0, st, a);
  else if (a.d.key_bits == 3)
    hipLaunchKernelGGL((tqk_attend_rows<D, VB, 3, false, TILED, NR>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((tqk_attend_rows<D, VB, 2, false, TILED, NR>), grid, block, 0, st, a);
}
template <int D, bool TILED, int NR>
void launch_rows_values(const MoreArgs& a, unsigned groups, hipStream_t st) {
  if (a.d.value_bits == 2)
    launch_rows_keys<D, 2, TILED, NR>(a, groups, st);
  else if (a.d.value_bits == 3)
    launch_rows_keys<D, 3, TILED, NR>(a, groups, st);
  else
    launch_rows_keys<D, 4, TILED, NR>(a, groups, st);
}
template <int D, bool TILED>
void launch_rows_tiled(const MoreArgs& a, unsigned groups, hipStream_t st) {
  if (a.per_item * (a.d.n_q_heads / a.d.n_kv_heads) <= 4)
    launch_rows_values<D, TILED, 4>(a, groups, st);
  else
    launch_rows_values<D, TILED, 8>(a, groups, st);
}
template <int D>
void launch_rows(const MoreArgs& a, unsigned groups, hipStream_t st) {
  if constexpr (D == TQK_D) {
    if (v_tiled(a.d.group_tokens, a.d.page_tokens, D, 0)) return launch_rows_tiled<D, true>(a, groups, st);
  }
  launch_rows_tiled<D, false>(a, groups, st);
}

}  // namespace
