// Attention of many rows over the coded groups that all sequences of a batch share
// (gfx950): the first part of tqk_attend_shared.
//
// A workgroup takes one kv head, up to 128 rows (queries times query heads, of any
// sequences) and a share of the prefix.  Its tokens are decoded once for all rows, 64
// at a time (32 at head_dim 256), into LDS: keys as fp16 pairs of mean + scale * level,
// a side-list entry's value over them, and the values' centroids by channel.  Four
// groups of 32 rows each go over them with 32 x 32 products, scores transposed (K Q^T),
// so that a row's statistics are a lane's registers and the weights are the operand of
// V^T P^T as they are; two waves share a row group, by tokens, or at head_dim 256 by
// channels.  Weights times norms are fp16 pairs, two products.  While a tile is
// multiplied the next one is decoded, and the one after it is on its way.
//
// 32768 tokens, 32 sequences, 32 / 8 heads of 128 (8 x 32 splits of 16 tiles): 73 us, 17 of
// them once (tables, first tiles, sums out through LDS) and 3.2 a tile.  No unit is full:
// vector issue half of the time, LDS 31 %, the matrix cores 23 %; the waves wait 47 % of
// theirs, at two waves a SIMD that all decode and multiply between two barriers a tile
// (3-bit values: 20 bytes of a lane in scratch).
#include "tqk_attend_few.h"

namespace {

typedef float f16_t __attribute__((ext_vector_type(16)));
constexpr int kPreRows = 128, kPreThreads = 512;

template <int D, int VB, bool TILED>
__global__ __launch_bounds__(kPreThreads, 2) void tqk_attend_prefix(MoreArgs a) {
  constexpr bool kWide = D == 256;          // two waves of a row group share channels, not tokens
  constexpr int TT = kWide ? 32 : 64;       // tokens of a tile
  constexpr int NB = TT / 32;               // blocks of a tile
  constexpr int CQ = D / 4, TG = kPreThreads / CQ, TPT = TT / TG;  // keys: four channels, TPT tokens a thread
  constexpr int KST = D + 8;                // halves of a key row in LDS
  constexpr int VST = TT + 4;               // halves of a channel's values in LDS
  constexpr int NK = D / 16;                // steps of a score product
  constexpr int NO = kWide ? D / 64 : D / 32;  // a wave's accumulator tiles of 32 channels
  constexpr int VROW = D * VB / 8;
  constexpr int kVThreads = TT / 4 * CQ;    // values: 4 tokens x 4 channels a thread
  static_assert(kVThreads <= kPreThreads && TPT * TG == TT, "the threads cover a tile");
  touch_args<MoreArgs>();
  const tqk_cache_desc& d = a.d;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lc = lane & 31, hl = lane >> 5;
  const int G = d.group_tokens, P = d.page_tokens, Hkv = d.n_kv_heads, Hq = d.n_q_heads, gq = Hq / Hkv, kb = d.key_bits;
  const int nblk = (G + 31) / 32;
  int x = blockIdx.x;
  const int split = x % a.n_splits;
  x /= a.n_splits;
  const int h = x % Hkv, row0 = x / Hkv * kPreRows;
  const int per = a.q_len * gq, all_rows = a.batch * per, n_rows = min(kPreRows, all_rows - row0);
  // this split's tiles
  const int blocks = a.shared / G * nblk, tiles = (blocks + NB - 1) / NB, each = (tiles + a.n_splits - 1) / a.n_splits;
  const int t0 = split * each, t1 = min(t0 + each, tiles);

  __shared__ __align__(16) uint16_t k_s[2][2][TT][KST];  // [buffer][half][token][channel]
  __shared__ __align__(16) uint16_t v_s[2][D][VST];      // [buffer][channel][token]
  __shared__ __align__(16) float norm_s[2][TT];
  constexpr int kLevCopies = 16, kCenCopies = VB == 4 ? 16 : 32;
  __shared__ __align__(128) float lev_s[256][kLevCopies][2];
  __shared__ __align__(128) uint32_t cen_s[1 << (2 * VB)][kCenCopies];
  // of the tiles ahead: rows of their tokens; their blocks' slot * Hkv + h, first entry,
  // entries, first token in the group and tokens
  constexpr int kRing = 4;
  struct Meta {
    int ob, lo, n, tok0, cnt;
  };
  __shared__ int row_s[kRing][TT];
  __shared__ Meta meta_s[kRing][NB];
  __shared__ float join_s[4][2][32];

  // ---- what the tables say of a tile ahead
  const int32_t* const bt = a.p.block_table;  // (every sequence's begins alike: the first one's)
  const int32_t* const gt = a.p.group_table;
  const bool listed = d.outliers_per_channel > 0;
  const int cap = listed ? d.outlier_cap : 1;
  const uint32_t* const oent = listed ? a.p.oent : reinterpret_cast<const uint32_t*>(a.p.ocount);
  // block j of tile t (the last one for those past it): its group and place there
  const uint32_t per_block = 0xFFFFFFFFu / (uint32_t)nblk + 1;  // 2^32 / nblk, over: exact below 2^28 blocks (1: 0)
  struct Place {
    int g, k;
    bool real;
  };
  auto place_of = [&](int t, int j) {
    const int blk = min(t * NB + j, blocks - 1), g = nblk == 1 ? blk : (int)__umulhi((uint32_t)blk, per_block);
    return Place{g, blk - g * nblk, t * NB + j < blocks};
  };
  const float per_page = 1.0f / (float)P;
  const int group_pages = G / P;
  // (pages inside a group by a product: fewer than 256 tokens, exact)
  auto page_in = [&](int o) { return (int)(((float)o + 0.5f) * per_page); };

  // A tile's chain of loads (group -> slot -> counts, page) a step a tile: what was asked
  // for while the last tile was multiplied goes into LDS, the next is asked for.
  const bool asks_rows = tid < TT, asks_meta = tid >= TT && tid < TT + NB;
  const int ask_j = asks_meta ? tid - TT : min(tid / 32, NB - 1);
  int r_page = 0, r_slot = 0, r_ob = 0, r_lo = 0, r_hi = 0;
  auto ask_slot = [&](int t) {
    if (asks_meta) r_slot = gt[place_of(t, ask_j).g];
  };
  auto ask = [&](int t) {  // (ask_slot(t) was before)
    const Place y = place_of(t, ask_j);
    if (asks_rows) {
      r_page = bt[y.g * group_pages + page_in(min(32 * y.k + tid % 32, G - 1))];
    } else if (asks_meta) {
      r_ob = r_slot * Hkv + h;
      const int32_t* oc = a.p.ocount + (size_t)r_ob * TQK_NOB;
      r_lo = oc[max(y.k - 1, 0)];
      r_hi = oc[y.k];
    }
  };
  auto keep = [&](int t) {
    if (asks_rows) {
      const int o = min(32 * place_of(t, ask_j).k + tid % 32, G - 1);
      row_s[t & (kRing - 1)][tid] = (r_page - page_in(o)) * P + o;
    } else if (asks_meta) {
      const Place y = place_of(t, ask_j);
      const int lo = listed && y.k > 0 ? min(max(r_lo, 0), cap) : 0;
      meta_s[t & (kRing - 1)][ask_j] = Meta{r_ob, lo, listed && y.real ? max(min(r_hi, cap) - lo, 0) : 0, 32 * y.k,
                                            y.real ? min(32, G - 32 * y.k) : 0};
    }
  };

  // the first three tiles' at once, a thread a token, and the chains of the next two begun
  if (t0 < t1) {
    for (int i = tid; i < 3 * TT; i += kPreThreads) {
      const int t = t0 + i / TT;
      const Place y = place_of(t, i % TT / 32);
      const int o = min(32 * y.k + i % 32, G - 1), pg = page_in(o);
      row_s[t & (kRing - 1)][i % TT] = (bt[y.g * group_pages + pg] - pg) * P + o;
    }
    if (tid < 3 * NB) {
      const int t = t0 + tid / NB, j = tid % NB;
      const Place y = place_of(t, j);
      const int ob = gt[y.g] * Hkv + h;
      const int32_t* oc = a.p.ocount + (size_t)ob * TQK_NOB;
      const int lo_ = oc[max(y.k - 1, 0)], hi_ = oc[y.k], lo = listed && y.k > 0 ? min(max(lo_, 0), cap) : 0;
      meta_s[t & (kRing - 1)][j] = Meta{ob, lo, listed && y.real ? max(min(hi_, cap) - lo, 0) : 0, 32 * y.k,
                                        y.real ? min(32, G - 32 * y.k) : 0};
    }
    ask_slot(t0 + 3);
    ask(t0 + 3);
    ask_slot(t0 + 4);
  }
  __shared__ float lev1_s[16], cen1_s[16];
  if (tid < 16) lev1_s[tid] = key_level(d.key_grid, tid);
  if (tid >= 64 && tid < 64 + (1 << VB)) cen1_s[tid - 64] = a.p.vcent[tid - 64];
  __syncthreads();

  // ---- a tile's loads: codes, statistics, norms, entries
  const size_t head = (size_t)h * d.n_pages * P;
  const int cq = tid % CQ, tg = tid / CQ, my_blk = tg * TPT / 32;
  // keys: the dword of a row that holds this thread's four channels' codes
  const int krow = D * kb / 8, kbit = 32 * kb * (cq / 8) + 4 * kb * (cq % 8), kbyte = min(kbit / 8, krow - 4), kshift = kbit - 8 * kbyte;
  const int pairs_mask = (1 << (2 * kb)) - 1;
  uint32_t kw[TPT], vw[TILED ? VB : 4], ent = 0;
  f4_t sc, mu;
  float nrm = 0.f;
  constexpr int kEntThreads = kPreThreads / NB;
  auto load = [&](int t) {
    const int* rows = row_s[t & (kRing - 1)];
    const int ob = meta_s[t & (kRing - 1)][my_blk].ob;
    sc = *reinterpret_cast<const f4_t*>(a.p.gscale + (size_t)ob * D + 4 * cq);
    mu = *reinterpret_cast<const f4_t*>(a.p.gmean + (size_t)ob * D + 4 * cq);
#pragma unroll
    for (int i = 0; i < TPT; ++i)
      __builtin_memcpy(&kw[i], a.p.kcodes + (head + rows[tg * TPT + i]) * krow + kbyte, 4);
    if (tid < kVThreads) {
      const int tq = tid / CQ, c4 = cq;  // tokens 4 tq .., channels 4 c4 ..
      if constexpr (TILED) {
        const int tok = 4 * tq;  // unit (lg, c) of a 16-token tile: 4 tokens x 8 channels
        const uint32_t* src = reinterpret_cast<const uint32_t*>(a.p.vcodes + (head + rows[tok & ~15]) * VROW +
                                                                v_unit_offset(tok / 4 % 4, c4 / 2, VROW));
#pragma unroll
        for (int e = 0; e < VB; ++e) vw[e] = src[e];
      } else {
        const int bit = 4 * VB * c4, byte = min(bit / 8, VROW - 4), shift = bit - 8 * byte;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t y;
          __builtin_memcpy(&y, a.p.vcodes + (head + rows[4 * tq + e]) * VROW + byte, 4);
          vw[e] = y >> shift;
        }
      }
    }
    if (tid < TT) nrm = a.p.vnorm[head + rows[tid]];
    const int j = tid / kEntThreads, e = tid % kEntThreads;
    ent = oent[(size_t)meta_s[t & (kRing - 1)][j].ob * cap + min(meta_s[t & (kRing - 1)][j].lo + e, cap - 1)];
  };
  // ---- into LDS
  const int lev_copy = lane % kLevCopies, cen_copy = lane % kCenCopies;
  auto decode = [&](int t) {
    const int buf = t & 1;
#pragma unroll
    for (int i = 0; i < TPT; ++i) {
      const uint32_t w = kw[i] >> kshift;
      const float2 l0 = *reinterpret_cast<const float2*>(lev_s[w & pairs_mask][lev_copy]);
      const float2 l1 = *reinterpret_cast<const float2*>(lev_s[(w >> (2 * kb)) & pairs_mask][lev_copy]);
      const float k[4] = {fmaf(sc[0], l0.x, mu[0]), fmaf(sc[1], l0.y, mu[1]), fmaf(sc[2], l1.x, mu[2]), fmaf(sc[3], l1.y, mu[3])};
      u32x2_t hi, lo;
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        // (towards zero: a key past 65504 leaves the rest to its second half)
        const h2_t y = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(k[e], k[e + 1]));
        hi[e / 2] = __builtin_bit_cast(uint32_t, y);
        lo[e / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float)y.x, -1.f, k[e]), fmaf((float)y.y, -1.f, k[e + 1])));
      }
      const int tok = tg * TPT + i;
      *reinterpret_cast<u32x2_t*>(&k_s[buf][0][tok][4 * cq]) = hi;
      *reinterpret_cast<u32x2_t*>(&k_s[buf][1][tok][4 * cq]) = lo;
    }
    if (tid < kVThreads) {
      const int tq = tid / CQ, c4 = cq;
      if constexpr (TILED) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // channel nt = 4 (c4 % 2) + c of the unit: its token pairs side by side
          u32x2_t y;
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const int b0 = (2 * c + f) * 2 * VB, b1 = (2 * (4 + c) + f) * 2 * VB;  // (even and odd c4)
            auto field = [&](int bit) {
              uint32_t z = vw[bit / 32] >> (bit % 32);
              if (bit % 32 + 2 * VB > 32) z |= vw[bit / 32 + 1] << (32 - bit % 32);
              return z;
            };
            y[f] = cen_s[(c4 & 1 ? field(b1) : field(b0)) & ((1 << (2 * VB)) - 1)][cen_copy];
          }
          *reinterpret_cast<u32x2_t*>(&v_s[buf][4 * c4 + c][4 * tq]) = y;
        }
      } else {
        uint32_t two[4][2];  // [token][channel pair]
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int f = 0; f < 2; ++f) two[e][f] = cen_s[(vw[e] >> (2 * VB * f)) & ((1 << (2 * VB)) - 1)][cen_copy];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t sel = c % 2 ? 0x07060302u : 0x05040100u;
          *reinterpret_cast<u32x2_t*>(&v_s[buf][4 * c4 + c][4 * tq]) =
              u32x2_t{__builtin_amdgcn_perm(two[1][c / 2], two[0][c / 2], sel), __builtin_amdgcn_perm(two[3][c / 2], two[2][c / 2], sel)};
        }
      }
    }
    if (tid < TT) norm_s[buf][tid] = tid % 32 < meta_s[t & (kRing - 1)][tid / 32].cnt ? nrm : 0.f;  // (none: whatever norm stands there)
  };
  // side-list entries over the decoded keys
  auto patch = [&](int t, uint32_t first) {
    const int j = tid / kEntThreads, buf = t & 1;
    const Meta& m = meta_s[t & (kRing - 1)][j];
    for (int e = tid % kEntThreads; e < m.n; e += kEntThreads) {
      const uint32_t y = e < kEntThreads ? first : oent[(size_t)m.ob * cap + min(m.lo + e, cap - 1)];
      const int tok = (int)((y & 0xFFFFu) / D) - m.tok0, ch = (int)(y & (D - 1));
      if ((unsigned)tok < 32u) {
        k_s[buf][0][32 * j + tok][ch] = (uint16_t)(y >> 16);
        k_s[buf][1][32 * j + tok][ch] = 0;
      }
    }
  };

  // ---- this wave's rows: 32 rg + lane % 32
  const int rg = wave & 3, part = wave >> 2;
  const bool works = 32 * rg < n_rows;
  h8_t qf[NK];
  {
    const int r = row0 + min(32 * rg + lc, n_rows - 1);
    const int b = r / per, t = r % per / gq, g = r % gq;
    const uint16_t* const qp = a.q + b * a.q_stride[0] + (h * gq + g) * a.q_stride[1] + t * a.q_stride[2];
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[s] = *reinterpret_cast<const h8_t*>(qp + 16 * s + 8 * hl);
  }
  const float c = d.sm_scale * 1.4426950408889634f;
  float m_run = -INFINITY, l_run = 0.f;
  f16_t O[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) O[i][e] = 0.f;
  auto across = [](float y, bool is_max) {
    const auto z = __builtin_amdgcn_permlane32_swap(fbits(y), fbits(y), false, false);
    return is_max ? fmaxf(bitsf(z[0]), bitsf(z[1])) : bitsf(z[0]) + bitsf(z[1]);
  };
  auto multiply = [&](int t) {
    const int buf = t & 1, blk = kWide ? 0 : part;
    const int cnt = __builtin_amdgcn_readfirstlane(meta_s[t & (kRing - 1)][blk].cnt);
    if (!works || cnt == 0) return;
    // (the pair's halves in sums of their own: two chains of products)
    f16_t S, low;
#pragma unroll
    for (int e = 0; e < 16; ++e) S[e] = low[e] = 0.f;
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      const h8_t hi = *reinterpret_cast<const h8_t*>(&k_s[buf][0][32 * blk + lc][16 * s + 8 * hl]);
      const h8_t lo = *reinterpret_cast<const h8_t*>(&k_s[buf][1][32 * blk + lc][16 * s + 8 * hl]);
      S = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, qf[s], S, 0, 0, 0);
      low = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo, qf[s], low, 0, 0, 0);
    }
    S += low;
    // token of element e: 8 (e / 4) + 4 hl + e % 4
    if (cnt < 32) {
#pragma unroll
      for (int e = 0; e < 16; ++e) S[e] = 8 * (e / 4) + 4 * hl + e % 4 < cnt ? S[e] : -INFINITY;
      asm volatile("");  // (one branch for the sixteen)
    }
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, S[e]);
    mx *= c;
    if (__any(mx > m_run + kFewLazy)) {
      mx = across(mx, true);
      const float m_new = fmaxf(m_run, mx);
      const float f = m_new == -INFINITY ? 1.f : above_zero(__builtin_amdgcn_exp2f(m_run - m_new));
      m_run = m_new;
      l_run *= f;
#pragma unroll
      for (int i = 0; i < NO; ++i) O[i] *= f;
    }
    const float at = m_run == -INFINITY ? 0.f : m_run;
    h8_t ph[2], pl[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f4_t nv = *reinterpret_cast<const f4_t*>(&norm_s[buf][32 * blk + 8 * q + 4 * hl]);
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float w = __builtin_amdgcn_exp2f(fmaf(S[4 * q + e], c, -at));
        l_run += w;
        y[e] = w * nv[e];
      }
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const h2_t z = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(y[e], y[e + 1]));
        const h2_t r = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(fmaf((float)z.x, -1.f, y[e]), fmaf((float)z.y, -1.f, y[e + 1])));
        ph[q / 2][4 * (q % 2) + e] = z.x;
        ph[q / 2][4 * (q % 2) + e + 1] = z.y;
        pl[q / 2][4 * (q % 2) + e] = r.x;
        pl[q / 2][4 * (q % 2) + e + 1] = r.y;
      }
    }
    // V^T P^T, 16 tokens a step: a lane's are 4 hl .. + 3 and 8 + 4 hl .. + 3, as its weights'
#pragma unroll
    for (int i = 0; i < NO; ++i) {
      const int ch = (kWide ? 128 * part : 0) + 32 * i + lc;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        union { h8_t h; u32x2_t u[2]; } y;
        y.u[0] = *reinterpret_cast<const u32x2_t*>(&v_s[buf][ch][32 * blk + 16 * s + 4 * hl]);
        y.u[1] = *reinterpret_cast<const u32x2_t*>(&v_s[buf][ch][32 * blk + 16 * s + 8 + 4 * hl]);
        O[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y.h, pl[s], O[i], 0, 0, 0);
        O[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y.h, ph[s], O[i], 0, 0, 0);
      }
    }
  };

  if (t0 < t1) load(t0);
  // ---- tables: levels of a pair of key codes; a pair of value codes' centroids, scaled
  // so that their fp16 roundings lose least (best of 128 scales)
  float up;
  {
    float cen[1 << VB];
#pragma unroll
    for (int i = 0; i < (1 << VB); ++i) cen[i] = cen1_s[i];
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
    up = __shfl(at, first ? __builtin_ctzll(first) : 0, 64);
    for (int i = tid; i < (1 << (2 * VB)) * kCenCopies; i += kPreThreads) {
      const int e = i / kCenCopies;
      cen_s[e][i % kCenCopies] = pk_f16(cen1_s[e & ((1 << VB) - 1)] * up, cen1_s[e >> VB] * up);
    }
  }
  for (int i = tid; i < (1 << (2 * kb)) * kLevCopies; i += kPreThreads) {
    const int e = i / kLevCopies;
    lev_s[e][i % kLevCopies][0] = lev1_s[k_code_even(e, kb)];
    lev_s[e][i % kLevCopies][1] = lev1_s[k_code_odd(e, kb)];
  }

  __syncthreads();
  if (t0 < t1) {
    decode(t0);
    uint32_t now = ent;
    load(t0 + 1);
    __syncthreads();
    patch(t0, now);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      // (tiles past the split's last are decoded too, of rows that there are, and left)
      // (half of the waves multiply first: a SIMD has one of each at a time)
      if (part != 0) multiply(t);
      decode(t + 1);
      now = ent;
      keep(t + 3);
      load(t + 2);
      ask(t + 4);
      ask_slot(t + 5);
      if (part == 0) multiply(t);
      __syncthreads();
      patch(t + 1, now);
      __syncthreads();
    }
  }

  // ---- the two waves of a row group joined (by tokens), and the sums written by rows
  // through LDS: still centroids' (the join rotates the sum of all splits back)
  float* const o_s = reinterpret_cast<float*>(&k_s[0][0][0][0]);  // [row][D + 4], 64 rows at a time at head_dim 256
  constexpr int OST = D + 4, kPass = kWide ? 64 : kPreRows;
  static_assert(kPass * OST * 4 <= (int)sizeof(k_s), "the accumulators fit");
  float l_all = across(l_run, false);
  auto place = [&](int my, int i, int q) { return &o_s[(my + lc) * OST + (kWide ? 128 * part : 0) + 32 * i + 8 * q + 4 * hl]; };
  if constexpr (!kWide) {
    if (part == 1 && works) {
#pragma unroll
      for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f4_t*>(place(32 * rg, i, q)) = f4_t{O[i][4 * q], O[i][4 * q + 1], O[i][4 * q + 2], O[i][4 * q + 3]};
      if (hl == 0) {
        join_s[rg][0][lc] = m_run;
        join_s[rg][1][lc] = l_all;
      }
    }
    __syncthreads();
    if (part == 0 && works) {
      const float m1 = join_s[rg][0][lc], l1 = join_s[rg][1][lc], M = fmaxf(m_run, m1);
      const float f0 = m_run == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(m_run - M));
      const float f1 = m1 == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(m1 - M));
      m_run = M;
      l_all = l_all * f0 + l1 * f1;
#pragma unroll
      for (int i = 0; i < NO; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f4_t* const at = reinterpret_cast<f4_t*>(place(32 * rg, i, q));
          f4_t y = *at;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = O[i][4 * q + e] * f0 + y[e] * f1;
          *at = y;
        }
    }
  }
  // row r of the workgroup among the partial results
  auto row_at = [&](int r) {
    const int rr = row0 + r, b = rr / per, t = rr % per / gq, hq = h * gq + rr % gq;
    return (a.split0 + split) * a.rows + ((long long)b * Hq + hq) * a.t_len + t;
  };
  if (part == 0 && works && hl == 0 && 32 * rg + lc < n_rows) {
    const long long o = row_at(32 * rg + lc);
    a.part_ml[2 * o] = m_run;
    a.part_ml[2 * o + 1] = l_all;
  }
  const float down = 1.f / up;
#pragma unroll
  for (int first = 0; first < kPreRows; first += kPass) {
    if constexpr (kWide) {
      __syncthreads();
      const int my = 32 * rg - first;
      if (works && my >= 0 && my < kPass) {
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f4_t*>(place(my, i, q)) = f4_t{O[i][4 * q], O[i][4 * q + 1], O[i][4 * q + 2], O[i][4 * q + 3]};
      }
    }
    __syncthreads();
    constexpr int kPieces = D / 4;
    for (int i = tid; i < min(n_rows - first, kPass) * kPieces; i += kPreThreads) {
      const int r = i / kPieces, p = i % kPieces;
      f4_t y = *reinterpret_cast<const f4_t*>(&o_s[r * OST + 4 * p]);
      y *= down;
      *reinterpret_cast<f4_t*>(a.part_acc + row_at(first + r) * D + 4 * p) = y;
    }
  }
}

template <int D, bool TILED>
void launch_prefix(const MoreArgs& a, unsigned groups, hipStream_t st) {
  if (a.d.value_bits == 2)
    hipLaunchKernelGGL((tqk_attend_prefix<D, 2, TILED>), dim3(groups), dim3(kPreThreads), 0, st, a);
  else if (a.d.value_bits == 3)
    hipLaunchKernelGGL((tqk_attend_prefix<D, 3, TILED>), dim3(groups), dim3(kPreThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tqk_attend_prefix<D, 4, TILED>), dim3(groups), dim3(kPreThreads), 0, st, a);
}

}  // namespace

void tqk_launch_prefix(const MoreArgs& a, unsigned groups, hipStream_t st) {
  if (a.d.head_dim == 64)
    launch_prefix<64, false>(a, groups, st);
  else if (a.d.head_dim == 256)
    launch_prefix<256, false>(a, groups, st);
  else if (v_tiled(a.d.group_tokens, a.d.page_tokens, TQK_D, 0))
    launch_prefix<TQK_D, true>(a, groups, st);
  else
    launch_prefix<TQK_D, false>(a, groups, st);
}
