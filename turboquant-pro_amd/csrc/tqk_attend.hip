// Attention of one or more new queries a sequence over the two-tier cache, with
// a sliding window and first tokens that stay visible (gfx950).
//
// Few queries: tqk_attend_codes reads the codes of the tokens that they see and
// nothing else.  Many queries (fp16 caches): what they see is reconstructed as
// dense keys (fp16 pairs) and fp16 values in the workspace, a GiB at a time, and the
// kernels of tqk_attention run over it.  fp32 caches: every query is an item of its own of
// the VALU decode (WIN instances of tqk_decode_kernels.h).
#include "tqk_attend.h"
#include "tqk_attn.h"
#include "tqk_decode_kernels.h"

namespace {

constexpr int kMostItems = 4096;  // fp32 caches: queries a launch (bounds the partials and the grid)
// Rows (queries times query heads of a kv head) attended on codes.  A workgroup of
// that kernel takes 16 rows and reads the codes again for the next 16; dense keys
// and values are made once, however few the queries.  8 sequences of 8192 tokens, 8
// kv heads of 128, window 4096, codes and dense: 32 rows 38 and 105 us, 64 rows 52
// and 108, 128 rows 100 and 117; one sequence of 16384: 128 rows 29 and 53; head_dim
// 256, 4 sequences: 128 rows 121 and 148, 64: 256 rows 46 and 48.
constexpr int kFewMost = 128;
// Bytes of keys and values reconstructed at a time: sequences, or kv heads of one,
// go one slice after another through the same workspace.  A slice of this size alone
// fills the chip (1 GiB is 170 us of writes), and a workspace of every sequence would
// be six times the codes' own size.  Where one kv head of one sequence needs more
// (1.4 million tokens at head_dim 128), the codes are attended, however many rows.
constexpr size_t kMostDense = (size_t)1 << 30;

// Coded groups that one query sees at most, past `max_len` tokens of cache: the
// first tokens', and the window's less what the hot window holds of it.  A cache
// with coded groups has at least W + 1 - G uncoded tokens; the first of T
// queries stands T - 1 before the last.
int most_groups(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  const int G = d->group_tokens, all = n_groups_of(t->max_len, d->hot_window, G);
  if (t->window == 0 || t->window >= t->max_len) return all;
  const long long hot = (long long)d->hot_window + 2 - G - t->q_len;
  const long long cold = (long long)t->window - (hot > 0 ? hot : 0);
  long long n = ((long long)t->sinks + G - 1) / G + (cold > 0 ? (cold + G - 2) / G + 1 : 0);
  return n < all ? (int)n : all;
}

// ---- reconstruction of what a chunk's queries see ---------------------------
// Rows [0, kept.sinks) and from the window on, moved down by kept.gap
// (tqk_attn.h), 64 tokens of a kv head a step: keys as grid value with the
// side-list's over it, an fp16 pair (a single fp16 moves a score of 60 by 0.01: the
// result was three times as far off, and a chunk a fifth faster), values as
// (cent[code] @ Pi) * norm and hot tokens as they are, in fp16 (half a step of a value
// in the result, as its own rounding; a pair would be a third product of tiles).
// PolarQuant keys are rotated as the values, and pairs (single: 141 us of 184 at
// head_dim 128, 378 of 432 at 256, and infinities past 65504); their centroids'
// roundings stay, and at 256 Pi's: up to 1.7e-3 of the result where a score of 60
// decides.  Pi is an fp16 pair up to head_dim 128 (fp16 at 256) and the centroids are
// scaled against their roundings, summed in fp32 by the matrix cores: the rotation
// costs a wave 32 products a step where the ordered sums of tqk_dequant_dense took 2 D
// VALU operations a value.
// Bound: the chain of a step's loads and barriers, and each workgroup's set-up (64 KiB
// of Pi split into pairs, the codebook's scale), beside the rows' writes (6 D bytes a
// token and kv head): two windows of 4096 and 8 kv heads of 128, a step a workgroup,
// 40 us of a chunk's 184 (1.4 TB/s); two whole caches of 16384, 100 to 114 us (2).
constexpr int kGather = 64;  // tokens a step
static_assert(kGather == kMaxKeys, "a step lies on one side of the gap");

struct GatherArgs {
  tqk_cache_desc d;
  tqk_cache_ptrs p;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  uint16_t* k;
  uint16_t* k_lo;  // what the keys' rounding left
  uint16_t* v;
  int q_len, max_len, window, sinks;
  int rows;   // rows of a sequence and kv head
  int steps;  // of kGather rows
  int units;  // seqs * heads * steps
  int b0, h0, heads;  // the slice's first sequence and kv head, and its kv heads
};

template <int VB, int D>
__global__ __launch_bounds__(kThreads) void tqk_gather_seen(GatherArgs a) {
  constexpr int CH = D / 8;                    // 8-channel pieces of a row
  constexpr int NT = D / 64, NK = D / 32;      // a wave's column tiles, steps of a product
  constexpr int VROW = D * VB / 8;
  const tqk_cache_desc& d = a.d;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, ln = lane & 15, lg = lane >> 4;
  const int G = d.group_tokens, P = d.page_tokens, Hkv = d.n_kv_heads, kb = d.key_bits;
  const bool polar = d.key_grid == 2;
  __shared__ __align__(16) uint16_t k_s[kGather][D], kl_s[kGather][D];
  __shared__ __align__(16) uint16_t c_s[kGather * D];  // centroids, then rotated values
  __shared__ int row_s[kGather];   // row in the head's pages; -1: a hot token
  __shared__ int slot_s[kGather];
  __shared__ float norm_s[2][kGather];  // value norms, key norms (PolarQuant keys)
  __shared__ float lev_s[16], cen_s[16];
  if (tid < 16) lev_s[tid] = key_level(d.key_grid == 1, tid);
  // centroids near 1, at the scale of 64 over a power of two whose fp16 roundings
  // lose least (the first of equals): 2^-12 of a centroid becomes about 2^-14
  float up;
  {
    const float g = (D == 64 ? 8.f : 16.f) * (1.0f + (float)lane * (1.0f / 64));
    float err = 0.f;
#pragma unroll
    for (int i = 0; i < (1 << VB); ++i) {
      const float y = a.p.vcent[i] * g, r = y - (float)(_Float16)y;
      err = fmaf(r, r, err);
    }
    err *= __builtin_amdgcn_rcpf(g * g);
    const float best = -wave_reduce<true>(-err);
    const uint64_t first = __builtin_amdgcn_ballot_w64(err == best);
    up = (D == 64 ? 8.f : 16.f) * (1.0f + (float)(first ? __builtin_ctzll(first) : 0) * (1.0f / 64));
  }
  const float down = 1.f / up;
  if (tid < (1 << VB)) cen_s[tid] = a.p.vcent[tid] * up;
  // Pi, up to head_dim 128 as fp16 pairs (there are no registers for more): columns e = 16 (NT wave + nt) + ln, rows 32 ks + 8 lg .. + 7 (a row of Pi^T)
  constexpr bool kPairs = D <= 128;
  h8_t pf[NT][NK], pl[kPairs ? NT : 1][kPairs ? NK : 1];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      const float* r = a.p.pi_t + (size_t)(16 * (NT * wave + nt) + ln) * D + 32 * ks + 8 * lg;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pf[nt][ks][e] = (_Float16)r[e];
        if constexpr (kPairs) pl[nt][ks][e] = (_Float16)(r[e] - (float)pf[nt][ks][e]);
      }
    }
  // place of a row's 16-byte piece: turned by the row, against bank conflicts
  auto at = [](int t, int c) { return (t * CH + (c ^ (t & 7))) * 8; };

  for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
    const int step = unit % a.steps, bh = unit / a.steps, h = a.h0 + bh % a.heads, b = a.b0 + bh / a.heads;
    const int n = min(a.seq_lens[b], a.max_len);
    const int m = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
    const KeptRows kept(n, m, 0, min(a.sinks, n), a.window);
    const int r0 = step * kGather, t0 = r0 < kept.sinks ? r0 : r0 + kept.gap;
    const int nt_ = min(kGather, n - t0);  // tokens of this step
    if (nt_ <= 0) continue;                // (the same for every thread)
    const int ng = n_groups_of(n, d.hot_window, G);
    const size_t head = (size_t)h * d.n_pages * P;
    const size_t ring = ((size_t)b * Hkv + h) * d.hot_ring;
    __syncthreads();  // the last step's LDS is read
    if (tid < kGather) {
      const int t = t0 + min(tid, nt_ - 1);
      const bool cold = t < ng * G;
      row_s[tid] = -1;
      if (cold) {
        const int row = a.p.block_table[(size_t)b * d.max_pages_per_seq + t / P] * P + t % P;
        row_s[tid] = row;
        slot_s[tid] = a.p.group_table[(size_t)b * d.max_groups_per_seq + t / G];
        norm_s[0][tid] = a.p.vnorm[head + row] * down;
        norm_s[1][tid] = polar ? a.p.knorm[head + row] * down : 0.f;
      }
    }
    __syncthreads();
    uint16_t* const ko = a.k + ((size_t)bh * a.rows + r0) * D;
    uint16_t* const klo = a.k_lo + ((size_t)bh * a.rows + r0) * D;
    uint16_t* const vo = a.v + ((size_t)bh * a.rows + r0) * D;

    // eight codes of a row from channel 8 c on, 4-bit keys' nibbles in order
    auto codes8 = [&](const uint8_t* row, int bits, int c, bool key) -> uint32_t {
      const uint8_t* s = row + c * bits;
      uint32_t w = 0;
      if (bits == 4) {
        w = *reinterpret_cast<const uint32_t*>(s);
        if (key) w = __builtin_bswap32(__builtin_bitreverse32(w));
      } else {
        for (int i = 0; i < bits; ++i) w |= (uint32_t)s[i] << (8 * i);
      }
      return w;
    };
    auto put_centroids = [&](const uint8_t* rows, int bits, int row_bytes, bool key) {
      for (int i = tid; i < nt_ * CH; i += kThreads) {
        const int t = i / CH, c = i % CH;
        if (row_s[t] < 0) continue;
        const uint32_t w = codes8(rows + (head + row_s[t]) * row_bytes, bits, c, key);
        h8_t x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (_Float16)cen_s[(w >> (VB * e)) & ((1 << VB) - 1)];
        *reinterpret_cast<h8_t*>(c_s + at(t, c)) = x;
      }
    };
    // c_s @ Pi times the norms, back into c_s, then out (hot rows from the ring);
    // keys as pairs, the second halves by way of kl_s
    uint16_t* const cl_s = &kl_s[0][0];
    auto rotate_out = [&](auto pair, uint16_t* out, uint16_t* out_lo, const float* norm, const uint16_t* hot) {
      constexpr bool kPair = decltype(pair)::value;
      __syncthreads();
      f4_t acc[NT][4];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][tt] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
          const h8_t x = *reinterpret_cast<const h8_t*>(c_s + at(16 * tt + ln, 4 * ks + lg));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {  // transposed: a lane gets four channels of one token
            if constexpr (kPairs)
              acc[nt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[nt][ks], x, acc[nt][tt], 0, 0, 0);
            acc[nt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf[nt][ks], x, acc[nt][tt], 0, 0, 0);
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const float f = norm[16 * tt + ln];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
          h4_t y, z;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = acc[nt][tt][e] * f;
            y[e] = (_Float16)(kPair ? fminf(fmaxf(x, -65504.f), 65504.f) : x);
            z[e] = (_Float16)(x - (float)y[e]);
          }
          const int ch = 16 * (NT * wave + nt) + 4 * lg;
          *reinterpret_cast<h4_t*>(c_s + at(16 * tt + ln, ch / 8) + ch % 8) = y;
          if constexpr (kPair) *reinterpret_cast<h4_t*>(cl_s + at(16 * tt + ln, ch / 8) + ch % 8) = z;
        }
      }
      __syncthreads();
      for (int i = tid; i < nt_ * CH; i += kThreads) {
        const int t = i / CH, c = i % CH;
        const uint4* src = row_s[t] < 0 ? reinterpret_cast<const uint4*>(hot + (ring + (t0 + t) % d.hot_ring) * D + 8 * c)
                                        : reinterpret_cast<const uint4*>(c_s + at(t, c));
        *reinterpret_cast<uint4*>(out + (size_t)t * D + 8 * c) = *src;
        if constexpr (kPair)
          *reinterpret_cast<uint4*>(out_lo + (size_t)t * D + 8 * c) =
              row_s[t] < 0 ? make_uint4(0u, 0u, 0u, 0u) : *reinterpret_cast<const uint4*>(cl_s + at(t, c));
      }
    };

    const uint16_t* const hot_k = static_cast<const uint16_t*>(a.p.hot_k);
    if (polar) {
      put_centroids(a.p.kcodes, VB, k_row_bytes(VB, D), true);
      rotate_out(std::true_type{}, ko, klo, norm_s[1], hot_k);
      __syncthreads();
    } else {
      for (int i = tid; i < nt_ * CH; i += kThreads) {
        const int t = i / CH, c = i % CH;
        if (row_s[t] < 0) {
          *reinterpret_cast<uint4*>(&k_s[t][8 * c]) =
              *reinterpret_cast<const uint4*>(hot_k + (ring + (t0 + t) % d.hot_ring) * D + 8 * c);
          *reinterpret_cast<uint4*>(&kl_s[t][8 * c]) = make_uint4(0u, 0u, 0u, 0u);
          continue;
        }
        const uint32_t w = codes8(a.p.kcodes + (head + row_s[t]) * k_row_bytes(kb, D), kb, c, true);
        const size_t mb = ((size_t)slot_s[t] * Hkv + h) * D + 8 * c;
        h8_t x, y;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 sc = *reinterpret_cast<const float4*>(a.p.gscale + mb + e);
          const float4 mu = *reinterpret_cast<const float4*>(a.p.gmean + mb + e);
          const float scv[4] = {sc.x, sc.y, sc.z, sc.w}, muv[4] = {mu.x, mu.y, mu.z, mu.w};
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const float k = fmaf(scv[f], lev_s[(w >> (kb * (e + f))) & ((1u << kb) - 1u)], muv[f]);
            // (a code near 65504 may stand for more: the rest goes into the second half,
            // and so does an infinity or a NaN)
            x[e + f] = (_Float16)fminf(fmaxf(k, -65504.f), 65504.f);
            y[e + f] = (_Float16)(k - (float)x[e + f]);
          }
        }
        *reinterpret_cast<h8_t*>(&k_s[t][8 * c]) = x;
        *reinterpret_cast<h8_t*>(&kl_s[t][8 * c]) = y;
      }
    }
    if (D == TQK_D && v_tiled(G, P, D, 0)) {
      // unit (lg, c) of a 16-token tile: tokens 4 lg .. + 3 x channels 8 c .. + 7
      const int tile = tid >> 6, ul = (tid >> 4) & 3, uc = tid & 15;
      if (16 * tile < nt_ && row_s[16 * tile] >= 0) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(a.p.vcodes + (head + row_s[16 * tile]) * VROW +
                                                                v_unit_offset(ul, uc, VROW));
        uint32_t w[VB];
#pragma unroll
        for (int i = 0; i < VB; ++i) w[i] = src[i];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          h8_t x;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = (_Float16)cen_s[stream_code<VB>(w, 4 * e + t)];
          *reinterpret_cast<h8_t*>(c_s + at(16 * tile + 4 * ul + t, uc)) = x;
        }
      }
    } else {
      put_centroids(a.p.vcodes, VB, VROW, false);
    }
    if (!polar) {
      __syncthreads();
      if (d.outliers_per_channel > 0) {
        // the side-list entries of the step's tokens, group by group
        const int end = min(t0 + nt_, ng * G);
        for (int g = t0 / G; g * G < end; ++g) {
          const int lo_t = max(t0, g * G), hi_t = min(end, (g + 1) * G);
          const size_t ob = (size_t)slot_s[lo_t - t0] * Hkv + h;
          const int32_t* oc = a.p.ocount + ob * TQK_NOB;
          const int q = (lo_t - g * G) / TQK_OBLK;
          const int lo = min(q > 0 ? oc[q - 1] : 0, d.outlier_cap);
          const int hi = min(oc[(hi_t - 1 - g * G) / TQK_OBLK], d.outlier_cap);
          for (int e = lo + tid; e < hi; e += kThreads) {
            const uint32_t ent = a.p.oent[ob * d.outlier_cap + e], pos = ent & 0xFFFFu;
            const int t = g * G + (int)(pos / D);
            if (t >= lo_t && t < hi_t) {
              k_s[t - t0][pos % D] = (uint16_t)(ent >> 16);
              kl_s[t - t0][pos % D] = 0;
            }
          }
        }
        __syncthreads();
      }
      for (int i = tid; i < nt_ * CH; i += kThreads) {
        reinterpret_cast<uint4*>(ko)[i] = reinterpret_cast<const uint4*>(&k_s[0][0])[i];
        reinterpret_cast<uint4*>(klo)[i] = reinterpret_cast<const uint4*>(&kl_s[0][0])[i];
      }
    }
    rotate_out(std::false_type{}, vo, nullptr, norm_s[0], static_cast<const uint16_t*>(a.p.hot_v));
  }
}

template <int D>
void launch_gather(const GatherArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.units < 2048 ? a.units : 2048));
  if (a.d.value_bits == 2)
    hipLaunchKernelGGL((tqk_gather_seen<2, D>), grid, dim3(kThreads), 0, st, a);
  else if (a.d.value_bits == 3)
    hipLaunchKernelGGL((tqk_gather_seen<3, D>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tqk_gather_seen<4, D>), grid, dim3(kThreads), 0, st, a);
}

struct AttendPlan {
  Plan pl;
  int items;  // queries a launch
  size_t ws_bytes;
};

// The VALU decode's plan (fp32 caches).
AttendPlan attend_plan(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  AttendPlan ap{};
  const long long items = (long long)t->batch * t->q_len;
  ap.items = (int)(items < kMostItems ? items : kMostItems);
  ap.pl = plan_groups(d, ap.items, most_groups(d, t), t->max_len < d->hot_window ? t->max_len : d->hot_window);
  const size_t ns = (size_t)(ap.pl.n_cold_splits + ap.pl.n_hot_splits);
  ap.ws_bytes = (size_t)ap.items * d->n_q_heads * ns * sizeof(float) * (2 + d->head_dim) + 256;
  return ap;
}

// Rows that a sequence's queries see at most, in whole tiles.
int kept_rows(const tqk_attend_desc* t) {
  const long long tile = kMaxKeys, all = ((long long)t->max_len + tile - 1) / tile * tile;
  if (t->window == 0 || t->window >= t->max_len) return (int)all;
  const long long sinks = t->sinks < t->max_len ? t->sinks : t->max_len;
  const long long rows = (sinks + tile - 1) / tile * tile + ((long long)t->window + t->q_len + tile - 2) / tile * tile + tile;
  return (int)(rows < all ? rows : all);
}

// Bytes of the reconstructed keys (pairs) and values of a sequence and kv head.
size_t dense_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t) { return (size_t)6 * kept_rows(t) * d->head_dim; }

// Whether the queries go over reconstructed keys and values.
bool dense_path(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  return !d->input_f32 && t->out_type == 1 && (long long)t->q_len * (d->n_q_heads / d->n_kv_heads) > kFewMost &&
         dense_bytes(d, t) <= kMostDense;
}

// Sequences and kv heads reconstructed at a time: as many sequences as fit, or of
// one sequence as many kv heads, in slices of about one size.
struct Slice {
  int seqs, heads;
  Slice(const tqk_cache_desc* d, const tqk_attend_desc* t) {
    auto even = [](int n, size_t most) {
      if (most >= (size_t)n) return n;
      const int count = (n + (int)most - 1) / (int)most;
      return (n + count - 1) / count;
    };
    const size_t one = dense_bytes(d, t), fit = one ? kMostDense / one : (size_t)INT32_MAX;
    heads = even(d->n_kv_heads, fit);
    seqs = heads < d->n_kv_heads ? 1 : even(t->batch, fit / d->n_kv_heads);
  }
};

// Attention over the reconstruction of some sequences' kv heads.
tqk_attn_desc dense_desc(const tqk_cache_desc* d, const tqk_attend_desc* t, int seqs, int heads) {
  tqk_attn_desc a{};
  a.batch = seqs;
  a.n_q_heads = heads * (d->n_q_heads / d->n_kv_heads);
  a.n_kv_heads = heads;
  a.head_dim = d->head_dim;
  a.q_len = t->q_len;
  a.kv_len = t->max_len;
  a.window = t->window;
  a.sinks = t->sinks;
  a.type = 1;
  a.sm_scale = d->sm_scale;
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = t->q_stride[i];
    a.o_stride[i] = t->o_stride[i];
  }
  const int64_t row = d->head_dim, head = row * kept_rows(t);
  a.k_stride[0] = a.v_stride[0] = head * heads;
  a.k_stride[1] = a.v_stride[1] = head;
  a.k_stride[2] = a.v_stride[2] = row;
  return a;
}

// Workspace of the attention over a slice, the last ones (which are smaller) too.
size_t slice_attention_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t, const Slice& sl) {
  size_t most = 0;
  for (int seqs : {sl.seqs, t->batch % sl.seqs})
    for (int heads : {sl.heads, d->n_kv_heads % sl.heads}) {
      const tqk_attn_desc a = dense_desc(d, t, seqs, heads);
      const size_t need = seqs && heads ? tqk_attention_workspace_bytes(&a) : 0;
      if (need > most) most = need;
    }
  return most;
}

int check_attend(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  const int rc = tqk_check_desc(d);
  if (rc != TQK_OK) return rc;
  if (!t || t->batch < 0 || t->q_len < 0 || t->max_len < 0 || t->window < 0 || t->sinks < 0) return TQK_EINVAL;
  if (t->out_type != 0 && t->out_type != 1) return TQK_EUNSUPPORTED;
  if (t->q_len > (1 << 28) || t->max_len > (1 << 30) || t->batch > counter_seqs(*d)) return TQK_EINVAL;
  if ((long long)t->batch * t->q_len > (1LL << 30)) return TQK_EINVAL;
  if (!(d->sm_scale > 0.f)) return TQK_EINVAL;
  // (the fp16 caches' kernels hold a head's rows in 32 bits)
  if (!d->input_f32 && (long long)d->n_pages * d->page_tokens > INT32_MAX) return TQK_EUNSUPPORTED;
  // (a side-list without room for one entry: its loads have no place to go)
  if (d->outliers_per_channel > 0 && d->outlier_cap < 1) return TQK_EINVAL;
  // (the tables reach as far as the longest sequence may)
  const int groups = n_groups_of(t->max_len, d->hot_window, d->group_tokens);
  if (groups > d->max_groups_per_seq || (long long)groups * (d->group_tokens / d->page_tokens) > d->max_pages_per_seq)
    return TQK_EINVAL;
  for (int i = 0; i < 3; ++i)
    if (t->q_stride[i] % 8 || t->o_stride[i] % 8) return TQK_EINVAL;
  return TQK_OK;
}

// Every buffer that a cache of this form has.
bool have_buffers(const tqk_cache_desc& d, const tqk_cache_ptrs& p) {
  const bool keys = d.key_grid == 2 ? p.knorm != nullptr : p.gscale && p.gmean;
  return keys && p.kcodes && p.vcodes && p.vnorm && p.ocount && (d.outliers_per_channel == 0 || p.oent) && p.hot_k &&
         p.hot_v && p.block_table && p.group_table && p.vcent && p.pi && p.pi_t;
}

template <int GQ, int D>
void launch_valu(const SplitArgs<true>& a, dim3 grid, hipStream_t st) {
  if (a.d.value_bits == 2)
    hipLaunchKernelGGL((tqk_decode_split_valu<GQ, 2, D, true>), grid, dim3(kThreads), 0, st, a);
  else if (a.d.value_bits == 3)
    hipLaunchKernelGGL((tqk_decode_split_valu<GQ, 3, D, true>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tqk_decode_split_valu<GQ, 4, D, true>), grid, dim3(kThreads), 0, st, a);
}

template <int GQ>
void launch_split(const SplitArgs<true>& a, dim3 grid, hipStream_t st) {
  if (a.d.head_dim == 64)
    launch_valu<GQ, 64>(a, grid, st);
  else if (a.d.head_dim == 128)
    launch_valu<GQ, 128>(a, grid, st);
  else
    launch_valu<GQ, 256>(a, grid, st);
}

template <int D>
void launch_join(const JoinArgs<true>& m, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((tqk_merge<D, true>), grid, dim3(2 * D), 0, st, m);
}

}  // namespace

extern "C" {

size_t tqk_attend_workspace_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  if (check_attend(d, t) != TQK_OK) return 0;
  if (!t->batch || !t->q_len) return 0;
  if (dense_path(d, t)) {
    const Slice sl(d, t);
    return (size_t)sl.seqs * sl.heads * dense_bytes(d, t) + ((slice_attention_bytes(d, t, sl) + 255) & ~(size_t)255);
  }
  if (!d->input_f32) return tqk_few_workspace_bytes(d, t);
  return attend_plan(d, t).ws_bytes;
}

int tqk_attend(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
               const int32_t* seq_lens, const int32_t* q_lens, void* out, void* workspace,
               size_t workspace_bytes, void* stream) {
  const int rc = check_attend(d, t);
  if (rc != TQK_OK) return rc;
  if (!t->batch || !t->q_len) return TQK_OK;
  if (!p || !q || !seq_lens || !out || (((uintptr_t)q | (uintptr_t)out) & 15) || !have_buffers(*d, *p)) return TQK_EINVAL;
  if (!workspace || ((uintptr_t)workspace & 15)) return TQK_EWORKSPACE;
  const bool dense = dense_path(d, t);
  if (!dense && !d->input_f32) return tqk_run_few(d, p, t, q, seq_lens, q_lens, out, workspace, workspace_bytes, stream);
  if (workspace_bytes < tqk_attend_workspace_bytes(d, t)) return TQK_EWORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dense) {
    const Slice sl(d, t);
    const int gq = d->n_q_heads / d->n_kv_heads;
    const size_t attn_bytes = slice_attention_bytes(d, t, sl);
    GatherArgs g{};
    g.d = *d;
    g.p = *p;
    g.seq_lens = seq_lens;
    g.q_lens = q_lens;
    g.k = static_cast<uint16_t*>(workspace);
    g.q_len = t->q_len;
    g.max_len = t->max_len;
    g.window = t->window;
    g.sinks = t->sinks;
    g.rows = kept_rows(t);
    g.steps = g.rows / kGather;
    for (g.b0 = 0; g.b0 < t->batch; g.b0 += sl.seqs)
      for (g.h0 = 0; g.h0 < d->n_kv_heads; g.h0 += sl.heads) {
        const int seqs = t->batch - g.b0 < sl.seqs ? t->batch - g.b0 : sl.seqs;
        g.heads = d->n_kv_heads - g.h0 < sl.heads ? d->n_kv_heads - g.h0 : sl.heads;
        const tqk_attn_desc a = dense_desc(d, t, seqs, g.heads);
        const size_t rows = (size_t)seqs * a.k_stride[0];
        g.k_lo = g.k + rows;
        g.v = g.k_lo + rows;
        if (t->max_len > 0) {
          g.units = seqs * g.heads * g.steps;
          if (d->head_dim == 64)
            launch_gather<64>(g, st);
          else if (d->head_dim == 128)
            launch_gather<128>(g, st);
          else
            launch_gather<256>(g, st);
          if (hipGetLastError() != hipSuccess) return TQK_EHIP;
        }
        const long long at_q = g.b0 * t->q_stride[0] + (long long)g.h0 * gq * t->q_stride[1];
        const long long at_o = g.b0 * t->o_stride[0] + (long long)g.h0 * gq * t->o_stride[1];
        const int arc = tqk_run_attention(&a, static_cast<const uint16_t*>(q) + at_q, g.k, g.v, seq_lens + g.b0,
                                          q_lens ? q_lens + g.b0 : nullptr, nullptr, static_cast<uint16_t*>(out) + at_o,
                                          g.v + rows, attn_bytes, 1, g.k_lo, stream);
        if (arc != TQK_OK) return arc;
      }
    return TQK_OK;
  }
  const AttendPlan ap = attend_plan(d, t);
  const Plan& pl = ap.pl;
  const int gq = d->n_q_heads / d->n_kv_heads;
  const int n_splits = pl.n_cold_splits + pl.n_hot_splits;
  SplitArgs<true> a{};
  a.d = *d;
  a.p = *p;
  a.q = q;
  a.seq_lens = seq_lens;
  const size_t per = (size_t)ap.items * d->n_q_heads * n_splits;
  a.pm = static_cast<float*>(workspace);
  a.pl = a.pm + per;
  a.pacc = a.pl + per;
  a.n_cold_splits = pl.n_cold_splits;
  a.n_hot_splits = pl.n_hot_splits;
  a.groups_per_split = pl.groups_per_split;
  a.hot_per_split = pl.hot_per_split;
  a.batch = t->batch;
  a.w.q_lens = q_lens;
  a.w.q_len = t->q_len;
  a.w.max_len = t->max_len;
  a.w.window = t->window >= t->max_len ? 0 : t->window;
  a.w.sinks = t->sinks < t->max_len ? t->sinks : t->max_len;
  a.w.out_type = t->out_type;
  for (int i = 0; i < 3; ++i) {
    a.w.q_stride[i] = t->q_stride[i];
    a.w.o_stride[i] = t->o_stride[i];
  }
  const long long items = (long long)t->batch * t->q_len;
  for (long long i0 = 0; i0 < items; i0 += ap.items) {
    const int n = (int)(items - i0 < ap.items ? items - i0 : ap.items);
    a.w.item0 = (int)i0;
    const dim3 grid(n_splits, d->n_kv_heads, n);
    switch (gq) {
      case 1: launch_split<1>(a, grid, st); break;
      case 2: launch_split<2>(a, grid, st); break;
      case 3: case 4: launch_split<4>(a, grid, st); break;
      default: launch_split<8>(a, grid, st); break;
    }
    if (hipGetLastError() != hipSuccess) return TQK_EHIP;
    JoinArgs<true> m{};
    m.pm = a.pm;
    m.pl = a.pl;
    m.pacc = a.pacc;
    m.pi = p->pi;
    m.n_cold_splits = pl.n_cold_splits;
    m.n_splits = n_splits;
    m.n_q_heads = d->n_q_heads;
    m.n_kv_heads = d->n_kv_heads;
    m.out = static_cast<float*>(out);
    m.w = a.w;
    m.seq_lens = seq_lens;
    const dim3 jg(d->n_kv_heads, n);
    if (d->head_dim == 64)
      launch_join<64>(m, jg, st);
    else if (d->head_dim == 128)
      launch_join<128>(m, jg, st);
    else
      launch_join<256>(m, jg, st);
    if (hipGetLastError() != hipSuccess) return TQK_EHIP;
  }
  return TQK_OK;
}

}  // extern "C"
