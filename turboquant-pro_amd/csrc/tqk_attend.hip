// Attention of one or more new queries a sequence over the two-tier cache, with
// a sliding window and first tokens that stay visible (gfx950).
//
// Few queries: every query is an item of its own of the decode kernels (WIN
// instances of tqk_decode_kernels.h), which read the codes of the groups that
// it sees and nothing else.  Many queries (fp16 caches): the visible groups are
// reconstructed once as dense fp16 keys and values in the workspace, and
// tqk_attention runs over them.
#include "tqk_decode_kernels.h"

namespace {

constexpr int kMostItems = 4096;  // queries a launch (bounds the partials and the grid)

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

struct AttendPlan {
  Plan pl;
  int items;  // queries a launch
  size_t ws_bytes;
};

AttendPlan attend_plan(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  AttendPlan ap{};
  const long long items = (long long)t->batch * t->q_len;
  ap.items = (int)(items < kMostItems ? items : kMostItems);
  const int n = most_groups(d, t);
  ap.pl = plan_groups(d, ap.items, n, t->max_len < d->hot_window ? t->max_len : d->hot_window);
  if (mfma_path(*d) && n > 0) {
    // A window's few groups in equal shares of blocks: s splits of g groups, each
    // wave an eighth of a split's blocks (wave_blocks), by the same cost in
    // groups per wave as plan_groups, with the mid-group starts on top.
    const int nblk = d->group_tokens / 32, ncu = device_cus();
    const long long pairs = (long long)ap.items * d->n_kv_heads;
    double best = 1e30;
    for (int s = 1; s <= n; ++s) {
      int g = (n + s - 1) / s;
      while ((g * nblk) % kMWaves) ++g;
      if (g > kMaxGPS) continue;
      const long long rounds = (pairs * ((n + g - 1) / g) + ncu - 1) / ncu;
      const double cost = (double)rounds * ((double)g / kMWaves + 0.45);
      if (cost < best - 1e-9) {
        best = cost;
        ap.pl.groups_per_split = g;
        ap.pl.wave_blocks = g * nblk / kMWaves;
        ap.pl.n_cold_splits = ap.pl.n_hot_splits = (n + g - 1) / g;
      }
    }
  }
  const size_t ns = (size_t)(ap.pl.n_cold_splits + ap.pl.n_hot_splits);
  ap.ws_bytes = (size_t)ap.items * d->n_q_heads * ns * sizeof(float) * (2 + d->head_dim) + 256;
  return ap;
}

// Whether the queries go over reconstructed keys and values.
bool dense_path(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  return !d->input_f32 && t->out_type == 1 && t->q_len > 8;
}

tqk_attn_desc dense_desc(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  tqk_attn_desc a{};
  a.batch = t->batch;
  a.n_q_heads = d->n_q_heads;
  a.n_kv_heads = d->n_kv_heads;
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
  const int64_t row = d->head_dim, head = row * t->max_len;
  a.k_stride[0] = a.v_stride[0] = head * d->n_kv_heads;
  a.k_stride[1] = a.v_stride[1] = head;
  a.k_stride[2] = a.v_stride[2] = row;
  return a;
}

int check_attend(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  const int rc = tqk_check_desc(d);
  if (rc != TQK_OK) return rc;
  if (!t || t->batch < 0 || t->q_len < 0 || t->max_len < 0 || t->window < 0 || t->sinks < 0) return TQK_EINVAL;
  if (t->out_type != 0 && t->out_type != 1) return TQK_EUNSUPPORTED;
  if (t->q_len > (1 << 28) || t->max_len > (1 << 30) || t->batch > counter_seqs(*d)) return TQK_EINVAL;
  if ((long long)t->batch * t->q_len > (1LL << 30)) return TQK_EINVAL;
  if (!(d->sm_scale > 0.f)) return TQK_EINVAL;
  return TQK_OK;
}

template <int GQ, int KB>
void launch_mfma_kb(const SplitArgs<true>& a, dim3 g1, hipStream_t st) {
  if (a.d.key_grid == 2)  // PolarQuant keys: value_bits == key_bits
    hipLaunchKernelGGL((tqk_decode_split_mfma<GQ, KB, KB, true, true>), g1, dim3(kMThreads), 0, st, a);
  else if (a.d.value_bits == 2)
    hipLaunchKernelGGL((tqk_decode_split_mfma<GQ, 2, KB, false, true>), g1, dim3(kMThreads), 0, st, a);
  else if (a.d.value_bits == 3)
    hipLaunchKernelGGL((tqk_decode_split_mfma<GQ, 3, KB, false, true>), g1, dim3(kMThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tqk_decode_split_mfma<GQ, 4, KB, false, true>), g1, dim3(kMThreads), 0, st, a);
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
  if (mfma_path(a.d)) {
    const dim3 g1(grid.x * grid.y * grid.z);  // over (split, kv head, item)
    if (a.d.key_bits == 4)
      launch_mfma_kb<GQ, 4>(a, g1, st);
    else if (a.d.key_bits == 3)
      launch_mfma_kb<GQ, 3>(a, g1, st);
    else
      launch_mfma_kb<GQ, 2>(a, g1, st);
  } else if (a.d.head_dim == 64) {
    launch_valu<GQ, 64>(a, grid, st);
  } else if (a.d.head_dim == 128) {
    launch_valu<GQ, 128>(a, grid, st);
  } else {
    launch_valu<GQ, 256>(a, grid, st);
  }
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
    const tqk_attn_desc a = dense_desc(d, t);
    return 4 * (size_t)t->batch * a.k_stride[0] + ((tqk_attention_workspace_bytes(&a) + 255) & ~(size_t)255);
  }
  return attend_plan(d, t).ws_bytes;
}

int tqk_attend(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
               const int32_t* seq_lens, const int32_t* q_lens, void* out, void* workspace,
               size_t workspace_bytes, void* stream) {
  const int rc = check_attend(d, t);
  if (rc != TQK_OK) return rc;
  if (!t->batch || !t->q_len) return TQK_OK;
  if (!p || !q || !seq_lens || !out) return TQK_EINVAL;
  if (d->key_grid == 2 && !p->knorm) return TQK_EINVAL;
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < tqk_attend_workspace_bytes(d, t))
    return TQK_EWORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dense_path(d, t)) {
    const tqk_attn_desc a = dense_desc(d, t);
    uint16_t* k = static_cast<uint16_t*>(workspace);
    uint16_t* v = k + (size_t)t->batch * a.k_stride[0];
    uint16_t* ws = v + (size_t)t->batch * a.k_stride[0];
    if (t->max_len > 0) {
      const int rd = tqk_dequant_dense(d, p, t->batch, seq_lens, t->max_len, 1, k, v, stream);
      if (rd != TQK_OK) return rd;
    }
    return tqk_attention(&a, q, k, v, seq_lens, q_lens, nullptr, out, ws, tqk_attention_workspace_bytes(&a), stream);
  }
  const AttendPlan ap = attend_plan(d, t);
  const Plan& pl = ap.pl;
  const int gq = d->n_q_heads / d->n_kv_heads;
  const bool mfma = mfma_path(*d);
  // one split of 4 or 8 heads: the split kernel ends with the output itself
  const bool direct = mfma && pl.n_cold_splits == 1 && gq > 2;
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
  a.wave_blocks = pl.wave_blocks;
  a.hot_per_split = pl.hot_per_split;
  a.batch = t->batch;
  a.out = direct ? static_cast<float*>(out) : nullptr;
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
    const dim3 grid(mfma ? pl.n_cold_splits : n_splits, d->n_kv_heads, n);
    switch (gq) {
      case 1: launch_split<1>(a, grid, st); break;
      case 2: launch_split<2>(a, grid, st); break;
      case 3: case 4: launch_split<4>(a, grid, st); break;
      default: launch_split<8>(a, grid, st); break;
    }
    if (hipGetLastError() != hipSuccess) return TQK_EHIP;
    if (direct) continue;
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
