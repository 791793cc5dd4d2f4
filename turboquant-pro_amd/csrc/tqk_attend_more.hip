// Attention over the codes of an fp16 cache of more kinds than a window's (gfx950): over
// listed groups, with the weight that every coded group received, and over a prefix that
// all sequences share.  The plans, joins and entry points; tqk_attend_rows.h has the
// kernel of up to eight rows of a sequence, tqk_attend_prefix.hip that of 128 rows of any.
//
// Listed groups: a workgroup's blocks are those of its list, nothing else is read.
//
// Weights: softmax_j = 2^(s_j - M) / L with a row's maximum M and sum L, which are
// known when its splits are joined.  A wave writes each block's own maximum and sum
// beside its partial results (8 bytes a row and block of 32 tokens: 10 of the step's
// 170 us); workgroups beside the join's add 2^(m - M) l / L over a kv head's rows and a
// group's blocks, in one order and 64 bits: no atomics.
//
// A shared prefix: rows of all sequences over one copy of its codes, then each
// sequence's rows over its other tokens; one join takes both.
//
// The joins are latency, the chain lengths -> partial results -> output: 4 to 5 us a
// launch, 6 to 8 with the groups' weights (their chain is one longer), 9 for a shared
// prefix (the rotation).  In launches of their own, so that nothing has to be zero
// before a call; an arrival counter a row would save part of that.
//
// An ordinary tqk_attend step stays with tqk_attend_codes, whose outputs it has had;
// up to eight rows tqk_attend_rows is faster (32 / 8 heads of 128, 16 sequences of 32768
// tokens: 175 for 189 us) and closer, and more rows go sixteen a workgroup there.
#include "tqk_attend_few.h"

namespace {

// Bytes of blocks' maxima and sums at a time: more queries go in slices.
constexpr long long kMostBlockBytes = (long long)256 << 20;

struct JoinMoreArgs {
  const float* part_acc;  // [split][row][D]
  const float* part_ml;   // [split][row][2]
  const int32_t* seq_lens;
  const int32_t* q_lens;
  void* out;
  long long rows;
  long long o_stride[3];
  int n_splits, n_q_heads, q_len, max_len, out_type, t0, t_len;
};

// The partial results of a row joined: NW waves a row, wave w the splits w, w + NW, ..,
// eight of them on their way at a time (one after another they are a chain of loads:
// 23 splits 8.7 us, where four waves take 4), D / 64 channels a lane.
template <int D, int NW>
__device__ void join_rows(const JoinMoreArgs& a, unsigned block) {
  constexpr int E = D / 64, kAhead = 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = wave % NW;
  const long long row = (long long)block * (4 / NW) + wave / NW;
  __shared__ float acc_s[4][D], ml_s[4][2];
  const bool real = row < a.rows;
  const long long from = real ? row : 0;
  float M = -INFINITY, l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int s0 = w; s0 < a.n_splits; s0 += NW * kAhead) {
    float x[kAhead][E], m_[kAhead], l_[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const long long o = min(s0 + u * NW, a.n_splits - 1) * a.rows + from;
      m_[u] = a.part_ml[2 * o];
      l_[u] = a.part_ml[2 * o + 1];
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = a.part_acc[o * D + E * lane + e];
    }
    float top = M;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) top = fmaxf(top, m_[u]);  // (a repeated last split: none below)
    const float f0 = M == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(M - top));
    l *= f0;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= f0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s0 + u * NW < a.n_splits) {
        const float f = m_[u] == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(m_[u] - top));
        l = fmaf(l_[u], f, l);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(x[u][e], f, acc[e]);
      }
    }
    M = top;
  }
  if constexpr (NW > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) acc_s[wave][E * lane + e] = acc[e];
    if (lane == 0) {
      ml_s[wave][0] = M;
      ml_s[wave][1] = l;
    }
    __syncthreads();
    if (w != 0) return;
    float top = M;
#pragma unroll
    for (int u = 1; u < NW; ++u) top = fmaxf(top, ml_s[wave + u][0]);
    const float f0 = M == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(M - top));
    l *= f0;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= f0;
#pragma unroll
    for (int u = 1; u < NW; ++u) {
      const float mu = ml_s[wave + u][0], f = mu == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(mu - top));
      l = fmaf(ml_s[wave + u][1], f, l);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(acc_s[wave + u][E * lane + e], f, acc[e]);
    }
    M = top;
  }
  if (!real) return;
  const int t = a.t0 + (int)(row % a.t_len);
  const long long bh = row / a.t_len;
  const int hq = (int)(bh % a.n_q_heads), b = (int)(bh / a.n_q_heads);
  const int n = min(a.seq_lens[b], a.max_len);
  const int m = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
  const bool any = t < m && n - m + t >= 0 && l != 0.f;  // (listed groups may leave a query nothing)
  const long long o = b * a.o_stride[0] + hq * a.o_stride[1] + t * a.o_stride[2] + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y = any ? acc[e] / l : 0.f;
    if (a.out_type == 0) static_cast<float*>(a.out)[o + e] = y;
    else static_cast<_Float16*>(a.out)[o + e] = (_Float16)y;
  }
}

template <int D, int NW>
__global__ __launch_bounds__(256) void tqk_join_more(JoinMoreArgs a) {
  touch_args<JoinMoreArgs>();
  join_rows<D, NW>(a, blockIdx.x);
}

// The same where the first `pre` splits hold sums of centroids (of a shared prefix): four
// rows a workgroup, four waves each (a wave a row was a chain of loads: 16 us for 33
// splits of 1024 rows); the centroids' sums over all of the row's weights as an fp16
// pair, times Pi's, by the matrix cores.
template <int D>
__global__ __launch_bounds__(1024) void tqk_join_shared(JoinMoreArgs a, const float* pi_t, int pre) {
  touch_args<JoinMoreArgs>();
  constexpr int E = D / 64, NM = D / 32, kAhead = 8, NW = 4, NR = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ln = lane & 15, lg = lane >> 4;
  const int w = wave % NW, r = wave / NW;
  __shared__ __align__(16) uint16_t c_s[2 * NR][D + 8];  // first halves, then second ones
  __shared__ __align__(16) float y_s[NR][D + 4], acc_s[NR][NW][2][D];
  __shared__ float ml_s[NR][NW][2];
  const long long row = (long long)blockIdx.x * NR + r;
  const long long from = row < a.rows ? row : a.rows - 1;
  float M = -INFINITY, l = 0.f, acc[2][E];  // [0] centroids' sums, [1] values'
#pragma unroll
  for (int e = 0; e < E; ++e) acc[0][e] = acc[1][e] = 0.f;
  auto add = [&](auto kind, int s_from, int s_to) {
    constexpr int k = decltype(kind)::value;
    for (int s0 = s_from + w; s0 < s_to; s0 += NW * kAhead) {
      float x[kAhead][E], m_[kAhead], l_[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const long long o = min(s0 + u * NW, s_to - 1) * a.rows + from;
        m_[u] = a.part_ml[2 * o];
        l_[u] = a.part_ml[2 * o + 1];
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = a.part_acc[o * D + E * lane + e];
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) top = fmaxf(top, s0 + u * NW < s_to ? m_[u] : -INFINITY);
      const float f0 = M == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(M - top));
      l *= f0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        acc[0][e] *= f0;
        acc[1][e] *= f0;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s0 + u * NW < s_to) {
          const float f = m_[u] == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(m_[u] - top));
          l = fmaf(l_[u], f, l);
#pragma unroll
          for (int e = 0; e < E; ++e) acc[k][e] = fmaf(x[u][e], f, acc[k][e]);
        }
      }
      M = top;
    }
  };
  add(std::integral_constant<int, 1>{}, pre, a.n_splits);
  add(std::integral_constant<int, 0>{}, 0, pre);
  // Pi^T's rows 16 wave + ln, on their way meanwhile
  f4_t pr[NM][2];
  if (wave < D / 16) {
#pragma unroll
    for (int mm = 0; mm < NM; ++mm)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        pr[mm][e] = *reinterpret_cast<const f4_t*>(pi_t + (size_t)(16 * wave + ln) * D + 32 * mm + 8 * lg + 4 * e);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) acc_s[r][w][k][E * lane + e] = acc[k][e];
  if (lane == 0) {
    ml_s[r][w][0] = M;
    ml_s[r][w][1] = l;
  }
  __syncthreads();
  float inv = 0.f, rest[E];
  if (w == 0) {
    float top = M;
#pragma unroll
    for (int u = 1; u < NW; ++u) top = fmaxf(top, ml_s[r][u][0]);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[0][e] = acc[1][e] = 0.f;
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float mu = ml_s[r][u][0], f = mu == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(mu - top));
      l = fmaf(ml_s[r][u][1], f, l);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[k][e] = fmaf(acc_s[r][u][k][E * lane + e], f, acc[k][e]);
    }
    inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      rest[e] = acc[1][e] * inv;
      const float y = acc[0][e] * inv;
      const _Float16 hi = (_Float16)y;
      c_s[r][E * lane + e] = __builtin_bit_cast(uint16_t, hi);
      c_s[NR + r][E * lane + e] = f2h(y - (float)hi);
    }
  }
  __syncthreads();
  if (wave < D / 16) {
    f4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int mm = 0; mm < NM; ++mm) {
      h8_t ph, pl;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = pr[mm][e / 4][e % 4];
        ph[e] = (_Float16)y;
        pl[e] = (_Float16)(y - (float)ph[e]);
      }
      const h8_t c8 = *reinterpret_cast<const h8_t*>(&c_s[ln % (2 * NR)][32 * mm + 8 * lg]);
      sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(c8, pl, sum, 0, 0, 0);
      sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(c8, ph, sum, 0, 0, 0);
    }
    // rows 4 lg + e of the product: first halves in lanes of lg 0, second ones of lg 1
#pragma unroll
    for (int e = 0; e < NR; ++e) {
      const float z = sum[e] + __shfl_xor(sum[e], 16, 64);
      if (lg == 0) y_s[e][16 * wave + ln] = z;
    }
  }
  __syncthreads();
  if (row >= a.rows || w != 0) return;
  const int t = (int)(row % a.t_len);
  const long long bh = row / a.t_len;
  const int hq = (int)(bh % a.n_q_heads), b = (int)(bh / a.n_q_heads);
  const int n = min(a.seq_lens[b], a.max_len);
  const int m = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
  const bool any = t < m && n - m + t >= 0;
  const long long o = b * a.o_stride[0] + hq * a.o_stride[1] + t * a.o_stride[2] + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y = any ? y_s[r][E * lane + e] + rest[e] : 0.f;
    if (a.out_type == 0) static_cast<float*>(a.out)[o + e] = y;
    else static_cast<_Float16*>(a.out)[o + e] = (_Float16)y;
  }
}

struct WeightArgs {
  tqk_cache_desc d;
  const float* block_ml;  // [row][blocks][2]
  float* weights;         // [sequence][kv head][max_groups_per_seq]
  int window, sinks, blocks, nblk, chunks;
  unsigned join_blocks;  // workgroups that join rows; those behind them add weights up
};

// weights += what the launch's queries gave every group.  A thread a block of 32 tokens
// (a workgroup: whole groups of them), rows one after another.  A row's maximum and sum
// over its splits are found here once more, by a thread a row, so that no launch waits
// for the join's (4.5 us of a step).
constexpr int kWeightRows = 256;  // at a time
__device__ void group_weights(const JoinMoreArgs& ja, const WeightArgs& a, unsigned block) {
  const tqk_cache_desc& d = a.d;
  const int G = d.group_tokens, Hkv = d.n_kv_heads, gq = d.n_q_heads / Hkv;
  const int chunk = block % a.chunks, h = block / a.chunks % Hkv, b = block / a.chunks / Hkv, tid = threadIdx.x;
  const int per = 256 / a.nblk;  // groups of a workgroup
  const int n = min(ja.seq_lens[b], ja.max_len), ng = n_groups_of(n, d.hot_window, G);
  const int m = ja.q_lens ? min(max(ja.q_lens[b], 0), ja.q_len) : ja.q_len;
  const int g = chunk * per + tid / a.nblk, k = tid % a.nblk;
  const int first = g * G + 32 * k, last = first + min(32, G - 32 * k) - 1;
  const bool mine = tid < per * a.nblk && g < ng;
  const int t_begin = max(ja.t0, m - n), t_end = min(m, ja.t0 + ja.t_len), sinks = min(a.sinks, max(n, 0));
  const int each = max(t_end - t_begin, 0), rows = gq * each;
  if (chunk * per >= ng || rows == 0) return;  // (the whole workgroup)
  const long long at = mine ? g * a.nblk + k : 0;
  __shared__ float M_s[kWeightRows], L_s[kWeightRows];
  __shared__ double sum_s[256];
  double sum = 0.0;
  for (int r0 = 0; r0 < rows; r0 += kWeightRows) {
    const int n_rows = min(kWeightRows, rows - r0);
    __syncthreads();  // (the rows before are read)
    if (tid < n_rows) {
      const int i = (r0 + tid) / each, t = t_begin + (r0 + tid) % each;
      const float* const ml = ja.part_ml + 2 * (((long long)b * d.n_q_heads + h * gq + i) * ja.t_len + t - ja.t0);
      float M = -INFINITY, L = 0.f;
      for (int s0 = 0; s0 < ja.n_splits; s0 += 8) {
        float m_[8], l_[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float* const y = ml + 2 * min(s0 + u, ja.n_splits - 1) * ja.rows;
          m_[u] = y[0];
          l_[u] = s0 + u < ja.n_splits ? y[1] : 0.f;
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < 8; ++u) top = fmaxf(top, m_[u]);
        L *= M == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(M - top));
#pragma unroll
        for (int u = 0; u < 8; ++u)
          L = fmaf(l_[u], m_[u] == -INFINITY ? 0.f : above_zero(__builtin_amdgcn_exp2f(m_[u] - top)), L);
        M = top;
      }
      M_s[tid] = M;
      L_s[tid] = L;
    }
    __syncthreads();
    int i = r0 / each, t = t_begin + r0 % each;
    for (int j0 = 0; j0 < n_rows; j0 += 8) {  // (eight rows' numbers on their way at once, summed in order)
      float m_[8], l_[8];
      int p[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const long long row = ((long long)b * d.n_q_heads + h * gq + i) * ja.t_len + t - ja.t0;
        p[u] = j0 + u < n_rows ? n - m + t : -1;
        m_[u] = a.block_ml[(row * a.blocks + at) * 2];
        l_[u] = a.block_ml[(row * a.blocks + at) * 2 + 1];
        if (j0 + u + 1 < n_rows && ++t == t_end) {
          t = t_begin;
          ++i;
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int lo = a.window > 0 && a.window <= p[u] ? p[u] - a.window + 1 : 0;
        // (only blocks that this row sees were visited)
        const bool seen = mine && first <= p[u] && (min(last, p[u]) >= lo || first < sinks);
        const int j = min(j0 + u, kWeightRows - 1);
        if (seen && l_[u] != 0.f) sum += (double)(__builtin_amdgcn_exp2f(m_[u] - M_s[j]) * l_[u] / L_s[j]);
      }
    }
  }
  sum_s[tid] = sum;
  __syncthreads();
  if (mine && k == 0) {
    double y = 0.0;
    for (int i = 0; i < a.nblk; ++i) y += sum_s[tid + i];
    float* const w = a.weights + ((long long)b * Hkv + h) * d.max_groups_per_seq + g;
    *w = (float)((double)*w + y);
  }
}

struct JoinWeightArgs {
  JoinMoreArgs j;
  WeightArgs w;
};
template <int D, int NW>
__global__ __launch_bounds__(256) void tqk_join_weights(JoinWeightArgs a) {
  touch_args<JoinWeightArgs>();
  if (blockIdx.x < a.w.join_blocks) join_rows<D, NW>(a.j, blockIdx.x);
  else group_weights(a.j, a.w, blockIdx.x - a.w.join_blocks);
}

// (few rows: a workgroup each; many, whose waves hide each other's loads, four)
bool join_apart(const JoinMoreArgs& a) { return a.n_splits > 4 && a.rows <= 4096; }
unsigned join_blocks(const JoinMoreArgs& a) { return (unsigned)(join_apart(a) ? a.rows : (a.rows + 3) / 4); }

// `w`: with the weights of `blocks` workgroups, or null
template <int D>
void launch_join_rows(const JoinMoreArgs& a, const WeightArgs* w, unsigned blocks, hipStream_t st) {
  if (w) {
    const JoinWeightArgs x{a, *w};
    const dim3 grid(w->join_blocks + blocks);
    if (join_apart(a))
      hipLaunchKernelGGL((tqk_join_weights<D, 4>), grid, dim3(256), 0, st, x);
    else
      hipLaunchKernelGGL((tqk_join_weights<D, 1>), grid, dim3(256), 0, st, x);
  } else if (join_apart(a)) {
    hipLaunchKernelGGL((tqk_join_more<D, 4>), dim3(join_blocks(a)), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((tqk_join_more<D, 1>), dim3(join_blocks(a)), dim3(256), 0, st, a);
  }
}
void launch_join(const JoinMoreArgs& a, const WeightArgs* w, unsigned blocks, int D, hipStream_t st) {
  if (D == 64)
    launch_join_rows<64>(a, w, blocks, st);
  else if (D == TQK_D)
    launch_join_rows<TQK_D>(a, w, blocks, st);
  else
    launch_join_rows<256>(a, w, blocks, st);
}

void launch_rows(MoreArgs a, long long groups, hipStream_t st) {
  const tqk_cache_desc& d = a.d;
  const long long blocks = (d.group_tokens + 31) / 32, n_waves = (long long)a.n_splits * kFewWaves;
  const long long most = ((long long)a.max_len / d.group_tokens + 2) * blocks, listed = (long long)a.n_list * blocks;
  a.by.splits = few_div(a.n_splits, groups);
  a.by.heads = few_div(d.n_kv_heads, groups);
  a.by.items = few_div(a.q_items, groups);
  a.by.heads_of = few_div(d.n_q_heads / d.n_kv_heads, 8);
  a.by.group = few_div(d.group_tokens, a.max_len);
  a.by.blocks = few_div(blocks, listed > most ? listed : most);
  a.by.waves = few_div(n_waves, listed + most + d.hot_window + n_waves);
  a.by.per_page = 1.0f / (float)d.page_tokens;
  a.by.group_pages = d.group_tokens / d.page_tokens;
  if (a.d.head_dim == 64)
    tqk_launch_rows_64(a, (unsigned)groups, st);
  else if (a.d.head_dim == TQK_D)
    tqk_launch_rows_128(a, (unsigned)groups, st);
  else
    tqk_launch_rows_256(a, (unsigned)groups, st);
}

size_t partial_bytes(long long rows, int splits, int D) { return (size_t)splits * rows * (D + 2) * sizeof(float) + 256; }

constexpr long long kMostGroups = 1LL << 22;  // workgroups of a launch (512 threads each: fewer than 2^32)

// Queries, kv heads and sequences of a launch, and its splits.
struct MorePlan {
  int per_item, q_items, n_splits;
  long long pairs;  // workgroups of a split
};
// Queries of a launch, `per_item` of them a workgroup: more go in slices.
int launch_queries(const tqk_cache_desc* d, const tqk_attend_desc* t, int per_item) {
  const long long fit = kMostGroups / ((long long)t->batch * d->n_kv_heads) * per_item;
  return fit < t->q_len ? (int)fit : t->q_len;
}
MorePlan more_plan(const tqk_cache_desc* d, long long batch, int queries, int most_per_item, long long tokens, double join) {
  MorePlan mp{};
  const int gq = d->n_q_heads / d->n_kv_heads;
  mp.per_item = 8 / gq < queries ? 8 / gq : queries;
  if (mp.per_item > most_per_item) mp.per_item = most_per_item;
  mp.q_items = (queries + mp.per_item - 1) / mp.per_item;
  mp.pairs = batch * mp.q_items * d->n_kv_heads;
  mp.n_splits = few_splits(mp.pairs, (tokens + 31) / 32 + 1, join);
  if (mp.pairs * mp.n_splits > kMostGroups && mp.n_splits > 1) mp.n_splits = mp.pairs < kMostGroups ? (int)(kMostGroups / mp.pairs) : 1;
  return mp;
}

// Tokens that one workgroup's rows see at most of a window.
long long window_tokens(const tqk_attend_desc* t, int per_item) {
  if (t->window > 0 && t->window < t->max_len) {
    const long long w = (long long)t->window + per_item + t->sinks + 64;
    if (w < t->max_len) return w;
  }
  return t->max_len;
}

MoreArgs more_args(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
                   const int32_t* seq_lens, const int32_t* q_lens, void* out) {
  MoreArgs a{};
  a.d = *d;
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.out = out;
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = t->q_stride[i];
    a.o_stride[i] = t->o_stride[i];
  }
  a.q_len = t->q_len;
  a.max_len = t->max_len;
  a.window = t->window;
  a.sinks = t->sinks;
  a.out_type = t->out_type;
  a.batch = t->batch;
  a.t_len = t->q_len;
  return a;
}

JoinMoreArgs join_args(const MoreArgs& a, int splits) {
  JoinMoreArgs j{};
  j.part_acc = a.part_acc;
  j.part_ml = a.part_ml;
  j.seq_lens = a.seq_lens;
  j.q_lens = a.q_lens;
  j.out = a.out;
  j.rows = a.rows;
  for (int i = 0; i < 3; ++i) j.o_stride[i] = a.o_stride[i];
  j.n_splits = splits;
  j.n_q_heads = a.d.n_q_heads;
  j.q_len = a.q_len;
  j.max_len = a.max_len;
  j.out_type = a.out_type;
  j.t0 = a.t0;
  j.t_len = a.t_len;
  return j;
}

int checked(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
            const int32_t* seq_lens, const void* out, const void* workspace) {
  if (!p || !q || !seq_lens || !out || (((uintptr_t)q | (uintptr_t)out) & 15) || !tqk_have_buffers(*d, *p)) return TQK_EINVAL;
  if (!workspace || ((uintptr_t)workspace & 15)) return TQK_EWORKSPACE;
  return TQK_OK;
}
int check_more(const tqk_cache_desc* d, const tqk_attend_desc* t, bool windowed) {
  const int rc = tqk_check_attend(d, t);
  if (rc != TQK_OK) return rc;
  if (d->input_f32) return TQK_EUNSUPPORTED;
  if (!windowed && (t->window || t->sinks)) return TQK_EINVAL;
  if ((long long)t->batch * d->n_q_heads * t->q_len > INT32_MAX / 2) return TQK_EINVAL;
  if ((long long)t->batch * d->n_kv_heads > kMostGroups) return TQK_EINVAL;  // (a launch has a query of each)
  return TQK_OK;
}

// The rows of t_len queries at a time (mp: the plan of so many), and the join of their splits.
size_t item_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t, const MorePlan& mp, int t_len) {
  return mp.n_splits > 1 ? partial_bytes((long long)t->batch * d->n_q_heads * t_len, mp.n_splits, d->head_dim) : 16;
}
int run_items(MoreArgs a, const MorePlan& mp, int t_len, void* workspace, void* stream) {
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  a.per_item = mp.per_item;
  a.n_splits = mp.n_splits;
  a.direct = mp.n_splits == 1;
  a.part_acc = static_cast<float*>(workspace);
  for (a.t0 = 0; a.t0 < a.q_len; a.t0 += t_len) {
    a.t_len = a.q_len - a.t0 < t_len ? a.q_len - a.t0 : t_len;
    a.q_items = (a.t_len + a.per_item - 1) / a.per_item;
    a.rows = (long long)a.batch * a.d.n_q_heads * a.t_len;
    a.part_ml = a.part_acc + (size_t)mp.n_splits * a.rows * a.d.head_dim;
    launch_rows(a, (long long)a.batch * a.q_items * a.d.n_kv_heads * a.n_splits, st);
    if (!a.direct) launch_join(join_args(a, mp.n_splits), nullptr, 0, a.d.head_dim, st);
    if (hipGetLastError() != hipSuccess) return TQK_EHIP;
  }
  return TQK_OK;
}

// ---- listed groups ----------------------------------------------------------
int check_list(const tqk_cache_desc* d, const tqk_attend_desc* t, const tqk_group_list* l) {
  const int rc = check_more(d, t, false);
  if (rc != TQK_OK) return rc;
  if (!l || l->n < 0 || l->n > (1 << 24)) return TQK_EINVAL;
  return TQK_OK;
}
struct ListPlan {
  int t_len;  // queries of a slice
  MorePlan mp;
};
ListPlan list_plan(const tqk_cache_desc* d, const tqk_attend_desc* t, const tqk_group_list* l) {
  const int G = d->group_tokens, nblk = (G + 31) / 32;
  const long long groups = n_groups_of(t->max_len, d->hot_window, G);
  const long long listed = l->n < groups ? l->n : groups;  // (more: of one twice)
  const long long hot = t->max_len < d->hot_window ? t->max_len : d->hot_window;
  const int most = l->stride[2] ? 1 : INT32_MAX;  // (a list a query: a workgroup each)
  const int t_len = launch_queries(d, t, l->stride[2] ? 1 : 8 / (d->n_q_heads / d->n_kv_heads));
  return ListPlan{t_len, more_plan(d, t->batch, t_len, most, 32 * listed * nblk + hot, 2.0)};
}

// ---- weights ----------------------------------------------------------------
struct WeightPlan {
  int t_len;   // queries of a slice
  int blocks;  // blocks of a row
  MorePlan mp;
};
WeightPlan weight_plan(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  WeightPlan w{};
  const int G = d->group_tokens, nblk = (G + 31) / 32, ng = n_groups_of(t->max_len, d->hot_window, G);
  w.blocks = ng * nblk;
  const long long one = (long long)t->batch * d->n_q_heads * w.blocks * 8;  // bytes of a query
  long long fit = one ? kMostBlockBytes / one : t->q_len;
  fit = fit < 1 ? 1 : fit;
  const int gq = d->n_q_heads / d->n_kv_heads, per = 8 / gq, most = launch_queries(d, t, per);
  w.t_len = fit < most ? (int)fit : most;
  // (whole workgroups where a slice ends)
  if (w.t_len < t->q_len && w.t_len > per) w.t_len = w.t_len / per * per;
  w.mp = more_plan(d, t->batch, w.t_len, INT32_MAX, window_tokens(t, per), 0.0);
  return w;
}
int weight_chunks(const tqk_cache_desc* d, const tqk_attend_desc* t) {  // workgroups of a (sequence, kv head)'s sums
  const int nblk = (d->group_tokens + 31) / 32, per = 256 / nblk;
  return (n_groups_of(t->max_len, d->hot_window, d->group_tokens) + per - 1) / per;
}
int check_weights(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  const int rc = check_more(d, t, true);
  if (rc != TQK_OK) return rc;
  const long long pairs = (long long)t->batch * d->n_kv_heads;
  // (and the join's workgroups: fewer than 2^24)
  if (pairs > 65535 || pairs * weight_chunks(d, t) >= 1 << 23) return TQK_EINVAL;
  return TQK_OK;
}
size_t weight_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t, const WeightPlan& w) {
  const long long rows = (long long)t->batch * d->n_q_heads * w.t_len;
  return partial_bytes(rows, w.mp.n_splits, d->head_dim) + (size_t)rows * w.blocks * 8;
}

// ---- a shared prefix ---------------------------------------------------------
struct SharedPlan {
  bool once;            // the prefix is read once
  long long pre_pairs;  // workgroups of a split of the prefix
  int pre_splits;
  MorePlan rest;  // what follows it, or (not `once`) every sequence for itself
};
// Whether reading the prefix once pays: it takes launches of its own and a set-up, about
// 28 us, and 3.2 a tile of its workgroups; each sequence for itself finds the others'
// codes in cache, a block of 32 tokens and 8 rows 1.0 ns of the whole card (0.7 at
// head_dim 64, 4 at 256; 16 rows of tqk_run_few a fifth more, whose weights are single
// fp16 numbers, 2.9e-4 of the result for 2.1e-4).  Each for itself and once, us, 32 / 8
// heads of 128: a prefix of 32768 tokens, 4 sequences 46 and 87, 8 73 and 88, 32 near
// 300 and 108; 4096 tokens, 64 sequences 84 and 78; 2048 tokens, 32 sequences 29 and 54;
// head_dim 256, 16 / 8 heads, 4096 tokens, 4 sequences 44 and 79, 16 81 and 79.
// (Measured with 3- and 4-bit values, 4-bit keys and a side-list of 2 %: other forms of
// the cache are taken to cost the same.)
SharedPlan shared_plan(const tqk_cache_desc* d, const tqk_attend_desc* t, int groups) {
  SharedPlan s{};
  const int gq = d->n_q_heads / d->n_kv_heads, tokens = groups * d->group_tokens, cus = device_cus();
  const int blocks = groups * ((d->group_tokens + 31) / 32), tiles = d->head_dim == 256 ? blocks : (blocks + 1) / 2;
  const long long rows = (long long)t->q_len * gq;  // of a workgroup each for itself: 8, or 16 a pass
  const double block = (d->head_dim == 64 ? 0.7e-3 : d->head_dim == TQK_D ? 1.0e-3 : 4.0e-3) * (rows > 8 ? 1.2 : 1.0);
  const double each = (double)t->batch * ((rows + 15) / 16) * d->n_kv_heads * blocks * block * 256.0 / cus;
  const double first = d->head_dim == 256 ? 38.0 : 28.0, tile = 3.2;
  if (each > first + tile) {
    s.pre_pairs = ((long long)t->batch * t->q_len * gq + 127) / 128 * d->n_kv_heads;
    // rounds of the workgroups that fit (one a CU) times a split's tiles and the set-up
    // and joining of about five tiles' time
    long long best = INT64_MAX, once = 0;
    for (int n = 1; n <= 64 && n <= tiles; ++n) {
      const long long rounds = (s.pre_pairs * n + cus - 1) / cus, run = (tiles + n - 1) / n;
      if (rounds * (run + 5) < best) {
        best = rounds * (run + 5);
        once = rounds * run;
        s.pre_splits = n;
      }
    }
    s.once = each > first + (double)once * tile;
  }
  s.rest = more_plan(d, t->batch, t->q_len, INT32_MAX, t->max_len - (s.once ? tokens : 0), s.once ? 0.0 : 2.0);
  return s;
}
bool shared_fits(const tqk_cache_desc* d, const tqk_attend_desc* t, const SharedPlan& s) {
  if (!s.once && s.rest.q_items > 1) return tqk_few_fits(d, t);
  return s.pre_pairs * s.pre_splits <= kMostGroups && s.rest.pairs * s.rest.n_splits <= kMostGroups;
}
int check_shared(const tqk_cache_desc* d, const tqk_attend_desc* t, int32_t groups) {
  const int rc = check_more(d, t, false);
  if (rc != TQK_OK) return rc;
  if (d->key_grid == 2) return TQK_EUNSUPPORTED;
  if (groups < 1 || groups > n_groups_of(t->max_len, d->hot_window, d->group_tokens)) return TQK_EINVAL;
  return TQK_OK;
}

}  // namespace

extern "C" {

size_t tqk_attend_groups_workspace_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t, const tqk_group_list* l) {
  if (check_list(d, t, l) != TQK_OK || !t->batch || !t->q_len) return 0;
  const ListPlan lp = list_plan(d, t, l);
  return item_bytes(d, t, lp.mp, lp.t_len);
}

int tqk_attend_groups(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t,
                      const tqk_group_list* l, const void* q, const int32_t* seq_lens, const int32_t* q_lens,
                      const int32_t* groups, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_list(d, t, l);
  if (rc != TQK_OK) return rc;
  if (!t->batch || !t->q_len) return TQK_OK;
  rc = checked(d, p, t, q, seq_lens, out, workspace);
  if (rc != TQK_OK) return rc;
  if (l->n > 0 && !groups) return TQK_EINVAL;
  if (workspace_bytes < tqk_attend_groups_workspace_bytes(d, t, l)) return TQK_EWORKSPACE;
  MoreArgs a = more_args(d, p, t, q, seq_lens, q_lens, out);
  // (a list of none: any pointer, which is not read)
  a.groups = groups ? groups : reinterpret_cast<const int32_t*>(seq_lens);
  for (int i = 0; i < 3; ++i) a.g_stride[i] = l->stride[i];
  a.n_list = l->n;
  const ListPlan lp = list_plan(d, t, l);
  return run_items(a, lp.mp, lp.t_len, workspace, stream);
}

size_t tqk_attend_weights_workspace_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t) {
  if (check_weights(d, t) != TQK_OK || !t->batch || !t->q_len) return 0;
  return weight_bytes(d, t, weight_plan(d, t));
}

int tqk_attend_weights(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, const void* q,
                       const int32_t* seq_lens, const int32_t* q_lens, void* out, float* weights, void* workspace,
                       size_t workspace_bytes, void* stream) {
  int rc = check_weights(d, t);
  if (rc != TQK_OK) return rc;
  if (!t->batch || !t->q_len) return TQK_OK;
  rc = checked(d, p, t, q, seq_lens, out, workspace);
  if (rc != TQK_OK) return rc;
  if (!weights) return TQK_EINVAL;
  const WeightPlan w = weight_plan(d, t);
  if (workspace_bytes < weight_bytes(d, t, w)) return TQK_EWORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int nblk = (d->group_tokens + 31) / 32, chunks = weight_chunks(d, t);
  MoreArgs a = more_args(d, p, t, q, seq_lens, q_lens, out);
  a.per_item = w.mp.per_item;
  a.n_splits = w.mp.n_splits;
  a.blocks = w.blocks;
  a.part_acc = static_cast<float*>(workspace);
  for (a.t0 = 0; a.t0 < t->q_len; a.t0 += w.t_len) {
    a.t_len = t->q_len - a.t0 < w.t_len ? t->q_len - a.t0 : w.t_len;
    a.q_items = (a.t_len + a.per_item - 1) / a.per_item;
    a.rows = (long long)t->batch * d->n_q_heads * a.t_len;
    a.part_ml = a.part_acc + (size_t)a.n_splits * a.rows * d->head_dim;
    a.block_ml = a.part_ml + (size_t)a.n_splits * a.rows * 2;
    launch_rows(a, (long long)t->batch * a.q_items * d->n_kv_heads * a.n_splits, st);
    const JoinMoreArgs j = join_args(a, a.n_splits);
    WeightArgs g{};
    g.d = *d;
    g.block_ml = a.block_ml;
    g.weights = weights;
    g.window = t->window;
    g.sinks = t->sinks;
    g.blocks = w.blocks;
    g.nblk = nblk;
    g.chunks = chunks;
    g.join_blocks = join_blocks(j);
    launch_join(j, chunks ? &g : nullptr, (unsigned)(chunks * t->batch * d->n_kv_heads), d->head_dim, st);
    if (hipGetLastError() != hipSuccess) return TQK_EHIP;
  }
  return TQK_OK;
}

size_t tqk_attend_shared_workspace_bytes(const tqk_cache_desc* d, const tqk_attend_desc* t, int32_t groups) {
  if (check_shared(d, t, groups) != TQK_OK || !t->batch || !t->q_len) return 0;
  const SharedPlan s = shared_plan(d, t, groups);
  if (!shared_fits(d, t, s)) return 0;
  if (!s.once) return s.rest.q_items > 1 ? tqk_few_workspace_bytes(d, t) : item_bytes(d, t, s.rest, t->q_len);
  return partial_bytes((long long)t->batch * d->n_q_heads * t->q_len, s.pre_splits + s.rest.n_splits, d->head_dim);
}

int tqk_attend_shared(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_attend_desc* t, int32_t groups,
                      const void* q, const int32_t* seq_lens, const int32_t* q_lens, void* out, void* workspace,
                      size_t workspace_bytes, void* stream) {
  int rc = check_shared(d, t, groups);
  if (rc != TQK_OK) return rc;
  if (!t->batch || !t->q_len) return TQK_OK;
  rc = checked(d, p, t, q, seq_lens, out, workspace);
  if (rc != TQK_OK) return rc;
  const SharedPlan s = shared_plan(d, t, groups);
  if (!shared_fits(d, t, s)) return TQK_EINVAL;
  if (workspace_bytes < tqk_attend_shared_workspace_bytes(d, t, groups)) return TQK_EWORKSPACE;
  if (!s.once) {  // (more than eight rows: sixteen a workgroup)
    if (s.rest.q_items > 1) return tqk_run_few(d, p, t, q, seq_lens, q_lens, out, workspace, workspace_bytes, stream);
    return run_items(more_args(d, p, t, q, seq_lens, q_lens, out), s.rest, t->q_len, workspace, stream);
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int splits = s.pre_splits + s.rest.n_splits;
  MoreArgs a = more_args(d, p, t, q, seq_lens, q_lens, out);
  a.rows = (long long)t->batch * d->n_q_heads * t->q_len;
  a.part_acc = static_cast<float*>(workspace);
  a.part_ml = a.part_acc + (size_t)splits * a.rows * d->head_dim;
  a.n_splits = s.pre_splits;
  a.shared = groups * d->group_tokens;
  tqk_launch_prefix(a, (unsigned)(s.pre_pairs * s.pre_splits), st);
  a.skip = a.shared;
  a.split0 = s.pre_splits;
  a.per_item = s.rest.per_item;
  a.q_items = s.rest.q_items;
  a.n_splits = s.rest.n_splits;
  launch_rows(a, s.rest.pairs * s.rest.n_splits, st);
  const JoinMoreArgs j = join_args(a, splits);
  const dim3 grid((unsigned)((a.rows + 3) / 4));
  if (d->head_dim == 64)
    hipLaunchKernelGGL(tqk_join_shared<64>, grid, dim3(1024), 0, st, j, p->pi_t, s.pre_splits);
  else if (d->head_dim == TQK_D)
    hipLaunchKernelGGL(tqk_join_shared<TQK_D>, grid, dim3(1024), 0, st, j, p->pi_t, s.pre_splits);
  else
    hipLaunchKernelGGL(tqk_join_shared<256>, grid, dim3(1024), 0, st, j, p->pi_t, s.pre_splits);
  return hipGetLastError() == hipSuccess ? TQK_OK : TQK_EHIP;
}

}  // extern "C"
