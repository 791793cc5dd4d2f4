// Which coded groups a query attends, and which ones stay in the cache (gfx950).
//
// tqk_score_groups: score = max over a kv head's query heads of sum_i q_i mid_i +
// spread |q_i| half_i from a group's scale and zero point.  16 lanes take a group,
// D / 16 channels each.  In 64 bits, where products of fp16 and fp32 are exact, so that
// the order of the sum decides no choice but between equals.
// tqk_pick_groups: the largest scores of a query by a search over the bits of the
// ordered 64-bit keys, which each thread holds in registers: a count of the keys from a
// threshold on for each bit, until exactly as many as wanted are left.
// tqk_evict_groups: the same choice by the weights' sums over the heads, then the table
// rows, weights and lengths; tqk_rotate_ring turns the uncoded tokens' places.
//
// All of them are chains of a few dependent loads and of the search's counts, not
// bytes.  Measured: 127 groups of 16 sequences and 8 heads (16.6 MB of levels) chosen in
// 11 us by one launch; 511 groups of one sequence 5 and 8 us; an eviction from the same
// 16 sequences 8, their rings (33.5 MB, read and written) 10.
#include "tqk_attend.h"
#include "tqk_wave.h"

namespace {

struct ScoreArgs {
  tqk_cache_desc d;
  tqk_cache_ptrs p;
  const uint16_t* q;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  double* scores;  // [sequence][kv head][query][most]
  int32_t* groups;
  long long q_stride[3];
  int batch, q_len, max_len, top, first, last, most;
  int t0, t_len;  // the queries of this launch
  float spread;
};

// A query's position: n - m + t, negative for none.
__device__ __forceinline__ int position(int n, const int32_t* q_lens, int q_len, int b, int t) {
  const int m = q_lens ? min(max(q_lens[b], 0), q_len) : q_len;
  return t < m ? n - m + t : -1;
}

// x over the 16 lanes of a row (rotations), in every lane
__device__ __forceinline__ double row_sum(double x) {
  auto ror = [](double v, auto n) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    constexpr int c = 0x120 + decltype(n)::value;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, c, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), c, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  x += ror(x, std::integral_constant<int, 8>{});
  x += ror(x, std::integral_constant<int, 4>{});
  x += ror(x, std::integral_constant<int, 2>{});
  x += ror(x, std::integral_constant<int, 1>{});
  return x;
}

// A group's levels of a lane's channels, E ln .. for ln of 16 lanes, and its score.
template <int D>
struct GroupLevels {
  static constexpr int E = D / 16;
  f4_t sc[E / 4], mu[E / 4];
  double mid[E], half[E];
  __device__ __forceinline__ void load(const ScoreArgs& a, int b, int h, int g) {
    const int slot = a.p.group_table[(size_t)b * a.d.max_groups_per_seq + g];
    const size_t at = ((size_t)slot * a.d.n_kv_heads + h) * D + E * (threadIdx.x & 15);
#pragma unroll
    for (int e = 0; e < E / 4; ++e) {
      sc[e] = *reinterpret_cast<const f4_t*>(a.p.gscale + at + 4 * e);
      mu[e] = *reinterpret_cast<const f4_t*>(a.p.gmean + at + 4 * e);
    }
  }
  __device__ __forceinline__ void ready(const ScoreArgs& a) {
    // nf4: levels -1 .. 1 of the scale; uniform: 0 .. 2^bits - 1 of the step
    const double steps = a.d.key_grid == 1 ? 0.5 * (double)((1 << a.d.key_bits) - 1) : 0.0;
    const double width = (a.d.key_grid == 1 ? steps : 1.0) * (double)a.spread;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      mid[e] = fma((double)sc[e / 4][e % 4], steps, (double)mu[e / 4][e % 4]);
      half[e] = (double)sc[e / 4][e % 4] * width;
    }
  }
  // query t's, in every lane of the 16
  __device__ __forceinline__ double score(const ScoreArgs& a, int b, int h, int t) const {
    const int gq = a.d.n_q_heads / a.d.n_kv_heads;
    const uint16_t* const qp = a.q + b * a.q_stride[0] + (long long)h * gq * a.q_stride[1] + t * a.q_stride[2] + E * (threadIdx.x & 15);
    double best = 0.0;
#pragma unroll 4
    for (int i = 0; i < gq; ++i) {
      double y = 0.0;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
        const h4_t q4 = *reinterpret_cast<const h4_t*>(qp + i * a.q_stride[1] + e);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const double q = (double)(float)q4[k];
          y = fma(q, mid[e + k], fma(fabs(q), half[e + k], y));
        }
      }
      y = row_sum(y);
      best = i == 0 || y > best || y != y ? y : best;  // (a NaN stays one)
    }
    return best;
  }
};

constexpr int kScoreGroups = 16;  // groups of a workgroup: four waves of four

template <int D>
__global__ __launch_bounds__(256) void tqk_score_groups(ScoreArgs a) {
  touch_args<ScoreArgs>();
  const int Hkv = a.d.n_kv_heads;
  int x = blockIdx.x;
  const int chunks = (a.most + kScoreGroups - 1) / kScoreGroups;
  const int g0 = x % chunks * kScoreGroups, g = g0 + threadIdx.x / 16;
  x /= chunks;
  const int h = x % Hkv, b = x / Hkv;
  const int n = min(a.seq_lens[b], a.max_len), ng = n_groups_of(n, a.d.hot_window, a.d.group_tokens);
  if (g0 >= ng) return;  // (the whole workgroup)
  GroupLevels<D> levels;
  levels.load(a, b, h, min(g, ng - 1));
  levels.ready(a);
  for (int t = a.t0; t < a.t0 + a.t_len; ++t) {
    const double y = levels.score(a, b, h, t);
    if ((threadIdx.x & 15) == 0 && g < ng) a.scores[(((size_t)b * Hkv + h) * a.t_len + t - a.t0) * a.most + g] = y;
  }
}

// Order-preserving key of a score: 1 or more; no number above all.
__device__ __forceinline__ uint64_t key_of(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  if (x != x) return ~0ull;
  return (u >> 63) ? ~u : u | 1ull << 63;
}

__device__ __forceinline__ int popcount64(uint64_t x) { return __popcll(x); }

// The choice of `top` of c candidates by NT threads: thread tid holds the keys of the
// candidates tid, tid + NT, ..., KPL of them in registers (KPL 0: asked again of `load`).
// emit(i, chosen, rank among the chosen, rank among the others) for every candidate,
// ranks in the order of the candidates.
template <int NT, int KPL, class Load, class Emit>
__device__ void pick(int c, int top, int first, int last, int tid, int (*count_s)[NT / 64 + 1], Load load, Emit emit) {
  constexpr int NW = NT / 64;
  const int wave = tid >> 6, lane = tid & 63;
  const int steps = (c + NT - 1) / NT;
  auto always = [&](int i) { return i < first || i >= c - last; };
  const int forced = min(first, c) + min(last, max(c - first, 0));
  const bool all = c <= top;
  const int need = all ? 0 : top - forced;  // of the other c - forced > need
  uint64_t keys[KPL > 0 ? KPL : 1];
  if constexpr (KPL > 0) {
#pragma unroll
    for (int j = 0; j < KPL; ++j) keys[j] = load(min(j * NT + tid, max(c - 1, 0)));  // (all on their way at once)
#pragma unroll
    for (int j = 0; j < KPL; ++j) {
      const int i = j * NT + tid;
      keys[j] = !all && i < c && !always(i) ? keys[j] : 0ull;
    }
  }
  auto key = [&](int j) -> uint64_t {
    if constexpr (KPL > 0) return keys[j];
    const int i = j * NT + tid;
    return !all && i < c && !always(i) ? load(i) : 0ull;
  };
  // a number of the workgroup: the sum of its waves'
  int turn = 0;
  auto total = [&](int mine) {
    if constexpr (NW == 1) return mine;
    turn ^= 1;
    if (lane == 0) count_s[turn][wave] = mine;
    __syncthreads();
    int y = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) y += count_s[turn][w];
    return y;
  };
  auto count_from = [&](uint64_t v) {
    int mine = 0;
    if constexpr (KPL > 0) {
#pragma unroll
      for (int j = 0; j < KPL; ++j)
        if (j < steps) mine += popcount64(__builtin_amdgcn_ballot_w64(keys[j] >= v));
    } else {
      for (int j = 0; j < steps; ++j) mine += popcount64(__builtin_amdgcn_ballot_w64(key(j) >= v));
    }
    return total(mine);
  };
  uint64_t v = ~0ull;  // keys above it are chosen
  int ties = 0;        // and that many equal to it, the first ones
  if (need > 0) {
    v = 0;
    int at = c, bit = 63;  // keys from v on
    if constexpr (NW == 1 && KPL > 0) {
      // (scores are of one sign and nearly one size: the bits that all keys have are
      // the threshold's)
      uint64_t one = 0, diff = 0;
#pragma unroll
      for (int j = 0; j < KPL; ++j) one = keys[j] ? keys[j] : one;
      const uint64_t some = __builtin_amdgcn_ballot_w64(one != 0);
      const int from = some ? __builtin_ctzll(some) : 0;
      one = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(one >> 32), from) << 32 |
            (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)one, from);
#pragma unroll
      for (int j = 0; j < KPL; ++j) diff |= keys[j] ? keys[j] ^ one : 0;
      uint32_t hi = (uint32_t)(diff >> 32);
#pragma unroll
      for (int o = 32; o; o >>= 1) hi |= (uint32_t)__shfl_xor((int)hi, o, 64);
      if (hi) {
        bit = 63 - __builtin_clz(hi);
        v = bit == 63 ? 0 : one >> (bit + 1) << (bit + 1);
      }
    }
    for (; bit >= 0 && at != need; --bit) {
      const uint64_t higher = v | 1ull << bit;
      const int n = count_from(higher);
      if (n >= need) {
        v = higher;
        at = n;
      }
    }
    if (at == need) ties = INT32_MAX;  // (every key equal to v too)
    else ties = need - (v == ~0ull ? 0 : count_from(v + 1));
  }
  // in order: ranks by ballots, a stretch of NT candidates at a time
  int n_equal = 0, n_in = 0;
  auto body = [&](int j) {
    const int i = j * NT + tid;
    const bool real = i < c;
    const uint64_t k = key(j);
    const bool open = real && !all && !always(i);
    const uint64_t below = (1ull << lane) - 1;
    const uint64_t eq = __builtin_amdgcn_ballot_w64(open && need > 0 && k == v);
    int before = popcount64(eq & below), sum = popcount64(eq);
    if constexpr (NW > 1) {
      turn ^= 1;
      if (lane == 0) count_s[turn][wave] = sum;
      __syncthreads();
      sum = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        before += w < wave ? count_s[turn][w] : 0;
        sum += count_s[turn][w];
      }
    }
    const bool tied = ((eq >> lane) & 1) && n_equal + before < ties;
    n_equal += sum;
    const bool in = real && (all || always(i) || (open && need > 0 && (k > v || tied)));
    const uint64_t ins = __builtin_amdgcn_ballot_w64(in);
    int rank = popcount64(ins & below), n = popcount64(ins);
    if constexpr (NW > 1) {
      turn ^= 1;
      if (lane == 0) count_s[turn][wave] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        rank += w < wave ? count_s[turn][w] : 0;
        n += count_s[turn][w];
      }
    }
    if (real) emit(i, in, n_in + rank, i - n_in - rank);
    n_in += n;
  };
  if constexpr (KPL > 0) {
#pragma unroll
    for (int j = 0; j < KPL; ++j)
      if (j < steps) body(j);
  } else {
    for (int j = 0; j < steps; ++j) body(j);
  }
}

template <int NT, int KPL>
__global__ __launch_bounds__(NT) void tqk_pick_groups(ScoreArgs a) {
  touch_args<ScoreArgs>();
  __shared__ int count_s[2][NT / 64 + 1];
  const tqk_cache_desc& d = a.d;
  const int tid = threadIdx.x;
  const long long row = blockIdx.x;
  const int t = a.t0 + (int)(row % a.t_len);
  const long long bh = row / a.t_len;
  const int b = (int)(bh / d.n_kv_heads);
  const int n = min(a.seq_lens[b], a.max_len), p = position(n, a.q_lens, a.q_len, b, t);
  const int c = p < 0 ? 0 : min(n_groups_of(n, d.hot_window, d.group_tokens), p / d.group_tokens + 1);
  const double* const s = a.scores + (size_t)row * a.most;
  int32_t* const out = a.groups + (bh * a.q_len + t) * a.top;
  pick<NT, KPL>(c, a.top, a.first, a.last, tid, count_s, [&](int i) { return key_of(s[i]); },
                [&](int i, bool in, int rank, int) {
                  if (in) out[rank] = i;
                });
  for (int i = min(c, a.top) + tid; i < a.top; i += NT) out[i] = -1;
}

// Both in one for few rows over few groups: a workgroup a kv head of a sequence, 64
// groups at a time, the next ones on their way; then a wave a query.  127 groups, 4
// rows, 128 workgroups 11.6 us, where the two kernels take 16.5; but 511 groups 28 to 16,
// 187 groups of 21 rows 31 to 17: one workgroup's loads and 64-bit products then bound it.
constexpr int kTogether = 128, kTogetherRows = 8;
template <int D>
__global__ __launch_bounds__(1024) void tqk_choose_groups(ScoreArgs a) {
  touch_args<ScoreArgs>();
  __shared__ double score_s[kTogetherRows][kTogether];
  const tqk_cache_desc& d = a.d;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x % d.n_kv_heads, b = blockIdx.x / d.n_kv_heads;
  const int n = min(a.seq_lens[b], a.max_len), ng = n_groups_of(n, d.hot_window, d.group_tokens);
  if (ng > a.top) {  // (else every candidate is chosen)
    GroupLevels<D> now, next;
    now.load(a, b, h, min(tid / 16, ng - 1));
    for (int g0 = 0; g0 < ng; g0 += 64) {
      if (g0 + 64 < ng) next.load(a, b, h, min(g0 + 64 + tid / 16, ng - 1));
      const int g = g0 + tid / 16;
      now.ready(a);
      for (int t = 0; t < a.q_len; ++t) {
        const double y = now.score(a, b, h, t);
        if ((tid & 15) == 0 && g < ng) score_s[t][g] = y;
      }
      now = next;
    }
    __syncthreads();
  }
  if (wave >= a.q_len) return;
  const int t = wave, p = position(n, a.q_lens, a.q_len, b, t);
  const int c = p < 0 ? 0 : min(ng, p / d.group_tokens + 1);
  int32_t* const out = a.groups + ((long long)blockIdx.x * a.q_len + t) * a.top;
  auto key = [&](int i) { return key_of(score_s[t][i]); };
  auto emit = [&](int i, bool in, int rank, int) {
    if (in) out[rank] = i;
  };
  pick<64, kTogether / 64>(c, a.top, a.first, a.last, lane, nullptr, key, emit);
  for (int i = min(c, a.top) + lane; i < a.top; i += 64) out[i] = -1;
}

struct EvictArgs {
  tqk_cache_desc d;
  float* weights;
  int32_t* seq_lens;
  int32_t* block_table;
  int32_t* group_table;
  int32_t* kept;
  double* scores;   // [sequence][max_groups_per_seq]
  int32_t* order;   // [sequence][max_groups_per_seq]: what stands in a place, formerly
  int32_t* pages;   // [sequence][max_pages_per_seq]: the former table
  int32_t* slots;   // [sequence][max_groups_per_seq]: the former table
  int32_t* turn;    // [sequence]: tokens by which the ring turns
  int keep, first, last;
};

// KPL: candidates that a lane of the first wave holds; 0: all waves choose.
template <int KPL>
__global__ __launch_bounds__(1024) void tqk_evict(EvictArgs a) {
  touch_args<EvictArgs>();
  constexpr int NT = 1024, kAhead = 4;
  __shared__ int count_s[2][NT / 64 + 1];
  const tqk_cache_desc& d = a.d;
  const int b = blockIdx.x, tid = threadIdx.x, G = d.group_tokens, mg = d.max_groups_per_seq, Hkv = d.n_kv_heads;
  const int n = a.seq_lens[b], ng = min(n_groups_of(n, d.hot_window, G), mg), per = G / d.page_tokens;
  const int n_in = min(ng, a.keep), gone = ng - n_in;
  __syncthreads();  // (the length is read before it is written)
  if (tid == 0) {
    a.turn[b] = (int)((long long)gone * G % d.hot_ring);
    a.seq_lens[b] = n - gone * G;
  }
  int32_t* const kept = a.kept + (size_t)b * a.keep;
  for (int i = n_in + tid; i < a.keep; i += NT) kept[i] = -1;
  float* const w = a.weights + (size_t)b * Hkv * mg;
  const long long all = (long long)Hkv * mg;
  if (gone == 0) {
    for (int i = tid; i < n_in; i += NT) kept[i] = i;
    for (long long i = tid; i < all; i += NT)
      if (i % mg >= ng) w[i] = 0.f;
    return;
  }
  double* const s = a.scores + (size_t)b * mg;
  int32_t* const bt = a.block_table + (size_t)b * d.max_pages_per_seq;
  int32_t* const gt = a.group_table + (size_t)b * mg;
  int32_t* const order = a.order + (size_t)b * mg;
  int32_t* const pages = a.pages + (size_t)b * d.max_pages_per_seq;
  int32_t* const slots = a.slots + (size_t)b * mg;
  for (int i = tid; i < ng; i += NT) {
    double y = 0.0;
    for (int h0 = 0; h0 < Hkv; h0 += 8) {  // (eight heads' weights on their way at once; summed in order)
      float x[8];
#pragma unroll
      for (int h = 0; h < 8; ++h) x[h] = w[(size_t)min(h0 + h, Hkv - 1) * mg + i];
#pragma unroll
      for (int h = 0; h < 8; ++h) y += h0 + h < Hkv ? (double)x[h] : 0.0;
    }
    s[i] = y;
    slots[i] = gt[i];
  }
  for (int i = tid; i < ng * per; i += NT) pages[i] = bt[i];
  __syncthreads();
  auto key = [&](int i) { return key_of(s[i]); };
  auto emit = [&](int i, bool in, int rank, int other) {
    order[in ? rank : n_in + other] = i;
    if (in) kept[rank] = i;
  };
  if constexpr (KPL > 0) {
    if (tid < 64) pick<64, KPL>(ng, a.keep, a.first, a.last, tid, nullptr, key, emit);
  } else {
    pick<NT, 0>(ng, a.keep, a.first, a.last, tid, count_s, key, emit);
  }
  __syncthreads();
  for (int i = tid; i < ng; i += NT) gt[i] = slots[order[i]];
  for (int i = tid; i < ng * per; i += NT) bt[i] = pages[order[i / per] * per + i % per];
  // the weights: a place's comes from no earlier one, so a stretch at a time in order
  for (long long i0 = 0; i0 < all; i0 += NT * kAhead) {
    float x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const long long i = i0 + u * NT + tid;
      const int g = (int)(i % mg);
      x[u] = i < all && g < n_in ? w[i - g + order[g]] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const long long i = i0 + u * NT + tid;
      if (i < all) w[i] = x[u];
    }
  }
}

// The rings' places: token t at t % ring, after `turn` tokens less at (t - turn) % ring.
// A workgroup takes a column of `cb` bytes of one (sequence, head)'s keys or values.
constexpr int kRingBytes = 65536;
struct RingArgs {
  uint8_t* ring[2];
  const int32_t* turn;
  int rows, row_bytes, cb, heads;
};
__global__ __launch_bounds__(256) void tqk_rotate_ring(RingArgs a) {
  __shared__ __align__(16) uint8_t col_s[kRingBytes];
  const int cols = a.row_bytes / a.cb, tid = threadIdx.x;
  int x = blockIdx.x;
  const int col = x % cols;
  x /= cols;
  const int which = x & 1;
  x >>= 1;  // (sequence, head)
  const int turn = a.turn[x / a.heads];
  if (turn == 0) return;  // (the same for every thread)
  uint8_t* const at = a.ring[which] + (size_t)x * a.rows * a.row_bytes + col * a.cb;
  const int pieces = a.cb / 16;
  for (int i = tid; i < a.rows * pieces; i += 256)
    *reinterpret_cast<u32x4_t*>(col_s + 16 * i) =
        *reinterpret_cast<const u32x4_t*>(at + (size_t)(i / pieces) * a.row_bytes + 16 * (i % pieces));
  __syncthreads();
  for (int i = tid; i < a.rows * pieces; i += 256) {
    int from = i / pieces + turn;
    from -= from >= a.rows ? a.rows : 0;
    *reinterpret_cast<u32x4_t*>(at + (size_t)(i / pieces) * a.row_bytes + 16 * (i % pieces)) =
        *reinterpret_cast<const u32x4_t*>(col_s + 16 * (from * pieces + i % pieces));
  }
}

// ---- plans and checks ---------------------------------------------------------
constexpr int kMostListed = 1 << 24;  // entries of a list (its places are counted in 32 bits)
// Scores and workgroups of a launch: more queries go in slices.
constexpr long long kMostScoreBytes = (long long)256 << 20, kMostRows = INT32_MAX / 1024, kMostScoreGroups = INT32_MAX / 256;

long long score_chunks(const tqk_cache_desc* d, int max_len) {
  return (n_groups_of(max_len, d->hot_window, d->group_tokens) + kScoreGroups - 1) / kScoreGroups;
}

int check_select(const tqk_cache_desc* d, const tqk_select_desc* s) {
  if (!s) return TQK_EINVAL;
  tqk_attend_desc t{};
  t.batch = s->batch;
  t.q_len = s->q_len;
  t.max_len = s->max_len;
  t.out_type = 1;
  for (int i = 0; i < 3; ++i) t.q_stride[i] = s->q_stride[i];
  const int rc = tqk_check_attend(d, &t);
  if (rc != TQK_OK) return rc;
  if (d->input_f32 || d->key_grid == 2) return TQK_EUNSUPPORTED;
  if (s->top < 1 || s->top > kMostListed || s->first < 0 || s->last < 0 || (long long)s->first + s->last > s->top) return TQK_EINVAL;
  if (!(s->spread >= 0.f) || s->spread > 3.0e38f) return TQK_EINVAL;
  const long long pairs = (long long)s->batch * d->n_kv_heads;  // (a launch has at least one query of each)
  if (pairs > kMostRows || pairs * score_chunks(d, s->max_len) > kMostScoreGroups) return TQK_EINVAL;
  return TQK_OK;
}

struct SelectPlan {
  int most, t_len;
  size_t ws_bytes;
};
SelectPlan select_plan(const tqk_cache_desc* d, const tqk_select_desc* s) {
  SelectPlan sp{};
  sp.most = n_groups_of(s->max_len, d->hot_window, d->group_tokens);
  const long long pairs = (long long)s->batch * d->n_kv_heads, one = pairs * sp.most * 8;
  long long fit = one ? kMostScoreBytes / one : s->q_len;
  fit = fit < kMostRows / pairs ? fit : kMostRows / pairs;
  fit = fit < 1 ? 1 : fit;
  sp.t_len = fit < s->q_len ? (int)fit : s->q_len;
  sp.ws_bytes = (size_t)one * sp.t_len + 16;
  return sp;
}

size_t evict_bytes(const tqk_cache_desc* d, int batch) {
  return (size_t)batch * ((size_t)d->max_groups_per_seq * 16 + (size_t)d->max_pages_per_seq * 4 + 4) + 16;
}
int ring_columns(const tqk_cache_desc* d) {  // bytes of a column, 0: none fits
  const int row = d->head_dim * (d->input_f32 ? 4 : 2);
  for (int cb = row < 128 ? row : 128; cb >= 16; cb /= 2)
    if ((long long)cb * d->hot_ring <= kRingBytes) return cb;
  return 0;
}
// Workgroups that turn the rings.
long long ring_groups(const tqk_cache_desc* d, int batch, int cb) {
  return (long long)batch * d->n_kv_heads * 2 * (d->head_dim * (d->input_f32 ? 4 : 2) / cb);
}

}  // namespace

extern "C" {

size_t tqk_select_groups_workspace_bytes(const tqk_cache_desc* d, const tqk_select_desc* s) {
  if (check_select(d, s) != TQK_OK || !s->batch || !s->q_len) return 0;
  return select_plan(d, s).ws_bytes;
}

int tqk_select_groups(const tqk_cache_desc* d, const tqk_cache_ptrs* p, const tqk_select_desc* s, const void* q,
                      const int32_t* seq_lens, const int32_t* q_lens, int32_t* groups, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const int rc = check_select(d, s);
  if (rc != TQK_OK) return rc;
  if (!s->batch || !s->q_len) return TQK_OK;
  if (!p || !q || !seq_lens || !groups || ((uintptr_t)q & 15) || !p->gscale || !p->gmean || !p->group_table) return TQK_EINVAL;
  const SelectPlan sp = select_plan(d, s);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < sp.ws_bytes) return TQK_EWORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  ScoreArgs a{};
  a.d = *d;
  a.p = *p;
  a.q = static_cast<const uint16_t*>(q);
  a.seq_lens = seq_lens;
  a.q_lens = q_lens;
  a.scores = static_cast<double*>(workspace);
  a.groups = groups;
  for (int i = 0; i < 3; ++i) a.q_stride[i] = s->q_stride[i];
  a.batch = s->batch;
  a.q_len = s->q_len;
  a.max_len = s->max_len;
  a.top = s->top;
  a.first = s->first;
  a.last = s->last;
  a.spread = s->spread;
  a.most = sp.most;
  const long long pairs = (long long)s->batch * d->n_kv_heads, chunks = score_chunks(d, s->max_len);
  if (sp.most <= kTogether && s->q_len * (d->n_q_heads / d->n_kv_heads) <= kTogetherRows) {
    const dim3 grid((unsigned)pairs);
    if (d->head_dim == 64)
      hipLaunchKernelGGL(tqk_choose_groups<64>, grid, dim3(1024), 0, st, a);
    else if (d->head_dim == 128)
      hipLaunchKernelGGL(tqk_choose_groups<128>, grid, dim3(1024), 0, st, a);
    else
      hipLaunchKernelGGL(tqk_choose_groups<256>, grid, dim3(1024), 0, st, a);
    return hipGetLastError() == hipSuccess ? TQK_OK : TQK_EHIP;
  }
  for (a.t0 = 0; a.t0 < s->q_len; a.t0 += sp.t_len) {
    a.t_len = s->q_len - a.t0 < sp.t_len ? s->q_len - a.t0 : sp.t_len;
    if (sp.most > s->top) {  // (else every candidate is chosen)
      const dim3 grid((unsigned)(pairs * chunks));
      if (d->head_dim == 64)
        hipLaunchKernelGGL(tqk_score_groups<64>, grid, dim3(256), 0, st, a);
      else if (d->head_dim == 128)
        hipLaunchKernelGGL(tqk_score_groups<128>, grid, dim3(256), 0, st, a);
      else
        hipLaunchKernelGGL(tqk_score_groups<256>, grid, dim3(256), 0, st, a);
    }
    const dim3 rows((unsigned)(pairs * a.t_len));
    if (sp.most <= 64 * 8)
      hipLaunchKernelGGL((tqk_pick_groups<64, 8>), rows, dim3(64), 0, st, a);
    else if (sp.most <= 64 * 16)
      hipLaunchKernelGGL((tqk_pick_groups<64, 16>), rows, dim3(64), 0, st, a);
    else if (sp.most <= 1024 * 16)
      hipLaunchKernelGGL((tqk_pick_groups<1024, 16>), rows, dim3(1024), 0, st, a);
    else
      hipLaunchKernelGGL((tqk_pick_groups<1024, 0>), rows, dim3(1024), 0, st, a);
    if (hipGetLastError() != hipSuccess) return TQK_EHIP;
  }
  return TQK_OK;
}

size_t tqk_evict_groups_workspace_bytes(const tqk_cache_desc* d, int32_t batch) {
  if (tqk_check_desc(d) != TQK_OK || batch < 1) return 0;
  return evict_bytes(d, batch);
}

int tqk_evict_groups(const tqk_cache_desc* d, const tqk_cache_ptrs* p, int32_t batch, int32_t keep, int32_t first,
                     int32_t last, float* weights, int32_t* seq_lens, int32_t* block_table, int32_t* group_table,
                     int32_t* kept, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = tqk_check_desc(d);
  if (rc != TQK_OK) return rc;
  if (d->zero_point == 2) return TQK_EUNSUPPORTED;
  if (batch < 0 || batch > 65535 || keep < 0 || keep > kMostListed || first < 0 || last < 0 || (long long)first + last > keep) return TQK_EINVAL;
  // (a sequence as long as its groups' table has its pages)
  if ((long long)d->max_groups_per_seq * (d->group_tokens / d->page_tokens) > d->max_pages_per_seq) return TQK_EINVAL;
  const int cb = ring_columns(d);
  if (!cb) return TQK_EUNSUPPORTED;
  // (before anything is rewritten)
  if (ring_groups(d, batch, cb) > INT32_MAX / 256) return TQK_EINVAL;
  if (!batch) return TQK_OK;
  if (!p || !p->hot_k || !p->hot_v || !weights || !seq_lens || !block_table || !group_table || (keep > 0 && !kept))
    return TQK_EINVAL;
  if ((((uintptr_t)p->hot_k | (uintptr_t)p->hot_v) & 15) || block_table != p->block_table || group_table != p->group_table)
    return TQK_EINVAL;
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < evict_bytes(d, batch)) return TQK_EWORKSPACE;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  EvictArgs a{};
  a.d = *d;
  a.weights = weights;
  a.seq_lens = seq_lens;
  a.block_table = block_table;
  a.group_table = group_table;
  a.kept = kept;
  const size_t mg = (size_t)batch * d->max_groups_per_seq;
  a.scores = static_cast<double*>(workspace);
  a.order = reinterpret_cast<int32_t*>(a.scores + mg);
  a.slots = a.order + mg;
  a.pages = a.slots + mg;
  a.turn = a.pages + (size_t)batch * d->max_pages_per_seq;
  a.keep = keep;
  a.first = first;
  a.last = last;
  const dim3 grid((unsigned)batch), block(1024);
  if (d->max_groups_per_seq <= 64 * 2)
    hipLaunchKernelGGL(tqk_evict<2>, grid, block, 0, st, a);
  else if (d->max_groups_per_seq <= 64 * 8)
    hipLaunchKernelGGL(tqk_evict<8>, grid, block, 0, st, a);
  else
    hipLaunchKernelGGL(tqk_evict<0>, grid, block, 0, st, a);
  if (hipGetLastError() != hipSuccess) return TQK_EHIP;
  RingArgs r{};
  r.ring[0] = static_cast<uint8_t*>(p->hot_k);
  r.ring[1] = static_cast<uint8_t*>(p->hot_v);
  r.turn = a.turn;
  r.rows = d->hot_ring;
  r.row_bytes = d->head_dim * (d->input_f32 ? 4 : 2);
  r.cb = cb;
  r.heads = d->n_kv_heads;
  hipLaunchKernelGGL(tqk_rotate_ring, dim3((unsigned)ring_groups(d, batch, cb)), dim3(256), 0, st, r);
  return hipGetLastError() == hipSuccess ? TQK_OK : TQK_EHIP;
}

}  // extern "C"
