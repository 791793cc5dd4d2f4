// Attention over dense keys and values with a sliding window and a few first
// tokens that stay visible (gfx950).
//
// Query t of a sequence with m queries and n keys stands at p = n - m + t and
// sees the keys j of [start, p] with j > p - window or j < start + sinks:
//   out = sum_j softmax_j(scale q . k_j) v_j
// by one pass over the visible keys with a running maximum and sum.  A key tile
// that no row of a workgroup sees is never read.
//
// tqk_attn_tiles: prompts and chunks.  The rows of one kv head are its query
// heads' rows side by side (row = t * heads + head), 32 a wave, 128 a workgroup;
// 64 keys at a time go through LDS.  Scores are computed transposed, K Q^T, so
// that a lane holds one row's scores and its running maximum and sum are plain
// registers, and the weights are already laid out as the operand of V^T P^T (the
// order of the keys inside a product is free: both operands take the order the
// scores come in).  V^T comes from LDS by transposing reads.
// Bound: the matrix cores and, as closely, LDS reads (16 KiB of K and V for
// 32 x 64 scores a wave).  A prompt of 8192 tokens, 32 heads of 128, window 4096:
// 464 to 480 us, 860 to 890 TFLOP/s (a large library product: 1200); head_dim 256, 16
// heads, 4096 tokens: 284 us, 485 TFLOP/s, at one wave a SIMD, which leaves the softmax
// nothing to hide behind (two waves spill: 442 us).  Few rows: HBM and the join.
//
// The weights are rounded to the inputs' type, as the matrix cores take them (pairs
// would be a second product of the two): 2.9e-4 off 64 bits in fp16, where the output's
// rounding alone is 2.1e-4 off, and 2.1e-3 in bf16, where it is 1.6e-3.
#include "tqk_attn.h"
#include "tqk_wave.h"

namespace {

typedef float f16v_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef short s8_t __attribute__((ext_vector_type(8)));

constexpr int kTileThreads = 256;
constexpr int kRows = 32;      // rows a wave
constexpr int kTileRows = 128; // rows a workgroup
// keys a tile: at head_dim 256 half as many, which leaves the accumulators their
// registers; so at head_dim 128 with keys in pairs, which leaves LDS to two
// workgroups (a chunk of 512 over a window of 4096, 4 sequences: 300 us, with 64
// keys 407; at head_dim 64 178, with 64 keys 163)
template <int D, bool PAIR = false>
constexpr int kTileKeys = D == 256 || (D == 128 && PAIR) ? 32 : 64;
// The running maximum follows the scores only when one exceeds it by this much
// (log2 units): weights stay at most 2^8, far inside fp16's range, and the
// accumulators are rescaled a few times a row instead of every tile.
constexpr float kLazy = 8.0f;

struct AttnArgs {
  tqk_attn_desc d;
  const void* q;
  const void* k;
  const void* v;
  const void* k_lo;  // PAIR: what the keys' rounding left
  const int32_t* kv_lens;
  const int32_t* q_lens;
  const int32_t* kv_starts;
  void* out;
  float* part_ml;   // [split][row][2]: running maximum (log2 units) and sum
  float* part_acc;  // [split][row][D]
  int row_tiles;    // row tiles of a (sequence, kv head)
  int n_splits;
  long long rows;   // rows of all sequences and heads
  int compact;      // keys and values hold only the first tiles and those from the first visible one on
};

template <typename T>
struct Mma;
template <>
struct Mma<_Float16> {
  typedef h8_t v8;
  static __device__ __forceinline__ f16v_t m32(v8 a, v8 b, f16v_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f4_t m16(v8 a, v8 b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<__bf16> {
  typedef bf8_t v8;
  static __device__ __forceinline__ f16v_t m32(v8 a, v8 b, f16v_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f4_t m16(v8 a, v8 b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// whether a 16-bit pattern is an infinity or a NaN
template <typename T>
__device__ __forceinline__ bool not_finite2(uint32_t two) {
  constexpr uint32_t e = __is_same(T, __bf16) ? 0x7F80u : 0x7C00u;
  return (two & e) == e || ((two >> 16) & e) == e;
}
template <typename T>
__device__ __forceinline__ bool not_finite(u4_t x) {
  return not_finite2<T>(x.x) || not_finite2<T>(x.y) || not_finite2<T>(x.z) || not_finite2<T>(x.w);
}

template <typename T>
__device__ __forceinline__ u4_t only_finite(u4_t x) {
  constexpr uint32_t e = __is_same(T, __bf16) ? 0x7F80u : 0x7C00u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((x[i] & e) == e) x[i] &= 0xFFFF0000u;
    if (((x[i] >> 16) & e) == e) x[i] &= 0xFFFFu;
  }
  return x;
}

// a raw buffer of `bytes` from p on (32-bit data, no swizzle); past it loads give zeros
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const char* p, long long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), (short)0, (int)bytes, 0x00020000);
}
// this wave's loads into LDS are done
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ float max_half(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float sum_half(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// a number that is the same in every lane, in a scalar register
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What a sequence's queries see.
struct Seen {
  int n, m, start, sink_end, window;  // window 0: none
  __device__ __forceinline__ Seen(const AttnArgs& a, int b) {
    n = uni(a.kv_lens ? min(max(a.kv_lens[b], 0), a.d.kv_len) : a.d.kv_len);
    m = uni(a.q_lens ? min(max(a.q_lens[b], 0), a.d.q_len) : a.d.q_len);
    start = uni(a.kv_starts ? min(max(a.kv_starts[b], 0), n) : 0);
    sink_end = start + min(a.d.sinks, n - start);
    window = a.d.window > 0 && a.d.window < n ? a.d.window : 0;
  }
  __device__ __forceinline__ int low(int p) const { return window ? max(start, p - window + 1) : start; }
  __device__ __forceinline__ bool sees(int p, int lo, int j) const {
    return (j <= p) & ((j >= lo) | ((j < sink_end) & (j >= start)));
  }
};

// The key tiles that rows at positions [p_lo, p_hi] see: a run from the first
// visible tokens' tile, then one up to p_hi's.
template <int kKeys>
struct Tiles {
  int first, n_first, second, n;
  __device__ __forceinline__ Tiles(const Seen& s, int p_lo, int p_hi) {
    first = s.start / kKeys;
    if (p_hi < s.start) {  // nothing
      n_first = n = second = 0;
      return;
    }
    const int lo = max(s.low(p_lo), s.start);
    const int sink = min(s.sink_end, p_hi + 1);  // (no row sees past itself)
    n_first = sink > s.start ? (sink - 1) / kKeys + 1 - first : 0;
    second = max(lo / kKeys, first + n_first);
    n = n_first + max(0, p_hi / kKeys + 1 - second);
  }
  __device__ __forceinline__ int at(int i) const { return uni(kKeys * (i < n_first ? first + i : second + i - n_first)); }
};

// blockIdx -> item so that consecutive items, which share keys, go to one XCD
// (workgroups are dealt to the 8 XCDs, each with its own L2, one after another)
__device__ __forceinline__ int xcd_item(int x, int n) {
  const int c = x & 7, q = n >> 3, r = n & 7;
  return c * q + min(c, r) + (x >> 3);
}

template <int D>
struct TileGeom {
  static constexpr int CH = D / 8;  // 16-byte chunks a row
  // Chunk places in LDS.  K's rows are read 16 bytes a lane, 8 rows at a time
  // from one column of chunks: the column is turned by the row, so that they
  // fall in different banks.  V's are read 4 rows x 32 bytes at a time.
  static __device__ __forceinline__ int k_at(int row, int c) { return (row * CH + (c ^ (row & 7))) * 16; }
  static __device__ __forceinline__ int v_at(int row, int c) { return (row * CH + (c ^ ((row & 3) << 1))) * 16; }
};

// PAIR: keys as the sum of two fp16, a product each.
template <int D, typename T, bool PAIR>
__global__ __launch_bounds__(kTileThreads, D <= 128 ? 2 : 1) void tqk_attn_tiles(AttnArgs a) {
  typedef typename Mma<T>::v8 v8;
  constexpr int kKeys = kTileKeys<D, PAIR>, NU = kKeys / 32, NP = PAIR ? 2 : 1;
  constexpr int CH = D / 8, NST = kKeys * CH / kTileThreads;  // 16-byte chunks a thread stages of K, and of V
  constexpr int ND = D / 32, NK = D / 16;
  constexpr int kBytes = kKeys * D * 2;
  using TG = TileGeom<D>;
  __shared__ __align__(16) uint8_t k0_s[NP * kBytes], v0_s[kBytes], k1_s[NP * kBytes], v1_s[kBytes];
  __shared__ int odd_s;  // an infinity or a NaN among the values that only some rows see

  const int tid = threadIdx.x, wave = uni(tid >> 6), lane = tid & 63, ln = lane & 31, lh = lane >> 5;
  const int Hq = a.d.n_q_heads, Hkv = a.d.n_kv_heads, gq = uni(Hq / Hkv);
  int item = xcd_item(blockIdx.x, gridDim.x);
  const int split = uni(item % a.n_splits);
  item /= a.n_splits;
  const int tile = uni(a.row_tiles - 1 - item % a.row_tiles);  // the last rows, which see most, first
  item /= a.row_tiles;
  const int h = uni(item % Hkv), b = uni(item / Hkv);
  const Seen s(a, b);

  // this lane's row
  const int row = tile * kTileRows + wave * kRows + ln;
  const int t = row / gq, qh = h * gq + row % gq;
  const bool inside = t < a.d.q_len, real = t < s.m;
  const int p = s.n - s.m + t, lo = s.low(p);
  // the positions of the workgroup's rows and of the wave's
  const int t_lo = uni(tile * kTileRows / gq), t_hi = min(uni((tile * kTileRows + kTileRows - 1) / gq), s.m - 1);
  const int w_lo = uni((tile * kTileRows + wave * kRows) / gq);
  const int w_hi = min(uni((tile * kTileRows + wave * kRows + kRows - 1) / gq), s.m - 1);
  const int p_lo = s.n - s.m + t_lo, p_hi = s.n - s.m + t_hi;
  const int wp_lo = s.n - s.m + w_lo, wp_hi = s.n - s.m + w_hi;
  const int b_lo = s.low(p_lo);                           // the first key that a row of the workgroup sees by its window
  const int wl_lo = s.low(wp_lo), wl_hi = s.low(wp_hi);   // the wave's rows' first and last window start

  const Tiles<kKeys> tiles(s, p_lo, p_hi);
  int i0 = 0, i1 = t_lo < s.m ? tiles.n : 0;
  if (a.n_splits > 1) {
    const int n = i1;
    i0 = uni((int)((long long)n * split / a.n_splits));
    i1 = uni((int)((long long)n * (split + 1) / a.n_splits));
  }

  // Q^T as the second operand: row ln, channels 16 ks + 8 lh .. + 7
  v8 qf[NK];
  {
    const T* qp = static_cast<const T*>(a.q) + b * a.d.q_stride[0] + (long long)min(qh, Hq - 1) * a.d.q_stride[1] +
                  (long long)min(t, a.d.q_len - 1) * a.d.q_stride[2] + 8 * lh;
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) qf[ks] = *reinterpret_cast<const v8*>(qp + 16 * ks);
  }
  const float c = a.d.sm_scale * 1.4426950408889634f;  // scores in log2 units

  f16v_t O[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[i][r] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;  // (l_run: this lane's keys only)

  // A tile goes straight into LDS, 16 bytes a lane and no registers: thread tid
  // fills places tid + 256 i, rows 256 / CH apart, from the chunk that belongs
  // there.  The buffer resource starts at the tile's first row and ends with
  // the last key: rows past it are not read.
  const long long ks_ = a.d.k_stride[2] * 2, vs_ = a.d.v_stride[2] * 2;
  const char* const kb = static_cast<const char*>(a.k) + 2 * (b * a.d.k_stride[0] + h * a.d.k_stride[1]);
  const char* const lb = PAIR ? static_cast<const char*>(a.k_lo) + 2 * (b * a.d.k_stride[0] + h * a.d.k_stride[1]) : kb;
  const char* const vb = static_cast<const char*>(a.v) + 2 * (b * a.d.v_stride[0] + h * a.d.v_stride[1]);
  const KeptRows kept(s.n, s.m, s.start, s.sink_end, s.window);
  const int gap = a.compact ? uni(kept.gap) : 0, sink_rows = uni(kept.sinks);
  const int my_row = tid / CH, my_ch = tid % CH;
  const uint32_t k_off = (uint32_t)my_row * (uint32_t)ks_ + 16u * (uint32_t)(TG::k_at(my_row, my_ch) / 16 % CH);
  const uint32_t v_off = (uint32_t)my_row * (uint32_t)vs_ + 16u * (uint32_t)(TG::v_at(my_row, my_ch) / 16 % CH);
  // whether every row of the workgroup sees the whole tile
  auto whole = [&](int k0) {
    return k0 + kKeys - 1 <= p_lo && k0 >= s.start && (k0 >= s.low(p_hi) || k0 + kKeys <= s.sink_end);
  };
  auto load_tile = [&](uint8_t* kd, uint8_t* vd, int k0) {
    const long long r0 = k0 - (k0 >= sink_rows ? gap : 0);
    const long long rows = min(kKeys, s.n - k0);
    const __amdgpu_buffer_rsrc_t rk = tile_rsrc(kb + r0 * ks_, (rows - 1) * ks_ + 2 * D);
    const __amdgpu_buffer_rsrc_t rl = tile_rsrc(lb + r0 * ks_, (rows - 1) * ks_ + 2 * D);
    const __amdgpu_buffer_rsrc_t rv = tile_rsrc(vb + r0 * vs_, (rows - 1) * vs_ + 2 * D);
#pragma unroll
    for (int i = 0; i < NST; ++i) {
      typedef __attribute__((address_space(3))) void* lds;
      // (the whole offset in the operand that is held against the resource's end: the
      // scalar one is not, and a last tile of few rows ends before most steps)
      const int step = i * (kTileThreads / CH), at = 16 * kTileThreads * i + 1024 * wave;
      const int ko = (int)(k_off + (uint32_t)step * (uint32_t)ks_), vo = (int)(v_off + (uint32_t)step * (uint32_t)vs_);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds)(kd + at), 16, ko, 0, 0, 0);
      if constexpr (PAIR) __builtin_amdgcn_raw_ptr_buffer_load_lds(rl, (lds)(kd + kBytes + at), 16, ko, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds)(vd + at), 16, vo, 0, 0, 0);
    }
  };
  // The tile has arrived (every wave waits for its own loads).  Values that no
  // row of the workgroup sees count as zero, and an infinity or a NaN that some
  // rows see and others do not is set aside (a weight of zero times one of them
  // is no zero): a thread mends the chunks that it loaded.
  auto mend_tile = [&](uint8_t* vd, int k0) {
    if (whole(k0)) return;
#pragma unroll 1
    for (int i = 0; i < NST; ++i) {
      u4_t* x = reinterpret_cast<u4_t*>(vd + 16 * (tid + kTileThreads * i));
      const int j = k0 + my_row + i * (kTileThreads / CH);
      if (!s.sees(p_hi, b_lo, j)) {
        *x = u4_t{0u, 0u, 0u, 0u};
      } else if (not_finite<T>(*x)) {
        *x = only_finite<T>(*x);
        odd_s = 1;
      }
    }
  };
  auto attend_tile = [&](const uint8_t* k_t, const uint8_t* v_t, int k0) {
    // (a tile that none of the wave's rows sees: only its staging)
    if (!(w_lo < s.m && k0 <= wp_hi && (k0 + kKeys > wl_lo || k0 < s.sink_end))) return;
    // K Q^T: keys k0 + 32 u + 8 (r / 4) + 4 lh + r % 4 of row ln
    f16v_t S[NU];
    // (the reads run a few products ahead: a read's latency is several products)
    constexpr int kAhead = 4;
    v8 kf[NU * NK * NP];
#pragma unroll
    for (int i = 0; i < NU * NK * NP + kAhead; ++i) {
      if (i < NU * NK * NP) {  // (the second halves first)
        const int x = i / NP, half = NP - 1 - i % NP;
        kf[i] = *reinterpret_cast<const v8*>(k_t + half * kBytes + TG::k_at(32 * (x / NK) + ln, 2 * (x % NK) + lh));
      }
      if (i >= kAhead) {
        const int x = (i - kAhead) / NP, u = x / NK, ks = x % NK;
        if (ks == 0 && (i - kAhead) % NP == 0) S[u] = Mma<T>::m32(kf[i - kAhead], qf[ks], f16v_t{});
        else S[u] = Mma<T>::m32(kf[i - kAhead], qf[ks], S[u]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!(k0 + kKeys - 1 <= wp_lo && k0 >= s.start && (k0 >= wl_hi || k0 + kKeys <= s.sink_end))) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = k0 + 32 * u + 8 * (r / 4) + 4 * lh + r % 4;
          S[u][r] = s.sees(p, lo, j) ? S[u][r] : -INFINITY;
        }
    }
    float mx = S[0][0];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[u][r]);
    mx = max_half(mx) * c;
    if (__any(mx > m_run + kLazy)) {
      const float m_new = fmaxf(m_run, mx);
      const float f = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= f;
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[i][r] *= f;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    // V^T P^T, 16 keys a product; the weights rounded to the inputs' type
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        v8 pf;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = __builtin_amdgcn_exp2f(fmaf(S[u][8 * g + e], c, -m_use));
          pf[e] = (T)w;
          // (PAIR: the rounded weights, whose roundings cancel where few tokens weigh:
          // 6% of the error and 3% of the time; not where the keys' own is larger)
          l_run += PAIR ? (float)pf[e] : w;
        }
        // the lane's part of a transposing read: row ln % 16 / 4 of four, channels 4 (ln % 4)
        const int r0 = 32 * u + 16 * g + 4 * lh + (ln % 16) / 4;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          const int cc = 4 * i + 2 * (ln / 16) + (ln % 4) / 2;
          typedef __attribute__((address_space(3))) s4_t* lds4;
          const s4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(v_t + TG::v_at(r0, cc) + 8 * (ln % 2)));
          const s4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(v_t + TG::v_at(r0 + 8, cc) + 8 * (ln % 2)));
          const s8_t xy = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
          O[i] = Mma<T>::m32(__builtin_bit_cast(v8, xy), pf, O[i]);
        }
      }
  };

  if (tid == 0) odd_s = 0;
  __syncthreads();
  if (i0 < i1) {
    load_tile(k0_s, v0_s, tiles.at(i0));
    wait_loads();
    mend_tile(v0_s, tiles.at(i0));
  }
  __syncthreads();
  // two tiles a round, each in LDS of its own: one is computed while the next arrives
  for (int it = i0; it < i1; it += 2) {
    if (it + 1 < i1) load_tile(k1_s, v1_s, tiles.at(it + 1));
    attend_tile(k0_s, v0_s, tiles.at(it));
    if (it + 1 >= i1) break;
    wait_loads();
    mend_tile(v1_s, tiles.at(it + 1));
    __syncthreads();
    if (it + 2 < i1) load_tile(k0_s, v0_s, tiles.at(it + 2));
    attend_tile(k1_s, v1_s, tiles.at(it + 1));
    if (it + 2 < i1) {
      wait_loads();
      mend_tile(v0_s, tiles.at(it + 2));
    }
    __syncthreads();
  }

  const float l = sum_half(l_run);
  // a result that is not finite beside a sum that is: an infinity or a NaN among the
  // values of a whole tile, which a weight that rounds to zero may have turned into a NaN
  float zero = 0.f;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) zero = fmaf(O[i][r], 0.f, zero);
  const bool lost = __any(real && zero != 0.f && l == l);
  if (__builtin_expect(odd_s != 0 || lost, 0)) {
    // the infinities and NaN that a row sees are its result in their channels,
    // whatever their positive weights
    f16v_t odd[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) odd[i] = f16v_t{};
    for (int it = i0; it < i1; ++it) {
      const int k0 = tiles.at(it), rows = min(kKeys, s.n - k0);
      if (!lost && whole(k0)) continue;
      const char* const vt = vb + (k0 - (k0 >= sink_rows ? gap : 0)) * vs_;
      bool has = false;
      for (int x = lane; x < rows * CH; x += 64)
        has |= not_finite<T>(*reinterpret_cast<const u4_t*>(vt + x / CH * vs_ + 16 * (x % CH)));
      if (!__any(has)) continue;
      for (int j = 0; j < rows; ++j) {
        const bool vis = s.sees(p, lo, k0 + j);
        const T* vr = reinterpret_cast<const T*>(vt + j * vs_) + 4 * lh;
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            typedef T v4 __attribute__((ext_vector_type(4)));
            const v4 x = *reinterpret_cast<const v4*>(vr + 32 * i + 2 * r);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = (float)x[e];
              odd[i][r + e] += vis && !(fabsf(y) < INFINITY) ? y : 0.f;
            }
          }
      }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) O[i][r] = odd[i][r] == 0.f ? O[i][r] : odd[i][r];
  }

  if (!inside) return;
  if (a.n_splits == 1) {
    // rows that see nothing, and those past the sequence's queries: zero
    const float inv = real && l != 0.f ? 1.0f / l : 0.f;
    const bool dead = !real || l == 0.f;
    T* op = static_cast<T*>(a.out) + b * a.d.o_stride[0] + (long long)qh * a.d.o_stride[1] +
            (long long)t * a.d.o_stride[2] + 4 * lh;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        typedef T v4 __attribute__((ext_vector_type(4)));
        v4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (T)(dead ? 0.f : O[i][r + e] * inv);
        *reinterpret_cast<v4*>(op + 32 * i + 2 * r) = y;
      }
  } else {
    const long long at = (long long)split * a.rows + ((long long)b * Hq + qh) * a.d.q_len + t;
    if (lh == 0) {
      a.part_ml[2 * at] = m_run;
      a.part_ml[2 * at + 1] = real ? l : 0.f;
    }
    float* op = a.part_acc + at * D + 4 * lh;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<float4*>(op + 32 * i + 2 * r) = make_float4(O[i][r], O[i][r + 1], O[i][r + 2], O[i][r + 3]);
  }
}

// The splits of a row joined: one wave a row, D / 64 channels a lane.
template <int D, typename T>
__global__ __launch_bounds__(256) void tqk_attn_join(AttnArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  // every split's numbers by a lane of its own, then all accumulators in flight
  const bool in = lane < a.n_splits;
  const float2 ml = in ? *reinterpret_cast<const float2*>(&a.part_ml[2 * (lane * a.rows + row)]) : make_float2(0.f, 0.f);
  const float m = ml.y != 0.f ? ml.x : -INFINITY, M = wave_reduce<true>(m);
  const float f = ml.y != 0.f ? __builtin_amdgcn_exp2f(m - M) : 0.f;
  const float l = wave_reduce<false>(ml.y * f);
  const uint64_t live = __builtin_amdgcn_ballot_w64(ml.y != 0.f);
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.n_splits; ++s) {
    const float g = __shfl(f, s, 64);
    const float* src = a.part_acc + (s * a.rows + row) * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e)  // (an infinity stays one, however far behind its split's weights are)
      acc[e] = live >> s & 1 ? (fabsf(src[e]) < INFINITY ? fmaf(src[e], g, acc[e]) : acc[e] + src[e]) : acc[e];
  }
  const int t = (int)(row % a.d.q_len);
  const long long bh = row / a.d.q_len;
  T* op = static_cast<T*>(a.out) + bh / a.d.n_q_heads * a.d.o_stride[0] + bh % a.d.n_q_heads * a.d.o_stride[1] +
          t * a.d.o_stride[2] + E * lane;
  const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = (T)(l != 0.f ? acc[e] * inv : 0.f);
}

constexpr int64_t kMostStride = 1 << 23;  // elements between tokens of keys and values

struct AttnPlan {
  int row_tiles, n_splits;
  long long rows, items;
  size_t ws_bytes;
};

// Most key tiles that a row tile reads.
long long most_tiles(const tqk_attn_desc& d) {
  const int gq = d.n_q_heads / d.n_kv_heads;
  const long long tokens = d.q_len < kTileRows / gq + 2 ? d.q_len : kTileRows / gq + 2;
  long long keys = d.kv_len;
  if (d.window > 0 && d.window < d.kv_len) {
    keys = (long long)d.window + tokens + d.sinks + 2 * kMaxKeys;
    if (keys > d.kv_len) keys = d.kv_len;
  }
  const int tile = d.head_dim == 256 ? kTileKeys<256> : kTileKeys<128>;
  return (keys + tile - 1) / tile + 1;
}

AttnPlan make_plan(const tqk_attn_desc& d) {
  AttnPlan pl{};
  const int gq = d.n_q_heads / d.n_kv_heads;
  pl.rows = (long long)d.batch * d.n_q_heads * d.q_len;
  pl.row_tiles = (int)(((long long)d.q_len * gq + kTileRows - 1) / kTileRows);
  const long long pairs = (long long)d.batch * d.n_kv_heads * pl.row_tiles;
  // Few row tiles: the keys of each are split until the workgroups fill the
  // chip once (two a CU up to head_dim 128), at least four key tiles a split.
  const long long slots = (d.head_dim <= 128 ? 2 : 1) * (long long)device_cus();
  long long splits = 1;
  if (pairs * 2 <= slots) {
    splits = slots / pairs;
    const long long most = most_tiles(d) / 4;
    if (splits > most) splits = most;
    if (splits > 64) splits = 64;
    if (splits < 1) splits = 1;
  }
  pl.n_splits = (int)splits;
  pl.items = pairs * splits;
  pl.ws_bytes = splits > 1 ? (size_t)splits * pl.rows * (d.head_dim + 2) * sizeof(float) + 256 : 0;
  return pl;
}

int check_attn(const tqk_attn_desc* d) {
  if (!d) return TQK_EINVAL;
  if (!head_dim_ok(d->head_dim)) return TQK_EUNSUPPORTED;
  if (d->type != 1 && d->type != 2) return TQK_EUNSUPPORTED;
  if (d->batch < 0 || d->q_len < 0 || d->kv_len < 0 || d->window < 0 || d->sinks < 0) return TQK_EINVAL;
  if (d->q_len > (1 << 28) || d->kv_len > (1 << 30)) return TQK_EINVAL;
  if (d->n_q_heads < 1 || d->n_kv_heads < 1 || d->n_q_heads % d->n_kv_heads) return TQK_EINVAL;
  if (d->n_q_heads > 1024) return TQK_EUNSUPPORTED;
  if ((long long)d->q_len * (d->n_q_heads / d->n_kv_heads) > (1LL << 30)) return TQK_EINVAL;
  if (!(d->sm_scale > 0.f)) return TQK_EINVAL;  // (and not a NaN)
  for (int i = 0; i < 3; ++i)  // 16-byte accesses
    if (d->q_stride[i] % 8 || d->k_stride[i] % 8 || d->v_stride[i] % 8 || d->o_stride[i] % 8) return TQK_EINVAL;
  // (a key tile's rows within 32-bit byte offsets)
  if (d->k_stride[2] < 0 || d->v_stride[2] < 0 || d->k_stride[2] > kMostStride || d->v_stride[2] > kMostStride)
    return TQK_EINVAL;
  // (256 threads a workgroup: fewer than 2^32)
  if (d->batch && d->q_len && make_plan(*d).items > (1LL << 23)) return TQK_EINVAL;
  return TQK_OK;
}

template <int D, typename T>
void launch_tiles(const AttnArgs& a, long long items, hipStream_t st) {
  if constexpr (__is_same(T, _Float16)) {
    if (a.k_lo) hipLaunchKernelGGL((tqk_attn_tiles<D, T, true>), dim3((unsigned)items), dim3(kTileThreads), 0, st, a);
    else hipLaunchKernelGGL((tqk_attn_tiles<D, T, false>), dim3((unsigned)items), dim3(kTileThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL((tqk_attn_tiles<D, T, false>), dim3((unsigned)items), dim3(kTileThreads), 0, st, a);
  }
  if (a.n_splits > 1)
    hipLaunchKernelGGL((tqk_attn_join<D, T>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a);
}
template <typename T>
void launch_tiles(const AttnArgs& a, long long items, hipStream_t st) {
  if (a.d.head_dim == 64)
    launch_tiles<64, T>(a, items, st);
  else if (a.d.head_dim == 128)
    launch_tiles<128, T>(a, items, st);
  else
    launch_tiles<256, T>(a, items, st);
}

}  // namespace

extern "C" {

size_t tqk_attention_workspace_bytes(const tqk_attn_desc* d) {
  if (check_attn(d) != TQK_OK) return 0;
  if (!d->batch || !d->q_len) return 0;
  return make_plan(*d).ws_bytes;
}

int tqk_attention(const tqk_attn_desc* d, const void* q, const void* k, const void* v,
                  const int32_t* kv_lens, const int32_t* q_lens, const int32_t* kv_starts, void* out,
                  void* workspace, size_t workspace_bytes, void* stream) {
  return tqk_run_attention(d, q, k, v, kv_lens, q_lens, kv_starts, out, workspace, workspace_bytes, 0, nullptr, stream);
}

}  // extern "C"

int tqk_run_attention(const tqk_attn_desc* d, const void* q, const void* k, const void* v, const int32_t* kv_lens,
                      const int32_t* q_lens, const int32_t* kv_starts, void* out, void* workspace,
                      size_t workspace_bytes, int compact, const void* k_lo, void* stream) {
  const int rc = check_attn(d);
  if (rc != TQK_OK) return rc;
  if (!d->batch || !d->q_len) return TQK_OK;
  if (!q || !out || (d->kv_len && (!k || !v))) return TQK_EINVAL;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) return TQK_EINVAL;
  const AttnPlan pl = make_plan(*d);
  if (pl.ws_bytes && (!workspace || workspace_bytes < pl.ws_bytes || ((uintptr_t)workspace & 15)))
    return TQK_EWORKSPACE;
  AttnArgs a{};
  a.d = *d;
  a.q = q;
  a.k = k;
  a.v = v;
  a.k_lo = k_lo;
  a.kv_lens = kv_lens;
  a.q_lens = q_lens;
  a.kv_starts = kv_starts;
  a.out = out;
  a.row_tiles = pl.row_tiles;
  a.n_splits = pl.n_splits;
  a.rows = pl.rows;
  a.compact = compact;
  // the accumulators first: 16-byte stores
  a.part_acc = static_cast<float*>(workspace);
  a.part_ml = a.part_acc + (size_t)pl.n_splits * pl.rows * d->head_dim;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (d->type == 1)
    launch_tiles<_Float16>(a, pl.items, st);
  else
    launch_tiles<__bf16>(a, pl.items, st);
  return hipGetLastError() == hipSuccess ? TQK_OK : TQK_EHIP;
}
