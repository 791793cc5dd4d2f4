// Head norms, position rotation and the cache's head-major layout in one pass
// over the projection rows of new tokens (gfx950).
//
//   x^  = x * rsqrt(mean(x^2) + eps) * (w + offset)       queries and keys, optional
//   y_a = s (x^_a cos(p f_i) - x^_b sin(p f_i))
//   y_b = s (x^_b cos(p f_i) + x^_a sin(p f_i))           the pair (a, b) of frequency i
// with (a, b) = (i, i + R/2) or (2i, 2i + 1) over the first R channels; values
// are converted only.  Everything between the load and the store is fp32, the
// angle excepted: p f_i reaches 1e6 radians, where fp32 is 0.06 radians off, so
// it is taken in turns in 64 bits and only its fraction goes on in fp32.
//
// Bound: HBM, every element is read once and written once.  A wave takes one
// token (or, with few tokens, a part of its heads): its lanes compute the
// token's R/2 rotations once, one or two each, and hand them round through the
// wave's own LDS; then 64 lanes take 512 channels at a time, 8 a lane.  Four prompts
// of 8192 tokens, 32 query and 8 kv heads of 128, bf16 to fp16: 157 us, 5.1 TB/s (a
// large copy: 4.9); 16 single tokens: 4.2 us of a call's 15 on the host.
#include "tqk_common.h"

namespace {

constexpr int kRopeWaves = 4;    // waves a workgroup, each on its own
constexpr int kRopeUnroll = 4;   // rows of loads in flight a lane
constexpr int kRopeMaxBlocks = 1 << 20;

struct RopeArgs {
  tqk_rope_desc d;
  const void* qkv;
  const void* positions;
  const float* inv_freq;
  const void* q_weight;
  const void* k_weight;
  void* q;
  void* k;
  void* v;
  long long units;  // (token, part) pairs
  int parts;        // parts of a token's heads
  int part_rows;    // heads a part
};

// eight consecutive elements as fp32
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void load8(const _Float16* p, float (&x)[8]) {
  const h8_t a = *reinterpret_cast<const h8_t*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
}
__device__ __forceinline__ void load8(const __bf16* p, float (&x)[8]) {
  const bf8_t a = *reinterpret_cast<const bf8_t*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(_Float16* p, const float (&x)[8]) {
  h8_t a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (_Float16)x[i];
  *reinterpret_cast<h8_t*>(p) = a;
}
__device__ __forceinline__ void store8(__bf16* p, const float (&x)[8]) {
  bf8_t a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (__bf16)x[i];
  *reinterpret_cast<bf8_t*>(p) = a;
}

template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
// the sum over a head's lanes (D / 8 consecutive ones), in each of them
template <int D>
__device__ __forceinline__ float head_sum(float x) {
  x = add_dpp<0xB1>(x);   // quad_perm 1 0 3 2
  x = add_dpp<0x4E>(x);   // quad_perm 2 3 0 1
  x = add_dpp<0x141>(x);  // mirrored in eight lanes
  if constexpr (D >= 128) x = add_dpp<0x140>(x);  // mirrored in sixteen
  if constexpr (D >= 256) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  }
  return x;
}

template <int D, typename TI, typename TO, typename TW>
__global__ __launch_bounds__(64 * kRopeWaves) void tqk_norm_rope_rows(RopeArgs a) {
  constexpr int LPR = D / 8;       // lanes a head
  constexpr int RPW = 64 / LPR;    // heads a wave takes at a time
  const tqk_rope_desc& d = a.d;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane % LPR, lr = lane / LPR;
  const int Hq = d.n_q_heads, Hkv = d.n_kv_heads, T = d.tokens, R = d.rotary_dim;
  __shared__ float2 rot_s[kRopeWaves][D / 2];
  // this lane's weights: the same channels of every head
  float wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) wq[i] = wk[i] = 1.0f;
  if (a.q_weight) {
    load8(static_cast<const TW*>(a.q_weight) + 8 * li, wq);
#pragma unroll
    for (int i = 0; i < 8; ++i) wq[i] += d.weight_offset;
  }
  if (a.k_weight) {
    load8(static_cast<const TW*>(a.k_weight) + 8 * li, wk);
#pragma unroll
    for (int i = 0; i < 8; ++i) wk[i] += d.weight_offset;
  }
  // where the other half of this lane's pairs is (lanes past R: themselves)
  const bool rotated = 8 * li < R, second = 16 * li >= R;
  const int partner = !rotated || d.interleaved ? lane : second ? lane - R / 16 : lane + R / 16;

  for (long long unit = (long long)blockIdx.x * kRopeWaves + wave; unit < a.units;
       unit += (long long)gridDim.x * kRopeWaves) {
    const long long token = unit / a.parts;
    const int part = (int)(unit % a.parts);
    const int b = (int)(token / T), t = (int)(token % T);
    const long long pi = d.pos_per_token ? token : b;
    long long pos = d.pos_i64 ? static_cast<const long long*>(a.positions)[pi]
                              : (long long)static_cast<const int32_t*>(a.positions)[pi];
    if (!d.pos_per_token) pos += t;
    for (int i = lane; i < R / 2; i += 64) {
      const double turns = (double)pos * (double)a.inv_freq[i] * 0.15915494309189535;
      const float r = (float)(turns - rint(turns));
      float sn, cs;
      sincospif(2.0f * r, &sn, &cs);
      rot_s[wave][i] = make_float2(d.rope_scale * cs, d.rope_scale * sn);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // the rotations of this lane's eight channels: of pair 8 li + e (halves), or
    // of pairs 4 li + e / 2 (adjacent)
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = d.interleaved ? 4 * li + e / 2 : 8 * li + e - (second ? R / 2 : 0);
      const float2 c = rot_s[wave][rotated ? i : 0];
      cs[e] = rotated ? c.x : 1.0f;
      const bool minus = d.interleaved ? (e & 1) == 0 : !second;
      sn[e] = rotated ? (minus ? -c.y : c.y) : 0.0f;
    }
    __builtin_amdgcn_wave_barrier();  // read before the next token's are written
    const TI* row = static_cast<const TI*>(a.qkv) + b * d.batch_stride + t * d.token_stride;
    const int h_end = min((part + 1) * a.part_rows, Hq + 2 * Hkv);
    for (int h0 = part * a.part_rows; h0 < h_end; h0 += RPW * kRopeUnroll) {
      float x[kRopeUnroll][8];
#pragma unroll
      for (int u = 0; u < kRopeUnroll; ++u) {
        const int h = min(h0 + RPW * u + lr, h_end - 1);
        load8(row + (long long)h * D + 8 * li, x[u]);
      }
#pragma unroll
      for (int u = 0; u < kRopeUnroll; ++u) {
        const int h = h0 + RPW * u + lr;
        if (h0 + RPW * u >= h_end) break;
        const bool is_q = h < Hq, is_k = !is_q && h < Hq + Hkv;
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[u][e], x[u][e], ss);
        ss = head_sum<D>(ss);
        const bool norm = (is_q && a.q_weight) || (is_k && a.k_weight);
        // (the correctly rounded root and quotient: the norm is one number a head)
        const float inv = norm ? 1.0f / __builtin_sqrtf(ss * (1.0f / D) + d.eps) : 1.0f;
        float y[8], z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = norm ? x[u][e] * inv * (is_q ? wq[e] : wk[e]) : x[u][e];
        if (d.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = y[e ^ 1];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = __shfl(y[e], partner, 64);
        }
        // (past R: no rotation, whatever stands there)
        const bool turn = rotated && (is_q || is_k);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = turn ? fmaf(y[e], cs[e], z[e] * sn[e]) : y[e];
        if (h < h_end) {
          TO* out = is_q   ? static_cast<TO*>(a.q) + (((long long)b * Hq + h) * T + t) * D
                    : is_k ? static_cast<TO*>(a.k) + (((long long)b * Hkv + h - Hq) * T + t) * D
                           : static_cast<TO*>(a.v) + (((long long)b * Hkv + h - Hq - Hkv) * T + t) * D;
          store8(out + 8 * li, y);
        }
      }
    }
  }
}

template <int D, typename TI, typename TO>
void launch_rope_w(dim3 grid, hipStream_t st, const RopeArgs& a) {
  // weights in the rows' type or in fp32
  if (a.d.weight_type == 0)
    hipLaunchKernelGGL((tqk_norm_rope_rows<D, TI, TO, float>), grid, dim3(64 * kRopeWaves), 0, st, a);
  else
    hipLaunchKernelGGL((tqk_norm_rope_rows<D, TI, TO, TI>), grid, dim3(64 * kRopeWaves), 0, st, a);
}
template <int D, typename TI>
void launch_rope_o(dim3 grid, hipStream_t st, const RopeArgs& a) {
  if (a.d.out_type == 0)
    launch_rope_w<D, TI, float>(grid, st, a);
  else if (a.d.out_type == 1)
    launch_rope_w<D, TI, _Float16>(grid, st, a);
  else
    launch_rope_w<D, TI, __bf16>(grid, st, a);
}
template <int D>
void launch_rope(dim3 grid, hipStream_t st, const RopeArgs& a) {
  if (a.d.in_type == 0)
    launch_rope_o<D, float>(grid, st, a);
  else if (a.d.in_type == 1)
    launch_rope_o<D, _Float16>(grid, st, a);
  else
    launch_rope_o<D, __bf16>(grid, st, a);
}

bool type_ok(int t) { return t >= 0 && t <= 2; }

}  // namespace

extern "C" int tqk_norm_rope(const tqk_rope_desc* d, const void* qkv, const void* positions,
                             const float* inv_freq, const void* q_weight, const void* k_weight, void* q,
                             void* k, void* v, void* stream) {
  if (!d) return TQK_EINVAL;
  if (!head_dim_ok(d->head_dim)) return TQK_EUNSUPPORTED;
  if (d->batch < 0 || d->tokens < 0 || d->n_q_heads < 0 || d->n_kv_heads < 0) return TQK_EINVAL;
  if (d->n_q_heads > (1 << 20) || d->n_kv_heads > (1 << 20)) return TQK_EINVAL;
  if (!type_ok(d->in_type) || !type_ok(d->out_type)) return TQK_EINVAL;
  if (d->weight_type != 0 && d->weight_type != d->in_type) return TQK_EUNSUPPORTED;
  if (d->rotary_dim < 0 || d->rotary_dim > d->head_dim) return TQK_EINVAL;
  if (d->rotary_dim % 16) return TQK_EUNSUPPORTED;  // a lane's eight channels lie in one half
  if (d->pos_i64 < 0 || d->pos_i64 > 1 || d->pos_per_token < 0 || d->pos_per_token > 1 || d->interleaved < 0 ||
      d->interleaved > 1)
    return TQK_EINVAL;
  const int rows = d->n_q_heads + 2 * d->n_kv_heads;
  const long long tokens = (long long)d->batch * d->tokens;
  if (tokens == 0 || rows == 0) return TQK_OK;
  if (!qkv || !positions || (d->rotary_dim && !inv_freq)) return TQK_EINVAL;
  if ((d->n_q_heads && !q) || (d->n_kv_heads && (!k || !v))) return TQK_EINVAL;
  // 16-byte accesses
  const uintptr_t at = (uintptr_t)qkv | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_weight |
                       (uintptr_t)k_weight;
  if ((at & 15) || d->batch_stride % 8 || d->token_stride % 8) return TQK_EINVAL;
  RopeArgs a;
  a.d = *d;
  a.qkv = qkv;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.q = q;
  a.k = k;
  a.v = v;
  // With few tokens a token's heads go to several waves, down to the heads that
  // a wave takes at once, until there are 4 waves a SIMD.
  const int rpw = 64 / (d->head_dim / 8);
  const int steps = (rows + rpw - 1) / rpw;
  long long parts = (4096 + tokens - 1) / tokens;
  if (parts > steps) parts = steps;
  a.part_rows = (int)((steps + parts - 1) / parts) * rpw;
  a.parts = (rows + a.part_rows - 1) / a.part_rows;
  a.units = tokens * a.parts;
  const long long blocks = (a.units + kRopeWaves - 1) / kRopeWaves;
  const dim3 grid((unsigned)(blocks < kRopeMaxBlocks ? blocks : kRopeMaxBlocks));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (d->head_dim == 64)
    launch_rope<64>(grid, st, a);
  else if (d->head_dim == 128)
    launch_rope<128>(grid, st, a);
  else
    launch_rope<256>(grid, st, a);
  return hipGetLastError() == hipSuccess ? TQK_OK : TQK_EHIP;
}
