// Cross-lane helpers of the attention kernels.
#pragma once

#include <type_traits>

#include "tqk_common.h"

namespace {

// The wave's sum or maximum in every lane, on the VALU (rotations inside the
// 16-lane rows, then the two permlane swaps): a butterfly of ds_bpermute is six
// LDS round trips in a row.
template <bool IS_MAX>
__device__ __forceinline__ float wave_reduce(float x) {
  auto op = [](float a, float b) { return IS_MAX ? fmaxf(a, b) : a + b; };
  auto ror = [](float v, auto n) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + decltype(n)::value,
                                                                 0xF, 0xF, true));
  };
  x = op(x, ror(x, std::integral_constant<int, 8>{}));
  x = op(x, ror(x, std::integral_constant<int, 4>{}));
  x = op(x, ror(x, std::integral_constant<int, 2>{}));
  x = op(x, ror(x, std::integral_constant<int, 1>{}));
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r16 = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = op(__builtin_bit_cast(float, (uint32_t)r16[0]), __builtin_bit_cast(float, (uint32_t)r16[1]));
  const uint32_t w = __builtin_bit_cast(uint32_t, x);
  const auto r32 = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return op(__builtin_bit_cast(float, (uint32_t)r32[0]), __builtin_bit_cast(float, (uint32_t)r32[1]));
}

// A positive weight that fp32 holds as zero, as its smallest normal number: what an
// infinity needs to stay one, and nothing to a finite value.
__device__ __forceinline__ float above_zero(float w) { return w < 0x1p-126f ? 0x1p-126f : w; }

// two floats as fp16 pairs: {hi, hi}, {lo, lo}
__device__ __forceinline__ uint2 split_pair(float x0, float x1) {
  const _Float16 h0 = (_Float16)x0, h1 = (_Float16)x1;
  const _Float16 l0 = (_Float16)(x0 - (float)h0), l1 = (_Float16)(x1 - (float)h1);
  return make_uint2((uint32_t)__builtin_bit_cast(uint16_t, h0) |
                        ((uint32_t)__builtin_bit_cast(uint16_t, h1) << 16),
                    (uint32_t)__builtin_bit_cast(uint16_t, l0) |
                        ((uint32_t)__builtin_bit_cast(uint16_t, l1) << 16));
}

// Workgroup barrier for LDS data only: this wave's LDS operations complete
// (lgkmcnt 0), then s_barrier.  Unlike __syncthreads it leaves the wave's
// global loads in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // vmcnt 63, expcnt 7, lgkmcnt 0
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Orders LDS accesses of one wave across lanes.  A wave's LDS instructions
// execute in issue order, so program order is enough; this only stops the
// compiler from moving memory operations across the point (and, unlike a
// fence, does not wait for the wave's outstanding global loads).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

// Cross-lane helpers without LDS traffic.
__device__ __forceinline__ uint32_t fbits(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float bitsf(uint32_t x) { return __builtin_bit_cast(float, x); }
// max / sum over lanes {l, l^16, l^32, l^48}: the four token groups of a column
__device__ __forceinline__ float colgroup_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(fbits(x), fbits(x), false, false);
  x = fmaxf(bitsf(a[0]), bitsf(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(fbits(x), fbits(x), false, false);
  return fmaxf(bitsf(b[0]), bitsf(b[1]));
}
__device__ __forceinline__ float colgroup_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(fbits(x), fbits(x), false, false);
  x = bitsf(a[0]) + bitsf(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(fbits(x), fbits(x), false, false);
  return bitsf(b[0]) + bitsf(b[1]);
}
// fp16 pair (RNE) of two floats in one dword
__device__ __forceinline__ uint32_t pk_f16(float x, float y) {
  typedef float float2_t __attribute__((ext_vector_type(2)));
  typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
  const half2_t hv = __builtin_convertvector((float2_t){x, y}, half2_t);
  return __builtin_bit_cast(uint32_t, hv);
}
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

}  // namespace
