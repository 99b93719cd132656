// routed_common.hpp -- device helpers of the routed layers (route.hip,
// experts.hip, adapters.hip).
#pragma once
#include "device_common.hpp"

namespace w8a8 {

// Wave sums, returned wave-uniform; every lane of the wave must be active.  The
// additions' order is fixed: the DPP steps of wave_max_u32 inside the 16-lane
// rows, then the four rows in pairs.
__device__ __forceinline__ float wave_sum_f32(float v) {
  v += __uint_as_float(dpp_u32<0xB1>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<0x4E>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<0x141>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<0x140>(__float_as_uint(v)));
  const int u = __float_as_int(v);
  return (__int_as_float(__builtin_amdgcn_readlane(u, 0)) + __int_as_float(__builtin_amdgcn_readlane(u, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(u, 32)) + __int_as_float(__builtin_amdgcn_readlane(u, 48)));
}

__device__ __forceinline__ int wave_sum_i32(int v) {
  v += (int)dpp_u32<0xB1>((uint32_t)v);
  v += (int)dpp_u32<0x4E>((uint32_t)v);
  v += (int)dpp_u32<0x141>((uint32_t)v);
  v += (int)dpp_u32<0x140>((uint32_t)v);
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
         __builtin_amdgcn_readlane(v, 48);
}

// exp(x) as 2^(x log2 e) on v_exp_f32: the product's rounding error, which
// grows with |x|, is put back to first order.
__device__ __forceinline__ float exp_fast(float x) {
  const float t = x * 1.44269502f;
  const float lo = __builtin_fmaf(x, 1.44269502f, -t) + x * 1.92596303e-8f;  // log2 e in two parts
  const float e = __builtin_amdgcn_exp2f(t);
  // past the range of 2^t, where e is 0 or infinite, lo is no correction
  return e < __builtin_inff() && __builtin_fabsf(lo) < 1.0f ? __builtin_fmaf(e, lo * 0.693147182f, e) : e;
}

// exp(x) for x in [-128, 0], where the correction is small and neither part can
// overflow: exp_fast without its tests.
__device__ __forceinline__ float exp_above_m128(float x) {
  const float t = x * 1.44269502f;
  const float lo = __builtin_fmaf(x, 1.44269502f, -t) + x * 1.92596303e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, lo * 0.693147182f, e);
}

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// A BF16-valued output in its buffer's type.
__device__ __forceinline__ void store_routed(void* out, int out_dtype, size_t o, float v) {
  v = bf16_rne(v);
  if (out_dtype == W8A8_OUT_F32) ((float*)out)[o] = v;
  else ((uint16_t*)out)[o] = (uint16_t)(__float_as_uint(v) >> 16);
}

}  // namespace w8a8
