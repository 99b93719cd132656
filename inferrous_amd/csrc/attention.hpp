// attention.hpp -- what the kernels between the qkv and the o projection share:
// the cache's layout, the packed batch's sequences, and BF16 helpers.
#pragma once
#include "internal.hpp"
#include "tile_stream.hpp"

namespace w8a8 {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
// A maximum before the first score.  Finite, so that scores of -inf (f32 overflows) weigh nothing.
constexpr float kNoScore = -3.402823466e38f;

// Two f32 values as BF16, nearest even, NaN kept (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const v2bf p = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// An output value as f32 holding its BF16 value.
__device__ __forceinline__ float as_bf16(float a) { return bf16_lo(pack_bf16(a, 0.f)); }

// 2^x, x a finite exponent below 128 or -inf (v_exp_f32; results below 2^-126 are 0).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Division of an x below 2^24 by a d below 2^16: with e = inverse * d - 2^40 < d, x * e is
// below 2^40.  (near: of an x below 2^11 by a d up to 2^10, the same with 2^21.)  The
// kernels' code is fetched anew by each launch, and a division is about 40 instructions.
struct Divisor {
  uint32_t d, near_inverse;
  uint64_t inverse;
  explicit Divisor(uint32_t by) : d(by), near_inverse(((1u << 21) + by - 1) / by), inverse(((1ull << 40) + by - 1) / by) {}
  __device__ __forceinline__ uint32_t of(uint32_t x) const { return (uint32_t)(x * inverse >> 40); }
  __device__ __forceinline__ uint32_t near(uint32_t x) const { return x * near_inverse >> 21; }
};

// Rows [lo, hi) of sequence i of a batch of m rows.  Whatever `starts` holds,
// the range stays within the batch.
struct RowRange {
  uint32_t lo, hi;
};
__device__ __forceinline__ RowRange rows_of(const int32_t* starts, uint32_t i, uint32_t m) {
  if (!starts) return {0u, m};
  const int32_t a = starts[i], b = starts[i + 1];
  const uint32_t lo = a < 0 ? 0u : min((uint32_t)a, m), hi = b < 0 ? 0u : min((uint32_t)b, m);
  return {lo, max(lo, hi)};
}

// The unit-th of the units that sequences 0 .. n - 1 have count(i) of, in order:
// its sequence and its place there, the same in every lane.  False if there are
// fewer.  Whole waves call it; a wave looks at 64 sequences at a time.
template <class Count>
__device__ __forceinline__ bool find_unit(uint32_t unit, uint32_t n, Count count, uint32_t* seq, uint32_t* index) {
  if (n == 1) {
    *seq = 0;
    *index = unit;
    return unit < count(0u);
  }
  const int lane = threadIdx.x & 63;
  for (uint32_t base = 0; base < n; base += 64) {
    const uint32_t c = base + lane < n ? count(base + lane) : 0u;
    uint32_t sum = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t below = (uint32_t)__shfl_up((int)sum, o, kWave);
      sum += lane >= o ? below : 0u;
    }
    const uint64_t past = __ballot(sum > unit);
    if (past) {
      const int at = __builtin_ctzll(past);
      *seq = base + at;
      *index = unit - (uint32_t)__builtin_amdgcn_readlane((int)(sum - c), at);
      return true;
    }
    unit -= (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
  return false;
}

}  // namespace w8a8
