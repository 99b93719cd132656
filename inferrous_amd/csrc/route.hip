// route.hip -- the router of a layer of experts: logits to expert ids and
// weights.  No counterpart in the reference, whose layers are dense.
//
//   s = softmax(x) or 1 / (1 + exp(-x)) over a row of logits x[E];
//   c = s + bias (the bias counts in the choice only);
//   an expert whose logit is -inf or NaN, or whose c is NaN or -inf, is out;
//   with groups, a group's score is the largest c of its live experts or the
//   sum of the two largest, and only the experts of the top_groups best
//   groups stay;
//   the k largest c are chosen, equal ones lowest index first; slots that no
//   live expert is left for get id -1 and weight 0;
//   weight = s of the chosen (divided by the chosen ones' sum) * scale.
// Every score, sum and weight is held in f32.
#include "internal.hpp"
#include "routed_common.hpp"

namespace w8a8 {

// Order of choice: larger keys first.  0 is an expert that is out; -0 ties
// with +0.
__device__ __forceinline__ uint32_t choice_key(float c) {
  const uint32_t u = __float_as_uint(c + 0.0f);
  if (c != c || u == 0xff800000u) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kRouteWaves = 4;

// One wave per row, lane l holding experts l, l + 64, ... (NE of them).
template <int NE>
__global__ __launch_bounds__(64 * kRouteWaves) void route_rows(RouteArgs a) {
  __shared__ float sh[kRouteWaves][2 * 64 * NE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t row = blockIdx.x * kRouteWaves + wave;
  if (row >= a.m) return;  // the waves of a workgroup share nothing
  float* const score = sh[wave];
  float* const choice = sh[wave] + 64 * NE;
  const float ninf = -__builtin_inff();
  float x[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const uint32_t e = 64 * i + lane;
    x[i] = ninf;
    if (e < a.experts) {
      const size_t o = (size_t)row * a.experts + e;
      x[i] = a.bf16 ? __uint_as_float((uint32_t)((const uint16_t*)a.logits)[o] << 16) : ((const float*)a.logits)[o];
      if (x[i] != x[i]) x[i] = ninf;
    }
  }
  float s[NE];
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < NE; ++i) s[i] = 1.0f / (1.0f + expf(-x[i]));
  } else {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < NE; ++i) top = fmaxf(top, x[i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      // infinite logits share the row; a row that is all out has no score
      s[i] = x[i] == top ? (top == ninf ? 0.0f : 1.0f) : expf(x[i] - top);
      if (x[i] == ninf) s[i] = 0.f;
      sum += s[i];
    }
    sum = wave_sum_f32(sum);
#pragma unroll
    for (int i = 0; i < NE; ++i) s[i] = sum > 0.f ? s[i] / sum : 0.f;
  }
  uint32_t key[NE];
  float c[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const uint32_t e = 64 * i + lane;
    c[i] = s[i];
    if (a.bias && e < a.experts) c[i] = s[i] + a.bias[e];
    if (x[i] == ninf) c[i] = ninf;
    key[i] = choice_key(c[i]);
    score[e] = s[i];
    choice[e] = key[i] ? c[i] : ninf;
  }
  // this wave's own LDS writes, read back by its other lanes
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (a.groups > 1) {
    const uint32_t per = a.experts / a.groups;
    float best = ninf, second = ninf;
    if ((uint32_t)lane < a.groups)
      for (uint32_t j = 0; j < per; ++j) {
        const float v = choice[lane * per + j];
        if (v > best) second = best, best = v;
        else if (v > second) second = v;
      }
    const float group = a.group_top == 2 && second > ninf ? best + second : best;
    const uint32_t gk = choice_key(group);
    uint32_t ahead = 0;
    for (uint32_t g = 0; g < a.groups; ++g) {
      const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)gk, (int)g);
      ahead += other > gk || (other == gk && g < (uint32_t)lane);
    }
    const uint64_t keep = __ballot((uint32_t)lane < a.groups && ahead < a.top_groups);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const uint32_t e = 64 * i + lane;
      if (e < a.experts && !((keep >> (e / per)) & 1)) key[i] = 0;
    }
  }
  // k rounds: the largest key of the wave, then its lowest index
  int32_t id = -1;
  for (uint32_t j = 0; j < a.k; ++j) {
    uint32_t mine = key[0], at = lane;
#pragma unroll
    for (int i = 1; i < NE; ++i)
      if (key[i] > mine) mine = key[i], at = 64 * i + lane;
    const uint32_t top = wave_max_u32(mine);
    if (top == 0) break;
    const uint32_t e = ~wave_max_u32(mine == top ? ~at : 0u);
    if ((uint32_t)lane == j) id = (int32_t)e;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (64 * i + lane == e) key[i] = 0;
  }
  float w = id >= 0 ? score[id] : 0.f;
  if (a.renorm) {
    const float sum = wave_sum_f32(w);
    w = sum > 0.f ? w / sum : 0.f;
  }
  if ((uint32_t)lane < a.k) {
    a.ids[(size_t)row * a.k + lane] = id;
    a.weights[(size_t)row * a.k + lane] = w * a.scale;
  }
}

hipError_t launch_route(hipStream_t st, const RouteArgs& a) {
  const uint32_t grid = (a.m + kRouteWaves - 1) / kRouteWaves;
  auto k = a.experts <= 64    ? route_rows<1>
           : a.experts <= 128 ? route_rows<2>
           : a.experts <= 256 ? route_rows<4>
           : a.experts <= 512 ? route_rows<8>
                              : route_rows<16>;
  hipLaunchKernelGGL(k, dim3(grid), dim3(64 * kRouteWaves), 0, st, a);
  return hipGetLastError();
}

}  // namespace w8a8
