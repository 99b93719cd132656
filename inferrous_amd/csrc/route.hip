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
#include <type_traits>

#include "internal.hpp"
#include "routed_common.hpp"

namespace w8a8 {

// 1 / (1 + exp(-x)) to about two units of the last place: v_exp_f32 on a split
// product (exp_fast) and v_rcp_f32 with one Newton step, against 25 instructions
// of expf and a division.
__device__ __forceinline__ float sigmoid_f32(float x) {
  const float d = 1.0f + exp_fast(-x);
  const float r = __builtin_amdgcn_rcpf(d);
  return d < __builtin_inff() ? __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r) : 0.0f;
}

// Order of choice: larger keys first.  0 is an expert that is out; -0 ties
// with +0.
__device__ __forceinline__ uint32_t choice_key(float c) {
  const uint32_t u = __float_as_uint(c + 0.0f);
  if (c != c || u == 0xff800000u) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kRouteWaves = 4;

// One wave per row, lane l holding experts l, l + 64, ... (NE of them): more
// experts, groups or choices than route_quads takes.
// k rounds of whole-wave maxima bound it: 16384 rows of 384 experts, k = 8, 25 us (26 MB);
// 512 in 8 groups 46; 1024, k = 16, 92.
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
    for (int i = 0; i < NE; ++i) s[i] = sigmoid_f32(x[i]);
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
      s[i] = x[i] == top ? (top == ninf ? 0.0f : 1.0f) : exp_fast(x[i] - top);
      if (x[i] == ninf) s[i] = 0.f;
      sum += s[i];
    }
    sum = wave_sum_f32(sum);
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) s[i] *= inv;
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

// What bounds it is instructions: about 1900 a wave for its four rows.  16384 rows of
// 256 experts, k = 8, 4 of 8 groups: 11.7 us (17.8 MB; a copy of them takes 3.4); a wave
// a row, whose reductions serve one row each, 27.  64 rows: 6.3 us, the same chain
// once.
//
// 16 lanes a row, four rows a wave, lane l of a row holding its experts NV l ..
// NV l + NV - 1: a round's reductions are four DPP steps for four rows at once.
// For at most 16 NV = 256 experts, 16 groups and k <= 16.
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
  return __uint_as_float(dpp_u32<CTRL>(__float_as_uint(v)));
}
__device__ __forceinline__ float row_max_f32(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  return fmaxf(v, dpp_f32<0x140>(v));
}
__device__ __forceinline__ float row_sum_f32(float v) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x141>(v);
  return v + dpp_f32<0x140>(v);
}
__device__ __forceinline__ uint32_t row_min_u32(uint32_t v) {
  v = min(v, dpp_u32<0xB1>(v));
  v = min(v, dpp_u32<0x4E>(v));
  v = min(v, dpp_u32<0x141>(v));
  return min(v, dpp_u32<0x140>(v));
}
// The two largest of (a, b) and a lane at the other end of a DPP step.
template <int CTRL>
__device__ __forceinline__ void merge_two(float& a, float& b) {
  const float c = dpp_f32<CTRL>(a), d = dpp_f32<CTRL>(b);
  b = fmaxf(fminf(a, c), fmaxf(b, d));
  a = fmaxf(a, c);
}

// Lane (l + R) % 16's value, within the 16 lanes of a row.
template <int R>
__device__ __forceinline__ uint32_t row_rotate(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + R, 0xF, 0xF, false);  // row_ror
}
template <int R, class F>
__device__ __forceinline__ void each_rotation(F f) {
  if constexpr (R < 16) {
    f(std::integral_constant<int, R>{});
    each_rotation<R + 1>(f);
  }
}

template <int NV>
__global__ __launch_bounds__(256) void route_quads(RouteArgs a) {
  __shared__ __attribute__((aligned(16))) float sh[32][16 * NV];  // scores, choice scores
  __shared__ uint2 lists[16][16];                                 // a row's candidates: choice score, expert
  const int lane = threadIdx.x & 63, li = lane & 15;
  const uint32_t slot = threadIdx.x >> 4, row = blockIdx.x * 16 + slot;
  const uint32_t r = min(row, a.m - 1);  // lanes of rows past the last one follow it, and store nothing
  const float ninf = -__builtin_inff();
  float* const score = sh[slot];
  float x[NV], c[NV];
  // an expert past the last one reads the last one's logit, and is out
  const uint32_t last = a.experts - 1;
  const size_t base = (size_t)r * a.experts;
  float bias[NV];
  auto loads = [&](auto load) {
    if ((uint32_t)(li + 1) * NV <= a.experts) {  // every one of the lane's experts is there: whole vectors
#pragma unroll
      for (int i = 0; i < NV; ++i) load(i, (uint32_t)(li * NV + i));
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) load(i, min((uint32_t)(li * NV + i), last));
    }
  };
  if (a.bf16) {
    const uint16_t* const p = (const uint16_t*)a.logits + base;
    loads([&](int i, uint32_t e) { x[i] = __uint_as_float((uint32_t)p[e] << 16); });
  } else {
    const float* const p = (const float*)a.logits + base;
    loads([&](int i, uint32_t e) { x[i] = p[e]; });
  }
  if (a.bias) {
    loads([&](int i, uint32_t e) { bias[i] = a.bias[e]; });
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) bias[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((uint32_t)(li * NV + i) > last) x[i] = ninf;
  float top = ninf;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (x[i] != x[i]) x[i] = ninf;
    top = fmaxf(top, x[i]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) c[i] = sigmoid_f32(x[i]);
  } else {
    top = row_max_f32(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      c[i] = x[i] == top ? (top == ninf ? 0.0f : 1.0f) : x[i] == ninf ? 0.f : exp_fast(x[i] - top);
      sum += c[i];
    }
    sum = row_sum_f32(sum);
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) c[i] *= inv;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) score[li * NV + i] = c[i];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    c[i] += bias[i];
    if (x[i] == ninf || c[i] != c[i]) c[i] = ninf;
    c[i] += 0.0f;  // -0 ties with +0
  }
  if (a.groups > 1) {
    const uint32_t per = a.experts / a.groups, lanes = per / NV;
    if (per % NV == 0 && lanes <= 8 && (lanes & (lanes - 1)) == 0) {  // whole lanes, a power of two of them, a group
      float best = ninf, second = ninf;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        second = fmaxf(second, fminf(best, c[i]));
        best = fmaxf(best, c[i]);
      }
      if (lanes > 1) merge_two<0xB1>(best, second);
      if (lanes > 2) merge_two<0x4E>(best, second);
      if (lanes > 4) merge_two<0x141>(best, second);
      const float mine = a.group_top == 2 && second > ninf ? best + second : best;
      const uint32_t g = li / lanes;
      uint32_t ahead = 0;
      for (uint32_t o = 0; o < a.groups; ++o) {
        const float other = __shfl(mine, (int)((lane & 48) + o * lanes), kWave);
        ahead += other > mine || (other == mine && o < g);
      }
      if (ahead >= a.top_groups) {
#pragma unroll
        for (int i = 0; i < NV; ++i) c[i] = ninf;
      }
    } else {  // lane g scores group g, from LDS
      float* const choice = sh[16 + slot];
#pragma unroll
      for (int i = 0; i < NV; ++i) choice[li * NV + i] = c[i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      float best = ninf, second = ninf;
      if ((uint32_t)li < a.groups)
        for (uint32_t j = 0; j < per; ++j) {
          const float v = choice[li * per + j];
          second = fmaxf(second, fminf(best, v));
          best = fmaxf(best, v);
        }
      const float mine = a.group_top == 2 && second > ninf ? best + second : best;
      uint32_t ahead = 0;
      for (uint32_t o = 0; o < a.groups; ++o) {
        const float other = __shfl(mine, (int)((lane & 48) + o), kWave);
        ahead += other > mine || (other == mine && o < (uint32_t)li);
      }
      const uint32_t keep = (uint32_t)(__ballot((uint32_t)li < a.groups && ahead < a.top_groups) >> (lane & 48)) & 0xffff;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (!((keep >> ((uint32_t)(li * NV + i) / per & 15)) & 1)) c[i] = ninf;
    }
  }
  // A bound on the k-th best: the k-th of every lane's two largest.  What is not
  // below it, little more than k as a rule, goes to the row's lanes one each (LDS), and
  // each counts the ones ahead of it.  More than 16, as after many ties: k rounds.
  int32_t id = -1;
  float first = ninf, second = ninf;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    second = fmaxf(second, fminf(first, c[i]));
    first = fmaxf(first, c[i]);
  }
  uint32_t ahead1 = 0, ahead2 = 1;  // of the lane's first and second among the 32
  each_rotation<1>([&](auto n) {
    constexpr int R = decltype(n)::value;
    const float f = __uint_as_float(row_rotate<R>(__float_as_uint(first)));
    const float g = __uint_as_float(row_rotate<R>(__float_as_uint(second)));
    ahead1 += (f > first) + (g > first);
    ahead2 += (f > second) + (g > second);
  });
  // the smallest of those with fewer than k ahead: at least k values are not below it
  float bound = ahead2 < a.k ? second : ahead1 < a.k ? first : __builtin_inff();
  bound = -row_max_f32(-bound);
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) mine += c[i] >= bound && c[i] > ninf;
  uint32_t upto = mine;  // inclusive sums over the row's lanes
  {
    uint32_t t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)upto, 0x111, 0xF, 0xF, true);
    upto += t;
    t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)upto, 0x112, 0xF, 0xF, true);
    upto += t;
    t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)upto, 0x114, 0xF, 0xF, true);
    upto += t;
    t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)upto, 0x118, 0xF, 0xF, true);
    upto += t;
  }
  const uint32_t count = ~row_min_u32(~upto);  // the row's largest
  if (!__any(count > 16)) {
    uint2* const list = lists[slot];
    uint32_t at = upto - mine;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (c[i] >= bound && c[i] > ninf) list[at++] = make_uint2(__float_as_uint(c[i]), (uint32_t)(li * NV + i));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const bool on = (uint32_t)li < count;
    const uint2 own = on ? list[li] : make_uint2(0xff800000u, 0xffffu);
    const float v = __uint_as_float(own.x);
    uint32_t ahead = 0;  // candidates lie in the order of their index: of equal ones the lower lane is ahead
    each_rotation<1>([&](auto n) {
      constexpr int R = decltype(n)::value;
      const float o = __uint_as_float(row_rotate<R>(own.x));
      const uint32_t oi = row_rotate<R>(own.y);
      ahead += o > v || (o == v && oi < own.y);
    });
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (on && ahead < 16) list[ahead].y = own.y;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if ((uint32_t)li < min(count, a.k)) id = (int32_t)list[li].y;
  } else {
    for (uint32_t j = 0; j < a.k; ++j) {
      float most = c[0];
#pragma unroll
      for (int i = 1; i < NV; ++i) most = fmaxf(most, c[i]);
      most = row_max_f32(most);
      uint32_t at = 16 * NV;
#pragma unroll
      for (int i = NV - 1; i >= 0; --i)
        if (c[i] == most) at = li * NV + i;
      at = row_min_u32(at);
      if ((uint32_t)li == j && most > ninf) id = (int32_t)at;
      const uint32_t gone = at - li * NV;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (gone == (uint32_t)i) c[i] = ninf;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  float w = id >= 0 ? score[id] : 0.f;
  if (a.renorm) {
    const float sum = row_sum_f32(w);
    w = sum > 0.f ? w / sum : 0.f;
  }
  if (row < a.m && (uint32_t)li < a.k) {
    a.ids[(size_t)row * a.k + li] = id;
    a.weights[(size_t)row * a.k + li] = w * a.scale;
  }
}

hipError_t launch_route(hipStream_t st, const RouteArgs& a) {
  if (a.experts <= 256 && a.k <= 16 && a.groups <= 16) {
    auto k = a.experts <= 16    ? route_quads<1>
             : a.experts <= 32  ? route_quads<2>
             : a.experts <= 64  ? route_quads<4>
             : a.experts <= 128 ? route_quads<8>
                                : route_quads<16>;
    hipLaunchKernelGGL(k, dim3((a.m + 15) / 16), dim3(256), 0, st, a);
    return hipGetLastError();
  }
  const uint32_t grid = (a.m + kRouteWaves - 1) / kRouteWaves;
  auto k = a.experts <= 256   ? route_rows<4>
           : a.experts <= 512 ? route_rows<8>
                              : route_rows<16>;
  hipLaunchKernelGGL(k, dim3(grid), dim3(64 * kRouteWaves), 0, st, a);
  return hipGetLastError();
}

}  // namespace w8a8
