// experts.hip -- the routed experts' W8A8 SwiGLU products and their weighted
// sum.  No counterpart in the reference, whose layers are dense.
//
// Row t of q[m, H] (scale asc[t]) meets the experts e = ids[t, 0 .. k):
//   gate = RN(RN(f32(q . Wg[e]) * asc) * wsg[e]), up likewise (exact i32 sums);
//   act = gate / (1 + exp(-gate)) * up, in f32;
//   s_g = max(1e-8, max |act|) / 127 over each 128 columns g of act, NaN
//   ignored, and the codes round(act / s_g) of w8a8_quantize's rounding;
//   y = wsd[e] * sum_g s_g * f32(codes_g . Wd[e]_g);
//   out = bf16(residual + sum over the slots of weight * y).
// One scale to 128 columns, not one to a row: the codes of 128 columns are known
// once their own sums are, so no pass waits for a row's maximum.
#include <algorithm>
#include <cmath>

#include "experts.hpp"

namespace w8a8 {

// ------------------------------------------------------------ slot by slot
// act[slot, I]: a wave holds COLS columns (gate and up row each) of one slot.  The
// weight stream bounds it: 8 slots of hidden 4096, inner 1024 (67 MB) 10.3 us, 6.5
// TB/s, the rate of a stream that is only read.  One column a wave was level.
template <int COLS>
__global__ __launch_bounds__(256) void experts_act_slot(ExpertsArgs a, float* act) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t c0 = (blockIdx.x * 4 + wave) * COLS;
  if (c0 >= a.inter) return;
  const uint32_t slot = blockIdx.y, row = slot / a.k, e = (uint32_t)a.ids[slot];
  if (e >= a.experts) return;
  {
    const int8_t* const q = a.q + (size_t)row * a.hidden;
    const int8_t *g[COLS], *u[COLS];
    int sg[COLS], su[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const size_t n = (size_t)e * a.inter + min(c0 + c, a.inter - 1);
      g[c] = a.w_gate + n * a.hidden;
      u[c] = a.w_up + n * a.hidden;
      sg[c] = su[c] = 0;
    }
#pragma unroll 2
    for (uint32_t o = lane * 16; o < a.hidden; o += 1024) {
      const v4i x = load16(q + o);
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        sg[c] = dot16(load_nt16(g[c] + o), x, sg[c]);
        su[c] = dot16(load_nt16(u[c] + o), x, su[c]);
      }
    }
    int mg = 0, mu = 0;
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const int tg = wave_sum_i32(sg[c]), tu = wave_sum_i32(su[c]);
      if (lane == c) mg = tg, mu = tu;
    }
    if (lane < COLS && c0 + lane < a.inter) {
      const size_t n = (size_t)e * a.inter + c0 + lane;
      act[(size_t)slot * a.inter + c0 + lane] = act_f32(mg, mu, a.asc[row], a.ws_gate[n], a.ws_up[n]);
    }
  }
}

// Sixteen values of act (0 past inter), and their codes and the scale of their group
// of 128, which eight lanes hold.
__device__ __forceinline__ void load_act(const float* p, bool in, float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  if (in) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const v4f t = *(const v4f*)(p + i);
      v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
    }
  }
}
__device__ __forceinline__ v4i code_act(const float (&v)[16], float& s) {
  bool nan;
  uint32_t m = absmax_bits(v, kFloorBits, &nan);
  m = max(m, dpp_u32<0xB1>(m));
  m = max(m, dpp_u32<0x4E>(m));
  m = max(m, dpp_u32<0x141>(m));  // row_half_mirror: the eight lanes of a group
  s = __uint_as_float(m) / 127.0f;
  const float r = 1.0f / s;
  v4i q;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q[i] = (int)codes4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], s, r, nan || s < kFastScaleMin);
  return q;
}

// One column's weighted sum in the definition's order, a slot's whole sum before its
// wsd and its weight: what experts_down_slot makes of parts that were not finite.
__device__ __forceinline__ float down_in_order(const ExpertsArgs& a, const float* act, uint32_t row, uint32_t col,
                                               int lane) {
  float out = 0.f;
  for (uint32_t j = 0; j < a.k; ++j) {
    const uint32_t slot = row * a.k + j, e = (uint32_t)a.ids[slot];
    if (e >= a.experts) continue;
    const size_t n = (size_t)e * a.hidden + col;
    float sum = 0.f;
    for (uint32_t o0 = 0; o0 < a.inter; o0 += 1024) {
      const uint32_t o = o0 + lane * 16;
      const bool in = o < a.inter;
      float v[16], s;
      load_act(act + (size_t)slot * a.inter + o, in, v);
      const v4i q = code_act(v, s);
      sum += (float)dot16(load16(a.w_down + n * a.inter + (in ? o : 0)), q, 0) * s;
    }
    const float y = wave_sum_f32(sum) * a.ws_down[n];
    out += a.weights[slot] * y;
  }
  return out;
}

// out[t, c] over the row's slots.  The workgroup's eight waves first make the codes
// of eight slots' next 1024 columns of act, a wave a slot (16 values a lane, so
// that eight lanes hold a group of 128), and share them through LDS; meanwhile
// each wave's weights for its COLS columns are on their way.  A lane's 16 products
// lie in one group, so its part of a sum is scaled, by s, weight and wsd, before the
// lanes' parts are added.  Parts of both signs or of 0 make NaN of an infinite wsd or
// weight: a column that is not finite is summed again, in order.  8 slots of hidden
// 4096, inner 1024 (33.5 MB): 9.4 us, 3.6 TB/s: ids, then act and weights, codes, sums
// follow each other.  With the codes made by a launch of their own 10.8 + 2.5 us; one
// column a wave level.
template <int COLS>
__global__ __launch_bounds__(512) void experts_down_slot(ExpertsArgs a, const float* act) {
  __shared__ __attribute__((aligned(16))) v4i code[8][64];
  __shared__ float scale[8][8];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t c0 = (blockIdx.x * 8 + wave) * COLS, row = blockIdx.y;
  uint32_t col[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c) col[c] = min(c0 + c, a.hidden - 1);
  float total[COLS];
#pragma unroll
  for (int c = 0; c < COLS; ++c) total[c] = 0.f;
  for (uint32_t j0 = 0; j0 < a.k; j0 += 8) {
    uint32_t e[8];  // past the last slot, or without an expert: ~0
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t id = (uint32_t)a.ids[(size_t)row * a.k + min(j0 + j, a.k - 1)];
      e[j] = j0 + j < a.k && id < a.experts ? id : ~0u;
    }
    // this wave's slot
    const uint32_t slot = row * a.k + min(j0 + wave, a.k - 1);
    const uint32_t id = (uint32_t)a.ids[slot];
    const bool mine = j0 + wave < a.k && id < a.experts;
    const float weight = a.weights[slot];
    for (uint32_t o0 = 0; o0 < a.inter; o0 += 1024) {
      const uint32_t o = o0 + lane * 16;
      const bool in = o < a.inter;
      float v[16];
      load_act(act + (size_t)slot * a.inter + o, mine && in, v);
      v4i w[8][COLS];
      float ws[8][COLS];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          if (e[j] == ~0u) continue;
          const size_t n = (size_t)e[j] * a.hidden + col[c];
          w[j][c] = load_nt16(a.w_down + n * a.inter + (in ? o : 0));
          ws[j][c] = a.ws_down[n];
        }
      __builtin_amdgcn_sched_barrier(0);  // the weights are under way while the codes are made
      float s;
      code[wave][lane] = code_act(v, s);
      if ((lane & 7) == 0) scale[wave][lane >> 3] = s * weight;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const v4i x = code[j][lane];
        const float t = scale[j][lane >> 3];
#pragma unroll
        for (int c = 0; c < COLS; ++c)
          if (e[j] != ~0u) total[c] += (float)dot16(w[j][c], x, 0) * t * ws[j][c];
      }
      __syncthreads();
    }
  }
  float y = 0.f;
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    float t = wave_sum_f32(total[c]);
    if (!(__builtin_fabsf(t) < __builtin_inff())) t = down_in_order(a, act, row, col[c], lane);
    if (lane == c) y = t;
  }
  if (lane < COLS && c0 + lane < a.hidden) {
    const size_t o = (size_t)row * a.hidden + c0 + lane;
    store_routed(a.out, a.out_dtype, o, a.residual ? a.residual[o] + y : y);
  }
}

// Slot by slot every slot reads its expert's weights; expert by expert the experts
// that are met are read once, in four launches instead of two.  The slots' form
// runs while what it reads more costs less than those launches: about 140 MB.
// Measured on weights of each pass's own, slots / experts us: hidden 4096, inner 1024, 8
// of 64, 4 rows (69 MB more) 65.0 / 78.3, 6 rows (160 MB) 92.6 / 112; hidden 2048, inner
// 768, 8 of 128, 8 rows (58 MB) 51.5 / 59.3, 12 rows (127 MB) 73.4 / 70.6; hidden 4096,
// inner 2048, 2 of 16, 6 rows (80 MB) 55.6 / 61.9, 8 rows (138 MB) 70.9 / 66.4, 12 rows
// (282 MB) 101 / 71; hidden 2048, inner 1024, 2 of 8, 12 rows (102 MB) 28.9 / 32.9, 16 rows
// (151 MB) 36.0 / 33.0.  Of small experts the slots' form takes more than its bytes:
// hidden 512, inner 256, 4 of 32, 32 rows (38 MB) 18.3 / 18.9, 64 rows (88 MB) 31.8 / 19.0.
bool experts_by_slot(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter) {
  if (m > 64) return false;
  const double slots = (double)m * k;
  const double met = experts * (1.0 - std::pow(1.0 - std::min(1.0, (double)k / experts), (double)m));
  return (slots - met) * 3.0 * hidden * inter <= 140e6;
}

size_t experts_workspace_bytes(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter) {
  if (!experts_by_slot(m, k, experts, hidden, inter))
    return experts_tiles_workspace_bytes(m, k, experts, hidden, inter);
  return up256((size_t)m * k * inter * 4);  // act
}

hipError_t launch_experts(hipStream_t st, const ExpertsArgs& a, void* workspace) {
  if (!experts_by_slot(a.m, a.k, a.experts, a.hidden, a.inter)) return launch_experts_tiles(st, a, workspace);
  const uint32_t slots = a.m * a.k;
  float* const act = (float*)workspace;
  constexpr int CG = 2, CD = 2;
  hipLaunchKernelGGL(experts_act_slot<CG>, dim3((a.inter + 4 * CG - 1) / (4 * CG), slots), dim3(256), 0, st, a, act);
  hipLaunchKernelGGL(experts_down_slot<CD>, dim3((a.hidden + 8 * CD - 1) / (8 * CD), a.m), dim3(512), 0, st, a, act);
  return hipGetLastError();
}

}  // namespace w8a8
