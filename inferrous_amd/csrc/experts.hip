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
#include "experts.hpp"

namespace w8a8 {

// ------------------------------------------------------------ slot by slot
// act[slot, I]: a wave holds COLS columns (gate and up row each) of one slot.
template <int COLS>
__global__ __launch_bounds__(256) void experts_act_slot(ExpertsArgs a, float* act) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t c0 = (blockIdx.x * 4 + wave) * COLS;
  if (c0 >= a.inter) return;
  for (uint32_t slot = blockIdx.y; slot < a.m * a.k; slot += gridDim.y) {
    const uint32_t e = (uint32_t)a.ids[slot];
    if (e >= a.experts) continue;
    const uint32_t row = slot / a.k;
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

// codes[slot, I] and scales[slot, groups] of act: eight lanes of 16 values hold
// a group, a wave eight groups.
__global__ __launch_bounds__(64) void experts_codes(const float* act, uint32_t slots, uint32_t inter, int8_t* codes,
                                                    float* scales) {
  const int lane = threadIdx.x;
  const uint32_t c = blockIdx.x * 1024 + lane * 16, groups = (inter + 127) / 128;
  for (uint32_t slot = blockIdx.y; slot < slots; slot += gridDim.y) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.f;
    if (c < inter) {
      const float* const p = act + (size_t)slot * inter + c;
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const v4f t = *(const v4f*)(p + i);
        v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
      }
    }
    bool nan;
    uint32_t m = absmax_bits(v, kFloorBits, &nan);
    m = max(m, dpp_u32<0xB1>(m));
    m = max(m, dpp_u32<0x4E>(m));
    m = max(m, dpp_u32<0x141>(m));  // row_half_mirror: the eight lanes of a group
    const float s = __uint_as_float(m) / 127.0f, r = 1.0f / s;
    if (c < inter) {
      v4i out;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        out[i] = (int)codes4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], s, r, nan || s < kFastScaleMin);
      *(v4i*)(codes + (size_t)slot * inter + c) = out;
      if ((lane & 7) == 0) scales[(size_t)slot * groups + c / 128] = s;
    }
  }
}

// out[t, c] over the row's slots: a wave holds COLS columns of one row.  Each
// lane's 16 products lie in one group, so its part of a sum is scaled before
// the lanes' parts are added.
template <int COLS>
__global__ __launch_bounds__(256) void experts_down_slot(ExpertsArgs a, const int8_t* codes, const float* scales) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t c0 = (blockIdx.x * 4 + wave) * COLS, groups = (a.inter + 127) / 128;
  if (c0 >= a.hidden) return;
  for (uint32_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    float total[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) total[c] = 0.f;
    for (uint32_t j = 0; j < a.k; ++j) {
      const uint32_t slot = row * a.k + j, e = (uint32_t)a.ids[slot];
      if (e >= a.experts) continue;
      const float weight = a.weights[slot];
      float sum[COLS];
#pragma unroll
      for (int c = 0; c < COLS; ++c) sum[c] = 0.f;
      for (uint32_t o = lane * 16; o < a.inter; o += 1024) {
        const v4i x = load16(codes + (size_t)slot * a.inter + o);
        const float s = scales[(size_t)slot * groups + o / 128];
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          const size_t n = (size_t)e * a.hidden + min(c0 + c, a.hidden - 1);
          sum[c] += (float)dot16(load_nt16(a.w_down + n * a.inter + o), x, 0) * s;
        }
      }
#pragma unroll
      for (int c = 0; c < COLS; ++c)
        total[c] += sum[c] * (weight * a.ws_down[(size_t)e * a.hidden + min(c0 + c, a.hidden - 1)]);
    }
    float mine = 0.f;
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const float t = wave_sum_f32(total[c]);
      if (lane == c) mine = t;
    }
    if (lane < COLS && c0 + lane < a.hidden) {
      const size_t o = (size_t)row * a.hidden + c0 + lane;
      store_routed(a.out, a.out_dtype, o, a.residual ? a.residual[o] + mine : mine);
    }
  }
}

static size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// Slot by slot every slot reads its expert's weights; expert by expert they are
// read once, in more launches.
static bool by_slot(uint32_t m) { return m <= 4; }

size_t experts_workspace_bytes(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter) {
  if (!by_slot(m)) return experts_tiles_workspace_bytes(m, k, experts, hidden, inter);
  const size_t slots = (size_t)m * k;
  return up256(slots * inter * 4) + up256(slots * inter) + up256(slots * ((inter + 127) / 128) * 4);
}

hipError_t launch_experts(hipStream_t st, const ExpertsArgs& a, void* workspace) {
  if (!by_slot(a.m)) return launch_experts_tiles(st, a, workspace);
  const uint32_t slots = a.m * a.k;
  char* p = (char*)workspace;
  float* const act = (float*)p;
  int8_t* const codes = (int8_t*)(p += up256((size_t)slots * a.inter * 4));
  float* const scales = (float*)(p + up256((size_t)slots * a.inter));
  constexpr int CG = 2, CD = 2;
  const uint32_t ys = slots < 65535u ? slots : 65535u, yr = a.m < 65535u ? a.m : 65535u;
  hipLaunchKernelGGL(experts_act_slot<CG>, dim3((a.inter + 4 * CG - 1) / (4 * CG), ys), dim3(256), 0, st, a, act);
  hipLaunchKernelGGL(experts_codes, dim3((a.inter + 1023) / 1024, ys), dim3(64), 0, st, act, slots, a.inter, codes,
                     scales);
  hipLaunchKernelGGL(experts_down_slot<CD>, dim3((a.hidden + 4 * CD - 1) / (4 * CD), yr), dim3(256), 0, st, a, codes,
                     scales);
  return hipGetLastError();
}

}  // namespace w8a8
