// experts.hpp -- what the two forms of the routed experts' MLP share: slot by
// slot (experts.hip) and expert by expert (experts_tiles.hip).
#pragma once
#include "internal.hpp"
#include "routed_common.hpp"
#include "row_sort.hpp"

namespace w8a8 {

// The slots sorted by expert: position p of the sorted order holds slot order[p],
// slot i stands at pos[i] (-1: it has no expert); tiles of one expert's positions.
struct ExpertsPlan {
  uint32_t* order;
  int32_t* pos;
  RowTile* tiles;
  uint32_t* n_tiles;
};

// act of two projections, kept in f32 up to its codes.  exp(-gate) goes straight to
// v_exp_f32: its error, 2^-23.7 |gate|, is far below a code's step, 1 / 127 of the
// group's maximum, wherever act is not negligible.
__device__ __forceinline__ float act_f32(int32_t g, int32_t u, float asc, float wg, float wu) {
  const float gate = (float)g * asc * wg, up = (float)u * asc * wu;
  return gate * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(gate * -1.44269502f)) * up;
}

// Four codes of act at scale s, r = RN(1 / s): v r is within 2^-23 of v / s, 1.6e-5 of a
// code at most, so that only a value that close to a half takes the other neighbour;
// adding 1.5 * 2^23 rounds to the integer that is the low byte.  An infinite s
// gives zeros.  `slow` as in codes4.  Two instructions a value, where the correctly
// rounded quotients take eight.
__device__ __forceinline__ uint32_t act_codes4(float a, float b, float c, float d, float s, float r, bool slow) {
  if (slow) return pack4(a, b, c, d, s);
  auto bits = [&](float v) { return __float_as_uint(__builtin_fmaf(v, r, 12582912.0f)); };
  return __builtin_amdgcn_perm(bits(b), bits(a), 0x0c0c0400u) | __builtin_amdgcn_perm(bits(d), bits(c), 0x04000c0cu);
}

size_t experts_tiles_workspace_bytes(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter);
hipError_t launch_experts_tiles(hipStream_t st, const ExpertsArgs& a, void* workspace);

}  // namespace w8a8
