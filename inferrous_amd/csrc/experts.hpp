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

// act of two projections, kept in f32 up to its codes: SiLU from t = exp(-|gate|), in
// (0, 1], as gate * (gate < 0 ? t : 1) / (1 + t), the reciprocal by v_rcp_f32 and one
// Newton step: the divisor is never large, where v_rcp_f32 has no normal result.
// Below -128 t is 0.  About 3 units of the last place.
__device__ __forceinline__ float act_f32(int32_t g, int32_t u, float asc, float wg, float wu) {
  const float gate = (float)g * asc * wg, up = (float)u * asc * wu;
  const float t = exp_above_m128(__builtin_fmaxf(-__builtin_fabsf(gate), -128.0f)), d = 1.0f + t;
  float r = __builtin_amdgcn_rcpf(d);
  r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
  return gate * (gate < 0.f ? t : 1.0f) * r * up;
}

bool experts_by_slot(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter);

// How a call runs expert by expert, a function of its sizes.
struct ExpertsTilesForm {
  uint32_t bt, tiles;            // rows of a token tile, and how many tiles there can be
  uint32_t sort_blocks;          // workgroups of the sort
  bool gate_deep, down_deep;     // 32 rows: one workgroup a CU with twice the stages under way
  bool gate_tail, down_tail;     // the last stage of K is short
};
ExpertsTilesForm experts_tiles_form(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter);
size_t experts_tiles_workspace_bytes(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter);
hipError_t launch_experts_tiles(hipStream_t st, const ExpertsArgs& a, void* workspace);

}  // namespace w8a8
