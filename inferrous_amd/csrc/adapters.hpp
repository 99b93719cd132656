// adapters.hpp -- what the adapters' kernels share: row by row (adapters.hip)
// and in tiles of rows sorted by adapter (adapters_tiles.hip).
#pragma once
#include "internal.hpp"
#include "routed_common.hpp"
#include "row_sort.hpp"
#include "tile_stream.hpp"

namespace w8a8 {

// Values of a row of scaling * h: the ranks, padded to whole 32s.
__host__ __device__ constexpr uint32_t part_width(uint32_t rank) { return (rank + 31) / 32 * 32; }

// How a call runs, a function of its sizes.
struct AdapterPlan {
  bool gemv;        // few rows: the projection and the second product in one kernel
  bool fused;       // the rows are sorted by adapter, and the projection's tiles add the second product
  uint32_t values;  // (not fused) values of h that a wave sums: 1, 2 or 8
  uint32_t ranks;   // (fused) ranks of a tile of the first product: 32, 64, 128 or 256
  uint32_t tile;    // (fused) rows and columns of the projection's tiles: 128 or 256
  bool tail;        // (fused) the last stage of the projection's K is short
  uint32_t bt;      // (fused) rows of a tile of the first product
  uint32_t tiles;   // tiles at most
  uint32_t splits;  // shares of K of the first product, each with partial sums of its own
  uint32_t stages;  // 128-byte stages of an adapter row in a share
  size_t h, order, table, n_tiles, counts, scaled, bytes;  // workspace offsets
};
AdapterPlan adapter_plan(const AdapterArgs& a);

hipError_t launch_adapters_fused(hipStream_t st, const AdapterArgs& a, const AdapterPlan& p, char* workspace);

}  // namespace w8a8
