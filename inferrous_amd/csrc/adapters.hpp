// adapters.hpp -- what the adapters' kernels share: row by row (adapters.hip)
// and in tiles of rows sorted by adapter (adapters_tiles.hip).
#pragma once
#include "internal.hpp"
#include "routed_common.hpp"
#include "row_sort.hpp"
#include "tile_stream.hpp"

namespace w8a8 {

static inline size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// Values of a row of h's BF16 parts: the ranks, padded to whole 32s.
__host__ __device__ constexpr uint32_t part_width(uint32_t rank) { return (rank + 31) / 32 * 32; }

// How a call runs, a function of its sizes.
struct AdapterPlan {
  bool sorted;   // the rows are sorted by adapter, and the first product runs in tiles of them
  bool fused;    // the projection runs in tiles of the sorted rows, and adds the second product itself
  uint32_t bt;   // sorted: rows of a tile of the first product
  uint32_t tiles;   // sorted: tiles at most
  uint32_t splits;  // shares of K of the first product, each with partial sums of its own
  uint32_t stages;  // sorted: 128-byte stages of an adapter row in a share
  size_t h, order, table, n_tiles, counts, high, low, bytes;  // workspace offsets
};
AdapterPlan adapter_plan(const AdapterArgs& a);

hipError_t launch_adapters_sorted(hipStream_t st, const AdapterArgs& a, const AdapterPlan& p, char* workspace);
hipError_t launch_adapters_fused(hipStream_t st, const AdapterArgs& a, const AdapterPlan& p, char* workspace);

}  // namespace w8a8
