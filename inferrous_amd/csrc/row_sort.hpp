// row_sort.hpp -- a counting sort of items by a small class number that keeps
// the items' order, shared by the routed experts (slots by expert) and the
// adapters (rows by adapter).
//
// Classes are 0 .. classes - 1, classes <= kSortClasses; an item of any other
// number is of class `classes` where REST is set, and of none otherwise.  A
// workgroup of kSortWaves waves sorts up to kSortBlock items alone; more are
// sorted by several workgroups, whose counts a launch before theirs has taken.
// The order is a function of the items alone: positions come from counts and
// ballots; there are no atomics.
#pragma once
#include <algorithm>

#include "device_common.hpp"

namespace w8a8 {

constexpr int kSortWaves = 16;
constexpr uint32_t kSortClasses = 1024;
constexpr uint32_t kSortBlock = 4096;
constexpr int kSortRegs = kSortBlock / (64 * kSortWaves);  // items of a lane, held in registers

// Items of a workgroup: all of them; or 1024, which more workgroups share; or the
// most there can be, where the workgroups' counts would take longer to add.
static inline uint32_t sort_per_block(uint32_t items) {
  return items <= kSortBlock ? items : items <= 64 * kSortBlock ? 1024 : kSortBlock;
}
static inline uint32_t sort_blocks(uint32_t items) {
  const uint32_t per = sort_per_block(items);
  return per ? (items + per - 1) / per : 0;
}

template <bool REST>
__device__ __forceinline__ uint32_t sort_class(int32_t id, uint32_t classes) {
  return (uint32_t)id < classes ? (uint32_t)id : REST ? classes : ~0u;
}

// Items [begin, end) of a wave: the workgroup's in kSortWaves runs of whole 64s.
__device__ __forceinline__ void sort_run(uint32_t items, uint32_t per_block, int wave, uint32_t& begin, uint32_t& end) {
  const uint32_t b0 = min(blockIdx.x * per_block, items), b1 = min(b0 + per_block, items);
  const uint32_t run = ((b1 - b0 + 64 * kSortWaves - 1) / (64 * kSortWaves)) * 64;
  begin = min(b0 + wave * run, b1);
  end = min(begin + run, b1);
}

// The lane's items of its wave's run, as classes (~0: none), all loads together.
template <bool REST>
__device__ __forceinline__ void sort_load(const int32_t* ids, uint32_t classes, uint32_t begin, uint32_t end, int lane,
                                          uint32_t (&c)[kSortRegs]) {
  int32_t id[kSortRegs];
#pragma unroll
  for (int i = 0; i < kSortRegs; ++i) {
    const uint32_t at = begin + 64 * i + lane;
    id[i] = begin < end ? ids[min(at, end - 1)] : -1;
  }
#pragma unroll
  for (int i = 0; i < kSortRegs; ++i)
    c[i] = begin + 64 * i + lane < end ? sort_class<REST>(id[i], classes) : ~0u;
}

// The lanes of a wave that hold the same class as this one, by ballots over the bits
// of its number (none for a lane of no class).
__device__ __forceinline__ uint64_t sort_peers(uint32_t c, uint32_t n) {
  uint64_t peers = __ballot(c < n);
  for (uint32_t b = 0; (1u << b) < n; ++b) {
    const uint64_t set = __ballot((c >> b) & 1);
    peers &= ((c >> b) & 1) ? set : ~set;
  }
  return c < n ? peers : 0;
}

// Of every group of 64 that the wave's run has: up to 1024 items among 16 waves leave
// a wave one group or none.
__device__ __forceinline__ void sort_all_peers(const uint32_t (&c)[kSortRegs], uint32_t begin, uint32_t end, uint32_t n,
                                               uint64_t (&peers)[kSortRegs]) {
#pragma unroll
  for (int i = 0; i < kSortRegs; ++i) {
    peers[i] = 0;
    if (begin + 64 * i < end) peers[i] = sort_peers(c[i], n);
  }
}

// hist[class] of a wave's items.  One lane of each class adds its peers: atomics
// of 64 equal classes, which sorted requests bring, took 10 of the sort's 13 us at
// 4096 items of 7 classes.
__device__ __forceinline__ void sort_count(const uint32_t (&c)[kSortRegs], const uint64_t (&peers)[kSortRegs],
                                           uint32_t n, uint32_t* hist, int lane) {
  for (uint32_t e = lane; e < n; e += 64) hist[e] = 0;
#pragma unroll
  for (int i = 0; i < kSortRegs; ++i) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (peers[i] && (peers[i] >> lane) == 1) hist[c[i]] += (uint32_t)__popcll(peers[i]);
  }
}

// counts[workgroup][class] of a sort over several workgroups.
template <bool REST>
__global__ __launch_bounds__(64 * kSortWaves) void sort_counts(const int32_t* ids, uint32_t items, uint32_t per_block,
                                                               uint32_t classes, uint32_t* counts) {
  extern __shared__ uint32_t hist[];  // [kSortWaves][classes]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t n = classes + REST;
  uint32_t begin, end;
  sort_run(items, per_block, wave, begin, end);
  uint32_t c[kSortRegs];
  uint64_t peers[kSortRegs];
  sort_load<REST>(ids, classes, begin, end, lane, c);
  sort_all_peers(c, begin, end, n, peers);
  sort_count(c, peers, n, hist + wave * n, lane);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < n; e += 64 * kSortWaves) {
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) sum += hist[w * n + e];
    counts[(size_t)blockIdx.x * n + e] = sum;
  }
}

// Exclusive sums of v over the workgroup's threads; *all receives the total.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* part, uint32_t* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = (uint32_t)__shfl_up((int)s, o, kWave);
    if (lane >= o) s += t;
  }
  if (lane == 63) part[wave] = s;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    if (w < wave) before += part[w];
    total += part[w];
  }
  __syncthreads();
  *all = total;
  return before + s - v;
}

// Up to `rows` sorted positions of one class.
struct RowTile {
  uint32_t of, first, rows, pad;
};

// The table of the classes' tiles of up to bt positions, by every thread of one
// workgroup: thread e lists class e's.
__device__ __forceinline__ void list_tiles(uint32_t first, uint32_t total, uint32_t bt, uint32_t* part, RowTile* table,
                                           uint32_t* n_tiles) {
  uint32_t tiles;
  const uint32_t mine = (total + bt - 1) / bt, at = block_prefix(mine, part, &tiles);
  for (uint32_t i = 0; i < mine; ++i)
    table[at + i] = RowTile{(uint32_t)threadIdx.x, first + i * bt, (uint32_t)min(bt, total - i * bt), 0u};
  if (threadIdx.x == 0) *n_tiles = tiles;
}

// The sort's positions.  hist: [kSortWaves][classes + REST] words, part:
// [kSortWaves] of LDS; counts as sort_counts wrote them (unused by one
// workgroup).  firsts(first, total) is called once by every thread of the
// workgroup with its class's first position and item count (thread e: class e;
// 0 items past the last class), place(item, position) by each item's lane, with
// -1 for an item of no class.
template <bool REST, class Firsts, class Place>
__device__ __forceinline__ void sort_items(const int32_t* ids, uint32_t items, uint32_t per_block, uint32_t classes,
                                           const uint32_t* counts, uint32_t* hist, uint32_t* part, Firsts firsts,
                                           Place place) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t e = threadIdx.x, n = classes + REST;
  uint32_t begin, end;
  sort_run(items, per_block, wave, begin, end);
  uint32_t c[kSortRegs];
  uint64_t peers[kSortRegs];
  sort_load<REST>(ids, classes, begin, end, lane, c);
  sort_all_peers(c, begin, end, n, peers);
  sort_count(c, peers, n, hist + wave * n, lane);
  __syncthreads();
  uint32_t total = 0, before = 0;  // of class e: all its items, those of earlier workgroups
  if (e < n) {
    if (gridDim.x == 1) {
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) total += hist[w * n + e];
    } else {
      for (uint32_t b0 = 0; b0 < gridDim.x; b0 += 16) {
        uint32_t k[16];
#pragma unroll
        for (uint32_t b = 0; b < 16; ++b) k[b] = counts[(size_t)min(b0 + b, gridDim.x - 1) * n + e];
#pragma unroll
        for (uint32_t b = 0; b < 16; ++b) {
          if (b0 + b >= gridDim.x) k[b] = 0;
          if (b0 + b < blockIdx.x) before += k[b];
          total += k[b];
        }
      }
    }
  }
  uint32_t all;
  const uint32_t first = block_prefix(total, part, &all);
  if (e < n) {
    uint32_t p = first + before, k[kSortWaves];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) k[w] = hist[w * n + e];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      hist[w * n + e] = p;
      p += k[w];
    }
  }
  firsts(first, total);
  __syncthreads();
  // Each wave walks its run in order; peers take positions in their lanes' order.
  uint32_t* const next = hist + wave * n;
#pragma unroll
  for (int g = 0; g < kSortRegs; ++g) {
    if (begin + 64 * g >= end) break;
    const uint32_t i = begin + 64 * g + lane;
    const bool on = peers[g] != 0;
    uint32_t p = 0;
    if (on) p = next[c[g]] + (uint32_t)__popcll(peers[g] & ((1ull << lane) - 1));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (on && (peers[g] >> lane) == 1) next[c[g]] = p + 1;  // the last of its peers
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (i < end) place(i, on ? (int32_t)p : -1);
  }
}

}  // namespace w8a8
