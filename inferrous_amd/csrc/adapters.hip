// adapters.hip -- a low-rank BF16 adapter per row beside a shared W8A8
// projection, many adapters in one call.  No counterpart in the reference.
//
//   out[r][c] = bf16(residual + RN(RN(f32(q . w) * asc) * ws)
//                    + scaling[a] * sum_j B[a][c][j] * h[r][j]),
//   h[r][j] = sum_i A[a][j][i] * bf16(x[r][i]),   a = ids[r],
// a row whose id is outside [0, n_adapters) taking the projection alone.  h and
// both sums are held in f32.
//
// Here: rows as they are (a decode batch).  h by MFMA on the rows of each
// adapter, then out row by row from the projection's exact sums; rows sorted by
// adapter (prompts, and many rows): adapters_tiles.hip.
#include <algorithm>

#include "adapters.hpp"

namespace w8a8 {

// Rows up to which they are taken as they are.
constexpr uint32_t kDirectRows = 64;
// Waves of a workgroup of the first product: their blocks meet in its LDS.
constexpr int shrink_waves(int fn) { return fn == 8 ? 4 : 8; }

// Eight values of a row as BF16.
template <bool BF16>
__device__ __forceinline__ v4i row_frag(const void* x, size_t o) {
  if constexpr (BF16) {
    return *(const v4i*)((const uint16_t*)x + o);
  } else {
    const v4f a = *(const v4f*)((const float*)x + o), b = *(const v4f*)((const float*)x + o + 4);
    return v4i{(int)bf16_pair(a.x, a.y), (int)bf16_pair(a.z, a.w), (int)bf16_pair(b.x, b.y), (int)bf16_pair(b.z, b.w)};
  }
}

// h[split][row][j], partial sums over the split's share of K.  Workgroup (32 rows,
// leader; split): the adapter of the leader row, if no row before it among the 32
// has the same.  Its 32 x 32 FN block of products comes from
// v_mfma_f32_32x32x16_bf16 (adapter rows x token rows); lane l gives the op 8
// consecutive k of row l % 32 of each operand, k = 8 (l / 32) ..., straight from
// memory, and the splits' waves take 64-value steps of K in turn.
template <int FN, bool BF16>
__global__ __launch_bounds__(64 * shrink_waves(FN)) void adapters_shrink(AdapterArgs a, float* h, uint32_t leaders) {
  constexpr int W = shrink_waves(FN);
  __shared__ __attribute__((aligned(16))) float red[W][FN * 4][64][4];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t leader = blockIdx.x % leaders, row0 = blockIdx.x / leaders * 32, p = row0 + (lane & 31);
  const uint32_t row = p < a.m ? p : row0;
  const uint32_t id = p < a.m ? (uint32_t)a.ids[row] : ~0u;
  const uint32_t ad = (uint32_t)__builtin_amdgcn_readlane((int)id, (int)leader);
  const uint32_t rows = (uint32_t)__ballot(id == ad);
  if (ad >= a.adapters || (rows & ((1u << leader) - 1))) return;
  const uint32_t K = a.width, stride = W * gridDim.y;
  const size_t xo = (size_t)row * K + 8 * half;
  const uint16_t* w[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j)
    w[j] = a.a + ((size_t)ad * a.rank + min(32u * j + (lane & 31), a.rank - 1)) * K + 8 * half;
  v16f acc[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) acc[j] = v16f{};
  uint32_t s = blockIdx.y * W + wave;
#pragma unroll 2
  for (; s * 64 + 64 <= K; s += stride) {
    v4i x[4], wf[FN][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = row_frag<BF16>(a.x, xo + s * 64 + 16 * i);
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) wf[j][i] = *(const v4i*)(w[j] + s * 64 + 16 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[j] = mfma_bf16(wf[j][i], x[i], acc[j]);
  }
  for (uint32_t o = s * 64; o < K; o += 16) {  // the last, partial step; K % 16 == 0
    const v4i x = row_frag<BF16>(a.x, xo + o);
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[j] = mfma_bf16(*(const v4i*)(w[j] + o), x, acc[j]);
  }
  // lane l holds row l % 32 and the ranks 32 j + 8 (v / 4) + 4 (l / 32) + v % 4
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int v = 0; v < 16; v += 4)
      *(v4f*)red[wave][4 * j + v / 4][lane] = v4f{acc[j][v], acc[j][v + 1], acc[j][v + 2], acc[j][v + 3]};
  __syncthreads();
  for (int i = wave; i < FN * 4; i += W) {
    const uint32_t r = 8 * i + 4 * half;
    if (((rows >> (lane & 31)) & 1) && r < a.rank) {
      v4f sum = *(const v4f*)red[0][i][lane];
#pragma unroll
      for (int t = 1; t < W; ++t) sum += *(const v4f*)red[t][i][lane];
      *(v4f*)(h + ((size_t)blockIdx.y * a.m + row) * a.rank + r) = sum;
    }
  }
}

// out row by row from the projection's exact sums (`slabs` partial ones) and h: a
// thread holds a column, its adapter row one contiguous run.
__global__ __launch_bounds__(256) void adapters_expand(AdapterArgs a, const int32_t* acc, uint32_t slabs,
                                                       const float* h, uint32_t splits) {
  __shared__ float hs[kMaxRank];
  const uint32_t c = blockIdx.x * 256 + threadIdx.x, cc = min(c, a.n - 1);
  for (uint32_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    const uint32_t id = (uint32_t)a.ids[row];
    const size_t o = (size_t)row * a.n + cc;
    int32_t sum = acc[o];
    for (uint32_t s = 1; s < slabs; ++s) sum += acc[o + (size_t)s * a.m * a.n];
    float y = (float)sum * a.asc[row] * a.ws[cc];
    if (id < a.adapters) {
      for (uint32_t j = threadIdx.x; j < a.rank; j += 256) {
        float v = 0.f;
        for (uint32_t s = 0; s < splits; ++s) v += h[((size_t)s * a.m + row) * a.rank + j];
        hs[j] = v;
      }
      __syncthreads();
      const uint16_t* const b = a.b + ((size_t)id * a.n + cc) * a.rank;
      float d = 0.f;
#pragma unroll 2
      for (uint32_t j = 0; j < a.rank; j += 8) {
        const v4i bv = *(const v4i*)(b + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d = __builtin_fmaf(bf16_lo((uint32_t)bv[i]), hs[j + 2 * i], d);
          d = __builtin_fmaf(bf16_hi((uint32_t)bv[i]), hs[j + 2 * i + 1], d);
        }
      }
      y += a.scaling[id] * d;
      __syncthreads();
    }
    if (c < a.n) {
      if (a.residual) y += a.residual[o];
      store_routed(a.out, a.out_dtype, o, y);
    }
  }
}

// ------------------------------------------------------------------ plan
AdapterPlan adapter_plan(const AdapterArgs& a) {
  AdapterPlan p{};
  const uint32_t mean = a.m / std::min(a.m, a.adapters);
  p.sorted = a.m > kDirectRows;
  // The fused tiles multiply every adapter of 32 sorted rows with all of them.
  p.fused = p.sorted && mean >= 16;
  if (p.sorted) {
    const uint32_t all = (a.width * 2 + 127) / 128;  // stages of an adapter row
    p.bt = mean <= 48 ? 32 : 128;
    p.tiles = a.m / p.bt + std::min(a.m, a.adapters);
    // about 512 workgroups, each with eight stages at least
    const uint32_t want = std::max(1u, std::min(512 / std::max(1u, a.m / p.bt), 16u));
    p.stages = std::max((all + want - 1) / want, std::min(all, 8u));
    p.splits = (all + p.stages - 1) / p.stages;
  } else {
    const uint32_t steps = (a.width + 63) / 64, groups = (a.m + 31) / 32 * std::min(a.m, 32u);
    p.splits = std::max(1u, std::min(std::min(256 / groups, (steps + 2 * 8 - 1) / (2 * 8)), 8u));
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  p.h = take((size_t)p.splits * a.m * a.rank * 4);
  if (p.sorted) {
    const uint32_t blocks = sort_blocks(a.m), padded = (a.rank + 15) / 16 * 16;
    p.order = take((size_t)a.m * 4);
    p.table = take((size_t)p.tiles * sizeof(RowTile));
    p.n_tiles = take(4);
    p.counts = take(blocks > 1 ? (size_t)blocks * (a.adapters + 1) * 4 : 0);
    if (p.fused) {
      p.high = take((size_t)a.m * padded * 2);
      p.low = take((size_t)a.m * padded * 2);
    }
  }
  p.bytes = at;
  return p;
}

size_t adapters_workspace_bytes(const AdapterArgs& a) { return adapter_plan(a).bytes; }
bool adapters_fused(const AdapterArgs& a) { return adapter_plan(a).fused; }

hipError_t launch_adapters_before(hipStream_t st, const AdapterArgs& a, void* workspace) {
  const AdapterPlan p = adapter_plan(a);
  if (p.sorted) {
    const hipError_t e = launch_adapters_sorted(st, a, p, (char*)workspace);
    return e != hipSuccess || !p.fused ? e : launch_adapters_fused(st, a, p, (char*)workspace);
  }
  const uint32_t leaders = std::min(a.m, 32u);
  float* const h = (float*)((char*)workspace + p.h);
  const dim3 grid((a.m + 31) / 32 * leaders, p.splits);
  const int waves = shrink_waves(a.rank > 128 ? 8 : 1);
  auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(64 * waves), 0, st, a, h, leaders); };
  if (a.x_bf16) go(a.rank <= 32 ? adapters_shrink<1, true> : a.rank <= 64 ? adapters_shrink<2, true>
                   : a.rank <= 128 ? adapters_shrink<4, true> : adapters_shrink<8, true>);
  else go(a.rank <= 32 ? adapters_shrink<1, false> : a.rank <= 64 ? adapters_shrink<2, false>
          : a.rank <= 128 ? adapters_shrink<4, false> : adapters_shrink<8, false>);
  return hipGetLastError();
}

hipError_t launch_adapters_after(hipStream_t st, const AdapterArgs& a, const int32_t* acc, uint32_t slabs,
                                 const void* workspace) {
  const AdapterPlan p = adapter_plan(a);
  hipLaunchKernelGGL(adapters_expand, dim3((a.n + 255) / 256, std::min(a.m, 65535u)), dim3(256), 0, st, a, acc, slabs,
                     (const float*)((const char*)workspace + p.h), p.splits);
  return hipGetLastError();
}

}  // namespace w8a8
