// adapters.hip -- a low-rank BF16 adapter per row beside a shared W8A8
// projection, many adapters in one call.  No counterpart in the reference.
//
//   out[r][c] = bf16(residual + RN(RN(f32(q . w) * asc) * ws)
//                    + scaling[a] * sum_j B[a][c][j] * h[r][j]),
//   h[r][j] = sum_i A[a][j][i] * bf16(x[r][i]),   a = ids[r],
// a row whose id is outside [0, n_adapters) taking the projection alone.  h and
// both sums are held in f32.
//
// Here: row by row (decode batches, short prompts), out from the projection's exact
// sums; with the rows sorted by adapter (longer prompts): adapters_tiles.hip.
#include <algorithm>

#include "adapters.hpp"

namespace w8a8 {

// Eight values of an x row as loaded, and as f32: f32 rows rounded to BF16.
template <bool BF16>
struct Eight {
  v4i lo, hi;
  __device__ __forceinline__ void load(const void* x, size_t i) {
    const v4i* const p = (const v4i*)((const char*)x + i * (BF16 ? 2 : 4));
    lo = p[0];
    if constexpr (!BF16) hi = p[1];
  }
  __device__ __forceinline__ float operator[](int k) const {
    if constexpr (BF16) return k & 1 ? bf16_hi((uint32_t)lo[k / 2]) : bf16_lo((uint32_t)lo[k / 2]);
    return bf16_rne(__int_as_float(k < 4 ? lo[k] : hi[k - 4]));
  }
};

// h[row][j], J of them a wave: its lanes take runs of 8 values of K, so that every
// load is 1 KiB of an adapter row, and U runs are in flight together.  Rank 16, width
// 4096: 2.5 us for one row, a load's latency.
template <int J, bool BF16>
__global__ __launch_bounds__(256) void adapters_shrink(AdapterArgs a, float* h) {
  constexpr int U = J == 8 ? 2 : 8 / J;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t per_row = (a.rank + 4 * J - 1) / (4 * J), row = blockIdx.x / per_row;
  const uint32_t j0 = (blockIdx.x % per_row * 4 + wave) * J;
  if (j0 >= a.rank) return;
  const uint32_t id = (uint32_t)a.ids[row];
  if (id >= a.adapters) return;
  const size_t xo = (size_t)row * a.width, ao = ((size_t)id * a.rank + j0) * a.width;
  float sum[J];
#pragma unroll
  for (int j = 0; j < J; ++j) sum[j] = 0.f;
  auto add = [&](uint32_t i, auto runs) {
    constexpr int R = decltype(runs)::value;
    Eight<BF16> x[R];
    v4i w[R][J];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      x[u].load(a.x, xo + i + 512 * u);
#pragma unroll
      for (int j = 0; j < J; ++j) w[u][j] = *(const v4i*)(a.a + ao + (size_t)j * a.width + i + 512 * u);
    }
    __builtin_amdgcn_sched_barrier(0);  // every load is under way before the first use
#pragma unroll
    for (int u = 0; u < R; ++u)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sum[j] = __builtin_fmaf(bf16_lo((uint32_t)w[u][j][k]), x[u][2 * k], sum[j]);
          sum[j] = __builtin_fmaf(bf16_hi((uint32_t)w[u][j][k]), x[u][2 * k + 1], sum[j]);
        }
  };
  uint32_t i = 0;
  for (; i + 512 * U <= a.width; i += 512 * U) add(i + lane * 8, std::integral_constant<int, U>{});
  for (; i < a.width; i += 512)
    if (i + lane * 8 < a.width) add(i + lane * 8, std::integral_constant<int, 1>{});
  float mine = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const float t = wave_sum_f32(sum[j]);
    if (lane == j) mine = t;
  }
  if (lane < J) h[(size_t)row * a.rank + j0 + lane] = mine;  // rank % 8 == 0
}

// out row by row from the projection's exact sums (`slabs` partial ones) and h: a
// thread holds a column, its adapter row one contiguous run.  64 rows of 6144 columns,
// rank 32: 25 MB of adapter rows, mostly from L2, and four slabs in 5.6 us; the slabs'
// own epilogue kernel, 3.6 us, is left out.
__global__ __launch_bounds__(256) void adapters_expand(AdapterArgs a, const int32_t* __restrict__ acc, uint32_t slabs,
                                                       const float* __restrict__ h) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x, cc = min(c, a.n - 1);
  const size_t slab = (size_t)a.m * a.n;
  for (uint32_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    const uint32_t id = (uint32_t)a.ids[row];
    const size_t o = (size_t)row * a.n + cc;
    int32_t part[4];  // four slabs' loads together
#pragma unroll
    for (uint32_t s = 0; s < 4; ++s) part[s] = acc[o + min(s, slabs - 1) * slab];
    const float res = a.residual ? a.residual[o] : 0.f;
    float d = 0.f;
    if (id < a.adapters) {
      const uint16_t* const b = a.b + ((size_t)id * a.n + cc) * a.rank;
      for (uint32_t j0 = 0; j0 < a.rank; j0 += 32) {  // rank % 8 == 0
        v4i bv[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) bv[q] = *(const v4i*)(b + min(j0 + 8 * q, a.rank - 8));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t j = j0 + 8 * q;
          if (j >= a.rank) break;
          float hv[8];  // wave-uniform
#pragma unroll
          for (int i = 0; i < 8; ++i) hv[i] = h[(size_t)row * a.rank + j + i];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            d = __builtin_fmaf(bf16_lo((uint32_t)bv[q][i]), hv[2 * i], d);
            d = __builtin_fmaf(bf16_hi((uint32_t)bv[q][i]), hv[2 * i + 1], d);
          }
        }
      }
    }
    int32_t sum = part[0];
#pragma unroll
    for (uint32_t s = 1; s < 4; ++s) sum += s < slabs ? part[s] : 0;
    for (uint32_t s = 4; s < slabs; ++s) sum += acc[o + s * slab];
    float y = (float)sum * a.asc[row] * a.ws[cc];
    if (id < a.adapters) y += a.scaling[id] * d;
    if (c < a.n) store_routed(a.out, a.out_dtype, o, a.residual ? res + y : y);
  }
}

// Few rows: the projection by dot products and the second product with
// it, one launch less than the projection's own route and adapters_expand take.  A
// wave holds two columns of every row; each lane reads 16 bytes of a weight row at a
// time, and up to 8 ranks of a column's adapter row.
constexpr int kGemvCols = 2;
template <int M>
__global__ __launch_bounds__(256) void adapters_gemv(AdapterArgs a, const float* __restrict__ h) {
  constexpr int U = M == 1 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t c0 = (blockIdx.x * 4 + wave) * kGemvCols;
  if (c0 >= a.n) return;
  uint32_t id[M];
  const int8_t *w[kGemvCols], *q[M];
  int sum[M][kGemvCols];
#pragma unroll
  for (int r = 0; r < M; ++r) {
    id[r] = (uint32_t)a.ids[r];
    q[r] = a.q + (size_t)r * a.width;
#pragma unroll
    for (int c = 0; c < kGemvCols; ++c) sum[r][c] = 0;
  }
#pragma unroll
  for (int c = 0; c < kGemvCols; ++c) w[c] = a.w + (size_t)min(c0 + c, a.n - 1) * a.width;
  auto add = [&](uint32_t o, auto runs) {
    constexpr int R = decltype(runs)::value;
    v4i x[R][M], v[R][kGemvCols];
#pragma unroll
    for (int u = 0; u < R; ++u) {
#pragma unroll
      for (int c = 0; c < kGemvCols; ++c) v[u][c] = load_nt16(w[c] + o + 1024 * u);
#pragma unroll
      for (int r = 0; r < M; ++r) x[u][r] = load16(q[r] + o + 1024 * u);
    }
    __builtin_amdgcn_sched_barrier(0);  // every load is under way before the first use
#pragma unroll
    for (int u = 0; u < R; ++u)
#pragma unroll
      for (int r = 0; r < M; ++r)
#pragma unroll
        for (int c = 0; c < kGemvCols; ++c) sum[r][c] = dot16(v[u][c], x[u][r], sum[r][c]);
  };
  uint32_t o = 0;
  for (; o + 1024 * U <= a.width; o += 1024 * U) add(o + lane * 16, std::integral_constant<int, U>{});
  for (; o < a.width; o += 1024)
    if (o + lane * 16 < a.width) add(o + lane * 16, std::integral_constant<int, 1>{});
  int acc = 0;
  float delta = 0.f;
#pragma unroll
  for (int r = 0; r < M; ++r) {
    float d[kGemvCols];
#pragma unroll
    for (int c = 0; c < kGemvCols; ++c) d[c] = 0.f;
    if (id[r] < a.adapters && lane * 8u < a.rank) {  // rank <= 256
      const float* const hr = h + (size_t)r * a.rank + lane * 8;
      const v4f h0 = *(const v4f*)hr, h1 = *(const v4f*)(hr + 4);
#pragma unroll
      for (int c = 0; c < kGemvCols; ++c) {
        const v4i b = *(const v4i*)(a.b + ((size_t)id[r] * a.n + min(c0 + c, a.n - 1)) * a.rank + lane * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[c] = __builtin_fmaf(bf16_lo((uint32_t)b[i]), i < 2 ? h0[2 * i] : h1[2 * i - 4], d[c]);
          d[c] = __builtin_fmaf(bf16_hi((uint32_t)b[i]), i < 2 ? h0[2 * i + 1] : h1[2 * i - 3], d[c]);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kGemvCols; ++c) {
      const int t = wave_sum_i32(sum[r][c]);
      const float u = wave_sum_f32(d[c]);
      if (lane == r * kGemvCols + c) acc = t, delta = u;
    }
  }
  // lane kGemvCols r + c stores column c0 + c of row r
  const uint32_t row = lane / kGemvCols, c = c0 + lane % kGemvCols;
  if (row < (uint32_t)M && c < a.n) {
    const size_t at = (size_t)row * a.n + c;
    const uint32_t ad = (uint32_t)a.ids[row];
    float y = (float)acc * a.asc[row] * a.ws[c];
    if (ad < a.adapters) y += a.scaling[ad] * delta;
    store_routed(a.out, a.out_dtype, at, a.residual ? a.residual[at] + y : y);
  }
}

// ------------------------------------------------------------------ plan
// Few rows on a small projection: adapters_gemv, whose dot products per row cost
// less than a launch while the rows past the first make at most 2^20 * 100 of them.
// Measured, adapters_gemv / the projection's route and adapters_expand us: 4096 x 4096,
// rank 16, m = 2 / 3 / 4 9.6 / 9.8 / 10.5 against 12.4 / 12.3 / 12.6; 4096 x 12288 14.0 /
// 15.0 / 16.9 against 16.3; 24576 x 4096 22.3 / 24.7 / 28.6 against 22.3 / 22.0 / 22.0.
constexpr uint32_t kGemvRows = 4;
static bool gemv_leads(const AdapterArgs& a) {
  return a.m == 1 || (a.m <= kGemvRows && (uint64_t)(a.m - 1) * a.n * a.width <= (100u << 20));
}

// Row by row, every row reads its own adapter: m rank (n + width) values from L2,
// at about 10 TB/s, beside the projection.  The fused tiles read an adapter once,
// but run in the tiles' own time: 22 us more than the projection at width 4096, 43
// at 12288 until the tiles fill the card, and 1.5 us for each 32 ranks of every
// adapter after a tile's first.  Measured, rows / fused us at 4 adapters, on the same
// weights again: 4096 x 4096, rank 16, m = 512 (134 MB) 32.8 / 39.8, m = 1024 (268 MB) 53 /
// 41; rank 64, m = 128 (134 MB) 30 / 43, m = 512 63 / 46; 4096 x 12288, rank 16, m = 512
// (268 MB) 55 / 69, m = 1024 99 / 77; 24576 x 4096, rank 32, m = 80 (147 MB) 40 / 42, m = 128
// 49 / 43.  On weights of each pass's own: 35 / 44, 58 / 51; 30 / 48, 66 / 51; 65 / 96, 113
// / 100; 42 / 53, 50 / 55.
static bool fused_leads(const AdapterArgs& a) {
  if (gemv_leads(a)) return false;
  const double rows_us = (double)a.m * a.rank * ((double)a.n + a.width) * 2.0 / 10e6;
  const uint32_t mean = a.m / std::min(a.m, a.adapters), met = std::min(a.m, 256u) / std::min(mean, 256u);
  return rows_us > 8.0 + a.width / 400.0 + 1.5 * ((a.rank + 31) / 32) * (met > 1 ? met - 1 : 0);
}

AdapterPlan adapter_plan(const AdapterArgs& a) {
  AdapterPlan p{};
  const uint32_t mean = a.m / std::min(a.m, a.adapters);
  p.gemv = gemv_leads(a);
  p.fused = fused_leads(a);
  if (p.fused) {
    p.ranks = a.rank <= 32 ? 32 : a.rank <= 64 ? 64 : a.rank <= 128 ? 128 : 256;
    p.tile = (uint64_t)((a.m + 255) / 256) * ((a.n + 255) / 256) >= 192 ? 256 : 128;
    p.tail = a.width % 128 != 0;
    const uint32_t all = (a.width * 2 + 127) / 128;  // stages of an adapter row
    p.bt = mean <= 48 ? 32 : 128;
    p.tiles = a.m / p.bt + std::min(a.m, a.adapters);
    // about 512 workgroups, each with eight stages at least
    const uint32_t want = std::max(1u, std::min(512 / std::max(1u, a.m / p.bt), 16u));
    p.stages = std::max((all + want - 1) / want, std::min(all, 8u));
    p.splits = (all + p.stages - 1) / p.stages;
  } else {
    // few values: one a wave; many: eight, which share their loads of x (64 rows of
    // rank 32 at width 4096, one / two / eight: 3.9 / 4.3 / 6.9 us)
    p.values = a.m * a.rank <= 4096 ? 1 : a.m * a.rank <= 16384 ? 2 : 8;
    p.splits = 1;
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  p.h = take((size_t)p.splits * a.m * a.rank * 4);
  if (p.fused) {
    const uint32_t blocks = sort_blocks(a.m);
    p.order = take((size_t)a.m * 4);
    p.table = take((size_t)p.tiles * sizeof(RowTile));
    p.n_tiles = take(4);
    p.counts = take(blocks > 1 ? (size_t)blocks * (a.adapters + 1) * 4 : 0);
    p.scaled = take((size_t)a.m * part_width(a.rank) * 4);
  }
  p.bytes = at;
  return p;
}

size_t adapters_workspace_bytes(const AdapterArgs& a) { return adapter_plan(a).bytes; }
bool adapters_fused(const AdapterArgs& a) {
  const AdapterPlan p = adapter_plan(a);
  return p.gemv || p.fused;
}

hipError_t launch_adapters_before(hipStream_t st, const AdapterArgs& a, void* workspace) {
  const AdapterPlan p = adapter_plan(a);
  if (p.fused) return launch_adapters_fused(st, a, p, (char*)workspace);
  float* const h = (float*)((char*)workspace + p.h);
  const uint32_t J = p.values;
  const dim3 grid((a.rank + 4 * J - 1) / (4 * J) * a.m);
  auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(256), 0, st, a, h); };
  if (a.x_bf16) go(J == 1 ? adapters_shrink<1, true> : J == 2 ? adapters_shrink<2, true> : adapters_shrink<8, true>);
  else go(J == 1 ? adapters_shrink<1, false> : J == 2 ? adapters_shrink<2, false> : adapters_shrink<8, false>);
  if (p.gemv) {
    auto k = a.m == 1 ? adapters_gemv<1> : a.m == 2 ? adapters_gemv<2> : a.m == 3 ? adapters_gemv<3> : adapters_gemv<4>;
    hipLaunchKernelGGL(k, dim3((a.n + 4 * kGemvCols - 1) / (4 * kGemvCols)), dim3(256), 0, st, a, h);
  }
  return hipGetLastError();
}

hipError_t launch_adapters_after(hipStream_t st, const AdapterArgs& a, const int32_t* acc, uint32_t slabs,
                                 const void* workspace) {
  const AdapterPlan p = adapter_plan(a);
  hipLaunchKernelGGL(adapters_expand, dim3((a.n + 255) / 256, std::min(a.m, 65535u)), dim3(256), 0, st, a, acc, slabs,
                     (const float*)((const char*)workspace + p.h));
  return hipGetLastError();
}

}  // namespace w8a8
