// adapters_tiles.hip -- adapters beside a projection with the rows sorted by
// adapter (adapters.hip has the definition).
//
//   adapters_order          the sort, and the tiles: up to bt rows of one adapter;
//   adapters_shrink_tiles   h's partial sums, tile x share of K, by bf16 MFMA;
//   adapters_parts          h as two BF16 parts, high and low, whose products with
//                           B are exact: 16 bits of h count, not 8;
//   adapters_gemm           the projection over the sorted rows, its int8 sums
//                           scaled in their registers and the second product
//                           added to them by bf16 MFMA before the one store.
#include "adapters.hpp"

namespace w8a8 {

// Rows sorted by adapter, those without one last.
__global__ __launch_bounds__(64 * kSortWaves) void adapters_order(const int32_t* ids, uint32_t m, uint32_t per_block,
                                                                  uint32_t adapters, const uint32_t* counts,
                                                                  uint32_t bt, uint32_t* order, RowTile* table,
                                                                  uint32_t* n_tiles) {
  extern __shared__ uint32_t hist[];
  __shared__ uint32_t part[kSortWaves];
  sort_items<true>(
      ids, m, per_block, adapters, counts, hist, part,
      [&](uint32_t first, uint32_t total) {
        if (blockIdx.x == 0) list_tiles(first, threadIdx.x < adapters ? total : 0, bt, part, table, n_tiles);
      },
      [&](uint32_t row, int32_t p) { order[p] = row; });
}

// h[share][p or row][j] of a tile: the token operand's rows are gathered, K is the
// share's stages.  by_row: h is read row by row, not in the sorted order.
template <class T>
__global__ __launch_bounds__(64 * T::NW) void adapters_shrink_tiles(AdapterArgs a, const uint32_t* order,
                                                                    const RowTile* table, const uint32_t* n_tiles,
                                                                    float* h, uint32_t stages, bool by_row) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[T::LDS];
  if (blockIdx.x >= *n_tiles) return;
  const RowTile t = table[blockIdx.x];
  const uint32_t k0 = blockIdx.y * stages * 64, values = min(stages * 64, a.width - k0);
  constexpr size_t XB = T::OP == OP_BF16 ? 2 : 4;
  T s;
  s.run(
      lds, values * 2,
      [&](int r) {
        const uint32_t row = order[t.first + ((uint32_t)r < t.rows ? r : 0)];
        return (const int8_t*)a.x + ((size_t)row * a.width + k0) * XB;
      },
      [&](int r) {
        return (const int8_t*)(a.a + ((size_t)t.of * a.rank + min((uint32_t)r, a.rank - 1)) * a.width + k0);
      },
      [](int) { return (const float*)nullptr; }, 0);
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t wt0 = (wave / T::WAVES_N) * T::WT, wn0 = (wave % T::WAVES_N) * T::WN;
#pragma unroll
  for (int f = 0; f < T::FT; ++f) {
    const uint32_t r = wt0 + 32 * f + (lane & 31);
    if (r >= t.rows) continue;
    const uint32_t p = by_row ? order[t.first + r] : t.first + r;
    float* const to = h + ((size_t)blockIdx.y * a.m + p) * a.rank;
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 4) {
        const uint32_t n = wn0 + 32 * j + 2 * v + 4 * half;
        if (n < a.rank) *(v4f*)(to + n) = v4f{s.acc[f][j][v], s.acc[f][j][v + 1], s.acc[f][j][v + 2], s.acc[f][j][v + 3]};
      }
  }
}

// high + low = the sum of the shares, to 16 bits; rows padded with zeros to a
// multiple of 16 values.
__global__ __launch_bounds__(256) void adapters_parts(const float* h, uint32_t m, uint32_t rank, uint32_t splits,
                                                      uint16_t* high, uint16_t* low) {
  const uint32_t quads = (rank + 15) / 16 * 4;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)m * quads) return;
  const uint32_t j = (uint32_t)(i % quads) * 4;
  v4f s{};
  if (j < rank)
    for (uint32_t t = 0; t < splits; ++t) s += *(const v4f*)(h + ((size_t)t * m + i / quads) * rank + j);
  const uint32_t h0 = bf16_pair(s.x, s.y), h1 = bf16_pair(s.z, s.w);
  *(v2i*)(high + i * 4) = v2i{(int)h0, (int)h1};
  *(v2i*)(low + i * 4) = v2i{(int)bf16_pair(s.x - bf16_lo(h0), s.y - bf16_hi(h0)),
                             (int)bf16_pair(s.z - bf16_lo(h1), s.w - bf16_hi(h1))};
}

// M tiles of a strip: the tiles that an XCD runs at once share panels of both
// operands (gemm.hip).
constexpr uint32_t kStripTiles = 4;

template <class T>
__global__ __launch_bounds__(64 * T::NW, 2) void adapters_gemm(AdapterArgs a, const uint32_t* order,
                                                              const uint16_t* high, const uint16_t* low,
                                                              uint32_t tiles_m, uint32_t tiles_n, bool wide) {
  constexpr int STRIDE = T::WN + 4;  // f32 values of an LDS row, padded
  static_assert(T::NW * 32 * STRIDE * 4 <= T::LDS, "the epilogue reuses the rings");
  __shared__ __attribute__((aligned(1024))) int8_t lds[T::LDS];
  const uint32_t G = tiles_m * tiles_n;
  uint32_t at = blockIdx.x;
  if (G % 8 == 0) at = (at % 8) * (G / 8) + at / 8;
  const uint32_t strip = kStripTiles * tiles_n, s0 = at / strip * kStripTiles, in = at % strip;
  const uint32_t sm = min(kStripTiles, tiles_m - s0);
  const uint32_t m0 = (s0 + in % sm) * T::BT, n0 = in / sm * T::BN, K = a.width;
  T s;
  s.run(
      lds, K, [&](int r) { return a.q + (size_t)order[m0 + r < a.m ? m0 + r : m0] * K; },
      [&](int r) { return a.w + (size_t)(n0 + r < a.n ? n0 + r : n0) * K; }, [](int) { return (const float*)nullptr; },
      0);

  const int lane = threadIdx.x & 63, half = lane >> 5, tl = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t wt0 = m0 + (wave / T::WAVES_N) * T::WT, cw = n0 + (wave % T::WAVES_N) * T::WN;
  const uint32_t padded = (a.rank + 15) / 16 * 16;
  float* const mine = (float*)lds + wave * 32 * STRIDE;
  __syncthreads();  // every wave is done with the rings
#pragma unroll
  for (int f = 0; f < T::FT; ++f) {
    const uint32_t p = wt0 + 32 * f + tl, pc = p < a.m ? p : m0;
    const uint32_t row = order[pc];
    const uint32_t id = p < a.m ? (uint32_t)a.ids[row] : ~0u;
    const float asc = a.asc[row];
    // a block of columns at a time: what the sums leave of the registers
#pragma unroll
    for (int j = 0; j < T::FN; ++j) {
      float y[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const uint32_t c = cw + 32 * j + 8 * (v >> 2) + 4 * half + (v & 3);
        y[v] = (float)s.acc[f][j][v] * asc * a.ws[c < a.n ? c : a.n - 1];
      }
      each_adapter(id, id < a.adapters, [&](uint32_t ad, uint32_t rows) {
        const uint16_t* const b = a.b + ((size_t)ad * a.n + min(cw + 32 * j + tl, a.n - 1)) * a.rank + 8 * half;
        const size_t ho = (size_t)pc * padded + 8 * half;
        v16f d{};
#pragma unroll 2
        for (uint32_t k = 0; k < a.rank; k += 16) {
          const v4i hi = *(const v4i*)(high + ho + k), lo = *(const v4i*)(low + ho + k);
          const v4i bf = k + 8 * half < a.rank ? *(const v4i*)(b + k) : v4i{};
          d = mfma_bf16(bf, hi, d);
          d = mfma_bf16(bf, lo, d);
        }
        const float sc = a.scaling[ad];
        if ((rows >> tl) & 1) {
#pragma unroll
          for (int v = 0; v < 16; ++v) y[v] += sc * d[v];
        }
      });
      // 32 rows through the wave's own LDS: whole runs of a row to memory
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *(v4f*)(mine + tl * STRIDE + 32 * j + 2 * v + 4 * half) = v4f{y[v], y[v + 1], y[v + 2], y[v + 3]};
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (wide) {  // n % 8 == 0: 16-byte stores
      constexpr int PER = T::WN / 8, ROWS = 64 / PER;
#pragma unroll
      for (int i = 0; i < 32; i += ROWS) {
        const uint32_t r = i + lane / PER, c = (lane % PER) * 8;
        const uint32_t to = (uint32_t)__shfl((int)row, (int)r, kWave);
        if (wt0 + 32 * f + r >= a.m || cw + c >= a.n) continue;
        const size_t o = (size_t)to * a.n + cw + c;
        v4f lo = *(const v4f*)(mine + r * STRIDE + c), hi = *(const v4f*)(mine + r * STRIDE + c + 4);
        if (a.residual) {
          lo += *(const v4f*)(a.residual + o);
          hi += *(const v4f*)(a.residual + o + 4);
        }
        if (a.out_dtype == W8A8_OUT_F32) {
          float* const out = (float*)a.out + o;
          *(v4f*)out = v4f{bf16_rne(lo.x), bf16_rne(lo.y), bf16_rne(lo.z), bf16_rne(lo.w)};
          *(v4f*)(out + 4) = v4f{bf16_rne(hi.x), bf16_rne(hi.y), bf16_rne(hi.z), bf16_rne(hi.w)};
        } else {
          *(v4i*)((uint16_t*)a.out + o) = v4i{(int)bf16_pair(lo.x, lo.y), (int)bf16_pair(lo.z, lo.w),
                                             (int)bf16_pair(hi.x, hi.y), (int)bf16_pair(hi.z, hi.w)};
        }
      }
    } else {
      for (int r = 0; r < 32; ++r) {
        const uint32_t to = (uint32_t)__builtin_amdgcn_readlane((int)row, r);
        if (wt0 + 32 * f + r >= a.m) break;
#pragma unroll
        for (int c = lane; c < T::WN; c += 64) {
          if (cw + c >= a.n) continue;
          const size_t o = (size_t)to * a.n + cw + c;
          const float v = mine[r * STRIDE + c];
          store_routed(a.out, a.out_dtype, o, a.residual ? a.residual[o] + v : v);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ------------------------------------------------------------------ launches
namespace {
template <int BT, int BN, int WT, int WN, int SA, int SB>
void shrink_as(hipStream_t st, const AdapterArgs& a, const AdapterPlan& p, char* ws) {
  auto go = [&](auto tile) {
    using T = decltype(tile);
    hipLaunchKernelGGL(adapters_shrink_tiles<T>, dim3(p.tiles, p.splits), dim3(64 * T::NW), 0, st, a,
                       (const uint32_t*)(ws + p.order), (const RowTile*)(ws + p.table), (const uint32_t*)(ws + p.n_tiles),
                       (float*)(ws + p.h), p.stages, !p.fused);
  };
  if (a.x_bf16) go(TileStream<BT, BN, WT, WN, SA, SB, false, true, OP_BF16>{});
  else go(TileStream<BT, BN, WT, WN, SA, SB, false, true, OP_BF16_F32>{});
}

template <int BT, int BN, int WT, int WN, int SA, int SB>
void gemm_as(hipStream_t st, const AdapterArgs& a, const AdapterPlan& p, char* ws) {
  const uint32_t tm = (a.m + BT - 1) / BT, tn = (a.n + BN - 1) / BN;
  auto aligned = [](const void* q) { return ((uintptr_t)q & 15) == 0; };
  const bool wide = a.n % 8 == 0 && aligned(a.out) && aligned(a.residual);
  auto go = [&](auto tile) {
    using T = decltype(tile);
    hipLaunchKernelGGL(adapters_gemm<T>, dim3(tm * tn), dim3(64 * T::NW), 0, st, a, (const uint32_t*)(ws + p.order),
                       (const uint16_t*)(ws + p.high), (const uint16_t*)(ws + p.low), tm, tn, wide);
  };
  if (a.width % 128 == 0) go(TileStream<BT, BN, WT, WN, SA, SB, false, false>{});
  else go(TileStream<BT, BN, WT, WN, SA, SB, false, true>{});
}
}  // namespace

hipError_t launch_adapters_sorted(hipStream_t st, const AdapterArgs& a, const AdapterPlan& p, char* ws) {
  uint32_t* const counts = (uint32_t*)(ws + p.counts);
  const uint32_t blocks = sort_blocks(a.m), per = sort_per_block(a.m), lds = kSortWaves * (a.adapters + 1) * 4;
  if (blocks > 1)
    hipLaunchKernelGGL(sort_counts<true>, dim3(blocks), dim3(64 * kSortWaves), lds, st, a.ids, a.m, per, a.adapters,
                       counts);
  hipLaunchKernelGGL(adapters_order, dim3(blocks), dim3(64 * kSortWaves), lds, st, a.ids, a.m, per, a.adapters, counts,
                     p.bt, (uint32_t*)(ws + p.order), (RowTile*)(ws + p.table), (uint32_t*)(ws + p.n_tiles));
  const int rank = a.rank <= 32 ? 32 : a.rank <= 64 ? 64 : a.rank <= 128 ? 128 : 256;
  if (p.bt == 32) {
    if (rank == 32) shrink_as<32, 32, 32, 32, 4, 4>(st, a, p, ws);
    else if (rank == 64) shrink_as<32, 64, 32, 32, 4, 4>(st, a, p, ws);
    else if (rank == 128) shrink_as<32, 128, 32, 32, 3, 3>(st, a, p, ws);
    else shrink_as<32, 256, 32, 64, 3, 3>(st, a, p, ws);
  } else {
    if (rank == 32) shrink_as<128, 32, 32, 32, 3, 3>(st, a, p, ws);
    else if (rank == 64) shrink_as<128, 64, 32, 64, 3, 3>(st, a, p, ws);
    else if (rank == 128) shrink_as<128, 128, 64, 64, 3, 3>(st, a, p, ws);
    else shrink_as<128, 256, 64, 64, 2, 2>(st, a, p, ws);
  }
  return hipGetLastError();
}

hipError_t launch_adapters_fused(hipStream_t st, const AdapterArgs& a, const AdapterPlan& p, char* ws) {
  const size_t quads = (size_t)a.m * ((a.rank + 15) / 16 * 4);
  hipLaunchKernelGGL(adapters_parts, dim3((uint32_t)((quads + 255) / 256)), dim3(256), 0, st,
                     (const float*)(ws + p.h), a.m, a.rank, p.splits, (uint16_t*)(ws + p.high),
                     (uint16_t*)(ws + p.low));
  const uint64_t big = (uint64_t)((a.m + 255) / 256) * ((a.n + 255) / 256);
  if (big >= 192) gemm_as<256, 256, 64, 128, 2, 3>(st, a, p, ws);
  else gemm_as<128, 128, 64, 64, 2, 3>(st, a, p, ws);
  return hipGetLastError();
}

}  // namespace w8a8
