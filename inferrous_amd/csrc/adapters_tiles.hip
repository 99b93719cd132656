// adapters_tiles.hip -- adapters beside a projection with the rows sorted by
// adapter (adapters.hip has the definition).  4096 rows on 4096 x 12288, 6 adapters of
// rank 64, with a residual: 229-231 us a pass among others, the projection's tiles 193 at
// the least and 208-220 in a run of passes (the projection alone 175-183); the large int8
// library product's rate, 2.07 POPS, would take 203.
//
//   adapters_order          the sort, and the tiles: up to bt rows of one adapter;
//   adapters_shrink_tiles   h's partial sums, tile x share of K, by bf16 MFMA;
//   adapters_scale          scaling * h, the shares of K added;
//   adapters_gemm           the projection over the sorted rows, its int8 sums
//                           scaled in their registers and the second product
//                           added to them by bf16 MFMA before the one store: of
//                           scaling * h as three BF16 parts, whose sum is the f32
//                           value and whose products with B are exact.
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

// h[share][p][j] of a tile, in the sorted order: the token operand's rows are
// gathered, K is the share's stages.  4096 rows x 12288, rank 64: 26 us for 100 MB of x
// and 50 MB of adapter rows, 5.8 TB/s; fragments straight from memory took 105 us, a
// line for each 32 bytes.
template <class T>
__global__ __launch_bounds__(64 * T::NW) void adapters_shrink_tiles(AdapterArgs a, const uint32_t* order,
                                                                    const RowTile* table, const uint32_t* n_tiles,
                                                                    float* h, uint32_t stages) {
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
    float* const to = h + ((size_t)blockIdx.y * a.m + t.first + r) * a.rank;
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 4) {
        const uint32_t n = wn0 + 32 * j + 2 * v + 4 * half;
        if (n < a.rank) *(v4f*)(to + n) = v4f{s.acc[f][j][v], s.acc[f][j][v + 1], s.acc[f][j][v + 2], s.acc[f][j][v + 3]};
      }
  }
}

// scaling * the sum of the shares, without an infinite scaling (adapters_gemm); rows
// padded with zeros to a multiple of 32 values.
__device__ __forceinline__ bool infinite(float v) { return __builtin_fabsf(v) == __builtin_inff(); }
__global__ __launch_bounds__(256) void adapters_scale(AdapterArgs a, const uint32_t* order, const float* h,
                                                      uint32_t splits, float* scaled) {
  const uint32_t quads = part_width(a.rank) / 4;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)a.m * quads) return;
  const uint32_t p = (uint32_t)(i / quads), j = (uint32_t)(i % quads) * 4;
  const uint32_t id = (uint32_t)a.ids[order[p]];
  v4f s{};
  if (j < a.rank && id < a.adapters) {
#pragma unroll 4
    for (uint32_t t = 0; t < splits; ++t) s += *(const v4f*)(h + ((size_t)t * a.m + p) * a.rank + j);
    const float scaling = a.scaling[id];
    if (!infinite(scaling)) s *= scaling;
  }
  *(v4f*)(scaled + i * 4) = s;
}

// Three parts of v, BF16 values in their high halves: each holds the next 8 of v's 24
// bits, cut off, so that their sum is v.  An infinite B times a part of 0 would be NaN:
// such a part is 2^-48 v, far below f32's last bit of the products' sum.  Every part of
// an infinity or NaN is v.
__device__ __forceinline__ void split3(float v, uint32_t (&part)[3]) {
  const float least = v * 0x1p-48f;
  part[0] = __float_as_uint(v) & 0xffff0000u;
  float rest = v - __uint_as_float(part[0]);
  rest = rest != 0.f ? rest : least;
  part[1] = __float_as_uint(rest) & 0xffff0000u;
  rest -= __uint_as_float(part[1]);
  part[2] = __float_as_uint(rest != 0.f ? rest : least);
  if (!(__builtin_fabsf(v) < __builtin_inff())) part[0] = part[1] = part[2] = v != v ? 0x7fc00000u : __float_as_uint(v);
}

// M tiles of a strip: the tiles that an XCD runs at once share panels of both
// operands (gemm.hip).
constexpr uint32_t kStripTiles = 4;

// After the K loop the rings' memory holds, 32 ranks at a time, the tile's B rows of
// one adapter and its rows' three parts of h: one load from memory serves every
// wave, and the next ranks (or adapter) are in flight while the waves multiply.
// Rows of another adapter keep the value they had (a lane is one row).
template <class T>
__global__ __launch_bounds__(64 * T::NW, 2) void adapters_gemm(AdapterArgs a, const uint32_t* order,
                                                              const float* scaled, uint32_t tiles_m,
                                                              uint32_t tiles_n, bool wide) {
  constexpr int PAIR = 40;          // BF16 values of an LDS row of 32, padded
  constexpr int STRIDE = 64 + 4;    // f32 values of an LDS row of 64 columns, padded
  constexpr int THREADS = 64 * T::NW;
  constexpr int B_AT = 0, H_AT = T::BN * PAIR * 2, H_SIZE = T::BT * PAIR * 2, W_AT = H_AT + 3 * H_SIZE;
  constexpr int O_AT = W_AT + T::BN * 4;
  static_assert(O_AT + T::NW * 32 * STRIDE * 4 <= T::LDS, "the epilogue reuses the rings");
  static_assert(T::WN % 64 == 0 && T::BN * 4 % THREADS == 0 && T::BT * 4 % THREADS == 0, "whole loads");
  constexpr int LB = T::BN * 4 / THREADS, LH = T::BT * 8 / THREADS;  // 16-byte loads of a thread
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
  const uint32_t wt = (wave / T::WAVES_N) * T::WT, wn = (wave % T::WAVES_N) * T::WN;
  const uint32_t padded = part_width(a.rank), rows_in = min((uint32_t)T::BT, a.m - m0);
  // the wave's rows
  uint32_t row[T::FT], id[T::FT];
  float asc[T::FT], scaling[T::FT];
#pragma unroll
  for (int f = 0; f < T::FT; ++f) {
    const uint32_t r = wt + 32 * f + tl;
    row[f] = order[m0 + (r < rows_in ? r : 0)];
    id[f] = r < rows_in ? (uint32_t)a.ids[row[f]] : ~0u;
    asc[f] = a.asc[row[f]];
    scaling[f] = id[f] < a.adapters ? a.scaling[id[f]] : 0.f;
  }
  // the tile's ids, every wave alike: lane l's are rows l, l + 64, ...
  uint32_t tid[T::BT / 64];
#pragma unroll
  for (int i = 0; i < T::BT / 64; ++i) {
    const uint32_t r = lane + 64 * i;
    tid[i] = r < rows_in ? (uint32_t)a.ids[order[m0 + r]] : ~0u;
  }
  __syncthreads();  // every wave is done with the rings
  float* const tile_ws = (float*)(lds + W_AT);
  for (int c = threadIdx.x; c < T::BN; c += THREADS) tile_ws[c] = a.ws[min(n0 + c, a.n - 1)];
  __syncthreads();
  v16f y[T::FT][T::FN];
#pragma unroll
  for (int j = 0; j < T::FN; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const v4f w = *(const v4f*)(tile_ws + wn + 32 * j + 8 * q + 4 * half);
#pragma unroll
      for (int f = 0; f < T::FT; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[f][j][4 * q + i] = (float)s.acc[f][j][4 * q + i] * asc[f] * w[i];
    }
  // An infinite scaling multiplies the row's whole second product, as in the definition:
  // its row starts from 0 here (NaN where the projection is not finite).
  bool odd[T::FT], any_odd = false;
#pragma unroll
  for (int f = 0; f < T::FT; ++f) {
    odd[f] = infinite(scaling[f]);
    any_odd |= odd[f];
  }
  any_odd = __any(any_odd);
  auto times = [&](auto factor) {
#pragma unroll
    for (int f = 0; f < T::FT; ++f)
#pragma unroll
      for (int j = 0; j < T::FN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) y[f][j][v] = odd[f] ? y[f][j][v] * factor(f) : y[f][j][v];
  };
  if (any_odd) times([](int) { return 0.f; });
  // Rows are sorted by adapter, those without one last: the tile's adapters follow
  // each other, each from the row after the last one's.
  auto at_row = [&](uint32_t r) {  // the id of tile row r, wave-uniform
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < T::BT / 64; ++i)
      if ((r >> 6) == (uint32_t)i) v = (uint32_t)__builtin_amdgcn_readlane((int)tid[i], (int)(r & 63));
    return v;
  };
  auto count = [&](uint32_t ad) {
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < T::BT / 64; ++i) c += (uint32_t)__popcll(__ballot(tid[i] == ad));
    return c;
  };
  v4i rb[LB];
  v4f rh[LH];
  auto fetch = [&](uint32_t ad, uint32_t k) {
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const uint32_t t = threadIdx.x + i * THREADS, kk = k + (t & 3) * 8;
      rb[i] = kk < a.rank ? *(const v4i*)(a.b + ((size_t)ad * a.n + min(n0 + (t >> 2), a.n - 1)) * a.rank + kk) : v4i{};
    }
#pragma unroll
    for (int i = 0; i < LH; ++i) {
      const uint32_t t = threadIdx.x + i * THREADS, r = t >> 3;
      rh[i] = *(const v4f*)(scaled + (size_t)(m0 + (r < rows_in ? r : 0)) * padded + k + (t & 7) * 4);
    }
  };
  uint32_t r0 = 0, ad = at_row(0);
  if (ad < a.adapters) fetch(ad, 0);
  while (ad < a.adapters) {
    const uint32_t r1 = r0 + count(ad), next = r1 < rows_in ? at_row(r1) : ~0u;
    for (uint32_t k = 0; k < a.rank; k += 32) {
      __syncthreads();  // the last ranks are multiplied
#pragma unroll
      for (int i = 0; i < LB; ++i) {
        const uint32_t t = threadIdx.x + i * THREADS;
        *(v4i*)(lds + B_AT + (t >> 2) * PAIR * 2 + (t & 3) * 16) = rb[i];
      }
#pragma unroll
      for (int i = 0; i < LH; ++i) {
        const uint32_t t = threadIdx.x + i * THREADS;
        uint32_t q[4][3];
#pragma unroll
        for (int l = 0; l < 4; ++l) split3(rh[i][l], q[l]);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *(v2i*)(lds + H_AT + p * H_SIZE + (t >> 3) * PAIR * 2 + (t & 7) * 8) =
              v2i{(int)__builtin_amdgcn_perm(q[1][p], q[0][p], 0x07060302u),
                  (int)__builtin_amdgcn_perm(q[3][p], q[2][p], 0x07060302u)};
      }
      __syncthreads();
      if (k + 32 < a.rank) fetch(ad, k + 32);
      else if (next < a.adapters) fetch(next, 0);
#pragma unroll
      for (int f = 0; f < T::FT; ++f) {
        const bool on = id[f] == ad;
        if (!__ballot(on)) continue;
        v4i hp[3][2];
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            hp[p][i] = *(const v4i*)(lds + H_AT + p * H_SIZE + (wt + 32 * f + tl) * PAIR * 2 + 32 * i + 16 * half);
#pragma unroll
        for (int j = 0; j < T::FN; ++j) {
          v16f d = y[f][j];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const v4i b = *(const v4i*)(lds + B_AT + (wn + 32 * j + tl) * PAIR * 2 + 32 * i + 16 * half);
#pragma unroll
            for (int p = 0; p < 3; ++p) d = mfma_bf16(b, hp[p][i], d);
          }
#pragma unroll
          for (int v = 0; v < 16; ++v) y[f][j][v] = on ? d[v] : y[f][j][v];
        }
      }
    }
    r0 = r1;
    ad = next;
  }
  if (any_odd) times([&](int f) { return scaling[f]; });
  // 32 rows x 64 columns at a time through the wave's own LDS: whole runs of a row
  // to memory
  float* const mine = (float*)(lds + O_AT) + wave * 32 * STRIDE;
#pragma unroll
  for (int f = 0; f < T::FT; ++f)
#pragma unroll
    for (int j0 = 0; j0 < T::FN; j0 += 2) {
      const uint32_t cw = n0 + wn + 32 * j0, rw = wt + 32 * f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
          *(v4f*)(mine + tl * STRIDE + 32 * j + 2 * v + 4 * half) =
              v4f{y[f][j0 + j][v], y[f][j0 + j][v + 1], y[f][j0 + j][v + 2], y[f][j0 + j][v + 3]};
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (wide) {  // n % 8 == 0: 16-byte stores
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          const uint32_t r = i + (lane >> 3), c = (lane & 7) * 8;
          const uint32_t to = (uint32_t)__shfl((int)row[f], (int)r, kWave);
          if (rw + r >= rows_in || cw + c >= a.n) continue;
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
      } else if (cw + lane < a.n) {
        for (uint32_t r = 0; r < 32 && rw + r < rows_in; ++r) {
          const size_t o = (size_t)(uint32_t)__builtin_amdgcn_readlane((int)row[f], (int)r) * a.n + cw + lane;
          const float v = mine[r * STRIDE + lane];
          store_routed(a.out, a.out_dtype, o, a.residual ? a.residual[o] + v : v);
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
                       (float*)(ws + p.h), p.stages);
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
                       (const float*)(ws + p.scaled), tm, tn, wide);
  };
  if (p.tail) go(TileStream<BT, BN, WT, WN, SA, SB, false, true>{});
  else go(TileStream<BT, BN, WT, WN, SA, SB, false, false>{});
}
}  // namespace

hipError_t launch_adapters_fused(hipStream_t st, const AdapterArgs& a, const AdapterPlan& p, char* ws) {
  uint32_t* const counts = (uint32_t*)(ws + p.counts);
  const uint32_t blocks = sort_blocks(a.m), per = sort_per_block(a.m), lds = kSortWaves * (a.adapters + 1) * 4;
  if (blocks > 1)
    hipLaunchKernelGGL(sort_counts<true>, dim3(blocks), dim3(64 * kSortWaves), lds, st, a.ids, a.m, per, a.adapters,
                       counts);
  hipLaunchKernelGGL(adapters_order, dim3(blocks), dim3(64 * kSortWaves), lds, st, a.ids, a.m, per, a.adapters, counts,
                     p.bt, (uint32_t*)(ws + p.order), (RowTile*)(ws + p.table), (uint32_t*)(ws + p.n_tiles));
  const uint32_t rank = p.ranks;
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
  const size_t quads = (size_t)a.m * (part_width(a.rank) / 4);
  hipLaunchKernelGGL(adapters_scale, dim3((uint32_t)((quads + 255) / 256)), dim3(256), 0, st, a,
                     (const uint32_t*)(ws + p.order), (const float*)(ws + p.h), p.splits, (float*)(ws + p.scaled));
  if (p.tile == 256) gemm_as<256, 256, 64, 128, 2, 3>(st, a, p, ws);
  else gemm_as<128, 128, 64, 64, 2, 3>(st, a, p, ws);
  return hipGetLastError();
}

}  // namespace w8a8
