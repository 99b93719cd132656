// experts_tiles.hip -- the routed experts' MLP expert by expert: the slots
// sorted by expert, each expert's rows multiplied in tiles by MFMA, and the
// slots' products summed row by row.  The definition is in experts.hip.
//
// For 4096 rows x 8 of 64 experts, hidden 4096, inner 1024 (825 G operations; the
// large int8 library product's rate, 2.07 POPS, would take 398 us): 700-718 us.
//
//   experts_plan       sorts the slots (a counting sort that keeps their order)
//                      and lists the token tiles: up to BT rows of one expert;
//   experts_gate_up    a tile's gate and up sums over 128 columns of act, the
//                      SiLU product, and its codes and scale;
//   experts_down       a tile's y over BN columns, the stages of K being the
//                      128-column groups, each scaled into f32 sums;
//   experts_combine    out = residual + sum over a row's slots of weight * y.
//
// y goes through memory in f32, the pass's largest stream: a sum over slots is of
// f32 values, and a column much larger than its neighbours costs them nothing.
#include "experts.hpp"
#include "tile_stream.hpp"

namespace w8a8 {

// ------------------------------------------------------------------ plan
__global__ __launch_bounds__(64 * kSortWaves) void experts_plan(const int32_t* ids, uint32_t slots, uint32_t per_block,
                                                                uint32_t experts, const uint32_t* counts, uint32_t bt,
                                                                ExpertsPlan plan) {
  extern __shared__ uint32_t hist[];
  __shared__ uint32_t part[kSortWaves];
  sort_items<false>(
      ids, slots, per_block, experts, counts, hist, part,
      [&](uint32_t first, uint32_t total) {
        if (blockIdx.x == 0) list_tiles(first, total, bt, part, plan.tiles, plan.n_tiles);
      },
      [&](uint32_t slot, int32_t p) {
        plan.pos[slot] = p;
        if (p >= 0) plan.order[p] = slot;
      });
}

// The rows and the column tile of a workgroup, or false where it has none.  Each XCD
// takes a contiguous run of the work, a tile's columns next to each other.  Strips of
// 2, 4 or 8 tiles walking the columns together were slower: 4096 rows x 8 of 64
// experts, gate and up 323 against 349-352 us, down 293 against 304-317.
__device__ __forceinline__ bool own_tile(const ExpertsPlan& plan, uint32_t cols, RowTile& t, uint32_t& col) {
  const uint32_t work = *plan.n_tiles * cols, per = (work + 7) / 8;
  const uint32_t at = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || at >= work) return false;
  col = at % cols;
  t = plan.tiles[at / cols];
  return true;
}

// ------------------------------------------------------------------ gate, up
// Weight row r of the tile: 16 gate rows, then the 16 up rows of the same
// columns, in turn, so that a lane of a 32 x 32 block holds a column's gate sum
// (v < 8) and its up sum (v + 8).
// Few rows an expert: the weight stream bounds it, two workgroups a CU (81 experts of
// hidden 2048, inner 768 met by 128 slots, 255 MB: 40 us, 6.4 TB/s; one workgroup with
// four stages 45).  Many (256-row tiles, 550 G operations): 325 us at the least and 365
// in a run of passes, whose power lowers the clock.  The matrix cores are busy 55% of
// a CU's own time and the VALU, most of it the epilogue, 27%, one after the other;
// CUs are idle for 17% at the end.
template <class T>
__device__ __forceinline__ void gate_up_tile(const ExpertsArgs& a, const ExpertsPlan& plan, const RowTile& t,
                                             uint32_t group, int8_t* lds, int8_t* codes, float* scales) {
  constexpr int CSTRIDE = 144;  // bytes of a row of codes in LDS: 128 and a pad against bank conflicts
  constexpr int MAXES = T::WAVES_N * T::BT * 4;
  static_assert(T::BN == 256 && MAXES + T::BT * CSTRIDE <= T::LDS, "the epilogue reuses the rings");
  const uint32_t H = a.hidden, I = a.inter, c0 = group * 128, slots = a.m * a.k;
  const int8_t* const wg = a.w_gate + (size_t)t.of * I * H;
  const int8_t* const wu = a.w_up + (size_t)t.of * I * H;
  T s;
  s.run(
      lds, H,
      [&](int r) { return a.q + (size_t)(plan.order[t.first + ((uint32_t)r < t.rows ? r : 0)] / a.k) * H; },
      [&](int r) {
        const uint32_t c = c0 + (r >> 5) * 16 + (r & 15);
        return ((r & 16) ? wu : wg) + (size_t)(c < I ? c : c0) * H;
      },
      [](int) { return (const float*)nullptr; }, 0);

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wt0 = (wave / T::WAVES_N) * T::WT, wn = wave % T::WAVES_N;
  const int half = lane >> 5, tl = lane & 31;
  // columns of block j, values v and v + 8: cj + 8 (v / 4) + v % 4
  float gs[T::FN][8], us[T::FN][8];
#pragma unroll
  for (int j = 0; j < T::FN; ++j)
#pragma unroll
    for (int v = 0; v < 8; v += 4) {
      const uint32_t c = c0 + (wn * T::FN + j) * 16 + 4 * half + 2 * v;
      const size_t n = (size_t)t.of * I + (c < I ? c : c0);
#pragma unroll
      for (int i = 0; i < 4; ++i) gs[j][v + i] = a.ws_gate[n + i], us[j][v + i] = a.ws_up[n + i];
    }
  float act[T::FT][T::FN][8];
  uint32_t most[T::FT];
  bool nan[T::FT];
#pragma unroll
  for (int f = 0; f < T::FT; ++f) {
    const uint32_t r = wt0 + 32 * f + tl;
    const float asc = a.asc[plan.order[t.first + (r < t.rows ? r : 0)] / a.k];
    most[f] = kFloorBits;
#pragma unroll
    for (int j = 0; j < T::FN; ++j) {
      const bool in = c0 + (wn * T::FN + j) * 16 < I;  // I % 16 == 0: a block's columns are in or out together
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        act[f][j][v] = in ? act_f32(s.acc[f][j][v], s.acc[f][j][v + 8], asc, gs[j][v], us[j][v]) : 0.f;
        most[f] = max(most[f], abs_bits(act[f][j][v]));
      }
    }
    nan[f] = most[f] > kInfBits;
    if (nan[f]) {
      most[f] = kFloorBits;
#pragma unroll
      for (int j = 0; j < T::FN; ++j)
#pragma unroll
        for (int v = 0; v < 8; ++v) most[f] = max(most[f], abs_bits_no_nan(act[f][j][v]));
    }
    most[f] = halves_max_u32(most[f]);
  }
  uint32_t* const maxes = (uint32_t*)lds;  // [WAVES_N][BT]
  int8_t* const rows = lds + MAXES;        // [BT][CSTRIDE]
  __syncthreads();                         // every wave is done with the rings
#pragma unroll
  for (int f = 0; f < T::FT; ++f)
    if (half == 0) maxes[wn * T::BT + wt0 + 32 * f + tl] = most[f];
  __syncthreads();
#pragma unroll
  for (int f = 0; f < T::FT; ++f) {
    const uint32_t r = wt0 + 32 * f + tl;
    uint32_t m = maxes[r];
#pragma unroll
    for (int w = 1; w < T::WAVES_N; ++w) m = max(m, maxes[w * T::BT + r]);
    const float sc = __uint_as_float(m) / 127.0f, inv = 1.0f / sc;
    const bool slow = nan[f] || sc < kFastScaleMin;
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int v = 0; v < 8; v += 4)
        *(uint32_t*)(rows + r * CSTRIDE + (wn * T::FN + j) * 16 + 4 * half + 2 * v) =
            codes4(act[f][j][v], act[f][j][v + 1], act[f][j][v + 2], act[f][j][v + 3], sc, inv, slow);
    if (wn == 0 && half == 0 && r < t.rows) scales[(size_t)group * slots + t.first + r] = sc;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < T::BT * 8; i += 64 * T::NW) {
    const uint32_t r = i >> 3, c = c0 + (i & 7) * 16;
    if (r < t.rows && c < I)
      *(v4i*)(codes + (size_t)(t.first + r) * I + c) = *(const v4i*)(rows + r * CSTRIDE + (i & 7) * 16);
  }
}

// A tile of few rows, an expert's last, takes the form of its height: the K loop's
// time goes with the form's rows, not with those that are there.
struct NoForm {
  static constexpr int LDS = 0;
};
template <class T>
constexpr int lds_of() { return T::LDS; }
template <class T, class Half, class Quarter>
__global__ __launch_bounds__(64 * T::NW, 2) void experts_gate_up(ExpertsArgs a, ExpertsPlan plan, int8_t* codes,
                                                                 float* scales) {
  constexpr int kHalf = lds_of<Half>(), kQuarter = lds_of<Quarter>();
  constexpr int kMost = kHalf > kQuarter ? kHalf : kQuarter;
  __shared__ __attribute__((aligned(1024))) int8_t lds[T::LDS > kMost ? T::LDS : kMost];
  RowTile t;
  uint32_t group;
  if (!own_tile(plan, (a.inter + 127) / 128, t, group)) return;
  if constexpr (!std::is_same_v<Quarter, NoForm>) {
    static_assert(Quarter::NW == T::NW, "forms of one launch");
    if (t.rows <= (uint32_t)Quarter::BT) return gate_up_tile<Quarter>(a, plan, t, group, lds, codes, scales);
  }
  if constexpr (!std::is_same_v<Half, NoForm>) {
    static_assert(Half::NW == T::NW, "forms of one launch");
    if (t.rows <= (uint32_t)Half::BT) return gate_up_tile<Half>(a, plan, t, group, lds, codes, scales);
  }
  gate_up_tile<T>(a, plan, t, group, lds, codes, scales);
}

// ------------------------------------------------------------------ down
// At many rows no unit bounds it alone: in 256 x 256 tiles of 4096 rows x 8 of 64 experts,
// hidden 4096, inner 1024 (275 G operations, 287 us at the least, 309 in a run of passes)
// the matrix cores are busy 27% of a CU's own time, the VALU 38%, the loads' addressing
// 43%, and the vector cache waits for L2 58%: with one workgroup a CU and 8 stages a
// tile they follow each other.  128 x 128 tiles (two workgroups a CU): 309 and 337.
// When y was 16 bits wide: 128 x 256 and 256 x 128 tiles with three stages 310-333, 128 x
// 128 with four 393-410, against 313 and 287.
template <class T>
__device__ __forceinline__ void down_tile(const ExpertsArgs& a, const RowTile& t, uint32_t col, int8_t* lds,
                                          const int8_t* codes, const float* scales, float* y) {
  constexpr int STRIDE = 64 + 4;  // f32 values of an LDS row of 64 columns, padded
  static_assert(T::WN % 64 == 0 && T::GROUPED && T::NW * 32 * STRIDE * 4 <= T::LDS, "the epilogue reuses the rings");
  const uint32_t H = a.hidden, I = a.inter, c0 = col * T::BN, slots = a.m * a.k;
  const int8_t* const w = a.w_down + (size_t)t.of * H * I;
  T s;
  s.run(
      lds, I, [&](int r) { return codes + (size_t)(t.first + ((uint32_t)r < t.rows ? r : 0)) * I; },
      [&](int r) { return w + (size_t)(c0 + r < H ? c0 + r : c0) * I; },
      [&](int r) { return scales + t.first + ((uint32_t)r < t.rows ? r : 0); }, slots);

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wt0 = (wave / T::WAVES_N) * T::WT, half = lane >> 5, tl = lane & 31;
  __syncthreads();  // every wave is done with the rings
  float* const mine = (float*)lds + wave * 32 * STRIDE;
  // 32 rows x 64 columns at a time through the wave's own LDS, whole lines to memory
#pragma unroll
  for (int j0 = 0; j0 < T::FN; j0 += 2) {
    const uint32_t cw = c0 + (wave % T::WAVES_N) * T::WN + 32 * j0;
    float ws[2][16];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 4) {
        const uint32_t c = cw + 32 * j + 4 * half + 2 * v;  // H % 16 == 0: four columns are in or out together
        const float* const w4 = a.ws_down + (size_t)t.of * H + (c < H ? c : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) ws[j][v + i] = w4[i];
      }
#pragma unroll
    for (int f = 0; f < T::FT; ++f) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
          const auto& sum = s.sum[f][j0 + j];
          *(v4f*)(mine + tl * STRIDE + 32 * j + 2 * v + 4 * half) =
              v4f{sum[v] * ws[j][v], sum[v + 1] * ws[j][v + 1], sum[v + 2] * ws[j][v + 2], sum[v + 3] * ws[j][v + 3]};
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const uint32_t r = i + (lane >> 4), c = cw + (lane & 15) * 4, row = wt0 + 32 * f + r;
        if (row < t.rows && c < H)
          *(v4f*)(y + (size_t)(t.first + row) * H + c) = *(const v4f*)(mine + r * STRIDE + (lane & 15) * 4);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// A tile of few rows takes the lower form.
template <class T, class Half, class Quarter>
__global__ __launch_bounds__(64 * T::NW, 2) void experts_down(ExpertsArgs a, ExpertsPlan plan, const int8_t* codes,
                                                              const float* scales, float* y) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[T::LDS];
  RowTile t;
  uint32_t col;
  if (!own_tile(plan, (a.hidden + T::BN - 1) / T::BN, t, col)) return;
  if constexpr (!std::is_same_v<Quarter, NoForm>) {
    static_assert(Quarter::NW == T::NW && Quarter::BN == T::BN && Quarter::LDS <= T::LDS, "forms of one launch");
    if (t.rows <= (uint32_t)Quarter::BT) return down_tile<Quarter>(a, t, col, lds, codes, scales, y);
  }
  if constexpr (!std::is_same_v<Half, NoForm>) {
    static_assert(Half::NW == T::NW && Half::BN == T::BN && Half::LDS <= T::LDS, "forms of one launch");
    if (t.rows <= (uint32_t)Half::BT) return down_tile<Half>(a, t, col, lds, codes, scales, y);
  }
  down_tile<T>(a, t, col, lds, codes, scales, y);
}

// ------------------------------------------------------------------ sum
constexpr uint32_t kCombineRows = 1u << 22;  // workgroups: their threads stay below 2^32

// out[t, c .. c + 3] a thread, slots in order: the sum's order is fixed.  Eight
// slots' rows are under way together; their positions and weights, one row's,
// are wave-uniform.  NT: y is read past the caches, which it has outgrown: 4096 rows of
// 8 slots, hidden 4096, 570 MB in 102 us, 5.6 TB/s.
template <bool NT>
__global__ __launch_bounds__(256) void experts_combine(ExpertsArgs a, const int32_t* __restrict__ pos,
                                                       const float* __restrict__ y) {
  const uint32_t c = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (c >= a.hidden) return;
  for (uint32_t row = blockIdx.x; row < a.m; row += gridDim.x) {
    v4f sum{};
    for (uint32_t j0 = 0; j0 < a.k; j0 += 8) {
      v4f v[8];
      int32_t p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = pos[(size_t)row * a.k + min(j0 + j, a.k - 1)];
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // a slot without an expert reads a row that it does not use
        const v4f* const q = (const v4f*)(y + (size_t)max(p[j], 0) * a.hidden + c);
        v[j] = NT ? __builtin_nontemporal_load(q) : *q;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j0 + j >= a.k || p[j] < 0) continue;
        const float w = a.weights[(size_t)row * a.k + j0 + j];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(w, v[j][i], sum[i]);
      }
    }
    const size_t o = (size_t)row * a.hidden + c;
    if (a.residual) {
      const v4f r = *(const v4f*)(a.residual + o);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = r[i] + sum[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = bf16_rne(sum[i]);
    if (a.out_dtype == W8A8_OUT_F32) {
      *(v4f*)((float*)a.out + o) = sum;
    } else {
      const uint32_t lo = (__float_as_uint(sum[0]) >> 16) | (__float_as_uint(sum[1]) & 0xffff0000u);
      const uint32_t hi = (__float_as_uint(sum[2]) >> 16) | (__float_as_uint(sum[3]) & 0xffff0000u);
      *(v2i*)((uint16_t*)a.out + o) = v2i{(int)lo, (int)hi};
    }
  }
}

// ------------------------------------------------------------------ launches
// Rows of a token tile, by an expert's mean share of the slots: the smallest that
// holds it with room for the uneven shares of real routing.  An expert that takes
// two tiles reads its weights twice, which large experts (above 8 MiB) cannot
// afford; a tile too tall computes rows that are not there.  Measured on weights of
// each pass's own, tile rows: us, hidden 4096, inner 1024, 8 of 64: mean 16 32: 213, 64:
// 182; mean 25 64: 217, 128: 193; mean 42 64: 229, 128: 215; mean 128 128: 277, 256: 312;
// mean 150 128: 315, 256: 314.  Hidden 2048, inner 768, 8 of 128: mean 16 32: 140, 64:
// 139; mean 44 64: 161, 128: 176; mean 128 128: 239, 256: 244; mean 144 128: 251, 256: 260.
// Hidden 2000, inner 720, 3 of 20: mean 19 32: 46, 64: 55, 128: 48; mean 50 64: 58, 128:
// 57; mean 105 128: 63, 256: 75.
static uint32_t tile_rows(uint32_t slots, uint32_t experts, uint32_t hidden, uint32_t inter) {
  const uint32_t mean = slots / std::min(slots, experts);
  if (3ull * hidden * inter > (8u << 20)) return mean <= 12 ? 32 : mean <= 20 ? 64 : mean <= 128 ? 128 : 256;
  return mean <= 24 ? 32 : mean <= 48 ? 64 : mean <= 128 ? 128 : 256;
}

constexpr uint32_t kOnePerCu = 256;  // workgroups

ExpertsTilesForm experts_tiles_form(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter) {
  const uint32_t slots = m * k;
  ExpertsTilesForm f{};
  f.bt = tile_rows(slots, experts, hidden, inter);
  f.tiles = slots / f.bt + std::min(slots, experts);
  f.sort_blocks = sort_blocks(slots);
  f.gate_deep = f.bt == 32 && f.tiles * ((inter + 127) / 128) <= kOnePerCu;
  f.down_deep = f.bt == 32 && f.tiles * ((hidden + 255) / 256) <= kOnePerCu;
  f.gate_tail = hidden % 128 != 0;
  f.down_tail = inter % 128 != 0;
  return f;
}

namespace {
struct Layout {
  size_t order, pos, tiles, n_tiles, counts, codes, scales, y, bytes;
};
Layout layout(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter) {
  const size_t slots = (size_t)m * k;
  const ExpertsTilesForm f = experts_tiles_form(m, k, experts, hidden, inter);
  Layout l{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  l.order = take(slots * 4);
  l.pos = take(slots * 4);
  l.tiles = take((size_t)f.tiles * sizeof(RowTile));
  l.n_tiles = take(4);
  l.counts = take(f.sort_blocks > 1 ? (size_t)f.sort_blocks * experts * 4 : 0);
  l.codes = take(slots * inter);
  l.scales = take(slots * ((inter + 127) / 128) * 4);
  l.y = take(slots * hidden * 4);
  l.bytes = at;
  return l;
}

template <int BT, int WT, int WN, int SA, int SB, bool TAIL>
using GateUp = TileStream<BT, 256, WT, WN, SA, SB, false, TAIL>;
template <int BT, int BN, int WT, int SA, int SB, bool TAIL>
using Down = TileStream<BT, BN, WT, 64, SA, SB, true, TAIL>;

template <class T, class Half, class Quarter>
void gate_up_as(hipStream_t st, const ExpertsArgs& a, const ExpertsPlan& p, uint32_t tiles, int8_t* codes,
                float* scales) {
  const uint32_t grid = (tiles * ((a.inter + 127) / 128) + 7) / 8 * 8;
  hipLaunchKernelGGL((experts_gate_up<T, Half, Quarter>), dim3(grid), dim3(64 * T::NW), 0, st, a, p, codes, scales);
}

template <bool TAIL>
void gate_up(hipStream_t st, const ExpertsArgs& a, const ExpertsPlan& p, const ExpertsTilesForm& form, int8_t* codes,
             float* scales) {
  const uint32_t bt = form.bt, tiles = form.tiles;
  using T32 = GateUp<32, 32, 64, 2, 2, TAIL>;
  using T64 = GateUp<64, 64, 32, 4, 4, TAIL>;
  using T128 = GateUp<128, 64, 64, 3, 3, TAIL>;
  using T256 = GateUp<256, 64, 128, 2, 3, TAIL>;
  // 32 rows: two workgroups share a CU, or one has twice the stages under way
  if (form.gate_deep)
    gate_up_as<GateUp<32, 32, 64, 4, 4, TAIL>, NoForm, NoForm>(st, a, p, tiles, codes, scales);
  else if (bt == 32) gate_up_as<T32, NoForm, NoForm>(st, a, p, tiles, codes, scales);
  else if (bt == 64) gate_up_as<GateUp<64, 64, 64, 2, 2, TAIL>, T32, NoForm>(st, a, p, tiles, codes, scales);
  else if (bt == 128) gate_up_as<T128, T64, NoForm>(st, a, p, tiles, codes, scales);
  else gate_up_as<T256, T128, T64>(st, a, p, tiles, codes, scales);
}

template <class T, class Half = NoForm, class Quarter = NoForm>
void down_as(hipStream_t st, const ExpertsArgs& a, const ExpertsPlan& p, uint32_t tiles,
             const int8_t* codes, const float* scales, float* y) {
  const uint32_t grid = (tiles * ((a.hidden + T::BN - 1) / T::BN) + 7) / 8 * 8;
  hipLaunchKernelGGL((experts_down<T, Half, Quarter>), dim3(grid), dim3(64 * T::NW), 0, st, a, p, codes, scales, y);
}

template <bool TAIL>
void down(hipStream_t st, const ExpertsArgs& a, const ExpertsPlan& p, const ExpertsTilesForm& form,
          const int8_t* codes, const float* scales, float* y) {
  const uint32_t bt = form.bt, tiles = form.tiles;
  if (form.down_deep)
    down_as<Down<32, 256, 32, 4, 4, TAIL>>(st, a, p, tiles, codes, scales, y);
  else if (bt == 32) down_as<Down<32, 256, 32, 2, 2, TAIL>>(st, a, p, tiles, codes, scales, y);
  else if (bt == 64) down_as<Down<64, 128, 32, 3, 3, TAIL>>(st, a, p, tiles, codes, scales, y);
  else if (bt == 256)
    down_as<TileStream<256, 256, 64, 128, 2, 2, true, TAIL, OP_I8, true>, Down<128, 256, 64, 2, 2, TAIL>,
            Down<64, 256, 32, 2, 2, TAIL>>(st, a, p, tiles, codes, scales, y);
  else down_as<Down<128, 128, 64, 2, 2, TAIL>, Down<64, 128, 32, 2, 2, TAIL>>(st, a, p, tiles, codes, scales, y);
}
}  // namespace

size_t experts_tiles_workspace_bytes(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter) {
  return layout(m, k, experts, hidden, inter).bytes;
}

hipError_t launch_experts_tiles(hipStream_t st, const ExpertsArgs& a, void* workspace) {
  const uint32_t slots = a.m * a.k;
  const Layout l = layout(a.m, a.k, a.experts, a.hidden, a.inter);
  char* const p = (char*)workspace;
  const ExpertsPlan plan{(uint32_t*)(p + l.order), (int32_t*)(p + l.pos), (RowTile*)(p + l.tiles),
                         (uint32_t*)(p + l.n_tiles)};
  int8_t* const codes = (int8_t*)(p + l.codes);
  float* const scales = (float*)(p + l.scales);
  float* const y = (float*)(p + l.y);
  uint32_t* const counts = (uint32_t*)(p + l.counts);
  const ExpertsTilesForm form = experts_tiles_form(a.m, a.k, a.experts, a.hidden, a.inter);
  const uint32_t blocks = form.sort_blocks, per = sort_per_block(slots), lds = kSortWaves * a.experts * 4;
  if (blocks > 1)
    hipLaunchKernelGGL(sort_counts<false>, dim3(blocks), dim3(64 * kSortWaves), lds, st, a.ids, slots, per, a.experts,
                       counts);
  hipLaunchKernelGGL(experts_plan, dim3(blocks), dim3(64 * kSortWaves), lds, st, a.ids, slots, per, a.experts, counts,
                     form.bt, plan);
  if (form.gate_tail) gate_up<true>(st, a, plan, form, codes, scales);
  else gate_up<false>(st, a, plan, form, codes, scales);
  if (form.down_tail) down<true>(st, a, plan, form, codes, scales, y);
  else down<false>(st, a, plan, form, codes, scales, y);
  // Measured, y past the caches / through them us: 25 MB (1100 rows of 3 slots, hidden 2000)
  // 8.4 / 7.7; hidden 4096, 8 slots, 67 MB 14.0 / 13.6, 134 MB 25.5 / 25.9, 197 MB 36.9 /
  // 37.8, 268 MB 47.0 / 53.8, 537 MB 102 / 130.
  const dim3 sums(std::min(a.m, kCombineRows), (a.hidden + 1023) / 1024);
  hipLaunchKernelGGL((size_t)slots * a.hidden * 4 >= 128u << 20 ? experts_combine<true> : experts_combine<false>, sums,
                     dim3(256), 0, st, a, plan.pos, y);
  return hipGetLastError();
}

}  // namespace w8a8
