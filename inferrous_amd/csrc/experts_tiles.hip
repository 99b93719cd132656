// experts_tiles.hip -- the routed experts' MLP expert by expert: the slots
// sorted by expert, each expert's rows multiplied in tiles by MFMA, and the
// slots' products summed row by row.  The definition is in experts.hip.
//
//   experts_plan       sorts the slots (a counting sort that keeps their order)
//                      and lists the token tiles: up to BT rows of one expert;
//   experts_gate_up    a tile's gate and up sums over 128 columns of act, the
//                      SiLU product, and its codes and scale;
//   experts_down       a tile's y over BN columns, the stages of K being the
//                      128-column groups, each scaled into f32 sums;
//   experts_combine    out = residual + sum over a row's slots of weight * y.
//
// y goes through memory as 16-bit fixed point against the largest magnitude of
// 64 columns of its row: half the bytes of f32, which would be the pass's largest
// stream, at an error below 2^-16 of that magnitude, 2^-8 of what BF16 would add.
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

// The token tile and column tile of a workgroup, or false past the last one.
// Each XCD takes a contiguous run of the live tiles, a token tile's columns next
// to each other.
__device__ __forceinline__ bool own_tile(const ExpertsPlan& plan, uint32_t cols, RowTile& t, uint32_t& col) {
  const uint32_t live = *plan.n_tiles * cols, per = (live + 7) / 8;
  const uint32_t at = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || at >= live) return false;
  t = plan.tiles[at / cols];
  col = at % cols;
  return true;
}

// ------------------------------------------------------------------ gate, up
// Weight row r of the tile: 16 gate rows, then the 16 up rows of the same
// columns, in turn, so that a lane of a 32 x 32 block holds a column's gate sum
// (v < 8) and its up sum (v + 8).
template <class T>
__global__ __launch_bounds__(64 * T::NW, T::NW == 8 ? 2 : 1) void experts_gate_up(ExpertsArgs a, ExpertsPlan plan,
                                                                                  int8_t* codes, float* scales) {
  constexpr int CSTRIDE = 144;  // bytes of a row of codes in LDS: 128 and a pad against bank conflicts
  constexpr int MAXES = T::WAVES_N * T::BT * 4;
  static_assert(T::BN == 256 && MAXES + T::BT * CSTRIDE <= T::LDS, "the epilogue reuses the rings");
  __shared__ __attribute__((aligned(1024))) int8_t lds[T::LDS];
  RowTile t;
  uint32_t group;
  if (!own_tile(plan, (a.inter + 127) / 128, t, group)) return;
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

// ------------------------------------------------------------------ down
// 16-bit fixed point of y against its block's largest finite magnitude: up to
// 32766, with codes of their own for the infinities and NaN.
constexpr float kYMost = 32766.0f;
__device__ __forceinline__ int y_code(float y, float inv) {
  if (__builtin_expect(!(__builtin_fabsf(y) < __builtin_inff()), 0)) return y != y ? -32768 : y > 0 ? 32767 : -32767;
  return (int)__builtin_rintf(y * inv);
}
__device__ __forceinline__ float y_value(int code, float s) {
  if (__builtin_expect(code == -32768, 0)) return __builtin_nanf("");
  if (__builtin_expect(code == 32767 || code == -32767, 0)) return code > 0 ? __builtin_inff() : -__builtin_inff();
  return (float)code * s;
}

template <class T>
__global__ __launch_bounds__(64 * T::NW, T::NW == 8 ? 2 : 1) void experts_down(ExpertsArgs a, ExpertsPlan plan,
                                                                               const int8_t* codes,
                                                                               const float* scales, int16_t* y,
                                                                               float* yscale) {
  constexpr int STRIDE = 144;  // bytes of a row of 64 codes in LDS, padded
  static_assert(T::WN == 64 && T::GROUPED && T::NW * T::WT * STRIDE <= T::LDS, "the epilogue reuses the rings");
  __shared__ __attribute__((aligned(1024))) int8_t lds[T::LDS];
  RowTile t;
  uint32_t col;
  if (!own_tile(plan, (a.hidden + T::BN - 1) / T::BN, t, col)) return;
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
  const uint32_t cw = c0 + (wave % T::WAVES_N) * 64;  // the wave's 64 columns
  float ws[T::FN][16];
#pragma unroll
  for (int j = 0; j < T::FN; ++j)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const uint32_t c = cw + 32 * j + 4 * half + 8 * (v >> 2) + (v & 3);
      ws[j][v] = a.ws_down[(size_t)t.of * H + (c < H ? c : H - 1)];
    }
  __syncthreads();  // every wave is done with the rings
  int8_t* const mine = lds + wave * T::WT * STRIDE;
  const uint32_t nb = (H + 63) / 64;
#pragma unroll
  for (int f = 0; f < T::FT; ++f) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float p = s.sum[f][j][v] * ws[j][v];
        s.sum[f][j][v] = p;
        const uint32_t c = cw + 32 * j + 4 * half + 8 * (v >> 2) + (v & 3), b = abs_bits(p);
        if (c < H && b < kInfBits) most = max(most, b);
      }
    most = halves_max_u32(most);
    const float big = __uint_as_float(most);
    const float sc = __builtin_fmaxf(big * (1.0f / kYMost), 0x1p-120f), inv = 1.0f / sc;
    const uint32_t r = wt0 + 32 * f + tl;
#pragma unroll
    for (int j = 0; j < T::FN; ++j)
#pragma unroll
      for (int v = 0; v < 16; v += 4) {
        int q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = y_code(s.sum[f][j][v + i], inv);
        v2i d;
        d.x = (q[0] & 0xffff) | (q[1] << 16);
        d.y = (q[2] & 0xffff) | (q[3] << 16);
        *(v2i*)(mine + (32 * f + tl) * STRIDE + (32 * j + 4 * half + 2 * v) * 2) = d;
      }
    if (half == 0 && r < t.rows && cw < H) yscale[(size_t)(t.first + r) * nb + cw / 64] = sc;
  }
  // the wave's own rows back, whole lines to memory
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < T::WT; i += 8) {
    const uint32_t r = i + (lane >> 3), c = cw + (lane & 7) * 8;
    if (wt0 + r < t.rows && c < H)
      *(v4i*)(y + (size_t)(t.first + wt0 + r) * H + c) = *(const v4i*)(mine + r * STRIDE + (lane & 7) * 16);
  }
}

// ------------------------------------------------------------------ sum
// out[t, c .. c + 7] a thread, slots in order: the sum's order is fixed.
__global__ __launch_bounds__(256) void experts_combine(ExpertsArgs a, const int32_t* pos, const int16_t* y,
                                                       const float* yscale) {
  const uint32_t H8 = a.hidden / 8, nb = (a.hidden + 63) / 64;
  const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (size_t)a.m * H8) return;
  const uint32_t row = (uint32_t)(at / H8), c = (uint32_t)(at % H8) * 8;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.f;
#pragma unroll 4
  for (uint32_t j = 0; j < a.k; ++j) {
    const int32_t p = pos[(size_t)row * a.k + j];
    if (p < 0) continue;
    const float w = a.weights[(size_t)row * a.k + j], s = yscale[(size_t)p * nb + c / 64];
    const v4i v = *(const v4i*)(y + (size_t)p * a.hidden + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum[2 * i] = __builtin_fmaf(w, y_value((int)(int16_t)(v[i] & 0xffff), s), sum[2 * i]);
      sum[2 * i + 1] = __builtin_fmaf(w, y_value(v[i] >> 16, s), sum[2 * i + 1]);
    }
  }
  const size_t o = (size_t)row * a.hidden + c;
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const v4f r = *(const v4f*)(a.residual + o + i);
#pragma unroll
      for (int l = 0; l < 4; ++l) sum[i + l] = r[l] + sum[i + l];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = bf16_rne(sum[i]);
  if (a.out_dtype == W8A8_OUT_F32) {
    float* const out = (float*)a.out + o;
    *(v4f*)out = v4f{sum[0], sum[1], sum[2], sum[3]};
    *(v4f*)(out + 4) = v4f{sum[4], sum[5], sum[6], sum[7]};
  } else {
    v4i out;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      out[i] = (int)((__float_as_uint(sum[2 * i]) >> 16) | (__float_as_uint(sum[2 * i + 1]) & 0xffff0000u));
    *(v4i*)((uint16_t*)a.out + o) = out;
  }
}

// ------------------------------------------------------------------ launches
static size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// Rows of a token tile: the smallest that holds an expert's mean share, so that
// few tiles are half empty and few experts take two where one would do.
static uint32_t tile_rows(uint32_t slots, uint32_t experts) {
  const uint32_t mean = slots / std::min(slots, experts);
  return mean <= 24 ? 32 : mean <= 48 ? 64 : mean <= 128 ? 128 : 256;
}

static uint32_t most_tiles(uint32_t slots, uint32_t experts, uint32_t bt) {
  return slots / bt + std::min(slots, experts);
}

namespace {
struct Layout {
  size_t order, pos, tiles, n_tiles, counts, codes, scales, y, yscale, bytes;
};
Layout layout(uint32_t m, uint32_t k, uint32_t experts, uint32_t hidden, uint32_t inter) {
  const size_t slots = (size_t)m * k;
  const uint32_t blocks = sort_blocks((uint32_t)slots);
  Layout l{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  l.order = take(slots * 4);
  l.pos = take(slots * 4);
  l.tiles = take((size_t)most_tiles((uint32_t)slots, experts, tile_rows((uint32_t)slots, experts)) * sizeof(RowTile));
  l.n_tiles = take(4);
  l.counts = take(blocks > 1 ? (size_t)blocks * experts * 4 : 0);
  l.codes = take(slots * inter);
  l.scales = take(slots * ((inter + 127) / 128) * 4);
  l.y = take(slots * hidden * 2);
  l.yscale = take(slots * ((hidden + 63) / 64) * 4);
  l.bytes = at;
  return l;
}

template <int BT, int WT, int WN, int SA, int SB>
void gate_up_as(hipStream_t st, const ExpertsArgs& a, const ExpertsPlan& p, uint32_t tiles, int8_t* codes,
                float* scales) {
  const uint32_t grid = (tiles * ((a.inter + 127) / 128) + 7) / 8 * 8;
  using Whole = TileStream<BT, 256, WT, WN, SA, SB, false, false>;
  using Tail = TileStream<BT, 256, WT, WN, SA, SB, false, true>;
  if (a.hidden % 128 == 0)
    hipLaunchKernelGGL(experts_gate_up<Whole>, dim3(grid), dim3(64 * Whole::NW), 0, st, a, p, codes, scales);
  else
    hipLaunchKernelGGL(experts_gate_up<Tail>, dim3(grid), dim3(64 * Whole::NW), 0, st, a, p, codes, scales);
}

template <int BT, int BN, int WT, int SA, int SB>
void down_as(hipStream_t st, const ExpertsArgs& a, const ExpertsPlan& p, uint32_t tiles, const int8_t* codes,
             const float* scales, int16_t* y, float* yscale) {
  const uint32_t grid = (tiles * ((a.hidden + BN - 1) / BN) + 7) / 8 * 8;
  using Whole = TileStream<BT, BN, WT, 64, SA, SB, true, false>;
  using Tail = TileStream<BT, BN, WT, 64, SA, SB, true, true>;
  if (a.inter % 128 == 0)
    hipLaunchKernelGGL(experts_down<Whole>, dim3(grid), dim3(64 * Whole::NW), 0, st, a, p, codes, scales, y, yscale);
  else
    hipLaunchKernelGGL(experts_down<Tail>, dim3(grid), dim3(64 * Whole::NW), 0, st, a, p, codes, scales, y, yscale);
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
  int16_t* const y = (int16_t*)(p + l.y);
  float* const yscale = (float*)(p + l.yscale);
  uint32_t* const counts = (uint32_t*)(p + l.counts);
  const uint32_t bt = tile_rows(slots, a.experts);
  const uint32_t tiles = most_tiles(slots, a.experts, bt);
  const uint32_t blocks = sort_blocks(slots), per = sort_per_block(slots), lds = kSortWaves * a.experts * 4;
  if (blocks > 1)
    hipLaunchKernelGGL(sort_counts<false>, dim3(blocks), dim3(64 * kSortWaves), lds, st, a.ids, slots, per, a.experts,
                       counts);
  hipLaunchKernelGGL(experts_plan, dim3(blocks), dim3(64 * kSortWaves), lds, st, a.ids, slots, per, a.experts, counts,
                     bt, plan);
  if (bt == 32) gate_up_as<32, 32, 64, 4, 4>(st, a, plan, tiles, codes, scales);
  else if (bt == 64) gate_up_as<64, 64, 32, 4, 4>(st, a, plan, tiles, codes, scales);
  else if (bt == 128) gate_up_as<128, 64, 64, 3, 3>(st, a, plan, tiles, codes, scales);
  else gate_up_as<256, 64, 128, 2, 3>(st, a, plan, tiles, codes, scales);
  if (bt == 32) down_as<32, 256, 32, 4, 4>(st, a, plan, tiles, codes, scales, y, yscale);
  else if (bt == 64) down_as<64, 256, 32, 3, 3>(st, a, plan, tiles, codes, scales, y, yscale);
  else if (bt == 128) down_as<128, 256, 64, 2, 3>(st, a, plan, tiles, codes, scales, y, yscale);
  else down_as<256, 128, 64, 2, 3>(st, a, plan, tiles, codes, scales, y, yscale);
  const size_t threads = (size_t)a.m * (a.hidden / 8);
  hipLaunchKernelGGL(experts_combine, dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, st, a, plan.pos, y,
                     yscale);
  return hipGetLastError();
}

}  // namespace w8a8
