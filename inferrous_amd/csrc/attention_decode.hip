// attention_decode.hip -- one query row of each sequence over the 8-bit cache.
//
//   s_j = scale * q . (k_scale k_j),  o = sum_j exp(s_j - m) (v_scale v_j) / sum_j exp(s_j - m)
//
// The cache's bytes bound it: 2 * D a token and key/value head, read once.  A
// workgroup takes a sequence's key/value head, alone or with other workgroups that
// share its pages, and a wave one page at a time; up to 16 of the query heads that share the
// key/value head are the 16 columns of v_mfma_f32_16x16x32_bf16, which so
// costs the same for one head or 16.
//
// Everything stays in registers.  Scores are taken transposed, S^T = K Q^T, the
// tokens as rows: MFMA t's row r is token 16 (r / 4) + 4 t + r % 4 of the page,
// so that of the result (row 4 g + i in lane group g = lane / 16, register i)
// lane group g holds the tokens 16 g .. 16 g + 15 of the lane's head -- just
// what the second product O^T = V^T P^T wants of its second operand, while the
// values' first operand, 16 tokens of one column, is one 16-byte load of the
// transposed codes.  v_cvt_scalef32_pk_bf16_fp8 makes codes BF16 exactly, the
// page's scale included.
//
// The running maximum m of a head moves only when a page's exceeds it by more
// than 8 (in powers of two): probabilities stay below 2^8, and the sums are
// rescaled a few times, not once a page.  A probability goes into the second product
// as two BF16 values, what BF16 holds of it and what that leaves (together off by 2^-16),
// and as f32 into the sum that divides.  With the first alone, long rows' outputs were
// off by a quarter more than their own rounding; the second costs 0.4% where the bytes
// bound (64 sequences of up to 4096 tokens) and 3% where a row's chain does (5 of up to
// 65536, 14/2 heads of 64).
//
// 64 sequences of up to 4096 tokens, 32/8 heads of 128: 261 MB in 49.4 us (5.3 TB/s; a
// plain read of the same pages, a page a wave, 45 us).  One of 4001 tokens: 5.1 us and
// 3.6 for the join, both mostly latency.
#include <algorithm>

#include "attention.hpp"

namespace w8a8 {

constexpr uint32_t kDecodeWaves = 4;
constexpr uint32_t kDecodeHeads = 16;  // query heads of a workgroup

struct DecodeSplit {
  uint32_t tiles;   // workgroups a key/value head's query heads take
  uint32_t chunk;   // pages of a workgroup
  uint32_t splits;  // workgroups of the widest sequence
  uint32_t turn;    // units that a turn of the compute units takes, 0: in the order they have
};
// Divisors of the launch's numbers.
struct DecodeBy {
  Divisor kv_heads, tiles, splits, turn, heads;
  uint32_t group;
  DecodeBy(const DecodeArgs& a, const DecodeSplit& d)
      : kv_heads(a.kv_heads), tiles(d.tiles), splits(d.splits), turn(std::max(1u, d.turn)), heads(a.heads),
        group(a.heads / a.kv_heads) {}
};

constexpr uint32_t kMaxSplits = 64;
// Splits that a join of so many waves a head takes.
constexpr uint32_t join_splits(int waves) { return waves == 1 ? 16 : kMaxSplits; }

// Splits: two workgroups a compute unit where a wave keeps a page, but none where a row's
// pages are few, or not many and the splits two: a join costs its launch, about three
// pages of a wave.  In splits / alone, us, 32/8 heads of 128 unless said: 1 row of 12
// pages 8.0 / 6.9, of 16 8.1 / 8.2, of 24 8.0 / 10.8; 14/2 heads of 64, 1 row of 24
// 7.9 / 6.2, of 48 8.0 / 9.8.  Two splits, rows of all lengths up to so many pages, or all
// of so many: 24 rows, 16 10.4 / 9.2 and 14.6 / 10.9, 24 12.2 / 12.0 and 18.5 / 14.5, 64
// 25.0 / 25.7 and 39.3 / 31.6; 32 rows, 64 24.4 / 27.4 and 47.7 / 43.2.  Four, 16 rows,
// 64 13.8 / 21.4 and 26.3 / 26.9.  Three or four workgroups a compute unit: 10 to 70% slower.
// (All with a table as wide as the longest row.  The pages of a workgroup follow from the
// width alone, so a wider table leaves shorter rows to fewer workgroups: one row of 63 pages
// 7.8 at a width of 63, 9.6 at 512, 17.4 at 2048, eight of them 16.9, 28.2 and 28.3.)
//
// Turns: workgroups that share a compute unit start together, so the order decides
// which do.  Ranking the units takes each workgroup under a microsecond, paid back where
// one has two pages a wave to read, up to 64 units (a lane each) or 256 whole rows.  32/8
// heads of 128, in the rows' order / by pages, us: 8 sequences of up to 4096 tokens
// 12.3 / 10.9, 16 17.7 / 13.9, 32 29.9 / 24.4, 64 53.8 / 47.0, 64 of up to 600
// 10.8 / 10.1, 128 of up to 2000 52.4 / 47.8, 200 80.1 / 77.7.  More than 64 units of split
// rows, 14/2 heads of 64: 5 of up to 65536 13.5 / 15.6, 100 of up to 4096 15.5 / 16.5.
static DecodeSplit decode_split(uint32_t m, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t width) {
  DecodeSplit d;
  d.tiles = (heads / kv_heads + kDecodeHeads - 1) / kDecodeHeads;
  const uint64_t units = (uint64_t)m * kv_heads * d.tiles;
  const uint64_t most = std::min<uint64_t>(kMaxSplits, 512 / units);
  const uint32_t splits = most < 2 || (uint64_t)width * dim <= (most == 2 ? 24 : 12) * 128 ? 1 : (uint32_t)most;
  d.chunk = ((width + splits - 1) / splits + kDecodeWaves - 1) / kDecodeWaves * kDecodeWaves;
  d.splits = (width + d.chunk - 1) / d.chunk;
  d.turn = m > 1 && (m * d.splits <= 64 || (d.splits == 1 && m <= 256)) && d.chunk >= 8 ? std::max(1u, 256 / (kv_heads * d.tiles)) : 0;
  return d;
}

__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// Eight codes (two words) times a power of two as BF16.
__device__ __forceinline__ v4u widen(uint32_t a, uint32_t b, float s) {
  return v4u{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false)),
             __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true))};
}
// Four neighbouring outputs.
__device__ __forceinline__ void store4(const DecodeArgs& a, size_t at, v4f x) {
  const uint32_t lo = pack_bf16(x[0], x[1]), hi = pack_bf16(x[2], x[3]);
  if (a.out_dtype == W8A8_OUT_BF16)
    *(v2u*)((uint16_t*)a.out + at) = v2u{lo, hi};
  else
    *(v4u*)((float*)a.out + at) = v4u{lo << 16, lo & 0xffff0000u, hi << 16, hi & 0xffff0000u};
}

// Across the four lane groups of a head's column (rows of 16 lanes): a row beside
// its neighbour, then a half beside the other.
template <class Op>
__device__ __forceinline__ float across_groups(float v, Op op) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float groups_max(float v) {
  return across_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float groups_sum(float v) {
  return across_groups(v, [](float a, float b) { return a + b; });
}

// What divides a row's sum o by l: a row that saw no token (its maximum is -inf, below any
// that a score leaves) is 0, one whose scores are all -inf is 0 / 0 as its softmax is.
__device__ __forceinline__ float weight(float m, float l) { return m == -__builtin_inff() ? 0.f : 1.f / l; }

// A page's codes as the two products take them.
template <int D>
struct PageCodes {
  v4u k[4][D / 64], v[D / 16];
  float scale;  // of the keys in even lanes, of the values in odd ones
};

// The unit (a row's split) that workgroup `place` of a key/value head takes: by their
// pages, the most first in even turns of the compute units and the fewest first in odd ones.
__device__ __forceinline__ uint32_t unit_of_turn(const DecodeArgs& a, const DecodeSplit& d, const DecodeBy& by, uint32_t place, uint32_t* keys) {
  const uint32_t lane = threadIdx.x & 63, units = a.m * d.splits;
  const uint32_t n = by.turn.of(place), at = place - n * d.turn;
  const uint32_t rank = n * d.turn + (n % 2 ? min(d.turn, units - n * d.turn) - 1 - at : at);
  const auto key = [&](uint32_t u) {  // no two alike
    const uint32_t row = by.splits.of(u), first = (u - row * d.splits) * d.chunk;
    const uint32_t pages = u < units ? min(((uint32_t)max(a.lengths[row], 0) + kPageTokens - 1) / kPageTokens, a.width) : 0u;
    return (pages > first ? min(pages - first, d.chunk) : 0u) * 256 + (255 - u);
  };
  const auto before = [&](uint32_t mine, uint32_t others) {
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) sum += (uint32_t)__builtin_amdgcn_readlane((int)others, i) > mine;
    return sum;
  };
  if (units <= 64) {  // each wave for itself
    const uint32_t k = key(lane);
    return (uint32_t)__builtin_ctzll(__ballot(before(k, k) == rank));
  }
  const uint32_t k = key(threadIdx.x);
  keys[threadIdx.x] = k;
  __syncthreads();
  uint32_t sum = 0;
  for (uint32_t u = 0; u < units; u += 64) sum += before(k, keys[u + lane]);
  if (sum == rank) keys[256] = threadIdx.x;
  __syncthreads();
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)keys[256]);
}

// partial: of sequences with more pages than a chunk, of each row, head and split its
// unscaled sum o[D], then of each {m, l}.
template <int D>
__global__ __launch_bounds__(256, 3) void attention_decode_kernel(DecodeArgs a, DecodeSplit d, DecodeBy by, float* partial) {
  constexpr int HALVES = D / 64, TILES = D / 16;
  __shared__ float sh_m[4][16], sh_l[4][16];
  __shared__ float sh_o[4][16][D + 4];
  __shared__ uint32_t keys[257];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t group = by.group, among = by.kv_heads.of(blockIdx.x), h = blockIdx.x - among * a.kv_heads;
  uint32_t b = by.tiles.of(among);
  const uint32_t tile = among - b * d.tiles;
  if (d.turn) b = unit_of_turn(a, d, by, b, keys);
  const uint32_t row = by.splits.of(b), split = b - row * d.splits;
  const uint32_t head0 = h * group + tile * kDecodeHeads, live = min(kDecodeHeads, group - tile * kDecodeHeads);

  const int32_t* const table = a.table + (size_t)row * a.width;
  uint32_t p = split * d.chunk + wave;  // the wave's first page: it does not wait for the length
  // The numbers of the wave's next 64 pages, one a lane.  (Vector loads, as the
  // scales' are: a scalar load's result is waited for with all that are in flight,
  // and these miss the caches.)
  const auto ids_from = [&](uint32_t page) { return table[min(page + lane * kDecodeWaves, a.width - 1)]; };
  int32_t ids = ids_from(p);
  const uint32_t len = min((uint32_t)max(a.lengths[row], 0), a.width * kPageTokens);
  const uint32_t pages = (len + kPageTokens - 1) / kPageTokens, end = min(pages, (split + 1) * d.chunk);
  if (split != 0 && split * d.chunk >= pages) return;  // the sequence ends before
  const auto known = [&](int32_t i) { return i >= 0 && (uint32_t)i < a.pages; };

  const auto load = [&](PageCodes<D>& x, int32_t i) {
    const size_t at = (size_t)(known(i) ? i : 0) * a.kv_heads + h;
    const uint8_t* const codes = a.codes + at * page_head_bytes(D);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int f = 0; f < HALVES; ++f)
        x.k[t][f] = *(const v4u*)(codes + (16 * (c >> 2) + 4 * t + (c & 3)) * D + 64 * f + 16 * g);
#pragma unroll
    for (int t = 0; t < TILES; ++t)
      x.v[t] = *(const v4u*)(codes + kPageTokens * D + (16 * t + c) * kPageTokens + 16 * g);
    x.scale = a.scales[2 * at + (lane & 1)];
  };

  v4u q[2 * HALVES];
#pragma unroll
  for (int s = 0; s < 2 * HALVES; ++s) {
    q[s] = v4u{};
    if ((uint32_t)c < live)
      q[s] = *(const v4u*)(a.q + ((size_t)row * a.heads + head0 + c) * D + 64 * (s / 2) + 16 * g + 8 * (s % 2));
  }
  const float to_log2 = a.scale * kLog2e;
  float m = kNoScore, l = 0.f;
  v4f o[TILES] = {};
  // minus the first of a pair, and minus the second (in registers: as a constant of the
  // instruction, the first comes out as the second)
  uint32_t first = 0x0000bf80u, second = 0xbf800000u;
  asm("" : "+s"(first), "+s"(second));

  const auto attend = [&](PageCodes<D>& x, uint32_t page) {
    const float ks = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x.scale), 0));
    const float vs = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x.scale), 1));
    float s[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      v4f acc = {};
#pragma unroll
      for (int f = 0; f < HALVES; ++f) {
        acc = mfma16(widen(x.k[t][f].x, x.k[t][f].y, ks), q[2 * f], acc);
        acc = mfma16(widen(x.k[t][f].z, x.k[t][f].w, ks), q[2 * f + 1], acc);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = acc[i] * to_log2;
    }
    const uint32_t left = len - page * kPageTokens;  // tokens of the page, 64 but in the last one
    if (left < kPageTokens) {
      // what lies behind the last token may be any bytes, NaN among them
      const int mine = (int)left - 16 * g;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = i < mine ? s[i] : -__builtin_inff();
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int keep = mine - 4 * w;
          x.v[t][w] &= keep >= 4 ? ~0u : keep <= 0 ? 0u : ~0u >> 8 * (4 - keep);
        }
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    top = groups_max(top);
    if (__ballot(top > m + 8.f || m == kNoScore)) {
      const float to = fmaxf(m, top);
      const float f = to == m ? 1.f : exp2_fast(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[t] *= f;
    }
    // each probability in two BF16 parts
    v4u w[2], rest[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x0 = exp2_fast(s[2 * i] - m), x1 = exp2_fast(s[2 * i + 1] - m);
      l += x0 + x1;
      const uint32_t pair = pack_bf16(x0, x1);
      w[i / 4][i % 4] = pair;
      rest[i / 4][i % 4] = pack_bf16(__builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), __builtin_bit_cast(v2bf, first), x0, false),
                                     __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), __builtin_bit_cast(v2bf, second), x1, false));
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const v4u lo = widen(x.v[t].x, x.v[t].y, vs), hi = widen(x.v[t].z, x.v[t].w, vs);
      o[t] = mfma16(lo, w[0], o[t]);
      o[t] = mfma16(hi, w[1], o[t]);
      o[t] = mfma16(lo, rest[0], o[t]);
      o[t] = mfma16(hi, rest[1], o[t]);
    }
  };
  bool seen = false;  // a page with a token that counts
  for (uint32_t n = 0; p < end; p += kDecodeWaves, ++n) {
    if (n == 64) ids = ids_from(p), n = 0;
    const int32_t id = __builtin_amdgcn_readlane(ids, (int)n);
    if (!known(id)) continue;
    PageCodes<D> x;
    load(x, id);
    attend(x, p);
    seen = true;
  }
  if (!seen) m = -__builtin_inff();
  l = groups_sum(l);
  if (g == 0) sh_m[wave][c] = m, sh_l[wave][c] = l;
#pragma unroll
  for (int t = 0; t < TILES; ++t) *(v4f*)&sh_o[wave][c][16 * t + 4 * g] = o[t];
  __syncthreads();
  // the waves' parts of a head, joined by 16 threads of D / 16 columns each
  const uint32_t hd = threadIdx.x >> 4, part = threadIdx.x & 15;
  if (hd >= live) return;
  float mm = sh_m[0][hd];
#pragma unroll
  for (int w = 1; w < 4; ++w) mm = fmaxf(mm, sh_m[w][hd]);
  float ll = 0.f;
  v4f oo[D / 64] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float mw = sh_m[w][hd], f = mw == mm ? 1.f : exp2_fast(mw - mm);
    ll += sh_l[w][hd] * f;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) oo[j] += *(const v4f*)&sh_o[w][hd][64 * j + 4 * part] * f;
  }
  const size_t at = (size_t)row * a.heads + head0 + hd;
  if (pages > d.chunk) {
    float* const ml = partial + (size_t)a.m * a.heads * d.splits * D;
    if (part == 0) *(float2*)(ml + 2 * (at * d.splits + split)) = float2{mm, ll};
#pragma unroll
    for (int j = 0; j < D / 64; ++j) *(v4f*)(partial + (at * d.splits + split) * D + 64 * j + 4 * part) = oo[j];
    return;
  }
  const float r = weight(mm, ll);
#pragma unroll
  for (int j = 0; j < D / 64; ++j) store4(a, at * D + 64 * j + 4 * part, oo[j] * r);
}

// A row's head, of WAVES waves: the splits' parts joined, each by the D / 4 threads
// of a group, and the groups' results by the first.
template <int D, int WAVES>
__global__ __launch_bounds__(256) void attention_join_kernel(DecodeArgs a, DecodeSplit d, DecodeBy by, const float* partial) {
  constexpr uint32_t LANES = D / 4, GROUPS = 64 * WAVES / LANES, EACH = join_splits(WAVES) / GROUPS, HEADS = 4 / WAVES;
  __shared__ float sh_m[HEADS][GROUPS], sh_l[HEADS][GROUPS];
  __shared__ v4f sh_o[HEADS][GROUPS][LANES];
  const uint32_t mine = threadIdx.x / (64 * WAVES), i = threadIdx.x % LANES, group = threadIdx.x % (64 * WAVES) / LANES;
  const uint64_t at = (uint64_t)blockIdx.x * HEADS + mine;
  const bool real = at < (uint64_t)a.m * a.heads;
  const float* const ml = partial + (size_t)a.m * a.heads * d.splits * D;
  const uint32_t len = real ? min((uint32_t)max(a.lengths[by.heads.of((uint32_t)at)], 0), a.width * kPageTokens) : 0u;
  uint32_t splits = ((len + kPageTokens - 1) / kPageTokens + d.chunk - 1) / d.chunk;
  if (splits == 1) splits = 0;  // the output is there
  float2 part[EACH];
  v4f x[EACH];
  // (requested before the length is known; what a short sequence did not write is not used)
#pragma unroll
  for (uint32_t e = 0; e < EACH; ++e) {
    const uint32_t s = group + e * GROUPS;
    const size_t from = real && s < d.splits ? at * d.splits + s : 0;
    part[e] = *(const float2*)(ml + 2 * from);
    x[e] = *(const v4f*)(partial + from * D + 4 * i);
  }
#pragma unroll
  for (uint32_t e = 0; e < EACH; ++e)
    if (group + e * GROUPS >= splits) part[e] = float2{-__builtin_inff(), 0.f}, x[e] = v4f{};
  float m = part[0].x;
#pragma unroll
  for (uint32_t e = 1; e < EACH; ++e) m = fmaxf(m, part[e].x);
  float l = 0.f;
  v4f o = {};
#pragma unroll
  for (uint32_t e = 0; e < EACH; ++e) {
    const float f = part[e].x == m ? 1.f : exp2_fast(part[e].x - m);
    l += part[e].y * f;
    o += x[e] * f;
  }
  if (i == 0) sh_m[mine][group] = m, sh_l[mine][group] = l;
  sh_o[mine][group][i] = o;
  __syncthreads();
  if (group != 0 || splits == 0) return;
#pragma unroll
  for (uint32_t e = 1; e < GROUPS; ++e) m = fmaxf(m, sh_m[mine][e]);
  l = 0.f;
  o = v4f{};
#pragma unroll
  for (uint32_t e = 0; e < GROUPS; ++e) {
    const float f = sh_m[mine][e] == m ? 1.f : exp2_fast(sh_m[mine][e] - m);
    l += sh_l[mine][e] * f;
    o += sh_o[mine][e][i] * f;
  }
  store4(a, at * D + 4 * i, o * weight(m, l));
}

size_t attention_decode_partial_bytes(uint32_t m, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t width) {
  const DecodeSplit d = decode_split(m, heads, kv_heads, dim, width);
  return d.splits > 1 ? (size_t)m * heads * d.splits * (dim + 2) * sizeof(float) : 0;
}

uint64_t attention_decode_blocks(uint32_t m, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t width) {
  const DecodeSplit d = decode_split(std::max(1u, m), heads, kv_heads, dim, width);
  return std::max((uint64_t)m * kv_heads * d.tiles * d.splits, (uint64_t)m * heads);
}

template <int D>
static void launch_decode(hipStream_t st, const DecodeArgs& a, float* partial) {
  const DecodeSplit d = decode_split(a.m, a.heads, a.kv_heads, a.dim, a.width);
  const DecodeBy by(a, d);
  const dim3 grid(a.m * a.kv_heads * d.tiles * d.splits), block(256);
  hipLaunchKernelGGL(attention_decode_kernel<D>, grid, block, 0, st, a, d, by, partial);
  if (d.splits == 1) return;
  if (d.splits <= join_splits(1))
    hipLaunchKernelGGL((attention_join_kernel<D, 1>), dim3((a.m * a.heads + 3) / 4), block, 0, st, a, d, by,
                       (const float*)partial);
  else
    hipLaunchKernelGGL((attention_join_kernel<D, 4>), dim3(a.m * a.heads), block, 0, st, a, d, by,
                       (const float*)partial);
}

hipError_t launch_attention_decode(hipStream_t st, const DecodeArgs& a, void* workspace) {
  if (a.dim == 128)
    launch_decode<128>(st, a, (float*)workspace);
  else
    launch_decode<64>(st, a, (float*)workspace);
  return hipGetLastError();
}

}  // namespace w8a8
