// attention_decode.hip -- one query row of each sequence over the 8-bit cache.
//
//   s_j = scale * q . (k_scale k_j),  o = sum_j exp(s_j - m) (v_scale v_j) / sum_j exp(s_j - m)
//
// The cache's bytes bound it: 2 * D a token and key/value head, read once.  A
// workgroup takes a sequence's key/value head and a run of its pages, a wave
// every fourth page of the run; up to 16 of the query heads that share the
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
// rescaled a few times, not once a page.  A probability is rounded to BF16, and the
// sum that divides is that of the rounded ones.
#include <algorithm>

#include "attention.hpp"

namespace w8a8 {

constexpr uint32_t kDecodeWaves = 4;
constexpr uint32_t kDecodeHeads = 16;  // query heads of a workgroup

struct DecodeSplit {
  uint32_t tiles;   // workgroups a key/value head's query heads take
  uint32_t splits;  // runs of a sequence's pages
};

// Runs of pages: enough workgroups for twice the CUs where a run keeps eight
// pages of the widest sequence or more.
static DecodeSplit decode_split(uint32_t m, uint32_t heads, uint32_t kv_heads, uint32_t width) {
  DecodeSplit d;
  d.tiles = (heads / kv_heads + kDecodeHeads - 1) / kDecodeHeads;
  const uint64_t units = (uint64_t)m * kv_heads * d.tiles, want = 2 * 256;
  const uint32_t most = std::max(1u, std::min(64u, width / 8));
  d.splits = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(1, (want + units - 1) / units));
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
// Across the four lane groups of a head's column.
__device__ __forceinline__ float groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float groups_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

// partial: [m][kv_heads][tiles][splits] of {float m, l}[16] and O[16][D], or null
// with one split.
template <int D>
__global__ __launch_bounds__(256) void attention_decode_kernel(DecodeArgs a, DecodeSplit d, float* partial) {
  constexpr int HALVES = D / 64, TILES = D / 16;
  __shared__ float sh_m[4][16], sh_l[4][16];
  __shared__ float sh_o[4][16][D + 4];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t group = a.heads / a.kv_heads;
  uint32_t b = blockIdx.x;
  const uint32_t h = b % a.kv_heads;
  b /= a.kv_heads;
  const uint32_t tile = b % d.tiles;
  b /= d.tiles;
  const uint32_t split = b % d.splits, row = b / d.splits;
  const uint32_t head0 = h * group + tile * kDecodeHeads, live = min(kDecodeHeads, group - tile * kDecodeHeads);

  const int32_t* const table = a.table + (size_t)row * a.width;
  const uint32_t len = min((uint32_t)max(a.lengths[row], 0), a.width * kPageTokens);
  const uint32_t pages = (len + kPageTokens - 1) / kPageTokens, run = (pages + d.splits - 1) / d.splits;
  const uint32_t p0 = min(split * run, pages), p1 = min(p0 + run, pages);

  v4u q[2 * HALVES];
#pragma unroll
  for (int s = 0; s < 2 * HALVES; ++s) {
    q[s] = v4u{};
    if ((uint32_t)c < live)
      q[s] = *(const v4u*)(a.q + ((size_t)row * a.heads + head0 + c) * D + 64 * (s / 2) + 16 * g + 8 * (s % 2));
  }
  const float to_log2 = a.scale * kLog2e;
  const size_t head_bytes = page_head_bytes(D);
  float m = -__builtin_inff(), l = 0.f;
  v4f o[TILES] = {};
  for (uint32_t p = p0 + wave; p < p1; p += kDecodeWaves) {
    const int32_t id = table[p];
    if (id < 0 || (uint32_t)id >= a.pages) continue;
    const uint8_t* const codes = a.codes + ((size_t)id * a.kv_heads + h) * head_bytes;
    const float* const scales = a.scales + ((size_t)id * a.kv_heads + h) * 2;
    const float ks = scales[0], vs = scales[1];
    v4u k[4][HALVES], v[TILES];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int f = 0; f < HALVES; ++f)
        k[t][f] = *(const v4u*)(codes + (16 * (c >> 2) + 4 * t + (c & 3)) * D + 64 * f + 16 * g);
#pragma unroll
    for (int t = 0; t < TILES; ++t) v[t] = *(const v4u*)(codes + kPageTokens * D + (16 * t + c) * kPageTokens + 16 * g);
    float s[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      v4f acc = {};
#pragma unroll
      for (int f = 0; f < HALVES; ++f) {
        acc = mfma16(widen(k[t][f].x, k[t][f].y, ks), q[2 * f], acc);
        acc = mfma16(widen(k[t][f].z, k[t][f].w, ks), q[2 * f + 1], acc);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * t + i] = acc[i] * to_log2;
    }
    const uint32_t left = len - p * kPageTokens;  // tokens of the page, 64 but in the last one
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
          v[t][w] &= keep >= 4 ? ~0u : keep <= 0 ? 0u : ~0u >> 8 * (4 - keep);
        }
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    top = groups_max(top);
    if (__ballot(top > m + 8.f || m == -__builtin_inff())) {
      const float to = fmaxf(m, top);
      const float f = to == m ? 1.f : exp2_fast(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[t] *= f;
    }
    v4u w[2];
    const v2bf one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t pair = pack_bf16(exp2_fast(s[2 * i] - m), exp2_fast(s[2 * i + 1] - m));
      l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), one, l, false);
      w[i / 4][i % 4] = pair;
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      o[t] = mfma16(widen(v[t].x, v[t].y, vs), w[0], o[t]);
      o[t] = mfma16(widen(v[t].z, v[t].w, vs), w[1], o[t]);
    }
  }
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
  float ll = 0.f, oo[D / 16] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float mw = sh_m[w][hd], f = mw == mm ? 1.f : exp2_fast(mw - mm);
    ll += sh_l[w][hd] * f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) oo[j] += sh_o[w][hd][part * (D / 16) + j] * f;
  }
  if (partial) {
    float* const at = partial + (((size_t)row * a.kv_heads + h) * d.tiles + tile) * d.splits * (16 * (D + 2)) +
                      (size_t)split * (16 * (D + 2));
    if (part == 0) at[2 * hd] = mm, at[2 * hd + 1] = ll;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) at[32 + hd * D + part * (D / 16) + j] = oo[j];
    return;
  }
  const float r = ll == 0.f ? 0.f : 1.f / ll;
  const size_t at = ((size_t)row * a.heads + head0 + hd) * D + part * (D / 16);
#pragma unroll
  for (int j = 0; j < D / 16; j += 2) {
    const uint32_t pair = pack_bf16(oo[j] * r, oo[j + 1] * r);
    if (a.out_dtype == W8A8_OUT_BF16)
      *(uint32_t*)((uint16_t*)a.out + at + j) = pair;
    else
      *(v2u*)((float*)a.out + at + j) = v2u{pair << 16, pair & 0xffff0000u};
  }
}

// One wave for a row's head: the splits' parts joined.
template <int D>
__global__ __launch_bounds__(64) void attention_join_kernel(DecodeArgs a, DecodeSplit d, const float* partial) {
  const uint32_t row = blockIdx.x / a.heads, head = blockIdx.x % a.heads, group = a.heads / a.kv_heads;
  const uint32_t h = head / group, tile = head % group / kDecodeHeads, hd = head % group % kDecodeHeads;
  const float* const at = partial + (((size_t)row * a.kv_heads + h) * d.tiles + tile) * d.splits * (16 * (D + 2));
  const int lane = threadIdx.x;
  constexpr size_t step = 16 * (D + 2);
  const float m = (uint32_t)lane < d.splits ? at[lane * step + 2 * hd] : -__builtin_inff();
  const float l = (uint32_t)lane < d.splits ? at[lane * step + 2 * hd + 1] : 0.f;
  float mm = m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) mm = fmaxf(mm, __shfl_xor(mm, o, kWave));
  const float f = m == mm ? 1.f : exp2_fast(m - mm);
  float ll = l * f;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) ll += __shfl_xor(ll, o, kWave);
  float oo[D / 64] = {};
  for (uint32_t s = 0; s < d.splits; ++s) {
    const float fs = __shfl(f, (int)s, kWave);
#pragma unroll
    for (int j = 0; j < D / 64; ++j) oo[j] += at[s * step + 32 + hd * D + lane * (D / 64) + j] * fs;
  }
  const float r = ll == 0.f ? 0.f : 1.f / ll;
  const size_t to = ((size_t)row * a.heads + head) * D + lane * (D / 64);
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const uint32_t w = pack_bf16(oo[j] * r, 0.f);
    if (a.out_dtype == W8A8_OUT_BF16)
      ((uint16_t*)a.out)[to + j] = (uint16_t)w;
    else
      ((float*)a.out)[to + j] = bf16_lo(w);
  }
}

size_t attention_decode_partial_bytes(uint32_t m, uint32_t heads, uint32_t kv_heads, uint32_t dim, uint32_t width) {
  const DecodeSplit d = decode_split(m, heads, kv_heads, width);
  return d.splits > 1 ? (size_t)m * kv_heads * d.tiles * d.splits * 16 * (dim + 2) * sizeof(float) : 0;
}

uint64_t attention_decode_blocks(uint32_t m, uint32_t heads, uint32_t kv_heads, uint32_t width) {
  const DecodeSplit d = decode_split(std::max(1u, m), heads, kv_heads, width);
  return std::max((uint64_t)m * kv_heads * d.tiles * d.splits, (uint64_t)m * heads / 4);  // of 256 threads
}

hipError_t launch_attention_decode(hipStream_t st, const DecodeArgs& a, void* workspace) {
  const DecodeSplit d = decode_split(a.m, a.heads, a.kv_heads, a.width);
  float* const partial = d.splits > 1 ? (float*)workspace : nullptr;
  const dim3 grid(a.m * a.kv_heads * d.tiles * d.splits);
  auto go = [&](auto kernel, auto join) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a, d, partial);
    if (partial) hipLaunchKernelGGL(join, dim3(a.m * a.heads), dim3(64), 0, st, a, d, (const float*)partial);
  };
  if (a.dim == 128)
    go(attention_decode_kernel<128>, attention_join_kernel<128>);
  else
    go(attention_decode_kernel<64>, attention_join_kernel<64>);
  return hipGetLastError();
}

}  // namespace w8a8
