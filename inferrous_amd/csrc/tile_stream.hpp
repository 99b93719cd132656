// tile_stream.hpp -- the K loop of the routed layers' int8 MFMA kernels.
//
// A workgroup of NW waves holds BT token rows x BN weight rows, a wave WT x WN
// of them in 32 x 32 blocks of v_mfma_i32_32x32x32_i8.  The weights are the
// op's first operand and the tokens its second, so lane l of a block's 16 x i32
// result holds ONE token, l % 32, and the weight rows 8 (v / 4) + 4 (l / 32) +
// v % 4: a token's scale is one register, and a row's maximum is one over a
// lane's own values and one exchange between the wave's halves.
//
// K advances in 128-byte stages through two LDS rings filled by
// global_load_lds_dwordx4, tokens (SA slots) and weights (SB >= SA slots: those
// lines come from further away), one barrier per stage.  16-byte chunk c of LDS
// row r sits at chunk c ^ ((r >> 1) & 7), so that the 16 rows of a fragment read
// meet 16 bank groups.  Sub-step i of a stage covers bytes [32 i, 32 i + 32);
// lane l reads chunk 2 i + l / 32 of row l % 32, of both operands alike.
//
// Loads complete in issue order.  Batch kt is {tokens kt + SA - 1, weights kt +
// SB - 1}; at the end of stage kt at most the loads issued after tokens kt + 1
// may remain: the weight half of its batch when SB > SA, and the SA - 2
// batches after it.
//
// GROUPED: every stage is a group of K with a scale of its own per token; its
// i32 sums are scaled into f32 accumulators when the stage is done.  The scales
// (f32, one per token row of the wave) ride as one more load of the token ring.
//
// BLOCKED (with GROUPED): a stage's sums are made block by block, each from the
// stage's four fragments of its rows, and folded while the next block's are made:
// the i32 sums take two blocks of registers, not FT * FN, and a wave can hold 64 x
// 128 f32 sums.  A larger tile pulls fewer operand bytes per product.
//
// The op (OP) is the int8 one above or v_mfma_f32_32x32x16_bf16, whose fragments
// are 16 bytes a lane too and whose result has the same layout.  K is then the
// weight row's bytes, 2 a value.  OP_BF16_F32's token rows are f32, twice the
// bytes: a stage takes 256 of them, in two LDS sections of 128 a row, and a
// fragment is rounded to BF16 as it is read.
//
// TAIL (K need not be a multiple of 128): in the last stage a lane whose chunk
// lies past K reads zeros, for both operands (a BF16 weight may be infinite):
// nothing outside the operands is read, and the sums are unchanged.
#pragma once
#include <type_traits>

#include "device_common.hpp"

namespace w8a8 {

typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v16f __attribute__((ext_vector_type(16)));

// s_waitcnt with vmcnt = N and the other counters at their maximum.
template <int N>
__device__ __forceinline__ void await_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

#define W8A8_LDS(p) ((void __attribute__((address_space(3)))*)(p))

__device__ const v4i kZeros16 = {0, 0, 0, 0};

enum { OP_I8 = 0, OP_BF16 = 1, OP_BF16_F32 = 2 };
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v16f mfma_bf16(v4i a, v4i b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v16i mfma_op(v4i a, v4i b, v16i c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v16f mfma_op(v4i a, v4i b, v16f c) { return mfma_bf16(a, b, c); }

// Two f32 values as BF16, rounded to nearest even.
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  return (__float_as_uint(bf16_rne(a)) >> 16) | (__float_as_uint(bf16_rne(b)) & 0xffff0000u);
}

template <int BT_, int BN_, int WT_, int WN_, int SA_, int SB_, bool GROUPED_, bool TAIL_, int OP_ = OP_I8,
          bool BLOCKED_ = false>
struct TileStream {
  static constexpr int OP = OP_, TS = OP == OP_BF16_F32 ? 2 : 1;  // sections of a token row's stage
  using Acc = std::conditional_t<OP == OP_I8, v16i, v16f>;
  static constexpr int BT = BT_, BN = BN_, WT = WT_, WN = WN_, SA = SA_, SB = SB_;
  static constexpr bool GROUPED = GROUPED_, TAIL = TAIL_, BLOCKED = BLOCKED_;
  static constexpr int WAVES_N = BN / WN, NW = (BT / WT) * WAVES_N;
  static constexpr int FT = WT / 32, FN = WN / 32;
  static constexpr int LT = TS * BT / 8 / NW, LN = BN / 8 / NW;  // row loads per wave per stage
  static constexpr int LA = LT + (GROUPED ? 1 : 0), L = LA + LN;
  static constexpr int ASL = TS * BT * 128, BSL = BN * 128, SCL = GROUPED ? 256 : 0;
  static constexpr int RINGS = SA * ASL + SB * BSL;
  static constexpr int LDS = RINGS + NW * SA * SCL;
  static_assert(!GROUPED || OP == OP_I8, "scaled groups are of int8 sums");
  static_assert(LT >= 1 && BT % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole loads");
  static_assert(SA >= 2 && SB >= SA && SB <= 8 && (SA - 1) * LA + (SB - 1) * LN < 64, "ring depths");
  static_assert(LDS <= 160 * 1024, "LDS");
  static_assert(!BLOCKED || (GROUPED && SA == 2 && SB == 2), "blocks of grouped sums, two stages");

  Acc acc[BLOCKED ? 1 : FT][BLOCKED ? 2 : FN];
  v16f sum[GROUPED ? FT : 1][GROUPED ? FN : 1];

  // token_row(r) / weight_row(r): the first byte of tile row r (any row of the
  // operand for a tile row past its end); scale_row(r): where the wave's token
  // row r has its first group's scale, `scale_step` floats between groups.
  template <class TokenRow, class WeightRow, class ScaleRow>
  __device__ __forceinline__ void run(int8_t* lds, uint32_t K, TokenRow token_row, WeightRow weight_row,
                                      ScaleRow scale_row, size_t scale_step) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wt0 = (wave / WAVES_N) * WT, wn0 = (wave % WAVES_N) * WN;
    const uint32_t KT = TAIL ? (K + 127) / 128 : K / 128;
    int8_t* const lds_t = lds;
    int8_t* const lds_n = lds + SA * ASL;
    int8_t* const lds_s = lds + RINGS + wave * SA * SCL;
    auto lds_row = [&](int g) { return 8 * g + (lane >> 3); };
    auto chunk = [&](int g) { return (uint32_t)((lane & 7) ^ ((lds_row(g) >> 1) & 7)) * 16; };
    const int8_t *pt[LT], *pn[LN];
#pragma unroll
    for (int j = 0; j < LT; ++j) {  // LDS row BT + r is the second section of token row r
      const int r = lds_row(wave * LT + j);
      pt[j] = token_row(TS == 2 && r >= BT ? r - BT : r) + (r >= BT ? 128 : 0) + (TAIL ? 0 : chunk(wave * LT + j));
    }
#pragma unroll
    for (int j = 0; j < LN; ++j) pn[j] = weight_row(lds_row(wave * LN + j)) + (TAIL ? 0 : chunk(wave * LN + j));
    const float* ps = nullptr;
    if constexpr (GROUPED) ps = scale_row(wt0 + (lane % WT));
    auto load_t = [&](uint32_t kt, int j) {
      if (j == LT) {  // GROUPED: the stage's scales
        __builtin_amdgcn_global_load_lds((const void*)(ps + (size_t)kt * scale_step),
                                         W8A8_LDS(lds_s + (kt % SA) * SCL), 4, 0, 0);
        return;
      }
      const int8_t* p = pt[j] + (size_t)kt * (128 * TS);
      if constexpr (TAIL) {
        const uint32_t c = chunk(wave * LT + j), sec = lds_row(wave * LT + j) >= BT ? 128 : 0;
        p = kt * (128 * TS) + sec + c < K * TS ? p + c : (const int8_t*)&kZeros16;
      }
      __builtin_amdgcn_global_load_lds((const void*)p,
                                       W8A8_LDS(lds_t + (kt % SA) * ASL + (wave * LT + j) * 1024), 16, 0, 0);
    };
    auto load_n = [&](uint32_t kt, int j) {
      const int8_t* p = pn[j] + (size_t)kt * 128;
      if constexpr (TAIL) {
        const uint32_t c = chunk(wave * LN + j);
        p = kt * 128 + c < K ? p + c : (const int8_t*)&kZeros16;
      }
      __builtin_amdgcn_global_load_lds((const void*)p,
                                       W8A8_LDS(lds_n + (kt % SB) * BSL + (wave * LN + j) * 1024), 16, 0, 0);
    };
    const int fr = lane & 31, fh = lane >> 5;
    int off[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) off[i] = fr * 128 + (((2 * i + fh) ^ ((fr >> 1) & 7)) * 16);
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if constexpr (!BLOCKED) acc[f][j] = Acc{};
        if constexpr (GROUPED) sum[f][j] = v16f{};
      }
    if constexpr (BLOCKED) {
      auto loads = [&](uint32_t kt) {
#pragma unroll
        for (int j = 0; j < LA; ++j) load_t(kt, j);
#pragma unroll
        for (int j = 0; j < LN; ++j) load_n(kt, j);
      };
      auto fold_block = [&](const Acc& a, float ts, v16f& to) {
#pragma unroll
        for (int v = 0; v < 16; ++v) to[v] = __builtin_fmaf((float)a[v], ts, to[v]);
      };
      loads(0);
      for (uint32_t kt = 0; kt < KT; ++kt) {
        await_loads<0>();                     // stage kt landed
        __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's reads of stage kt - 1 returned
        __builtin_amdgcn_s_barrier();         // for every wave
        if (kt + 1 < KT) loads(kt + 1);
        const int8_t* const bt = lds_t + (kt % SA) * ASL + wt0 * 128;
        const int8_t* const bn = lds_n + (kt % SB) * BSL + wn0 * 128;
        v4i tf[FT][4], nf[4];
        float ts[FT];
#pragma unroll
        for (int f = 0; f < FT; ++f) {
          ts[f] = *(const float*)(lds_s + (kt % SA) * SCL + (32 * f + fr) * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) tf[f][i] = *(const v4i*)(bt + f * 4096 + off[i]);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) nf[i] = *(const v4i*)(bn + j * 4096 + off[i]);
#pragma unroll
          for (int f = 0; f < FT; ++f) {
            const int b = j * FT + f;
            Acc& d = acc[0][b & 1];
            d = mfma_op(nf[0], tf[f][0], Acc{});
#pragma unroll
            for (int i = 1; i < 4; ++i) d = mfma_op(nf[i], tf[f][i], d);
            if (b > 0) fold_block(acc[0][(b - 1) & 1], ts[(b - 1) % FT], sum[(b - 1) % FT][(b - 1) / FT]);
          }
        }
        constexpr int LAST = FT * FN - 1;
        fold_block(acc[0][LAST & 1], ts[LAST % FT], sum[LAST % FT][LAST / FT]);
      }
      return;
    } else {
    auto rd = [&](uint32_t kt, int i, v4i(&tf)[FT], v4i(&nf)[FN]) {
      const int8_t* bt = lds_t + (kt % SA) * ASL;
      const int8_t* bn = lds_n + (kt % SB) * BSL;
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        if constexpr (TS == 1) {
          tf[f] = *(const v4i*)(bt + (wt0 + 32 * f) * 128 + off[i]);
        } else {  // 16 values of the stage: half a section; a lane's 8 are two chunks
          const int8_t* const r = bt + ((i >> 1) * BT + wt0 + 32 * f + fr) * 128;
          const int c = 4 * (i & 1) + 2 * fh, key = (fr >> 1) & 7;
          const v4f a = *(const v4f*)(r + (c ^ key) * 16), b = *(const v4f*)(r + ((c + 1) ^ key) * 16);
          tf[f] = v4i{(int)bf16_pair(a.x, a.y), (int)bf16_pair(a.z, a.w), (int)bf16_pair(b.x, b.y),
                      (int)bf16_pair(b.z, b.w)};
        }
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) nf[j] = *(const v4i*)(bn + (wn0 + 32 * j) * 128 + off[i]);
    };
    // FT * FN MFMAs with the loads load(0) .. load(N - 1) issued evenly between
    // them; `first`: the sums start from zero.
    auto mm = [&](const v4i(&tf)[FT], const v4i(&nf)[FN], auto first, auto n, auto load) {
      constexpr int N = decltype(n)::value, MF = FT * FN;
#pragma unroll
      for (int i = 0; i < MF; ++i) {
        Acc& d = acc[i / FN][i % FN];
        d = mfma_op(nf[i % FN], tf[i / FN], decltype(first)::value ? Acc{} : d);
        const int lo = (i * N + MF - 1) / MF, hi = ((i + 1) * N + MF - 1) / MF;
        if (lo == hi) continue;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j >= lo && j < hi) load(j);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    using None = std::integral_constant<int, 0>;
    using LoadsT = std::integral_constant<int, LA>;
    using LoadsN = std::integral_constant<int, LN>;
    using First = std::integral_constant<bool, GROUPED>;
    auto nothing = [](int) {};
    float ts[FT];
    auto rd_scales = [&](uint32_t kt) {
      if constexpr (GROUPED) {
#pragma unroll
        for (int f = 0; f < FT; ++f) ts[f] = *(const float*)(lds_s + (kt % SA) * SCL + (32 * f + fr) * 4);
      }
    };
    auto fold = [&] {
      if constexpr (GROUPED) {
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) sum[f][j][v] = __builtin_fmaf((float)acc[f][j][v], ts[f], sum[f][j][v]);
      }
    };

#pragma unroll
    for (int s = 0; s < SB - 1; ++s) {
      if (s >= (int)KT) break;
      if (s < SA - 1)
#pragma unroll
        for (int j = 0; j < LA; ++j) load_t(s, j);
#pragma unroll
      for (int j = 0; j < LN; ++j) load_n(s, j);
    }
    if (KT >= (uint32_t)SB - 1) await_loads<(SA - 2) * LA + (SB - 2) * LN>();
    else await_loads<0>();
    __builtin_amdgcn_s_barrier();
    v4i t0[FT], n0[FN], t1[FT], n1[FN];
    if (SA - 1 < KT)
#pragma unroll
      for (int j = 0; j < LA; ++j) load_t(SA - 1, j);
    rd(0, 0, t0, n0);
    auto stage = [&](uint32_t kt, auto all) {
      constexpr bool ALL = decltype(all)::value;  // every load of this stage exists
      const bool more_n = ALL || kt + SB - 1 < KT, more_t = ALL || kt + SA < KT;
      rd(kt, 1, t1, n1);
      rd_scales(kt);
      mm(t0, n0, First{}, LoadsN{}, [&](int j) { if (more_n) load_n(kt + SB - 1, j); });
      rd(kt, 2, t0, n0);
      mm(t1, n1, std::false_type{}, None{}, nothing);
      rd(kt, 3, t1, n1);
      mm(t0, n0, std::false_type{}, None{}, nothing);
      if (more_n) await_loads<(SB > SA ? LN : 0) + (SA - 2) * L>();
      else await_loads<0>();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's reads of stage kt returned
      __builtin_amdgcn_s_barrier();         // all waves: stage kt + 1 landed, stage kt read
      rd(kt + 1, 0, t0, n0);
      mm(t1, n1, std::false_type{}, LoadsT{}, [&](int j) { if (more_t) load_t(kt + SA, j); });
      fold();
    };
    uint32_t kt = 0;
    constexpr uint32_t AHEAD = SB > SA ? SB - 1 : SA;
    for (; kt + AHEAD < KT; ++kt) stage(kt, std::true_type{});
    for (; kt + 1 < KT; ++kt) stage(kt, std::false_type{});
    rd(KT - 1, 1, t1, n1);
    rd_scales(KT - 1);
    mm(t0, n0, First{}, None{}, nothing);
    rd(KT - 1, 2, t0, n0);
    mm(t1, n1, std::false_type{}, None{}, nothing);
    rd(KT - 1, 3, t1, n1);
    mm(t0, n0, std::false_type{}, None{}, nothing);
    mm(t1, n1, std::false_type{}, None{}, nothing);
    fold();
    }
  }
};

// The larger of v and the other half of the wave's v, lane by lane.
__device__ __forceinline__ uint32_t halves_max_u32(uint32_t v) {
  const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)s[0], (uint32_t)s[1]);
}

}  // namespace w8a8
