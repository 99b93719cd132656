// attention_prefill.hip -- causal attention of whole prompts, packed one after
// another, with grouped heads, in BF16.
//
//   o_r = sum_{j <= r} exp(s_rj - m_r) v_j / sum_{j <= r} exp(s_rj - m_r),  s_rj = scale * q_r . k_j
//
// The matrix cores bound it: 4 D operations a query head, query and key.  A
// workgroup takes kRows rows of one key/value head, where a row is a pair of a
// query and one of the query heads that share the head, query first: whatever
// the group's size, the workgroup's queries are neighbours, so little of what
// it computes lies above the diagonal, and its keys and values are read once
// for the whole group.  A wave holds 32 rows.
//
// Scores are taken transposed, S^T = K Q^T (v_mfma_f32_32x32x16_bf16, keys as
// rows): lane l holds one row of the workgroup, l % 32, and of each 32 keys the
// 16 with (key / 4) % 2 == l / 32.  A row's maximum and sum are over a lane's own
// registers and one exchange between the wave's halves, the mask is one
// comparison per score with the lane's own limit, and the probabilities,
// packed to BF16 in place, are the second operand of O^T = V^T P^T when that
// product takes its keys in the same order: ds_read_b64_tr_b16 reads 4 keys of
// a column per lane from the row-major values.  No score touches LDS.
//
// Keys and values come 64 at a time through two LDS buffers filled by
// global_load_lds_dwordx4.  16-byte chunk c of row r sits at chunk c ^ swizzle(r).
#include <algorithm>

#include "attention.hpp"

namespace w8a8 {

constexpr int kTileKeys = 64, kPrefillWaves = 8;

// 16 keys of 32 columns of the values in LDS, as the first operand: lane l's
// column is l % 32 and its keys 4 (l / 32) + {0..3, 8..11}.
__device__ __forceinline__ v4u read_columns(const uint8_t* at0, const uint8_t* at1) {
  typedef __attribute__((address_space(3))) v4s* lds_v4s;
  const v2u a = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)at0));
  const v2u b = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)at1));
  return v4u{a.x, a.y, b.x, b.y};
}
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// The bits of a word's BF16 values that are infinities or NaN.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}
__device__ __forceinline__ v4u not_finite(v4u w) {
  return v4u{not_finite(w.x), not_finite(w.y), not_finite(w.z), not_finite(w.w)};
}

// Everything requested but the newest N loads has arrived.
template <int N>
__device__ __forceinline__ void arrived() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// A workgroup barrier that no access to LDS is moved across.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// 16 bytes a lane from `base` + `at` to LDS, at `to` + 16 * lane (base and to are the
// same in every lane).  In assembly: the compiler would make every later read of
// LDS wait for it.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(at), "s"(base), "s"(to) : "memory");
}

template <int D>
__global__ __launch_bounds__(64 * kPrefillWaves, 2) void attention_prefill_kernel(PrefillArgs a) {
  constexpr int NW = kPrefillWaves, ROWS = 32 * NW, CH = D / 8, STEPS = D / 16, COLS = D / 32;
  constexpr int TILE = kTileKeys * D * 2;  // bytes of a tile of keys, or of values
  constexpr int LOADS = TILE / 1024 / NW;  // of a wave for one of them
  static_assert(LOADS * NW * 1024 == TILE, "whole loads");
  __shared__ __align__(1024) uint8_t lds[6 * TILE];  // three tiles of keys, then of values
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t head = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
  uint32_t seq, tile;
  const auto count = [&](uint32_t s) {
    const RowRange r = rows_of(a.starts, s, a.m);
    return (uint32_t)(((uint64_t)(r.hi - r.lo) * group + ROWS - 1) / ROWS);
  };
  if (!find_unit(blockIdx.x / a.kv_heads, a.seqs, count, &seq, &tile)) return;
  tile = count(seq) - 1 - tile;  // the longest first
  const RowRange r = rows_of(a.starts, seq, a.m);
  const uint32_t len = r.hi - r.lo;

  // the lane's row: a query and a head
  const uint64_t rows = (uint64_t)len * group, first = (uint64_t)tile * ROWS;
  const uint64_t flat = first + 32 * wave + col;
  const bool mine = flat < rows;
  const uint32_t query = (uint32_t)((mine ? flat : rows - 1) / group), member = (uint32_t)((mine ? flat : rows - 1) % group);
  const uint32_t last_query = (uint32_t)((std::min<uint64_t>(first + ROWS, rows) - 1) / group);
  const uint32_t wave_first = (uint32_t)(std::min<uint64_t>(first + 32 * wave, rows - 1) / group);
  const uint32_t wave_last = (uint32_t)(std::min<uint64_t>(first + 32 * wave + 31, rows - 1) / group);
  const uint32_t tiles = last_query / kTileKeys + 1;    // of the workgroup
  const uint32_t own = wave_last / kTileKeys + 1;       // with a key that a row of the wave sees
  const uint32_t whole = (wave_first + 1) / kTileKeys;  // of those, without one that a row does not see

  v4u q[STEPS];
  {
    const uint16_t* const p = a.q + (size_t)(r.lo + query) * a.q_stride + (size_t)(head * group + member) * D;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) q[s] = *(const v4u*)(p + 16 * s + 8 * half);
  }

  const auto key_swizzle = [](int row) { return row & (CH - 1); };
  const auto value_swizzle = [](int row) { return D == 128 ? (row & 7) * 2 : (row & 3) * 2; };
  const uint16_t* const kbase = a.k + (size_t)r.lo * a.k_stride + (size_t)head * D;
  const uint16_t* const vbase = a.v + (size_t)r.lo * a.v_stride + (size_t)head * D;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  const auto load_tile = [&](uint32_t t, const uint16_t* base, size_t stride, uint32_t to, auto swizzle) {
    const uint32_t last = len - 1 - min(t * kTileKeys, len - 1);  // rows behind it are that one again
    const void* const from = base + (size_t)min(t * kTileKeys, len - 1) * stride;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int at = (wave * LOADS + j) * 64 + lane, row = at / CH, ch = at % CH;  // where it lands
      load_to_lds(from, min((uint32_t)row, last) * ((uint32_t)stride * 2) + (ch ^ swizzle(row)) * 16,
                  to + (wave * LOADS + j) * 1024);
    }
  };
  const auto load_keys = [&](uint32_t t) { load_tile(t, kbase, a.k_stride, lds0 + t % 3 * TILE, key_swizzle); };
  const auto load_values = [&](uint32_t t) { load_tile(t, vbase, a.v_stride, lds0 + (3 + t % 3) * TILE, value_swizzle); };

  // Where the lane's fragments lie in a tile: of the keys, step i's are at key_at ^
  // 32 i (its two chunks differ from the first step's in bits that the swizzle only
  // flips), of the values, 32 columns c's at value_at ^ 64 c.
  const uint32_t key_at = col * (2 * D) + (half ^ key_swizzle(col)) * 16;
  const int vrow = 4 * half + ((lane & 15) >> 2);
  const uint32_t value_at = vrow * (2 * D) + ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ value_swizzle(vrow)) * 16 + (lane & 1) * 8;

  const float to_log2 = a.scale * kLog2e;
  float m = -__builtin_inff(), l = 0.f;
  v16f o[COLS] = {}, s[2];
  v4u p[4];
  const auto scores = [&](uint32_t t) {
    const uint8_t* const kb = lds + t % 3 * TILE;
    s[0] = s[1] = v16f{};
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] = mfma32(*(const v4u*)(kb + (key_at ^ (32 * i)) + 32 * b * (2 * D)), q[i], s[b]);
  };
  const auto softmax = [&](uint32_t t, auto masked) {
    if (masked && t >= whole) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (t * kTileKeys + 32 * b + 8 * (i / 4) + 4 * half + i % 4 > query) s[b][i] = -__builtin_inff();
    }
    float top = s[0][0];  // v_med3 with infinity: a maximum without fmaxf's care for signalling NaN
#pragma unroll
    for (int i = 1; i < 32; ++i) top = __builtin_amdgcn_fmed3f(top, s[i / 16][i % 16], __builtin_inff());
    const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(__uint_as_float(other[0]), __uint_as_float(other[1])) * to_log2;
    if (__ballot(top > m + 8.f || m == -__builtin_inff())) {
      const float to = fmaxf(m, top);
      const float f = to == m ? 1.f : exp2_fast(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int c = 0; c < COLS; ++c) o[c] *= f;
    }
    const v2bf one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t pair = pack_bf16(exp2_fast(__builtin_fmaf(s[b][2 * i], to_log2, -m)),
                                        exp2_fast(__builtin_fmaf(s[b][2 * i + 1], to_log2, -m)));
        l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), one, l, false);
        p[2 * b + i / 4][i % 4] = pair;
      }
  };
  const auto values = [&](uint32_t t, int i, int c) {
    const uint8_t* const at = lds + (3 + t % 3) * TILE + (value_at ^ (64 * c)) + 16 * i * (2 * D);
    return read_columns(at, at + 8 * (2 * D));
  };
  const auto add_values = [&](uint32_t t) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < COLS; ++c) o[c] = mfma32(values(t, i, c), p[i], o[c]);
  };
  // The same for a tile that some of the rows see in part.
  const auto add_seen_values = [&](uint32_t t) {
    uint32_t odd = 0;  // values on the diagonal's tile that a zero probability would make NaN
#pragma unroll 1
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const v4u bad = not_finite(values(t, i, c));
        odd |= bad.x | bad.y | bad.z | bad.w;
      }
    if (!__ballot(odd != 0)) {
      add_values(t);
      return;
    }
    // what is finite first, then the rest key by key, and only into the rows that see the key
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const v4u v = values(t, i, c);
        o[c] = mfma32(v & ~not_finite(v), p[i], o[c]);
      }
#pragma unroll 1
      for (int key = 0; key < 16; ++key) {
        const int slot = (key >> 3) * 4 + (key & 3);  // of the lanes of half (key >> 2) & 1
        const uint32_t part = half == ((key >> 2) & 1) ? 0xffffu << 16 * (slot & 1) : 0u;
        const v4u only = {slot / 2 == 0 ? part : 0u, slot / 2 == 1 ? part : 0u, slot / 2 == 2 ? part : 0u,
                          slot / 2 == 3 ? part : 0u};
        const bool seen = t * kTileKeys + 16 * i + key <= query;
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          const v4u v = values(t, i, c);
          const v16f with = mfma32(v & not_finite(v) & only, p[i], o[c]);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[c][e] = seen ? with[e] : o[c][e];
        }
      }
    }
  };

  // Two waves share a SIMD.  Half of the waves run half a turn behind, so that one of
  // the two feeds the matrix cores (a tile's scores and the sums of the tile before)
  // while the other works on its softmax.  In turn t a wave requests keys t + 2 and
  // values t + 1, into the buffers that all waves left before the barrier; at the turn's
  // second barrier what it requested a turn ago has arrived, for all to read after
  // the next one.
  const bool behind = wave >= NW / 2;
  load_keys(0);
  load_keys(1);
  load_values(0);
  arrived<2 * LOADS>();
  if (behind) meet();
  uint32_t t = 0;
  // tiles that every row of the workgroup sees as a whole
  const uint32_t plain = (uint32_t)(first / group + 1) / kTileKeys;
  if (plain) {
    meet();
    load_keys(2);
    load_values(1);
    scores(0);
    arrived<2 * LOADS>();
    meet();
    softmax(0, std::false_type{});
#pragma unroll 1
    for (t = 1; t < plain; ++t) {
      meet();
      load_keys(t + 2);
      load_values(t + 1);
      __builtin_amdgcn_s_setprio(1);
      add_values(t - 1);
      scores(t);
      // reads of LDS run eight ahead of the products
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
      for (int i = 0; i < 4 * COLS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
#pragma unroll
      for (int i = 0; i < 2 * STEPS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_s_setprio(0);
      arrived<2 * LOADS>();
      meet();
      softmax(t, std::false_type{});
    }
  }
#pragma unroll 1
  for (; t <= tiles; ++t) {
    meet();
    if (t < tiles) {
      load_keys(t + 2);
      load_values(t + 1);
    }
    __builtin_amdgcn_s_setprio(1);
    if (t > 0 && t <= whole)
      add_values(t - 1);
    else if (t > 0 && t <= own)
      add_seen_values(t - 1);
    if (t < own) scores(t);
    __builtin_amdgcn_s_setprio(0);
    arrived<2 * LOADS>();
    meet();
    if (t < own) softmax(t, std::true_type{});
  }
  if (!behind) meet();
  arrived<0>();

  l += __shfl_xor(l, 32, kWave);
  if (!mine) return;
  const float inv = 1.f / l;
  const size_t at = ((size_t)(r.lo + query) * a.heads + head * group + member) * D;
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = pack_bf16(o[c][4 * i] * inv, o[c][4 * i + 1] * inv);
      const uint32_t y = pack_bf16(o[c][4 * i + 2] * inv, o[c][4 * i + 3] * inv);
      const size_t to = at + 32 * c + 8 * i + 4 * half;
      if (a.out_dtype == W8A8_OUT_BF16)
        *(v2u*)((uint16_t*)a.out + to) = v2u{x, y};
      else
        *(v4u*)((float*)a.out + to) = v4u{x << 16, x & 0xffff0000u, y << 16, y & 0xffff0000u};
    }
}

// Every tile has a row, and a sequence has at most one tile that is not full.
uint64_t attention_prefill_blocks(const PrefillArgs& a) {
  const uint64_t rows = (uint64_t)a.m * (a.heads / a.kv_heads);
  return std::min<uint64_t>(rows / (32 * kPrefillWaves) + a.seqs, rows) * a.kv_heads;
}

hipError_t launch_attention_prefill(hipStream_t st, const PrefillArgs& a) {
  const dim3 grid((uint32_t)attention_prefill_blocks(a)), block(64 * kPrefillWaves);
  if (a.dim == 128)
    hipLaunchKernelGGL(attention_prefill_kernel<128>, grid, block, 0, st, a);
  else
    hipLaunchKernelGGL(attention_prefill_kernel<64>, grid, block, 0, st, a);
  return hipGetLastError();
}

}  // namespace w8a8
