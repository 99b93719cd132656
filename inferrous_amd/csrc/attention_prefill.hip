// attention_prefill.hip -- causal attention of whole prompts, packed one after
// another, with grouped heads, in BF16.
//
//   o_r = sum_{j <= r} exp(s_rj - m_r) v_j / sum_{j <= r} exp(s_rj - m_r),  s_rj = scale * q_r . k_j
//
// Work: 4 D operations a query head, query and key below the diagonal.  A workgroup
// takes 256 (or 128) rows of one key/value head, where a row is a pair of a query
// and one of the query heads that share the head, query first: whatever the group's
// size, the workgroup's queries are neighbours, so little of what it computes lies
// above the diagonal, and its keys and values are read once for the whole group.  A
// wave holds 32 rows.
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
// A wave issues in order, so what keeps the matrix cores fed is the order.  It works on
// three neighbouring groups of 32 keys at once: the scores of the next, the softmax of
// this one, the sums of the last; one step is a product, the LDS reads for a product
// eight steps on, and one or two probabilities.  Keys and values come 64 at a time
// (global_load_lds_dwordx4, each a turn ahead of its use) through rings of three
// tiles, with one barrier a tile.  Only the tiles that a row of the workgroup sees in
// part, at the diagonal, are done plainly.
//
// The running maximum moves when the scores exceed it by more than 8 (in powers of two):
// probabilities stay below 2^8, and the sums are rescaled a few times, not once for
// every 32 keys.  A probability is rounded to BF16, which the second product takes
// at its rate (in two parts it would be half as many products again, and power bounds
// already), and the sum that divides is that of the rounded ones: against 64 bits the
// outputs are off by 0.0017, where their own rounding alone gives 0.0016.
//
// 32/8 heads of 128: one prompt of 4096 tokens 133 to 145 us (by the card; 136: 1010
// TFLOP/s), one of 16384 1942 us (1134 TFLOP/s, where a library product of 8192^3 reaches
// 1371); heads of 64, twice the exponentials for the same products: 92 and 1254 us (743
// and 877 TFLOP/s).  The matrix
// cores are busy in 58% of the cycles, and the clock is down to 1.95 of 2.4 GHz: each
// part of the loop that is left out (exponentials, reads of LDS, loads) gives its power
// back as clock, 5 to 12%, so that none of them is what the others wait for.  Waves that
// alternate between products and softmax, one barrier each: 2220 us.
#include <algorithm>

#include "attention.hpp"

namespace w8a8 {

constexpr int kTileKeys = 64;

// 16 keys of 32 columns of the values in LDS, as the first operand: lane l's
// column is l % 32 and its keys 4 (l / 32) + {0..3, 8..11}.
__device__ __forceinline__ v4u read_columns(uint32_t at0, uint32_t at1) {
  typedef __attribute__((address_space(3))) v4s* lds_v4s;
  const v2u a = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)at0));
  const v2u b = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)at1));
  return v4u{a.x, a.y, b.x, b.y};
}
__device__ __forceinline__ v4u read_row(uint32_t at) {
  return *(const __attribute__((address_space(3))) v4u*)(uintptr_t)at;
}
__device__ __forceinline__ void write_lds(uint32_t at, v2u x) {
  *(__attribute__((address_space(3))) v2u*)(uintptr_t)at = x;
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
// LDS wait for it.  (m0 takes the LDS address; the warning is that it is reserved.)
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(at), "s"(base), "s"(to) : "memory", "m0");
}

template <int D, int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void attention_prefill_kernel(PrefillArgs a, Divisor kv, Divisor members) {
  constexpr int ROWS = 32 * NW, CH = D / 8, STEPS = D / 16, COLS = D / 32;
  constexpr int TILE = kTileKeys * D * 2;  // bytes of a tile of keys, or of values
  constexpr int LOADS = TILE / 1024 / NW;  // of a wave for one of them
  static_assert(LOADS * NW * 1024 == TILE, "whole loads");
  __shared__ __align__(1024) uint8_t lds[6 * TILE];  // three tiles of keys, then of values
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t unit = kv.of(blockIdx.x), head = blockIdx.x - unit * kv.d, group = members.d;
  uint32_t seq, tile;
  const auto count = [&](uint32_t s) {
    const RowRange r = rows_of(a.starts, s, a.m);
    return (uint32_t)(((uint64_t)(r.hi - r.lo) * group + ROWS - 1) / ROWS);
  };
  if (!find_unit(unit, a.seqs, count, &seq, &tile)) return;
  tile = count(seq) - 1 - tile;  // the longest first
  const RowRange r = rows_of(a.starts, seq, a.m);
  const uint32_t len = r.hi - r.lo;

  // the lane's row: a query and a head
  const uint64_t rows = (uint64_t)len * group, first = (uint64_t)tile * ROWS;
  const uint32_t turns = members.of(tile), left = (tile - turns * group) * ROWS;  // of whole tiles of queries; below 2^18
  const uint32_t first_query = turns * ROWS + members.of(left), first_member = left - members.of(left) * group;
  const auto queries_on = [&](uint32_t row) { return members.near(first_member + row); };
  const auto query_of = [&](uint32_t row) { return min(first_query + queries_on(row), len - 1); };
  const bool mine = first + 32 * wave + col < rows;
  const uint32_t query = query_of(32 * wave + col), member = first_member + 32 * wave + col - queries_on(32 * wave + col) * group;
  const uint32_t last_query = query_of(ROWS - 1), wave_first = query_of(32 * wave), wave_last = query_of(32 * wave + 31);
  const uint32_t tiles = last_query / kTileKeys + 1;    // of the workgroup
  const uint32_t own = wave_last / kTileKeys + 1;       // with a key that a row of the wave sees
  const uint32_t whole = (wave_first + 1) / kTileKeys;  // of those, without one that a row does not see

  v4u q[STEPS];
  {
    const uint16_t* const p = a.q + (size_t)(r.lo + query) * a.q_stride + (size_t)(head * group + member) * D;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) q[s] = *(const v4u*)(p + 16 * s + 8 * half);
  }

  // 16-byte chunks of a row change places so that what one cycle of LDS serves, 256
  // bytes in 64 banks, lies in as many banks: a chunk of 16 rows of keys, four chunks of
  // four rows of values.
  const auto key_swizzle = [](int row) { return D == 128 ? row & 15 : (row >> 1) & 7; };
  const auto value_swizzle = [](int row) { return D == 128 ? (row & 3) * 4 : (row >> 1 & 1) * 4; };
  const uint16_t* const kbase = a.k + (size_t)r.lo * a.k_stride + (size_t)head * D;
  const uint16_t* const vbase = a.v + (size_t)r.lo * a.v_stride + (size_t)head * D;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  // Requests of the wave's part of a tile: row row0 of its first load, and 1024 / (2 D)
  // rows on for each more.  Rows behind the sequence, which no row sees, are a part of its last one.
  constexpr int APART = 1024 / (2 * D);
  const uint32_t row0 = wave * (LOADS * APART) + lane / CH;
  uint32_t key_from[LOADS], value_from[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int row = row0 + j * APART, ch = lane % CH;
    key_from[j] = row * ((uint32_t)a.k_stride * 2) + (ch ^ key_swizzle(row)) * 16;
    value_from[j] = row * ((uint32_t)a.v_stride * 2) + (ch ^ value_swizzle(row)) * 16;
  }
  const auto load_one = [&](uint32_t t, const uint16_t* base, uint32_t stride, uint32_t from, uint32_t to) {
    const uint32_t top = min(t * kTileKeys, len - 1), last = min(len - 1 - top, (uint32_t)kTileKeys - 1);
    load_to_lds(base + (size_t)top * stride, min(from, last * stride * 2 + (2 * D - 16)), to);
  };
  const auto load_key = [&](uint32_t t, int j) {
    load_one(t, kbase, (uint32_t)a.k_stride, key_from[j], lds0 + t % 3 * TILE + (wave * LOADS + j) * 1024);
  };
  const auto load_value = [&](uint32_t t, int j) {
    load_one(t, vbase, (uint32_t)a.v_stride, value_from[j], lds0 + (3 + t % 3) * TILE + (wave * LOADS + j) * 1024);
  };
  const auto load_keys = [&](uint32_t t) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load_key(t, j);
  };
  const auto load_values = [&](uint32_t t) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) load_value(t, j);
  };

  // Where the lane's fragments lie in a tile: of the keys, step i's are at key_at ^
  // 32 i (its two chunks differ from the first step's in bits that the swizzle only
  // flips), of the values, 32 columns c's at value_at ^ 64 c.
  const uint32_t key_at = col * (2 * D) + (half ^ key_swizzle(col)) * 16;
  const int vrow = 4 * half + ((lane & 15) >> 2);
  const uint32_t value_at = vrow * (2 * D) + ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ value_swizzle(vrow)) * 16 + (lane & 1) * 8;

  // in a scalar register: a product with a sum of three vector registers is slower
  const float to_log2 = __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(a.scale * kLog2e)));
  float m = kNoScore, l = 0.f;
  v16f o[COLS] = {}, s[2];
  v4u p[4];
  // v_med3 with infinity: a maximum without fmaxf's care for signalling NaN
  const auto larger = [](float x, float y) { return __builtin_amdgcn_fmed3f(x, y, __builtin_inff()); };
  const v2bf one = {(__bf16)1.f, (__bf16)1.f};
  const auto key = [&](uint32_t t, int b, int i) {
    return read_row(lds0 + t % 3 * TILE + (key_at ^ (32 * i)) + 32 * b * (2 * D));
  };
  // the largest of the lane's part of 32 keys' scores
  const auto top_of = [&](const v16f& x) {
    float tops[2] = {x[0], x[1]};
#pragma unroll
    for (int i = 2; i < 16; ++i) tops[i % 2] = larger(tops[i % 2], x[i]);
    return larger(tops[0], tops[1]);
  };
  // of the row, both of its lanes', as a power of two
  const auto both = [&](float top) {
    const auto other = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    return fmaxf(__uint_as_float(other[0]), __uint_as_float(other[1])) * to_log2;
  };
  // m, or a new one if the scores are far above it, and what sums so far are scaled by for that
  const auto raised = [&](float top) { return top > m + 8.f || m == kNoScore ? fmaxf(m, top) : m; };
  const auto factor = [&](float to) { return to == m ? 1.f : exp2_fast(m - to); };
  const auto rescale = [&](float f) {
    if (__ballot(f != 1.f)) {
#pragma unroll
      for (int c = 0; c < COLS; ++c) o[c] *= f;
    }
  };
  // probabilities of 32 keys, and their sum
  const auto soften = [&](const v16f& x, v4u* to) {
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t pair = pack_bf16(exp2_fast(__builtin_fmaf(x[2 * i], to_log2, -m)),
                                      exp2_fast(__builtin_fmaf(x[2 * i + 1], to_log2, -m)));
      sums[i % 2] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), one, sums[i % 2], false);
      to[i / 4][i % 4] = pair;
    }
    return sums[0] + sums[1];
  };
  const auto values = [&](uint32_t t, int i, int c) {
    const uint32_t at = lds0 + (3 + t % 3) * TILE + (value_at ^ (64 * c)) + 16 * i * (2 * D);
    return read_columns(at, at + 8 * (2 * D));
  };
  // adds a tile that some of the rows see in part
  const auto add_seen_values = [&](uint32_t t) {
    v4u v[2][COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) v[0][c] = values(t, 0, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < 3) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) v[(i + 1) % 2][c] = values(t, i + 1, c);
      }
      uint32_t odd = 0;  // bits 15 and 31 if there is a value that a probability of zero would make NaN
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const v4u x = (v[i % 2][c] & 0x7f807f80u) + 0x00800080u;
        odd |= x.x | x.y | x.z | x.w;
      }
      // what is finite first, then the rest key by key, and only into the rows that see the key
      const bool rest = __ballot(odd & 0x80008000u);
      if (rest) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) v[i % 2][c] &= ~not_finite(v[i % 2][c]);
      }
#pragma unroll
      for (int c = 0; c < COLS; ++c) o[c] = mfma32(v[i % 2][c], p[i], o[c]);
      if (!rest) continue;
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        v4u w = values(t, i, c);
        w &= not_finite(w);
#pragma unroll 1
        for (int key = 0; key < 16; ++key) {
          const int slot = (key >> 3) * 4 + (key & 3);  // of the lanes of half (key >> 2) & 1
          const uint32_t part = half == ((key >> 2) & 1) ? 0xffffu << 16 * (slot & 1) : 0u;
          const v4u only = {slot / 2 == 0 ? part : 0u, slot / 2 == 1 ? part : 0u, slot / 2 == 2 ? part : 0u,
                            slot / 2 == 3 ? part : 0u};
          const bool seen = t * kTileKeys + 16 * i + key <= query;
          const v16f with = mfma32(w & only, p[i], o[c]);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[c][e] = seen ? with[e] : o[c][e];
        }
      }
    }
  };

  load_keys(0);
  load_values(0);
  if (tiles > 1) load_keys(1);
  uint32_t t = 0;
  // tiles that every row of the workgroup sees as a whole
  const uint32_t plain = (first_query + 1) / kTileKeys;
  arrived<0>();
  meet();
  if (plain) {
    v16f s0, s1;
    v4u p0[2], p1[2], kf[STEPS], vf[STEPS];
    static_assert(STEPS == 2 * COLS, "a read for each product");
    uint32_t key_lies[STEPS], value_lies[COLS];  // in the tiles that are read next
    float next_m, next_f;  // for the keys whose scores come next
#pragma unroll
    for (int i = 0; i < STEPS; ++i) key_lies[i] = lds0 + (key_at ^ (32 * i));
#pragma unroll
    for (int c = 0; c < COLS; ++c) value_lies[c] = lds0 + (3 * TILE) + (value_at ^ (64 * c));
    const auto read_key = [&](int b, int i) { kf[i] = read_row(key_lies[i] + 32 * b * (2 * D)); };
    const auto read_value = [&](int b, int j) {
      const uint32_t at = value_lies[j % COLS] + (2 * b + j / COLS) * 16 * (2 * D);
      vf[j] = read_columns(at, at + 8 * (2 * D));
    };
    // Scores of the next 32 keys, sums of the last 32 and the softmax of those between,
    // in one stream: a product, the reads for one that is STEPS products away and a part
    // of the softmax in every step.
    const auto unit = [&](const v16f& now, v16f& next, const v4u* before, v4u* to, int bv, int bk, auto sum, auto load) {
      constexpr int EACH = 16 / (2 * STEPS);
      float sums[2] = {0.f, 0.f}, x[16], tops[2], top;
      m = next_m;
      const float f = next_f;
      next = v16f{};
      const auto pack = [&](int i) {
        const uint32_t pair = pack_bf16(x[2 * i], x[2 * i + 1]);
        sums[i % 2] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), one, sums[i % 2], false);
        to[i / 4][i % 4] = pair;
      };
#pragma unroll
      for (int k = 0; k < 2 * STEPS; ++k) {
        if (k < STEPS) {
          next = mfma32(kf[k], q[k], next);
          if (sum) read_value(bv, k);
        } else {
          const int j = k - STEPS;
          if (sum) o[j % COLS] = mfma32(vf[j], before[j / COLS], o[j % COLS]);
          read_key(bk, j);
        }
#pragma unroll
        for (int e = k * EACH; e < (k + 1) * EACH; ++e) {
          if (e % 2 == 0 && e) pack(e / 2 - 1);
          x[e] = exp2_fast(__builtin_fmaf(now[e], to_log2, -m));
        }
        constexpr int FROM = STEPS + STEPS / 4, MANY = 32 / STEPS;
        if (k >= FROM && k < FROM + STEPS / 2) {
#pragma unroll
          for (int e = (k - FROM) * MANY; e < (k - FROM + 1) * MANY; ++e)
            tops[e % 2] = e < 2 ? next[e] : larger(tops[e % 2], next[e]);
        }
        if (k == 2 * STEPS - 2) top = both(larger(tops[0], tops[1]));
        if (k == 2 * STEPS - 1) {
          next_m = raised(top);
          next_f = factor(next_m);
        }
        if (k % (STEPS / LOADS) == 1) load(k / (STEPS / LOADS));
        __builtin_amdgcn_sched_barrier(0);
      }
      pack(7);
      l = __builtin_fmaf(l, f, sums[0] + sums[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) asm volatile("" : "+v"(to[i]));
      asm volatile("" : "+v"(l), "+v"(next_m), "+v"(next_f));
      rescale(f);
    };
#pragma unroll
    for (int i = 0; i < STEPS; ++i) read_key(0, i);
    s0 = v16f{};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) s0 = mfma32(kf[i], q[i], s0);
    next_m = raised(both(top_of(s0)));
    next_f = 1.f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) read_key(1, i);
    uint32_t key_buffer = 0, value_buffer = 0;
    const auto keys_on = [&] {
      const uint32_t by = key_buffer == 2 ? (uint32_t)(-2 * TILE) : (uint32_t)TILE;
      key_buffer = key_buffer == 2 ? 0 : key_buffer + 1;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) key_lies[i] += by;
    };
    const auto values_on = [&] {
      const uint32_t by = value_buffer == 2 ? (uint32_t)(-2 * TILE) : (uint32_t)TILE;
      value_buffer = value_buffer == 2 ? 0 : value_buffer + 1;
#pragma unroll
      for (int c = 0; c < COLS; ++c) value_lies[c] += by;
    };
    keys_on();
    unit(s0, s1, p1, p0, 1, 0, std::false_type{}, [&](int j) { j < LOADS ? load_key(2, j) : load_value(1, j - LOADS); });
    unit(s1, s0, p0, p1, 0, 1, std::true_type{}, [](int) {});
#pragma unroll 1
    for (t = 1; t < plain; ++t) {
      arrived<0>();
      meet();
      keys_on();
      unit(s0, s1, p1, p0, 1, 0, std::true_type{}, [&](int j) { j < LOADS ? load_key(t + 2, j) : load_value(t + 1, j - LOADS); });
      values_on();
      unit(s1, s0, p0, p1, 0, 1, std::true_type{}, [](int) {});
    }
    // what is left of the last keys; the scores that were taken ahead are not used
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      read_value(1, j);
      o[j % COLS] = mfma32(vf[j], p1[j / COLS], o[j % COLS]);
    }
    arrived<0>();
    meet();
  }
#pragma unroll 1
  for (; t < tiles; ++t) {
    if (t + 1 < tiles) {
      load_keys(t + 2);
      load_values(t + 1);
    }
    if (t < own) {
      s[0] = s[1] = v16f{};
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = mfma32(key(t, b, i), q[i], s[b]);
      if (t >= whole) {
        const int seen = (int)(query - t * kTileKeys) - 4 * half;  // the last key, from the lane's first
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (32 * b + 8 * (i / 4) + i % 4 > seen) s[b][i] = -__builtin_inff();
      }
      const float to = raised(both(larger(top_of(s[0]), top_of(s[1])))), f = t ? factor(to) : 1.f;
      m = to;
      l = __builtin_fmaf(l, f, soften(s[0], p) + soften(s[1], p + 2));
#pragma unroll
      for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(p[i]));  // here: the scores would not fit beside the values
      rescale(f);
      add_seen_values(t);
    }
    if (t + 1 < tiles) {
      arrived<0>();
      meet();
    }
  }

  l += __shfl_xor(l, 32, kWave);
  const float inv = 1.f / l;
  if (a.out_dtype == W8A8_OUT_BF16) {
    // through LDS, so that a store's lanes write whole rows
    meet();
    const uint32_t part = lds0 + wave * (32 * 2 * D);
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        write_lds(part + col * (2 * D) + ((4 * c + i) ^ key_swizzle(col)) * 16 + 8 * half,
                  v2u{pack_bf16(o[c][4 * i] * inv, o[c][4 * i + 1] * inv), pack_bf16(o[c][4 * i + 2] * inv, o[c][4 * i + 3] * inv)});
#pragma unroll
    for (int j = 0; j < 32 / (64 / CH); ++j) {
      const uint32_t row = j * (64 / CH) + lane / CH;
      const uint32_t on = queries_on(32 * wave + row), of = first_member + 32 * wave + row - on * group;
      const v4u x = read_row(part + row * (2 * D) + ((lane % CH) ^ key_swizzle(row)) * 16);
      if (first + 32 * wave + row < rows)
        *(v4u*)((uint16_t*)a.out + ((size_t)(r.lo + first_query + on) * a.heads + head * group + of) * D +
                lane % CH * 8) = x;
    }
    return;
  }
  if (!mine) return;
  const size_t at = ((size_t)(r.lo + query) * a.heads + head * group + member) * D;
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = pack_bf16(o[c][4 * i] * inv, o[c][4 * i + 1] * inv);
      const uint32_t y = pack_bf16(o[c][4 * i + 2] * inv, o[c][4 * i + 3] * inv);
      *(v4u*)((float*)a.out + at + 32 * c + 8 * i + 4 * half) = v4u{x << 16, x & 0xffff0000u, y << 16, y & 0xffff0000u};
    }
}

// Workgroups of `waves` waves: each has a row, and all of a sequence's but its last
// are full.
static uint64_t prefill_blocks(const PrefillArgs& a, int waves) {
  const uint64_t rows = (uint64_t)a.m * (a.heads / a.kv_heads);
  return std::min<uint64_t>((rows + (uint64_t)a.seqs * (32 * waves - 1)) / (32 * waves), rows) * a.kv_heads;
}

// Half the rows a workgroup where the compute units have no second workgroup of whole
// ones to take: one wave a SIMD then ends sooner than two.  One sequence of 32/8 heads
// of 128, 128 rows / 256 rows a workgroup, us: 37 tokens 7.0 / 7.5, 200 10.5 / 12.1, 512
// 15.3 / 18.4, 1024 25.4 / 30.6, 1400 32.8 / 39.9, 2048 52.9 / 56.3, 2300 69.3 / 64.8,
// 4096 170 / 137.  (The bound counts a part of a workgroup for every sequence, so a batch
// of many short prompts gets 256 rows: 64 of 32 tokens, which fill half of them, 18.7.)
static int prefill_waves(const PrefillArgs& a) { return prefill_blocks(a, 8) <= 256 ? 4 : 8; }

uint64_t attention_prefill_blocks(const PrefillArgs& a) { return prefill_blocks(a, prefill_waves(a)); }

template <int D, int NW>
static void start_prefill(hipStream_t st, const PrefillArgs& a) {
  hipLaunchKernelGGL((attention_prefill_kernel<D, NW>), dim3((uint32_t)prefill_blocks(a, NW)), dim3(64 * NW), 0, st, a, Divisor(a.kv_heads),
                     Divisor(a.heads / a.kv_heads));
}

hipError_t launch_attention_prefill(hipStream_t st, const PrefillArgs& a) {
  const bool small = prefill_waves(a) == 4;
  if (a.dim == 128)
    small ? start_prefill<128, 4>(st, a) : start_prefill<128, 8>(st, a);
  else
    small ? start_prefill<64, 4>(st, a) : start_prefill<64, 8>(st, a);
  return hipGetLastError();
}

}  // namespace w8a8
