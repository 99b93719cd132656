// kv_cache.hip -- the cache of keys and values: what prepare_qk appends to it
// beside normalising and rotating the heads, and copies of its pages.
//
//   n = x / sqrt(mean(x^2) + eps) * gain         (a head's x[D]; optional)
//   (a', b') = (a cos - b sin, b cos + a sin)    (a, b: n's halves)
//   s = the smallest 2^e, e >= -100, with 448 * 2^e >= the page's largest |x|
//   code = e4m3(x / s), nearest even; NaN and infinities are NaN codes
// Norms, rotations and maxima are held in f32 and rounded once: to BF16 in the
// outputs, to e4m3 in the cache.
//
// A scale is a power of two, so that x / s is exact, a larger one later only
// shifts the codes that are there (exact but for e4m3's subnormals), and the
// readers' conversion to BF16 (v_cvt_scalef32_pk_bf16_fp8) applies it for free.
//
// Bytes bound both.  prepare_qk reads and writes each value once; everything of a page's
// head is one workgroup's, so that the scale needs no second pass, and each lane asks
// for all its rows before it uses the first.  4096 rows of five sequences, 32/8 heads of 128,
// BF16: 26.9 us for 111 MB (4.1 TB/s; a large copy reaches 4.93); one row 4.2 to 5 us, a chain
// of three dependent loads (the row's past, its page, the page's scale) and two barriers.
// copy_pages: 200 pages of 36 layers 350 us (5.4 TB/s), 16 KiB a workgroup.
#include <algorithm>
#include <type_traits>

#include "attention.hpp"

namespace w8a8 {

// The scale of a largest magnitude given as f32 bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ float page_scale(uint32_t top) {
  const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}
__device__ __forceinline__ float pow2_inverse(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }

// Four codes; |v| <= 448, or v is not finite.
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ uint32_t codes_times(uint32_t w, float f) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return codes_of(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
}

__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = abs_bits(x);
  return b < kInfBits ? b : 0u;
}

// A lane's share of a head: four values of each half, so that a rotation's
// pairs are in one lane.
struct Share {
  float lo[4], hi[4];
};

// What a lane reads for a share: loads of many shares are under way before the
// first is used.
template <int D, bool BF16IN>
struct Read {
  typename std::conditional<BF16IN, v2u, v4f>::type lo, hi;
  __device__ __forceinline__ void start(const void* rows, size_t at, int i) {
    const uint8_t* p = (const uint8_t*)rows + (at + 4 * i) * (BF16IN ? 2 : 4);
    lo = *(const decltype(lo)*)p;
    hi = *(const decltype(hi)*)(p + D / 2 * (BF16IN ? 2 : 4));
  }
  __device__ __forceinline__ Share share() const {
    Share x;
    if constexpr (BF16IN) {
      x.lo[0] = bf16_lo(lo.x), x.lo[1] = bf16_hi(lo.x), x.lo[2] = bf16_lo(lo.y), x.lo[3] = bf16_hi(lo.y);
      x.hi[0] = bf16_lo(hi.x), x.hi[1] = bf16_hi(hi.x), x.hi[2] = bf16_lo(hi.y), x.hi[3] = bf16_hi(hi.y);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x.lo[j] = lo[j], x.hi[j] = hi[j];
    }
    return x;
  }
};

// The lane's cosines and sines of a position; NaN if the table has no such row.
template <int D>
struct Angles {
  v4f c, s;
  bool known;
  __device__ __forceinline__ void start(const float* rope, uint32_t rope_rows, uint32_t pos, int i) {
    known = pos < rope_rows;
    const float* r = rope + (size_t)(known ? pos : 0u) * D + 4 * i;
    c = *(const v4f*)r, s = *(const v4f*)(r + D / 2);
  }
};

template <int D>
__device__ __forceinline__ void store_share(uint16_t* out, size_t at, int i, const Share& x) {
  uint16_t* p = out + at + 4 * i;
  *(v2u*)p = v2u{pack_bf16(x.lo[0], x.lo[1]), pack_bf16(x.lo[2], x.lo[3])};
  *(v2u*)(p + D / 2) = v2u{pack_bf16(x.hi[0], x.hi[1]), pack_bf16(x.hi[2], x.hi[3])};
}

// The sum over the D / 8 lanes of a head (8 or 16, within a DPP row).
template <int D>
__device__ __forceinline__ float head_sum(float v) {
  auto add = [&](auto other) { v = v + other; };
  add(__uint_as_float(dpp_u32<0xB1>(__float_as_uint(v))));
  add(__uint_as_float(dpp_u32<0x4E>(__float_as_uint(v))));
  add(__uint_as_float(dpp_u32<0x141>(__float_as_uint(v))));
  if constexpr (D == 128) add(__uint_as_float(dpp_u32<0x140>(__float_as_uint(v))));
  return v;
}

// The lane's gains, if there is a norm.
template <int D>
struct Gains {
  v4f a, b;
  __device__ __forceinline__ void start(const float* gain, int i) {
    if (gain) a = *(const v4f*)(gain + 4 * i), b = *(const v4f*)(gain + D / 2 + 4 * i);
  }
};

template <int D>
__device__ __forceinline__ void norm_rotate(Share& x, bool norm, const Gains<D>& g, float eps, const Angles<D>& r) {
  if (norm) {
    const auto mean = [&](float e) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(x.lo[j], x.lo[j], __builtin_fmaf(x.hi[j], x.hi[j], ss));
      return __builtin_fmaf(head_sum<D>(ss), 1.0f / D, e);
    };
    float v = mean(eps);
    // squares that lose bits below f32's normal numbers (v_rsq_f32 takes those for zeros) or
    // overflow: n is that of x times a power of two
    constexpr uint32_t LEAST = 0x0d800000u;  // 2^-100
    if (__builtin_expect(__ballot(__float_as_uint(v) - LEAST >= kInfBits - LEAST) != 0, 0)) {
      const float by = v < __uint_as_float(LEAST) ? 0x1p100f : v == __builtin_inff() ? 0x1p-70f : 1.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) x.lo[j] *= by, x.hi[j] *= by;
      v = mean(eps * by * by);
    }
    const float inv = __builtin_amdgcn_rsqf(v);  // one unit of the last place
#pragma unroll
    for (int j = 0; j < 4; ++j) x.lo[j] = x.lo[j] * inv * g.a[j], x.hi[j] = x.hi[j] * inv * g.b[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = x.lo[j], b = x.hi[j];
    x.lo[j] = r.known ? __builtin_fmaf(a, r.c[j], -(b * r.s[j])) : __builtin_nanf("");
    x.hi[j] = r.known ? __builtin_fmaf(b, r.c[j], a * r.s[j]) : __builtin_nanf("");
  }
}

constexpr uint32_t kPrepareHeads = 4;  // query heads that a group of lanes takes of one token

// A unit is the rows that one sequence brings to one page.  Of a unit, one
// workgroup takes a head's 64 x D keys or values (a whole block of the cache, so that
// its scale is one workgroup's).  The queries of GROUPS of its
// tokens and of kPrepareHeads heads are one workgroup's, too; if every sequence
// brings one row (ONE), GROUPS heads of it are.  D / 8 lanes hold a head.
template <int D, bool BF16IN, bool ONE>
__global__ __launch_bounds__(256) void prepare_qk_kernel(PrepareArgs a, Divisor parts, Divisor sets) {
  constexpr int LPH = D / 8, GROUPS = 256 / LPH, SLOTS = 64 / GROUPS;  // lanes of a head, heads in flight, tokens of a group
  __shared__ uint32_t red[4];
  __shared__ __align__(16) uint32_t turned[ONE ? 1 : D * kPageTokens / 4];  // the page's value codes
  const uint32_t unit = parts.of(blockIdx.x), part = blockIdx.x - unit * parts.d;
  const int tid = threadIdx.x, i = tid % LPH, group = tid / LPH;
  uint32_t seq = unit, index = 0, lo = unit, n = 1;
  if constexpr (!ONE) {
    const auto count = [&](uint32_t s) {
      const RowRange r = rows_of(a.starts, s, a.m);
      const uint32_t p = a.past ? (uint32_t)max(a.past[s], 0) : 0u, rows = r.hi - r.lo;
      return rows ? (p + rows - 1) / kPageTokens - p / kPageTokens + 1 : 0u;
    };
    if (!find_unit(unit, a.seqs, count, &seq, &index)) return;
    const RowRange r = rows_of(a.starts, seq, a.m);
    lo = r.lo;
    n = r.hi - r.lo;
  }
  const uint32_t past = a.past ? (uint32_t)max(a.past[seq], 0) : 0u;
  const uint32_t page = past / kPageTokens + index;  // of the sequence
  const uint32_t first = max(past, page * kPageTokens), last = min(past + n, (page + 1) * kPageTokens);
  const uint32_t n0 = first - page * kPageTokens, n1 = last - page * kPageTokens;  // the unit's slots of the page
  const uint32_t row0 = lo + (first - past);

  if (part >= 2 * a.kv_heads) {
    constexpr uint32_t TIMES = ONE ? 1 : kPrepareHeads, HEADS = ONE ? GROUPS : kPrepareHeads;
    const uint32_t part_q = part - 2 * a.kv_heads, tokens = sets.of(part_q), set = part_q - tokens * sets.d;
    const uint32_t t = ONE ? 0u : tokens * GROUPS + group, h0 = set * HEADS + (ONE ? group : 0u);
    if (t >= n1 - n0 || h0 >= a.heads) return;
    const size_t row = row0 + t;
    Read<D, BF16IN> in[TIMES];
    Angles<D> angles;
    Gains<D> gains;
#pragma unroll
    for (uint32_t j = 0; j < TIMES; ++j) in[j].start(a.q, row * a.q_stride + (size_t)min(h0 + j, a.heads - 1) * D, i);
    angles.start(a.rope, a.rope_rows, first + t, i);
    gains.start(a.q_gain, i);
#pragma unroll
    for (uint32_t j = 0; j < TIMES; ++j) {
      Share x = in[j].share();
      norm_rotate<D>(x, a.q_gain, gains, a.eps, angles);
      if (h0 + j < a.heads) store_share<D>(a.q_out, (row * a.heads + h0 + j) * D, i, x);
    }
    return;
  }

  // The keys of a head, or its values.  The page and what its scale was are asked for
  // before the rows.
  const bool keys = part < a.kv_heads;
  const uint32_t h = keys ? part : part - a.kv_heads;
  int32_t id = a.codes && page < a.width ? a.table[(size_t)seq * a.width + page] : -1;
  if ((uint32_t)id >= a.pages) id = -1;
  const size_t block = (size_t)max(id, 0) * a.kv_heads + h;
  uint8_t* const codes = a.codes + block * page_head_bytes(D) + (keys ? 0 : kPageTokens * D);
  float* const scale = a.scales + block * 2 + (keys ? 0 : 1);
  const float was = n0 && id >= 0 ? *scale : 0.f;  // of tokens that are there

  Share x[SLOTS] = {};
  uint32_t top = 0;
  const uint32_t s0 = SLOTS * group;
  if (s0 < n1 && s0 + SLOTS > n0) {  // the same for a head's lanes
    const auto row_of = [&](int j) { return min(max(s0 + j, n0), n1 - 1) - n0; };
    Read<D, BF16IN> in[SLOTS];
    uint16_t* const out = keys ? a.k_out : a.v_out;
    const void* const from = keys ? a.k : a.v;
    const size_t stride = keys ? a.k_stride : a.v_stride;
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) in[j].start(from, (row0 + row_of(j)) * stride + (size_t)h * D, i);
    if (keys) {
      Angles<D> angles[SLOTS];
      Gains<D> gains;
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) angles[j].start(a.rope, a.rope_rows, first + row_of(j), i);
      gains.start(a.k_gain, i);
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        x[j] = in[j].share();
        norm_rotate<D>(x[j], a.k_gain, gains, a.eps, angles[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) x[j] = in[j].share();
    }
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      if (s0 + j < n0 || s0 + j >= n1) continue;
      if (out) store_share<D>(out, ((row0 + (s0 + j - n0)) * (size_t)a.kv_heads + h) * D, i, x[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, max(finite_bits(x[j].lo[e]), finite_bits(x[j].hi[e])));
    }
  }
  if (id < 0) return;
  top = wave_max_u32(top);
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  const float now = fmaxf(page_scale(top), was), r = pow2_inverse(now);
  if (tid == 0) *scale = now;

  // a larger scale: the codes that are there move down
  if (n0 && now > was) {
    const float f = was * r;
    if (keys) {
      for (uint32_t w = tid; w < n0 * (D / 4); w += 256) ((uint32_t*)codes)[w] = codes_times(((uint32_t*)codes)[w], f);
    } else {
      for (uint32_t w = tid; w < D * (kPageTokens / 4); w += 256) {
        const uint32_t slot = w % (kPageTokens / 4) * 4;
        if (slot >= n0) continue;
        const uint32_t keep = n0 - slot < 4 ? 0xffffffffu << 8 * (n0 - slot) : 0u;  // later slots' bytes
        uint32_t* const p = (uint32_t*)codes + w;
        *p = (codes_times(*p, f) & ~keep) | (*p & keep);
      }
    }
  }
  if (keys) {
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      const uint32_t slot = s0 + j;
      if (slot < n0 || slot >= n1) continue;
      uint32_t* const p = (uint32_t*)(codes + slot * D) + i;
      p[0] = codes_of(x[j].lo[0] * r, x[j].lo[1] * r, x[j].lo[2] * r, x[j].lo[3] * r);
      p[D / 8] = codes_of(x[j].hi[0] * r, x[j].hi[1] * r, x[j].hi[2] * r, x[j].hi[3] * r);
    }
    return;
  }
  __syncthreads();  // a word of the values' codes may hold old tokens and new ones

  uint32_t held[8] = {};  // of each of the lane's columns, its slots' value codes
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) {
    const Share& y = x[j];
    const uint32_t a0 = codes_of(y.lo[0] * r, y.lo[1] * r, y.lo[2] * r, y.lo[3] * r);
    const uint32_t a1 = codes_of(y.hi[0] * r, y.hi[1] * r, y.hi[2] * r, y.hi[3] * r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      held[e] |= (a0 >> 8 * e & 0xffu) << 8 * j;
      held[4 + e] |= (a1 >> 8 * e & 0xffu) << 8 * j;
    }
  }
  if (!ONE && n1 - n0 == kPageTokens) {
    // a whole page of value codes leaves through LDS, 16 bytes a lane: straight from the
    // registers a store's lanes would write 4 bytes each of 64 lines
    constexpr int WORDS = kPageTokens / 4;  // of a column
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int column = 4 * i + e % 4 + e / 4 * (D / 2);
      if constexpr (SLOTS == 4)
        turned[column * WORDS + (group ^ (i & (WORDS - 1)))] = held[e];
      else
        ((uint16_t*)turned)[2 * (column * WORDS + (group / 2 ^ (i & (WORDS - 1)))) + group % 2] = (uint16_t)held[e];
    }
    __syncthreads();
#pragma unroll
    for (int at = 4 * tid; at < D * WORDS; at += 4 * 256) {
      const int column = at / WORDS, turn = column % (D / 2) / 4 & (WORDS - 1), word = at % WORDS;
      v4u x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = turned[column * WORDS + ((word + j) ^ turn)];
      *(v4u*)(codes + 4 * at) = x;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint8_t* const p = codes + (size_t)(4 * i + e % 4 + e / 4 * (D / 2)) * kPageTokens + s0;
    if (s0 >= n0 && s0 + SLOTS <= n1) {
      if constexpr (SLOTS == 4)
        *(uint32_t*)p = held[e];
      else
        *(uint16_t*)p = (uint16_t)held[e];
    } else {
#pragma unroll
      for (int j = 0; j < SLOTS; ++j)
        if (s0 + j >= n0 && s0 + j < n1) p[j] = (uint8_t)(held[e] >> 8 * j);
    }
  }
}

// Workgroups of a unit: those of the key/value heads, and sets of query heads (of whole
// rows, or of the tokens of one after another).
static uint32_t prepare_sets(const PrepareArgs& a) {
  const uint32_t heads = a.starts ? kPrepareHeads : 256 / (a.dim / 8);
  return (a.heads + heads - 1) / heads;
}
static uint32_t prepare_parts(const PrepareArgs& a) {
  return 2 * a.kv_heads + prepare_sets(a) * (a.starts ? kPageTokens * (a.dim / 8) / 256 : 1);
}

// Every unit has a row, and a sequence's pages hold 64 of its rows but for two.
uint64_t prepare_qk_blocks(const PrepareArgs& a) {
  const uint64_t units = a.starts ? std::min<uint64_t>(a.m, a.m / kPageTokens + (uint64_t)2 * a.seqs) : a.m;
  return units * prepare_parts(a);
}

template <int D, bool BF16IN>
static void start_prepare_qk(hipStream_t st, const PrepareArgs& a) {
  const dim3 grid((uint32_t)prepare_qk_blocks(a));
  const Divisor parts(prepare_parts(a)), sets(prepare_sets(a));
  if (a.starts)
    hipLaunchKernelGGL((prepare_qk_kernel<D, BF16IN, false>), grid, dim3(256), 0, st, a, parts, sets);
  else
    hipLaunchKernelGGL((prepare_qk_kernel<D, BF16IN, true>), grid, dim3(256), 0, st, a, parts, sets);
}

hipError_t launch_prepare_qk(hipStream_t st, const PrepareArgs& a) {
  if (a.dim == 128)
    a.bf16 ? start_prepare_qk<128, true>(st, a) : start_prepare_qk<128, false>(st, a);
  else
    a.bf16 ? start_prepare_qk<64, true>(st, a) : start_prepare_qk<64, false>(st, a);
  return hipGetLastError();
}

constexpr uint32_t kCopyBytes = 16384;  // of one workgroup

__global__ __launch_bounds__(256) void copy_pages_kernel(CopyPagesArgs a, uint32_t chunks) {
  const uint32_t chunk = blockIdx.x % chunks, pair = blockIdx.x / chunks % a.n, layer = blockIdx.x / chunks / a.n;
  const int32_t from = a.src[pair], to = a.dst[pair];
  if (from < 0 || to < 0 || (uint32_t)from >= a.pages || (uint32_t)to >= a.pages || from == to) return;
  const size_t bytes = a.kv_heads * page_head_bytes(a.dim);
  const size_t f = (size_t)layer * a.pages + from, t = (size_t)layer * a.pages + to;
  const uint8_t* const p = a.codes + f * bytes;
  uint8_t* const q = a.codes + t * bytes;
  const size_t at = (size_t)chunk * kCopyBytes + threadIdx.x * 16;
  v4u w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (at + j * 4096 < bytes) w[j] = __builtin_nontemporal_load((const v4u*)(p + at + j * 4096));
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (at + j * 4096 < bytes) __builtin_nontemporal_store(w[j], (v4u*)(q + at + j * 4096));
  if (chunk == 0)
    for (uint32_t s = threadIdx.x; s < 2 * a.kv_heads; s += 256)
      a.scales[t * 2 * a.kv_heads + s] = a.scales[f * 2 * a.kv_heads + s];
}

static uint32_t copy_chunks(const CopyPagesArgs& a) {
  return (uint32_t)((a.kv_heads * page_head_bytes(a.dim) + kCopyBytes - 1) / kCopyBytes);
}
uint64_t copy_pages_blocks(const CopyPagesArgs& a) { return (uint64_t)a.layers * a.n * copy_chunks(a); }

hipError_t launch_copy_pages(hipStream_t st, const CopyPagesArgs& a) {
  hipLaunchKernelGGL(copy_pages_kernel, dim3((uint32_t)copy_pages_blocks(a)), dim3(256), 0, st, a, copy_chunks(a));
  return hipGetLastError();
}

}  // namespace w8a8
