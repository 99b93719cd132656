// adapters.hip -- a low-rank BF16 adapter per row beside a shared W8A8
// projection, many adapters in one call.  No counterpart in the reference.
//
//   out[r][c] = bf16(residual + RN(RN(f32(q . w) * asc) * ws)
//                    + scaling[a] * sum_j B[a][c][j] * h[r][j]),
//   h[r][j] = sum_i A[a][j][i] * bf16(x[r][i]),   a = ids[r],
// a row whose id is outside [0, n_adapters) taking the projection alone.
// h and both sums are held in f32.
#include "internal.hpp"
#include "routed_common.hpp"

namespace w8a8 {


// h[row][j]: one wave per value.
__global__ __launch_bounds__(256) void adapters_shrink(AdapterArgs a, float* h) {
  const int lane = threadIdx.x & 63;
  const uint32_t j = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (j >= a.rank) return;
  for (uint32_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    const uint32_t id = (uint32_t)a.ids[row];
    if (id >= a.adapters) continue;
    const uint16_t* const w = a.a + ((size_t)id * a.rank + j) * a.width;
    float sum = 0.f;
    for (uint32_t o = lane * 8; o < a.width; o += 512) {
      const v4i av = *(const v4i*)(w + o);
      float x[8];
      if (a.x_bf16) {
        const v4i xv = *(const v4i*)((const uint16_t*)a.x + (size_t)row * a.width + o);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = bf16_lo((uint32_t)xv[i]), x[2 * i + 1] = bf16_hi((uint32_t)xv[i]);
      } else {
        const float* const p = (const float*)a.x + (size_t)row * a.width + o;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = bf16_rne(p[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum = __builtin_fmaf(bf16_lo((uint32_t)av[i]), x[2 * i], sum);
        sum = __builtin_fmaf(bf16_hi((uint32_t)av[i]), x[2 * i + 1], sum);
      }
    }
    sum = wave_sum_f32(sum);
    if (lane == 0) h[(size_t)row * a.rank + j] = sum;
  }
}

// out from the exact accumulators: one thread per column.
__global__ __launch_bounds__(256) void adapters_expand(AdapterArgs a, const int32_t* acc, const float* h) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.n) return;
  const float ws = a.ws[c];
  for (uint32_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    const size_t o = (size_t)row * a.n + c;
    float v = (float)acc[o] * a.asc[row] * ws;
    const uint32_t id = (uint32_t)a.ids[row];
    if (id < a.adapters) {
      const uint16_t* const b = a.b + ((size_t)id * a.n + c) * a.rank;
      const float* const hr = h + (size_t)row * a.rank;
      float d = 0.f;
      for (uint32_t j = 0; j < a.rank; j += 8) {
        const v4i bv = *(const v4i*)(b + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d = __builtin_fmaf(bf16_lo((uint32_t)bv[i]), hr[j + 2 * i], d);
          d = __builtin_fmaf(bf16_hi((uint32_t)bv[i]), hr[j + 2 * i + 1], d);
        }
      }
      v += a.scaling[id] * d;
    }
    if (a.residual) v += a.residual[o];
    store_routed(a.out, a.out_dtype, o, v);
  }
}

hipError_t launch_adapters_shrink(hipStream_t st, const AdapterArgs& a, float* h) {
  const uint32_t y = a.m < 65535u ? a.m : 65535u;
  hipLaunchKernelGGL(adapters_shrink, dim3((a.rank + 3) / 4, y), dim3(256), 0, st, a, h);
  return hipGetLastError();
}

hipError_t launch_adapters_expand(hipStream_t st, const AdapterArgs& a, const int32_t* acc, const float* h) {
  const uint32_t y = a.m < 65535u ? a.m : 65535u;
  hipLaunchKernelGGL(adapters_expand, dim3((a.n + 255) / 256, y), dim3(256), 0, st, a, acc, h);
  return hipGetLastError();
}

}  // namespace w8a8
