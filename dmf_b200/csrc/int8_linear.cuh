// The 8-bit product for rows that TMA cannot read (base or stride no multiple of 16 bytes), on the integer pipe:
//
//   out[m, n] = (sum_k x[m, k] w[n, k]) x_scale[m] w_scale[n] + bias[n]
//
// A block owns 64 x 64 outputs, a thread 4 x 4 of them; 64 bytes of k at a time lie in shared memory as words of four, which
// dp4a multiplies and adds to int32.  Bytes are read one by one.  16384 x 1152 x 3456 takes 1.7 ms here, against 51 us on the tensor
// cores: rows that this package makes start at multiples of 16 bytes, and the callers above the C entry copy others for large products.
#pragma once

#include <stdint.h>

#include "int8_types.cuh"
#include "sm100_ptx.cuh"

namespace dmf {

struct Int8LinearParams {
  const int8_t *x, *w;
  const float *x_scale, *w_scale;
  const void* bias;
  void* out;
  int64_t x_stride, w_stride, out_stride;
  int m, n, k;
  int out_dtype, bias_dtype;
};

constexpr int kAnyTile = 64, kAnyWords = 16;  // 64 bytes of k

__global__ void __launch_bounds__(256) int8_linear_any_kernel(const Int8LinearParams p) {
  __shared__ int sx[kAnyWords][kAnyTile + 1], sw[kAnyWords][kAnyTile + 1];
  grid_dependency_wait();
  grid_launch_dependents();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kAnyTile, n0 = static_cast<int64_t>(blockIdx.x) * kAnyTile;
  int acc[4][4] = {};
  auto word = [&](const int8_t* base, int64_t stride, int64_t row, int rows, int64_t k) -> int {
    uint32_t v = 0u;
    if (row < rows)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k + i < p.k) v |= static_cast<uint32_t>(static_cast<uint8_t>(base[row * stride + k + i])) << (8 * i);
    return static_cast<int>(v);
  };
  for (int64_t k0 = 0; k0 < p.k; k0 += 4 * kAnyWords) {
    for (int i = threadIdx.x; i < kAnyWords * kAnyTile; i += 256) {
      const int kw = i % kAnyWords, r = i / kAnyWords;
      sx[kw][r] = word(p.x, p.x_stride, m0 + r, p.m, k0 + 4 * kw);
      sw[kw][r] = word(p.w, p.w_stride, n0 + r, p.n, k0 + 4 * kw);
    }
    __syncthreads();
#pragma unroll
    for (int kw = 0; kw < kAnyWords; ++kw) {
      int a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = sx[kw][ty + 16 * i];
        b[i] = sw[kw][tx + 16 * i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    if (m >= p.m) continue;
    const float s = p.x_scale[m];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (n >= p.n) continue;
      const float b = p.bias != nullptr ? row_load(p.bias, p.bias_dtype, n) : 0.f;
      row_store(p.out, p.out_dtype, m * p.out_stride + n, fmaf(static_cast<float>(acc[i][j]) * s, p.w_scale[n], b));
    }
  }
}

}  // namespace dmf
