// Rows in 8 bits (include/dmf_int8.h): quantisation behind an activation, RMS norm and LayerNorm-modulate with the
// residual's addition in front and int8 rows with a scale each behind them, and back to 16 or 32 bits.
//
// Any width and alignment: one block per row, the row's values computed again from global memory in every pass (statistics,
// maximum, output).  Sums and the arithmetic are fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace dmf {

enum Int8RowOp { kRowQuantize = 0, kRowRms = 1, kRowLn = 2 };

struct Int8RowParams {
  const void *x, *add;                  // add: residual (RMS) or h (LayerNorm); nullptr: none
  void* sum;                            // the rounded sum, where there is something to add
  const void *weight;                   // RMS: (C)
  const void *gate, *shift, *scale;     // LayerNorm: (B, C)
  int8_t* q;
  float* row_scale;
  int64_t x_sb, x_sl, add_sb, add_sl, sum_sb, sum_sl, gate_sb, shift_sb, scale_sb, q_stride;
  int seqlen, channels;
  int x_dtype, add_dtype, sum_dtype, mod_dtype;   // mod: weight / gate, shift, scale
  int act;
  float eps;
};

constexpr int kRowThreads = 256;
constexpr float kRowTiny = 7.52316384526264e-37f;   // 2^-120: below it a row counts as zeros (127 / a stays finite)

__device__ __forceinline__ float row_load(const void* p, int dtype, int64_t i) {
  if (dtype == 0) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == 1) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void row_store(void* p, int dtype, int64_t i, float v) {
  if (dtype == 0) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == 1) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<float*>(p)[i] = v;
}

// GELU in its tanh form, 0.5 x (1 + tanh u) = x / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3); SiLU x / (1 + exp(-x))
__device__ __forceinline__ float row_act(float x, int act) {
  if (act == 0) return x;
  const float t = act == 1 ? 2.f * 0.7978845608028654f * fmaf(0.044715f * x, x * x, x) : x;
  return __fdividef(x, 1.f + __expf(-t));
}

// What a row's maximum makes of it.  `bits`: max of |y| as unsigned bit patterns, which order like the values with infinity
// and then NaN behind them, so a NaN is not lost as it is in fmaxf.
struct RowScale {
  float scale, inverse;
};
__device__ __forceinline__ RowScale row_scale_of(uint32_t bits) {
  const float a = __uint_as_float(bits);
  if (bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
  if (a < kRowTiny) return {0.f, 0.f};
  return {__fdiv_rn(a, 127.f), __fdiv_rn(127.f, a)};
}
__device__ __forceinline__ int row_quantize(float y, const RowScale& s) {
  return s.inverse == 0.f ? 0 : __float2int_rn(y * s.inverse);
}

// sums and maxima over the block, returned to every thread
__device__ __forceinline__ float row_block_sum(float v, float* red) {
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  __syncthreads();  // red is free
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) v += red[w];
  return v;
}
__device__ __forceinline__ uint32_t row_block_max(uint32_t v, float* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(v);
  __syncthreads();
  v = 0u;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) v = max(v, __float_as_uint(red[w]));
  return v;
}

template <int kOp>
__global__ void __launch_bounds__(kRowThreads) int8_row_any_kernel(const Int8RowParams p) {
  __shared__ float red[kRowThreads / 32];
  const int64_t row = blockIdx.x;
  const int64_t b = row / p.seqlen, l = row % p.seqlen;
  const int64_t x0 = b * p.x_sb + l * p.x_sl, add0 = b * p.add_sb + l * p.add_sl, sum0 = b * p.sum_sb + l * p.sum_sl;
  const float inv_c = 1.f / static_cast<float>(p.channels);
  auto z_at = [&](int c) -> float {
    const float x = row_load(p.x, p.x_dtype, x0 + c);
    if constexpr (kOp == kRowQuantize) return row_act(x, p.act);
    if (p.add == nullptr) return x;
    const float a = row_load(p.add, p.add_dtype, add0 + c);
    if constexpr (kOp == kRowRms) return a + x;
    return fmaf(row_load(p.gate, p.mod_dtype, b * p.gate_sb + c), a, x);
  };
  float mean = 0.f, r = 1.f;
  if constexpr (kOp == kRowLn) {
    float s = 0.f;
    for (int c = threadIdx.x; c < p.channels; c += kRowThreads) s += z_at(c);
    mean = row_block_sum(s, red) * inv_c;
  }
  if constexpr (kOp != kRowQuantize) {
    float s = 0.f;
    for (int c = threadIdx.x; c < p.channels; c += kRowThreads) {
      const float z = z_at(c) - mean;
      s = fmaf(z, z, s);
    }
    r = rsqrtf(row_block_sum(s, red) * inv_c + p.eps);
  }
  auto y_of = [&](float z, int c) -> float {
    if constexpr (kOp == kRowQuantize) return z;
    if constexpr (kOp == kRowRms) return z * r * row_load(p.weight, p.mod_dtype, c);
    return fmaf((z - mean) * r, 1.f + row_load(p.scale, p.mod_dtype, b * p.scale_sb + c),
                row_load(p.shift, p.mod_dtype, b * p.shift_sb + c));
  };
  uint32_t bits = 0u;
  for (int c = threadIdx.x; c < p.channels; c += kRowThreads)
    bits = max(bits, __float_as_uint(fabsf(y_of(z_at(c), c))));
  const RowScale s = row_scale_of(row_block_max(bits, red));
  // a thread reads and writes the same channels in every pass, so sum may be x or the residual
  for (int c = threadIdx.x; c < p.channels; c += kRowThreads) {
    const float z = z_at(c);
    if (kOp != kRowQuantize && p.sum != nullptr) row_store(p.sum, p.sum_dtype, sum0 + c, z);
    p.q[row * p.q_stride + c] = static_cast<int8_t>(row_quantize(y_of(z, c), s));
  }
  if (threadIdx.x == 0) p.row_scale[row] = s.scale;
}

__global__ void __launch_bounds__(kRowThreads)
int8_dequantize_any_kernel(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t out_stride, int dtype, int channels) {
  const int64_t row = blockIdx.x;
  const float s = scale[row];
  for (int c = threadIdx.x; c < channels; c += kRowThreads)
    row_store(out, dtype, row * out_stride + c, static_cast<float>(q[row * q_stride + c]) * s);
}

}  // namespace dmf
