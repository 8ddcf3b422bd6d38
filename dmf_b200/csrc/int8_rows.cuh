// Rows in 8 bits (include/dmf_int8.h): quantisation behind an activation, RMS norm and LayerNorm-modulate with the
// residual's addition in front and int8 rows with a scale each behind them, and back to 16 or 32 bits.
//
// HBM-bound: every tensor is read and written once, the row stays in registers between the statistics, the maximum and the
// output.  int8_row_group_kernel has a warp (rows of up to 1280 channels) or a block (wider ones, LayerNorm) take row after row,
// the loads of the next one under way while it works on the present one, and the per-channel vectors in shared memory.
// int8_row_block_kernel has a block per row: few rows, where latency counts, and wide ones without a sample's vectors, where
// blocks that come and go keep more loads under way than the loop's 64 registers allow (16384 x 4608: quantisation 38 us
// against 40, with GELU 55 against 68; gated LayerNorm 188 against 101).  Both move eight elements at a time.
// int8_row_single_kernel takes what these do not - odd widths, strides and alignments, mixed 16-bit types - in the same way, an
// element at a time, and int8_row_any_kernel what is then too wide for a block's registers, computing the row again from global
// memory in every pass.  Sums and the arithmetic are fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "int8_types.cuh"
#include "vec8.cuh"

namespace dmf {

enum Int8RowOp { kRowQuantize, kRowGelu, kRowSilu, kRowRms, kRowLn };
template <int kOp>
constexpr bool kIsNorm = kOp == kRowRms || kOp == kRowLn;
template <int kOp>
constexpr int kActOf = kOp == kRowGelu ? 1 : (kOp == kRowSilu ? 2 : 0);

struct Int8RowParams {
  const void *x, *add;                  // add: residual (RMS) or h (LayerNorm); nullptr: none
  void* sum;                            // the rounded sum, where there is something to add
  const void *weight;                   // RMS: (C)
  const void *gate, *shift, *scale;     // LayerNorm: (B, C)
  int8_t* q;
  float* row_scale;
  int64_t x_sb, x_sl, add_sb, add_sl, sum_sb, sum_sl, gate_sb, shift_sb, scale_sb, q_stride;
  int64_t rows;
  int seqlen, channels, batch;
  int x_dtype, add_dtype, sum_dtype, mod_dtype;   // mod: weight / gate, shift, scale
  float eps;
};

constexpr int kRowThreads = 256;
constexpr float kRowTiny = 7.52316384526264e-37f;   // 2^-120: below it a row counts as zeros (127 / a stays finite)

__device__ __forceinline__ float row_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// SiLU x / (1 + exp(-x)); GELU in its tanh form, 0.5 x (1 + tanh u) = x / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3).
// Both as x / (1 + 2^v): where 2^v overflows the result is 0 (of -infinity NaN, as the formulas have it).
template <int kAct>
__device__ __forceinline__ float row_act(float x) {
  constexpr float kLog2e = 1.4426950408889634f;
  if constexpr (kAct == 0) return x;
  constexpr float c1 = -2.f * 0.7978845608028654f * kLog2e;
  const float v = kAct == 1 ? x * fmaf(c1 * 0.044715f, x * x, c1) : -kLog2e * x;
  return x * row_rcp(1.f + fast_exp2(v));
}

// max(m, |a|, |b|), NaN if one of them is
__device__ __forceinline__ float row_max3(float m, float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return d;
}

// What a row's maximum makes of it.  `bits`: of the maximum of |y|; as unsigned numbers bit patterns order like the values, with
// infinity and then NaN behind them.
struct RowScale {
  float scale, inverse;
};
__device__ __forceinline__ float row_warp_sum(float v) {
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ RowScale row_scale_of(uint32_t bits) {
  const float a = __uint_as_float(bits);
  if (bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
  if (a < kRowTiny) return {0.f, 0.f};
  return {__fdiv_rn(a, 127.f), __fdiv_rn(127.f, a)};
}
// The nearest integer, ties to even, in the low byte of the result: adding 1.5 * 2^23 leaves it in the low mantissa bits.  (The
// conversion instruction shares its unit with the exponentials, at an eighth of the rate of an addition.)  Not for inverse = 0.
__device__ __forceinline__ uint32_t row_quantize(float y, float inverse) {
  return __float_as_uint(__fadd_rn(__fmul_rn(y, inverse), 12582912.f));
}
__device__ __forceinline__ uint32_t row_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Sums and maxima over the block, returned to every thread.  red: two rows of a word per warp, used in turn (`turn` counts), so
// that one barrier per reduction is enough: a row is written again only behind the barrier that follows its last reading.
__device__ __forceinline__ float row_block_sum(float v, float (*red)[32], int& turn) {
  float* r = red[turn++ & 1];
  v = row_warp_sum(v);
  if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) v += r[w];
  return v;
}
__device__ __forceinline__ uint32_t row_block_max(uint32_t v, float (*red)[32], int& turn) {
  float* r = red[turn++ & 1];
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = __uint_as_float(v);
  __syncthreads();
  v = 0u;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) v = max(v, __float_as_uint(r[w]));
  return v;
}

// Coherent, unlike ld_nc_v4: the sum may be written where its first term was read, and what a kernel reads may still be written by
// the grid before it when its own blocks start (a dependent launch), which rules out non-coherent loads anywhere in these kernels.
__device__ __forceinline__ uint4 ld_stream_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Eight consecutive elements as they lie in memory: one load of 16 bytes, or of 32 for fp32.
template <typename T>
struct Raw8 {
  uint4 a;
  __device__ __forceinline__ void load(const void* p, int64_t i) { a = ld_stream_v4(static_cast<const T*>(p) + i); }
  __device__ __forceinline__ void get(float (&f)[8]) const { unpack8<T>(a, f); }
  __device__ __forceinline__ static void put(void* p, int64_t i, const float (&f)[8]) { store8(static_cast<T*>(p) + i, f); }
};
template <>
struct Raw8<float> {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* p, int64_t i) {   // a whole sector per lane: two halves would be fetched twice
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(static_cast<const float*>(p) + i));
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(u[i]);
  }
  __device__ __forceinline__ static void put(void* p, int64_t i, const float (&f)[8]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(static_cast<float*>(p) + i), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                 : "memory");
  }
};

// eight channels of a per-channel vector whose type the launch knows
__device__ __forceinline__ void row_vec8(const void* p, int dtype, int64_t i, float (&f)[8]) {
  if (dtype == 0) unpack8<__nv_bfloat16>(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + i), f);
  else if (dtype == 1) unpack8<__half>(*reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + i), f);
  else {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7])
                 : "l"(static_cast<const float*>(p) + i));
  }
}

// row_act of eight elements, two to an instruction where there is one for two and with one reciprocal for two: 1 / d0 and 1 / d1
// are d1 r and d0 r with r = 1 / (d0 d1), which halves the reciprocals, whose unit bounds these activations (16 results a clock
// and SM, for them and the exponentials).  v is held at 63 so that the product stays finite; below that (|x| of 43 and more for SiLU,
// 7.6 for GELU) the result is x 2^-63 instead of next to nothing.  Two rules keep that from the row: row_far_to_zero first puts 0 for
// every x below kRowActFar, so that it is 2^-53 at most; and the caller takes row_act for a row whose maximum is below kRowActExact =
// 2^-40, so that it is less than 2^-13 of the maximum and rounds to 0 like the true result.
constexpr float kRowActExact = 9.094947017729282e-13f;   // 2^-40
constexpr float kRowActFar = -1024.f;                    // both activations of it are below 2^-1400
template <int kAct>
__device__ __forceinline__ void row_act8(float (&f)[8]) {
  constexpr float kLog2e = 1.4426950408889634f, c1 = -2.f * 0.7978845608028654f * kLog2e;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t x = pack_f2(f[i], f[i + 1]);
    uint64_t v;
    if constexpr (kAct == 1) v = mul2(x, fma2(pack_f2(c1 * 0.044715f, c1 * 0.044715f), mul2(x, x), pack_f2(c1, c1)));
    else v = mul2(pack_f2(-kLog2e, -kLog2e), x);
    float v0, v1, d0, d1;
    unpack_f2(v, v0, v1);
    unpack_f2(add2(pack_f2(1.f, 1.f), pack_f2(fast_exp2(fminf(v0, 63.f)), fast_exp2(fminf(v1, 63.f)))), d0, d1);
    const float r = row_rcp(d0 * d1);
    unpack_f2(mul2(x, mul2(pack_f2(d1, d0), pack_f2(r, r))), f[i], f[i + 1]);
  }
}

// 0, whose activation is 0, for each x below kRowActFar; -infinity stays, its row has no scale.  One minimum for two elements and a
// branch that ordinary rows do not take: 16384 x 4608 bf16 behind GELU 52.7 -> 54.6 us, behind SiLU 51.3 -> 52.3 (a select per element
// would be two instructions instead of half of one).
template <int NV>
__device__ __forceinline__ void row_far_to_zero(float (&z)[NV][8]) {
  float low = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < 8; i += 2) asm("min.f32 %0, %0, %1, %2;" : "+f"(low) : "f"(z[k][i]), "f"(z[k][i + 1]));
  if (low < kRowActFar) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (z[k][i] < kRowActFar && z[k][i] >= -3.402823466e38f) z[k][i] = 0.f;
  }
}

// A row in registers, thread `t` of `threads` holding eights t, t + threads, ...
template <int kOp, typename TX, typename TA, int NV>
struct RowLoads {
  static constexpr bool kAdd = !std::is_void<TA>::value;
  using TAdd = typename std::conditional<kAdd, TA, float>::type;
  Raw8<TX> x[NV];
  Raw8<TAdd> add[NV];
  __device__ __forceinline__ void start(const Int8RowParams& p, int64_t x0, int64_t add0, int t, int threads) {
    const int eights = p.channels >> 3;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * threads < eights) {
        x[k].load(p.x, x0 + 8 * (t + k * threads));
        if constexpr (kAdd) add[k].load(p.add, add0 + 8 * (t + k * threads));
      }
  }
};

// What both kernels do with a loaded row.
//   load_next: called once the loads are in z;  sum_up, max_up: over the row's threads
//   vec(which, c, f): eight channels of 0 gate, 1 weight or 1 + scale, 2 shift
template <int kOp, typename TX, typename TA, int NV, typename Next, typename SumUp, typename MaxUp, typename Vec>
__device__ __forceinline__ void row_in_registers(const Int8RowParams& p, RowLoads<kOp, TX, TA, NV>& loads, int64_t row, int64_t x0, int64_t sum0, int t,
                                                 int threads, Next&& load_next, SumUp&& sum_up, MaxUp&& max_up, Vec&& vec) {
  using Loads = RowLoads<kOp, TX, TA, NV>;
  constexpr bool kAdd = Loads::kAdd;
  using TSum = typename std::conditional<kOp == kRowLn, TX, typename Loads::TAdd>::type;
  const int eights = p.channels >> 3;
  float z[NV][8];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (t + k * threads < eights) {
      loads.x[k].get(z[k]);
      if constexpr (kAdd) {
        float a[8];
        loads.add[k].get(a);
        if constexpr (kOp == kRowRms) {
#pragma unroll
          for (int i = 0; i < 8; ++i) z[k][i] += a[i];
        } else {
          float g[8];
          vec(0, 8 * (t + k * threads), g);
#pragma unroll
          for (int i = 0; i < 8; ++i) z[k][i] = fmaf(g[i], a[i], z[k][i]);
        }
        Raw8<TSum>::put(p.sum, sum0 + 8 * (t + k * threads), z[k]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[k][i] = 0.f;
    }
  }
  load_next();
  if constexpr (kActOf<kOp> != 0) {
    row_far_to_zero<NV>(z);
#pragma unroll
    for (int k = 0; k < NV; ++k) row_act8<kActOf<kOp>>(z[k]);
  }
  if constexpr (kIsNorm<kOp>) {
    const float inv_c = 1.f / static_cast<float>(p.channels);
    if constexpr (kOp == kRowLn) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += z[k][i];
      const float mean = sum_up(s) * inv_c;
      s = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (t + k * threads < eights)
#pragma unroll
          for (int i = 0; i < 8; ++i) z[k][i] -= mean;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(z[k][i], z[k][i], s);
    const float r = rsqrtf(sum_up(s) * inv_c + p.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (t + k * threads < eights) {
        const int c = 8 * (t + k * threads);
        float w[8], b[8];
        vec(1, c, w);
        if constexpr (kOp == kRowLn) vec(2, c, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[k][i] = kOp == kRowLn ? fmaf(z[k][i] * r, w[i], b[i]) : z[k][i] * r * w[i];
      }
  }
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < 8; i += 2) top = row_max3(top, z[k][i], z[k][i + 1]);
  uint32_t bits = max_up(__float_as_uint(top));
  if constexpr (kActOf<kOp> != 0) {
    if (bits < __float_as_uint(kRowActExact)) {   // (the whole row alike)
      top = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (t + k * threads < eights) {
          Raw8<TX> x;
          x.load(p.x, x0 + 8 * (t + k * threads));
          x.get(z[k]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            z[k][i] = row_act<kActOf<kOp>>(z[k][i]);
            top = row_max3(top, z[k][i], z[k][i]);
          }
        }
      bits = max_up(__float_as_uint(top));
    }
  }
  const RowScale rs = row_scale_of(bits);
  int8_t* q = p.q + row * p.q_stride;
  const bool zeros = rs.inverse == 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (t + k * threads < eights) {
      uint2 out = make_uint2(0u, 0u);
      if (!zeros) {
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {   // row_quantize of two
          float a, b;
          unpack_f2(add2(mul2(pack_f2(z[k][i], z[k][i + 1]), pack_f2(rs.inverse, rs.inverse)), pack_f2(12582912.f, 12582912.f)), a, b);
          u[i] = __float_as_uint(a);
          u[i + 1] = __float_as_uint(b);
        }
        out = make_uint2(row_pack4(u[0], u[1], u[2], u[3]), row_pack4(u[4], u[5], u[6], u[7]));
      }
      *reinterpret_cast<uint2*>(q + 8 * (t + k * threads)) = out;
    }
  if (t == 0) p.row_scale[row] = rs.scale;
}

// Many rows.  kWarp: a warp per row, eight rows of a block at a time; else the whole block on one row.  grid (blocks over the rows
// of a sample, samples): block x owns rows [x * rows_per_block, ...) of sample y, so that the sample's vectors are staged once per
// block, as fp32.  (RMS norm and quantisation see all rows as one sample.)
constexpr int kGroupThreads = 512;      // most threads of a block that works on one row
template <int kOp, typename TA>
constexpr int kRowVectors = !kIsNorm<kOp> ? 0 : (kOp == kRowRms ? 1 : (std::is_void<TA>::value ? 2 : 3));

template <int kOp, typename TX, typename TA, int NV, bool kWarp>
__global__ void __launch_bounds__(kWarp ? kRowThreads : kGroupThreads) int8_row_group_kernel(const Int8RowParams p, int rows_per_block) {
  // kRowVectors x channels: [weight or 1 + scale | shift | gate], the first halves of all eights in front of the second ones, so that
  // a warp's 16-byte reads lie side by side
  extern __shared__ __align__(16) float s_vec[];
  __shared__ float red[2][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int t = kWarp ? threadIdx.x & 31 : threadIdx.x, threads = kWarp ? 32 : blockDim.x;
  const int64_t b0 = blockIdx.y;
  if constexpr (kRowVectors<kOp, TA> > 0) {
    for (int c = 8 * threadIdx.x; c < p.channels; c += 8 * blockDim.x) {
      float f[8];
      auto stage = [&](int which, const void* src, int64_t at, float plus) {
        row_vec8(src, p.mod_dtype, at + c, f);
        float* d = s_vec + which * p.channels + (c >> 1);
        *reinterpret_cast<float4*>(d) = make_float4(f[0] + plus, f[1] + plus, f[2] + plus, f[3] + plus);
        *reinterpret_cast<float4*>(d + (p.channels >> 1)) = make_float4(f[4] + plus, f[5] + plus, f[6] + plus, f[7] + plus);
      };
      if constexpr (kOp == kRowRms) {
        stage(0, p.weight, 0, 0.f);
      } else {
        stage(0, p.scale, b0 * p.scale_sb, 1.f);
        stage(1, p.shift, b0 * p.shift_sb, 0.f);
        if constexpr (kRowVectors<kOp, TA> == 3) stage(2, p.gate, b0 * p.gate_sb, 0.f);
      }
    }
    __syncthreads();
  }
  auto vec = [&](int which, int c, float (&f)[8]) {
    const float* v = s_vec + (which == 0 ? 2 : which - 1) * p.channels + (c >> 1);
    const float4 a = *reinterpret_cast<const float4*>(v), b = *reinterpret_cast<const float4*>(v + (p.channels >> 1));
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  };
  const int64_t per_sample = kOp == kRowLn ? p.seqlen : p.rows;
  const int64_t l0 = static_cast<int64_t>(blockIdx.x) * rows_per_block, l1 = min(per_sample, l0 + rows_per_block);
  constexpr int kStep = kWarp ? kRowThreads / 32 : 1;
  RowLoads<kOp, TX, TA, NV> loads;
  auto start = [&](int64_t l) {
    const int64_t b = kOp == kRowLn ? b0 : static_cast<unsigned>(l) / static_cast<unsigned>(p.seqlen);   // rows fit in 31 bits
    const int64_t i = kOp == kRowLn ? l : static_cast<unsigned>(l) % static_cast<unsigned>(p.seqlen);
    loads.start(p, b * p.x_sb + i * p.x_sl, b * p.add_sb + i * p.add_sl, t, threads);
  };
  int turn = 0;
  int64_t l = l0 + (kWarp ? threadIdx.x >> 5 : 0);
  if (l < l1) start(l);
  for (; l < l1; l += kStep) {
    const int64_t b = kOp == kRowLn ? b0 : static_cast<unsigned>(l) / static_cast<unsigned>(p.seqlen);   // rows fit in 31 bits
    const int64_t i = kOp == kRowLn ? l : static_cast<unsigned>(l) % static_cast<unsigned>(p.seqlen);
    row_in_registers<kOp, TX, TA, NV>(
        p, loads, b0 * per_sample + l, b * p.x_sb + i * p.x_sl, b * p.sum_sb + i * p.sum_sl, t, threads,
        [&] {
          if (l + kStep < l1) start(l + kStep);
        },
        [&](float v) { return kWarp ? row_warp_sum(v) : row_block_sum(v, red, turn); },
        [&](uint32_t v) { return kWarp ? __reduce_max_sync(0xffffffffu, v) : row_block_max(v, red, turn); }, vec);
  }
}

// A block per row, the vectors from global memory.
template <int kOp, typename TX, typename TA, int NV>
__global__ void __launch_bounds__(NV == 1 ? 1024 : kGroupThreads) int8_row_block_kernel(const Int8RowParams p) {
  __shared__ float red[2][32];
  grid_dependency_wait();
  grid_launch_dependents();
  int turn = 0;
  const int64_t row = blockIdx.x;
  const int64_t b = blockIdx.x / static_cast<unsigned>(p.seqlen), l = blockIdx.x % static_cast<unsigned>(p.seqlen);
  RowLoads<kOp, TX, TA, NV> loads;
  loads.start(p, b * p.x_sb + l * p.x_sl, b * p.add_sb + l * p.add_sl, threadIdx.x, blockDim.x);
  row_in_registers<kOp, TX, TA, NV>(
      p, loads, row, b * p.x_sb + l * p.x_sl, b * p.sum_sb + l * p.sum_sl, threadIdx.x, blockDim.x, [] {}, [&](float v) { return row_block_sum(v, red, turn); },
      [&](uint32_t v) { return row_block_max(v, red, turn); },
      [&](int which, int c, float (&f)[8]) {
        if (which == 0) row_vec8(p.gate, p.mod_dtype, b * p.gate_sb + c, f);
        else if (which == 2) row_vec8(p.shift, p.mod_dtype, b * p.shift_sb + c, f);
        else if (kOp == kRowRms) row_vec8(p.weight, p.mod_dtype, c, f);
        else {
          row_vec8(p.scale, p.mod_dtype, b * p.scale_sb + c, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] += 1.f;
        }
      });
}

// Rows that cannot be read as vectors: kWarps warps on a row, NE single elements per lane, c = thread of the row + k * threads; a
// block of eight warps has 8 / kWarps rows.  Bound by instruction issue (a load and a store for every element): quantisation of
// 11136 x 1919 23 us, of 1920 in vectors 13, residual + RMS norm 52 and 25, gated LayerNorm (samples of 128 rows) 92 and 31; a block per row took 37, 70 and
// 130, its barriers and divisions not spread over enough elements.
template <int kOp, int NE, int kWarps>
__global__ void __launch_bounds__(kRowThreads) int8_row_single_kernel(const Int8RowParams p) {
  constexpr int kThreads = 32 * kWarps;
  __shared__ float red[kRowThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int t = threadIdx.x % kThreads, group = threadIdx.x / kThreads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (8 / kWarps) + group;
  if (row >= p.rows) return;                           // (a group's warps alike: its barriers are its own)
  const int64_t b = static_cast<unsigned>(row) / static_cast<unsigned>(p.seqlen), l = static_cast<unsigned>(row) % static_cast<unsigned>(p.seqlen);
  auto up = [&](auto&& within, auto&& across, float v) -> float {   // over the row's threads
    v = within(v);
    if constexpr (kWarps > 1) {
      named_bar_sync(1 + group, kThreads);             // the last reduction has been read
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      named_bar_sync(1 + group, kThreads);
      v = red[group * kWarps];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) v = across(v, red[group * kWarps + w]);
    }
    return v;
  };
  auto sum_up = [&](float v) { return up([](float x) { return row_warp_sum(x); }, [](float x, float y) { return x + y; }, v); };
  auto max_up = [&](float v) {                          // of magnitudes and NaN
    return up([](float x) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x))); },
              [](float x, float y) { return row_max3(x, y, y); }, v);
  };
  // eight elements from k0 on; their type is decided once, so that the loads overlap
  auto load8 = [&](const void* src, int dtype, int64_t at, int k0, float (&f)[8]) {
    uint32_t u[8];
    const int64_t i0 = at + t + static_cast<int64_t>(k0) * kThreads;
    if (dtype == 2) {
      const uint32_t* s = static_cast<const uint32_t*>(src) + i0;
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = t + (k0 + k) * kThreads < p.channels ? s[k * kThreads] : 0u;
    } else {
      const uint16_t* s = static_cast<const uint16_t*>(src) + i0;
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = t + (k0 + k) * kThreads < p.channels ? s[k * kThreads] : 0u;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      f[k] = dtype == 0 ? __uint_as_float(u[k] << 16) : (dtype == 1 ? __half2float(__ushort_as_half(static_cast<unsigned short>(u[k]))) : __uint_as_float(u[k]));
  };
  float z[NE];
  const int64_t x0 = b * p.x_sb + l * p.x_sl, add0 = b * p.add_sb + l * p.add_sl, sum0 = b * p.sum_sb + l * p.sum_sl;
#pragma unroll
  for (int k0 = 0; k0 < NE; k0 += 8) {
    float x[8], v[8], g[8];
    load8(p.x, p.x_dtype, x0, k0, x);
    if (kIsNorm<kOp> && p.add != nullptr) {
      load8(p.add, p.add_dtype, add0, k0, v);
      if constexpr (kOp == kRowLn) load8(p.gate, p.mod_dtype, b * p.gate_sb, k0, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[k] = kOp == kRowLn ? fmaf(g[k], v[k], x[k]) : v[k] + x[k];
        if (t + (k0 + k) * kThreads < p.channels) row_store(p.sum, p.sum_dtype, sum0 + t + (k0 + k) * kThreads, x[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k0 + k] = row_act<kActOf<kOp>>(x[k]);     // 0 beyond the row
  }
  if constexpr (kIsNorm<kOp>) {
    const float inv_c = 1.f / static_cast<float>(p.channels);
    if constexpr (kOp == kRowLn) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < NE; ++k) s += z[k];
      const float mean = sum_up(s) * inv_c;
#pragma unroll
      for (int k = 0; k < NE; ++k)
        if (t + k * kThreads < p.channels) z[k] -= mean;
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NE; ++k) s = fmaf(z[k], z[k], s);
    const float r = rsqrtf(sum_up(s) * inv_c + p.eps);
#pragma unroll
    for (int k0 = 0; k0 < NE; k0 += 8) {
      float w[8], v[8];
      load8(kOp == kRowRms ? p.weight : p.scale, p.mod_dtype, kOp == kRowRms ? 0 : b * p.scale_sb, k0, w);
      if constexpr (kOp == kRowLn) load8(p.shift, p.mod_dtype, b * p.shift_sb, k0, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) z[k0 + k] = kOp == kRowLn ? fmaf(z[k0 + k] * r, 1.f + w[k], v[k]) : z[k0 + k] * r * w[k];   // 0 beyond
    }
  }
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < NE; k += 2) top = row_max3(top, z[k], z[k + 1]);
  const RowScale rs = row_scale_of(__float_as_uint(max_up(top)));
  int8_t* q = p.q + row * p.q_stride + t;
  if (rs.inverse == 0.f) {
#pragma unroll
    for (int k = 0; k < NE; ++k)
      if (t + k * kThreads < p.channels) q[k * kThreads] = 0;
  } else {
#pragma unroll
    for (int k = 0; k < NE; ++k)
      if (t + k * kThreads < p.channels) q[k * kThreads] = static_cast<int8_t>(row_quantize(z[k], rs.inverse));
  }
  if (t == 0) p.row_scale[row] = rs.scale;
}

template <int kOp>
__global__ void __launch_bounds__(kRowThreads) int8_row_any_kernel(const Int8RowParams p) {
  __shared__ float red[2][32];
  grid_dependency_wait();
  grid_launch_dependents();
  int turn = 0;
  const int64_t row = blockIdx.x;
  const int64_t b = blockIdx.x / static_cast<unsigned>(p.seqlen), l = blockIdx.x % static_cast<unsigned>(p.seqlen);
  const int64_t x0 = b * p.x_sb + l * p.x_sl, add0 = b * p.add_sb + l * p.add_sl, sum0 = b * p.sum_sb + l * p.sum_sl;
  const float inv_c = 1.f / static_cast<float>(p.channels);
  auto z_at = [&](int c) -> float {
    const float x = row_load(p.x, p.x_dtype, x0 + c);
    if constexpr (!kIsNorm<kOp>) return row_act<kActOf<kOp>>(x);
    if (p.add == nullptr) return x;
    const float a = row_load(p.add, p.add_dtype, add0 + c);
    if constexpr (kOp == kRowRms) return a + x;
    return fmaf(row_load(p.gate, p.mod_dtype, b * p.gate_sb + c), a, x);
  };
  float mean = 0.f, r = 1.f;
  if constexpr (kOp == kRowLn) {
    float s = 0.f;
    for (int c = threadIdx.x; c < p.channels; c += kRowThreads) s += z_at(c);
    mean = row_block_sum(s, red, turn) * inv_c;
  }
  if constexpr (kIsNorm<kOp>) {
    float s = 0.f;
    for (int c = threadIdx.x; c < p.channels; c += kRowThreads) {
      const float z = z_at(c) - mean;
      s = fmaf(z, z, s);
    }
    r = rsqrtf(row_block_sum(s, red, turn) * inv_c + p.eps);
  }
  auto y_of = [&](float z, int c) -> float {
    if constexpr (!kIsNorm<kOp>) return z;
    if constexpr (kOp == kRowRms) return z * r * row_load(p.weight, p.mod_dtype, c);
    return fmaf((z - mean) * r, 1.f + row_load(p.scale, p.mod_dtype, b * p.scale_sb + c),
                row_load(p.shift, p.mod_dtype, b * p.shift_sb + c));
  };
  uint32_t bits = 0u;
  for (int c = threadIdx.x; c < p.channels; c += kRowThreads)
    bits = max(bits, __float_as_uint(fabsf(y_of(z_at(c), c))));
  const RowScale s = row_scale_of(row_block_max(bits, red, turn));
  // a thread reads and writes the same channels in every pass, so sum may be x or the residual
  for (int c = threadIdx.x; c < p.channels; c += kRowThreads) {
    const float z = z_at(c);
    if (kIsNorm<kOp> && p.sum != nullptr) row_store(p.sum, p.sum_dtype, sum0 + c, z);
    p.q[row * p.q_stride + c] = static_cast<int8_t>(s.inverse == 0.f ? 0u : row_quantize(y_of(z, c), s.inverse) & 0xffu);
  }
  if (threadIdx.x == 0) p.row_scale[row] = s.scale;
}

// A warp per piece of a row: four eights per lane, their loads under way together.
constexpr int kDequantizeEights = 4 * 32;
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
int8_dequantize_kernel(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t out_stride, int64_t rows, int eights, int pieces) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / pieces;
  if (row >= rows) return;
  const int k0 = static_cast<int>(unit - row * pieces) * kDequantizeEights + (threadIdx.x & 31);
  const float s = scale[row];
  const uint2* src = reinterpret_cast<const uint2*>(q + row * q_stride);
  uint2 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = k0 + 32 * j < eights ? src[k0 + 32 * j] : make_uint2(0u, 0u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (k0 + 32 * j >= eights) break;
    // q + 128 in the low mantissa bits of 2^23 is 2^23 + 128 + q, exactly; the conversion instruction is slow
    const uint32_t u[2] = {v[j].x ^ 0x80808080u, v[j].y ^ 0x80808080u};
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (__uint_as_float(__byte_perm(u[i >> 2], 0x4b000000u, 0x7540 + (i & 3))) - 8388736.f) * s;
    Raw8<T>::put(out, row * out_stride + 8 * (k0 + 32 * j), f);
  }
}

// The same for rows that start anywhere, eight single elements per lane.
constexpr int kDequantizeSingles = 8 * 32;
__global__ void __launch_bounds__(kRowThreads)
int8_dequantize_any_kernel(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t out_stride, int dtype, int64_t rows, int channels,
                           int pieces) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
  const int64_t row = unit / pieces;
  if (row >= rows) return;
  const int c0 = static_cast<int>(unit - row * pieces) * kDequantizeSingles + (threadIdx.x & 31);
  const float s = scale[row];
  const int8_t* src = q + row * q_stride;
  int v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c0 + 32 * j < channels ? src[c0 + 32 * j] : 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c0 + 32 * j < channels) row_store(out, dtype, row * out_stride + c0 + 32 * j, static_cast<float>(v[j]) * s);
}

}  // namespace dmf
