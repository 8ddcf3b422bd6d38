/*
 * dmf_int8.h - C ABI of inference in 8-bit integers: the rows of an activation or a weight as int8 with one fp32 scale
 * per row, the norms in front of a product with their result in that form, and the product itself.
 *
 * Rows in 8 bits.  For a row y (fp32):  a = max|y|,  scale = a / 127,  q = y * (127 / a) rounded to the nearest integer,
 * ties to even; q is in [-127, 127] and stands for q * scale.  A row with a < 2^-120 (zeros included) is held as zeros with
 * scale 0; a row that holds a NaN or an infinity as zeros with scale NaN, so that whatever is computed from it is NaN.
 *
 *     dmf_int8_quantize     y = act(x)                                     act: none, GELU (tanh form), SiLU
 *     dmf_int8_rmsnorm      z = x (+ residual),  y = z rsqrt(mean(z^2) + eps) weight
 *     dmf_int8_ln_modulate  z = x (+ gate * h),  y = (z - mean z) rsqrt(var z + eps) (1 + scale) + shift
 *     dmf_int8_linear       out[m, n] = (sum_k x[m, k] w[n, k]) x_scale[m] w_scale[n] (+ bias[n])
 *     dmf_int8_dequantize   out[m, c] = q[m, c] scale[m]
 *
 * z is used as it is summed in fp32; what is written of it (`sum`) is its rounding to the stream's type.  The sums over k are
 * exact (int32), hence K <= 131071; N <= 2^30; elsewhere C <= 2^20.  At most 2^31 - 1 rows.
 *
 * These are the block's linear layers at sampling time (models/layers.py:119-154 qkv and proj, :157-167 the MLP, :187-201
 * the modulation and the adaLN forms in front of them), which the reference runs in 16 bits.
 *
 * Tensors: (B, L, C) with element strides for B and L and stride 1 for C, per-sample vectors (B, C) with an element stride for
 * B, 8-bit rows with an element stride per row (row b * L + l).  Any size from 1, any stride, any alignment that the
 * element type needs; where C, strides and the bases' alignment are multiples of eight elements the kernels read whole vectors.
 *
 * Return values: the DMF_ATTN_* status codes of dmf_attn.h.  No call allocates or synchronises; zero rows launch nothing.
 */
#ifndef DMF_INT8_H_
#define DMF_INT8_H_

#include <stddef.h>
#include <stdint.h>

#include "dmf_adaln.h"

#ifdef __cplusplus
extern "C" {
#endif

enum dmf_int8_dtype {
  DMF_INT8_BF16 = 0,
  DMF_INT8_FP16 = 1,
  DMF_INT8_F32 = 2
};

enum dmf_int8_act {
  DMF_INT8_ACT_NONE = 0,
  DMF_INT8_ACT_GELU = 1,
  DMF_INT8_ACT_SILU = 2
};

/* rows of a matrix in 8 bits: `values` with an element stride per row, one scale per row (contiguous) */
typedef struct dmf_int8_matrix {
  int8_t* values;
  int64_t stride;
  float* scale;
} dmf_int8_matrix;

typedef struct dmf_int8_quantize_args {
  int32_t batch, seqlen, channels;
  int32_t dtype;                /* of x (enum dmf_int8_dtype) */
  int32_t act;                  /* enum dmf_int8_act */
  int32_t reserved;
  dmf_rows x;
  dmf_int8_matrix out;          /* B * L rows */
  void* stream;                 /* cudaStream_t */
} dmf_int8_quantize_args;

typedef struct dmf_int8_rmsnorm_args {
  int32_t batch, seqlen, channels;
  int32_t dtype;                /* of x */
  int32_t stream_dtype;         /* of residual and sum */
  int32_t weight_dtype;
  float eps;
  int32_t reserved;
  dmf_rows x;
  dmf_rows residual, sum;       /* both or neither; sum may be residual itself */
  const void* weight;           /* (C), contiguous */
  dmf_int8_matrix out;
  void* stream;
} dmf_int8_rmsnorm_args;

typedef struct dmf_int8_ln_modulate_args {
  int32_t batch, seqlen, channels;
  int32_t stream_dtype;         /* of x and sum */
  int32_t dtype;                /* of h */
  int32_t mod_dtype;            /* of shift, scale and gate */
  float eps;
  int32_t reserved;
  dmf_rows x;
  dmf_rows h, sum;              /* with gate: all three or none; sum may be x itself */
  dmf_mod gate, shift, scale;
  dmf_int8_matrix out;
  void* stream;
} dmf_int8_ln_modulate_args;

typedef struct dmf_int8_linear_args {
  int32_t m, n, k;
  int32_t out_dtype;
  int32_t bias_dtype;           /* ignored without bias */
  int32_t reserved;
  dmf_int8_matrix x;            /* m rows of k */
  dmf_int8_matrix w;            /* n rows of k */
  const void* bias;             /* (n), contiguous, or NULL */
  void* out;                    /* m rows of n */
  int64_t out_stride;
  int32_t* status_word;         /* as in dmf_attn_fwd_args; may be NULL */
  void* stream;
} dmf_int8_linear_args;

typedef struct dmf_int8_dequantize_args {
  int64_t rows;
  int32_t channels;
  int32_t out_dtype;
  dmf_int8_matrix x;
  void* out;                    /* `rows` rows of `channels` */
  int64_t out_stride;
  void* stream;
} dmf_int8_dequantize_args;

int dmf_int8_quantize(const dmf_int8_quantize_args* args);
int dmf_int8_rmsnorm(const dmf_int8_rmsnorm_args* args);
int dmf_int8_ln_modulate(const dmf_int8_ln_modulate_args* args);
int dmf_int8_linear(const dmf_int8_linear_args* args);
int dmf_int8_dequantize(const dmf_int8_dequantize_args* args);

/*
 * Checking hook: the kernel template instance, and the cut of k, that dmf_int8_linear picks for m x k x n on the current device (on a
 * B200 where there is none), as text, for rows that the tensor cores can read.
 */
int dmf_int8_linear_kernel_name(int32_t m, int32_t n, int32_t k, char* buf, size_t len);

#ifdef __cplusplus
}
#endif

#endif /* DMF_INT8_H_ */
