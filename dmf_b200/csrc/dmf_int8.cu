// C ABI of inference in 8-bit integers (include/dmf_int8.h): validation and launches.
#include <cuda_runtime.h>

#include <cstring>

#include "dmf_attn.h"
#include "dmf_int8.h"
#include "int8_linear.cuh"
#include "int8_rows.cuh"

namespace {

using namespace dmf;

constexpr int kMaxChannels = 1 << 20;
constexpr int kMaxK = 131071;  // 128 * 128 * K stays below 2^31

int sm_count_of_current_device(int* sm_count) {
  static thread_local int cached_dev = -1, cached_sms = 0, cached_ok = 0;  // a thread rarely changes its device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    return DMF_ATTN_ERR_DEVICE;
  }
  if (dev != cached_dev) {
    int major = 0, sms = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      (void)cudaGetLastError();
      return DMF_ATTN_ERR_DEVICE;
    }
    cached_dev = dev;
    cached_sms = sms;
    cached_ok = (major == 10);
  }
  if (!cached_ok) return DMF_ATTN_ERR_DEVICE;
  *sm_count = cached_sms;
  return DMF_ATTN_OK;
}

int element_bytes(int dtype) { return dtype == DMF_INT8_F32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype == DMF_INT8_BF16 || dtype == DMF_INT8_FP16 || dtype == DMF_INT8_F32; }

int check_pointer(const void* p, int bytes) {
  if (p == nullptr) return DMF_ATTN_ERR_NULL;
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 ? DMF_ATTN_OK : DMF_ATTN_ERR_ALIGN;
}

int check_rows(const dmf_rows& t, int dtype) {
  if (t.stride_b < 0 || t.stride_l < 0) return DMF_ATTN_ERR_STRIDE;
  return check_pointer(t.ptr, element_bytes(dtype));
}

// `written`: rows that are written must not overlap
int check_matrix(const dmf_int8_matrix& t, int columns, bool written) {
  if (t.values == nullptr) return DMF_ATTN_ERR_NULL;
  if (t.stride < (written ? columns : 0)) return DMF_ATTN_ERR_STRIDE;
  return check_pointer(t.scale, 4);
}

int check_row_shape(int batch, int seqlen, int channels) {
  if (batch < 0 || seqlen < 0 || channels < 1 || channels > kMaxChannels) return DMF_ATTN_ERR_SHAPE;
  if (static_cast<int64_t>(batch) * seqlen > 0x7fffffff) return DMF_ATTN_ERR_SHAPE;  // rows are a grid dimension
  return DMF_ATTN_OK;
}

int launched() { return cudaGetLastError() == cudaSuccess ? DMF_ATTN_OK : DMF_ATTN_ERR_LAUNCH; }

template <int kOp>
int launch_rows(const Int8RowParams& p, int64_t rows, cudaStream_t stream) {
  int sms = 0, st = sm_count_of_current_device(&sms);
  if (st != DMF_ATTN_OK) return st;
  if (rows == 0) return DMF_ATTN_OK;
  int8_row_any_kernel<kOp><<<static_cast<unsigned>(rows), kRowThreads, 0, stream>>>(p);
  return launched();
}

void set_out(Int8RowParams* p, const dmf_int8_matrix& out) {
  p->q = out.values;
  p->q_stride = out.stride;
  p->row_scale = out.scale;
}

int run_quantize(const dmf_int8_quantize_args* a) {
  if (a == nullptr) return DMF_ATTN_ERR_NULL;
  if (!known_dtype(a->dtype)) return DMF_ATTN_ERR_DTYPE;
  if (a->act < DMF_INT8_ACT_NONE || a->act > DMF_INT8_ACT_SILU) return DMF_ATTN_ERR_SHAPE;
  int st = check_row_shape(a->batch, a->seqlen, a->channels);
  if (st != DMF_ATTN_OK) return st;
  const int64_t rows = static_cast<int64_t>(a->batch) * a->seqlen;
  if (rows > 0) {
    if ((st = check_rows(a->x, a->dtype)) != DMF_ATTN_OK) return st;
    if ((st = check_matrix(a->out, a->channels, true)) != DMF_ATTN_OK) return st;
  }
  Int8RowParams p = {};
  p.x = a->x.ptr; p.x_sb = a->x.stride_b; p.x_sl = a->x.stride_l; p.x_dtype = a->dtype;
  p.seqlen = a->seqlen; p.channels = a->channels; p.act = a->act;
  set_out(&p, a->out);
  return launch_rows<kRowQuantize>(p, rows, static_cast<cudaStream_t>(a->stream));
}

int run_rmsnorm(const dmf_int8_rmsnorm_args* a) {
  if (a == nullptr) return DMF_ATTN_ERR_NULL;
  if (!known_dtype(a->dtype) || !known_dtype(a->weight_dtype)) return DMF_ATTN_ERR_DTYPE;
  const bool add = a->residual.ptr != nullptr;
  if (add && !known_dtype(a->stream_dtype)) return DMF_ATTN_ERR_DTYPE;
  int st = check_row_shape(a->batch, a->seqlen, a->channels);
  if (st != DMF_ATTN_OK) return st;
  const int64_t rows = static_cast<int64_t>(a->batch) * a->seqlen;
  if (rows > 0) {
    if (add != (a->sum.ptr != nullptr)) return DMF_ATTN_ERR_NULL;
    if ((st = check_rows(a->x, a->dtype)) != DMF_ATTN_OK) return st;
    if (add && ((st = check_rows(a->residual, a->stream_dtype)) != DMF_ATTN_OK || (st = check_rows(a->sum, a->stream_dtype)) != DMF_ATTN_OK))
      return st;
    if ((st = check_pointer(a->weight, element_bytes(a->weight_dtype))) != DMF_ATTN_OK) return st;
    if ((st = check_matrix(a->out, a->channels, true)) != DMF_ATTN_OK) return st;
  }
  Int8RowParams p = {};
  p.x = a->x.ptr; p.x_sb = a->x.stride_b; p.x_sl = a->x.stride_l; p.x_dtype = a->dtype;
  p.add = a->residual.ptr; p.add_sb = a->residual.stride_b; p.add_sl = a->residual.stride_l; p.add_dtype = a->stream_dtype;
  p.sum = a->sum.ptr; p.sum_sb = a->sum.stride_b; p.sum_sl = a->sum.stride_l; p.sum_dtype = a->stream_dtype;
  p.weight = a->weight; p.mod_dtype = a->weight_dtype;
  p.seqlen = a->seqlen; p.channels = a->channels; p.eps = a->eps;
  set_out(&p, a->out);
  return launch_rows<kRowRms>(p, rows, static_cast<cudaStream_t>(a->stream));
}

int run_ln_modulate(const dmf_int8_ln_modulate_args* a) {
  if (a == nullptr) return DMF_ATTN_ERR_NULL;
  if (!known_dtype(a->stream_dtype) || !known_dtype(a->mod_dtype)) return DMF_ATTN_ERR_DTYPE;
  const bool add = a->h.ptr != nullptr;
  if (add && !known_dtype(a->dtype)) return DMF_ATTN_ERR_DTYPE;
  int st = check_row_shape(a->batch, a->seqlen, a->channels);
  if (st != DMF_ATTN_OK) return st;
  const int64_t rows = static_cast<int64_t>(a->batch) * a->seqlen;
  if (rows > 0) {
    if (add != (a->sum.ptr != nullptr) || add != (a->gate.ptr != nullptr)) return DMF_ATTN_ERR_NULL;
    if ((st = check_rows(a->x, a->stream_dtype)) != DMF_ATTN_OK) return st;
    if (add && ((st = check_rows(a->h, a->dtype)) != DMF_ATTN_OK || (st = check_rows(a->sum, a->stream_dtype)) != DMF_ATTN_OK)) return st;
    const dmf_mod* mods[] = {&a->shift, &a->scale, &a->gate};
    for (int i = 0; i < (add ? 3 : 2); ++i) {
      if (mods[i]->stride_b < 0) return DMF_ATTN_ERR_STRIDE;
      if ((st = check_pointer(mods[i]->ptr, element_bytes(a->mod_dtype))) != DMF_ATTN_OK) return st;
    }
    if ((st = check_matrix(a->out, a->channels, true)) != DMF_ATTN_OK) return st;
  }
  Int8RowParams p = {};
  p.x = a->x.ptr; p.x_sb = a->x.stride_b; p.x_sl = a->x.stride_l; p.x_dtype = a->stream_dtype;
  p.add = a->h.ptr; p.add_sb = a->h.stride_b; p.add_sl = a->h.stride_l; p.add_dtype = a->dtype;
  p.sum = a->sum.ptr; p.sum_sb = a->sum.stride_b; p.sum_sl = a->sum.stride_l; p.sum_dtype = a->stream_dtype;
  p.gate = a->gate.ptr; p.gate_sb = a->gate.stride_b;
  p.shift = a->shift.ptr; p.shift_sb = a->shift.stride_b;
  p.scale = a->scale.ptr; p.scale_sb = a->scale.stride_b;
  p.mod_dtype = a->mod_dtype;
  p.seqlen = a->seqlen; p.channels = a->channels; p.eps = a->eps;
  set_out(&p, a->out);
  return launch_rows<kRowLn>(p, rows, static_cast<cudaStream_t>(a->stream));
}

int run_linear(const dmf_int8_linear_args* a) {
  if (a == nullptr) return DMF_ATTN_ERR_NULL;
  if (!known_dtype(a->out_dtype) || (a->bias != nullptr && !known_dtype(a->bias_dtype))) return DMF_ATTN_ERR_DTYPE;
  if (a->m < 0 || a->n < 1 || a->k < 1 || a->k > kMaxK) return DMF_ATTN_ERR_SHAPE;
  int sms = 0, st = DMF_ATTN_OK;
  if (a->m > 0) {
    if ((st = check_matrix(a->x, a->k, false)) != DMF_ATTN_OK) return st;
    if ((st = check_matrix(a->w, a->k, false)) != DMF_ATTN_OK) return st;
    if (a->bias != nullptr && (st = check_pointer(a->bias, element_bytes(a->bias_dtype))) != DMF_ATTN_OK) return st;
    if (a->out_stride < a->n) return DMF_ATTN_ERR_STRIDE;
    if ((st = check_pointer(a->out, element_bytes(a->out_dtype))) != DMF_ATTN_OK) return st;
  }
  if ((st = sm_count_of_current_device(&sms)) != DMF_ATTN_OK) return st;
  if (a->m == 0) return DMF_ATTN_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  const int64_t tiles_m = (static_cast<int64_t>(a->m) + kAnyTile - 1) / kAnyTile, tiles_n = (static_cast<int64_t>(a->n) + kAnyTile - 1) / kAnyTile;
  // at most 65535 blocks fit in grid y: more rows go in slices
  constexpr int64_t kSlice = 65535;
  for (int64_t t0 = 0; t0 < tiles_m; t0 += kSlice) {
    Int8LinearParams p = {};
    const int64_t m0 = t0 * kAnyTile;
    p.x = a->x.values + m0 * a->x.stride; p.x_stride = a->x.stride; p.x_scale = a->x.scale + m0;
    p.w = a->w.values; p.w_stride = a->w.stride; p.w_scale = a->w.scale;
    p.bias = a->bias; p.bias_dtype = a->bias_dtype;
    p.out = static_cast<char*>(a->out) + m0 * a->out_stride * element_bytes(a->out_dtype);
    p.out_stride = a->out_stride; p.out_dtype = a->out_dtype;
    p.m = static_cast<int>(a->m - m0); p.n = a->n; p.k = a->k;
    const dim3 grid(static_cast<unsigned>(tiles_n), static_cast<unsigned>(tiles_m - t0 < kSlice ? tiles_m - t0 : kSlice));
    int8_linear_any_kernel<<<grid, 256, 0, stream>>>(p);
  }
  return launched();
}

int run_dequantize(const dmf_int8_dequantize_args* a) {
  if (a == nullptr) return DMF_ATTN_ERR_NULL;
  if (!known_dtype(a->out_dtype)) return DMF_ATTN_ERR_DTYPE;
  if (a->rows < 0 || a->rows > 0x7fffffff || a->channels < 1) return DMF_ATTN_ERR_SHAPE;
  int sms = 0, st = DMF_ATTN_OK;
  if (a->rows > 0) {
    if ((st = check_matrix(a->x, a->channels, false)) != DMF_ATTN_OK) return st;
    if (a->out_stride < a->channels) return DMF_ATTN_ERR_STRIDE;
    if ((st = check_pointer(a->out, element_bytes(a->out_dtype))) != DMF_ATTN_OK) return st;
  }
  if ((st = sm_count_of_current_device(&sms)) != DMF_ATTN_OK) return st;
  if (a->rows == 0) return DMF_ATTN_OK;
  int8_dequantize_any_kernel<<<static_cast<unsigned>(a->rows), kRowThreads, 0, static_cast<cudaStream_t>(a->stream)>>>(
      a->x.values, a->x.stride, a->x.scale, a->out, a->out_stride, a->out_dtype, a->channels);
  return launched();
}

}  // namespace

#define DMF_EXPORT extern "C" __attribute__((visibility("default")))
DMF_EXPORT int dmf_int8_quantize(const dmf_int8_quantize_args* args) { return run_quantize(args); }
DMF_EXPORT int dmf_int8_rmsnorm(const dmf_int8_rmsnorm_args* args) { return run_rmsnorm(args); }
DMF_EXPORT int dmf_int8_ln_modulate(const dmf_int8_ln_modulate_args* args) { return run_ln_modulate(args); }
DMF_EXPORT int dmf_int8_linear(const dmf_int8_linear_args* args) { return run_linear(args); }
DMF_EXPORT int dmf_int8_dequantize(const dmf_int8_dequantize_args* args) { return run_dequantize(args); }
