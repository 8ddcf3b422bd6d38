// C ABI of inference in 8-bit integers (include/dmf_int8.h), rows: quantisation, norms with 8-bit results, and the way back.
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "attn_launch.h"
#include "dmf_attn.h"
#include "dmf_int8.h"
#include "int8_launch.h"
#include "int8_rows.cuh"

namespace {

using namespace dmf;

constexpr int kMaxChannels = 1 << 20;

int check_rows(const dmf_rows& t, int dtype) {
  if (t.stride_b < 0 || t.stride_l < 0) return DMF_ATTN_ERR_STRIDE;
  return check_pointer(t.ptr, element_bytes(dtype));
}

int check_row_shape(int batch, int seqlen, int channels) {
  if (batch < 0 || seqlen < 0 || channels < 1 || channels > kMaxChannels) return DMF_ATTN_ERR_SHAPE;
  if (static_cast<int64_t>(batch) * seqlen > 0x7fffffff) return DMF_ATTN_ERR_SHAPE;  // rows are a grid dimension
  return DMF_ATTN_OK;
}

// ---- which kernel ----

// rows that start at multiples of eight elements' bytes, as the kernels read and write them: 16 bytes, of fp32 32
bool whole_vectors(const void* p, int dtype, int64_t stride_b, int batch, int64_t stride_l, int seqlen) {
  const int64_t unit = 8 * element_bytes(dtype);
  return reinterpret_cast<uintptr_t>(p) % unit == 0 && (batch == 1 || stride_b % 8 == 0) && (seqlen == 1 || stride_l % 8 == 0);
}

bool reads_vectors(const Int8RowParams& p, int op) {
  bool ok = p.channels % 8 == 0 && whole_vectors(p.x, p.x_dtype, p.x_sb, p.batch, p.x_sl, p.seqlen) &&
            reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && (p.rows == 1 || p.q_stride % 8 == 0);
  if (p.add != nullptr)
    ok = ok && whole_vectors(p.add, p.add_dtype, p.add_sb, p.batch, p.add_sl, p.seqlen) &&
         whole_vectors(p.sum, p.sum_dtype, p.sum_sb, p.batch, p.sum_sl, p.seqlen);
  if (op == kRowRms) ok = ok && whole_vectors(p.weight, p.mod_dtype, 0, 1, 0, 1);
  if (op == kRowLn) {
    ok = ok && whole_vectors(p.shift, p.mod_dtype, p.shift_sb, p.batch, 0, 1) && whole_vectors(p.scale, p.mod_dtype, p.scale_sb, p.batch, 0, 1);
    if (p.add != nullptr) ok = ok && whole_vectors(p.gate, p.mod_dtype, p.gate_sb, p.batch, 0, 1);
  }
  return ok;
}

// Blocks of a kernel that an SM holds.
int blocks_per_sm(int registers, int threads, int smem) {
  const int by_registers = 65536 / ((registers + 7) / 8 * 8 * threads), by_threads = 2048 / threads, by_smem = smem > 0 ? 227 * 1024 / (smem + 1280) : 32;
  int blocks = by_registers < by_threads ? by_registers : by_threads;
  if (by_smem < blocks) blocks = by_smem;
  return blocks > 1 ? blocks : 1;
}

// A kernel's registers per thread, asked for once.
template <typename Kernel>
int registers_of(Kernel kernel, std::atomic<int>& registers) {
  if (registers.load(std::memory_order_relaxed) != 0) return DMF_ATTN_OK;
  cudaFuncAttributes attr;
  if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess) {
    (void)cudaGetLastError();
    return DMF_ATTN_ERR_LAUNCH;
  }
  registers.store(attr.numRegs, std::memory_order_relaxed);
  return DMF_ATTN_OK;
}

constexpr int kWarpRowEights = 160;            // a warp's registers hold rows of up to 5 x 32 eights
constexpr int kMaxEights = 4 * kGroupThreads;  // a block's: 4 per thread

// The loop over rows where that fills the SMs; the LayerNorm form, whose blocks stay within a sample, also wants a few rows of a
// sample per block.
bool many_rows(const Int8RowParams& p, int op, int sms) {
  if (p.channels / 8 > 1024) return true;      // more than the threads of a block per row
  return p.rows >= 8ll * sms && (op != kRowLn || (p.seqlen >= 8 && p.batch <= 65535));
}

template <int kOp, typename TX, typename TA, int NV, bool kWarp>
int launch_group(const Int8RowParams& p, int threads, int sms, cudaStream_t stream) {
  static bool allowed[64];
  const auto kernel = int8_row_group_kernel<kOp, TX, TA, NV, kWarp>;
  const int smem = kRowVectors<kOp, TA> * p.channels * 4;
  constexpr int kOwnWords = 2 * 32 * 4;   // the kernel's static shared memory, which counts against the 48 KB that need no leave
  if (smem + kOwnWords > 48 * 1024 && !allow_smem(kernel, kRowVectors<kOp, TA> * kMaxEights * 32, allowed)) return DMF_ATTN_ERR_LAUNCH;
  static std::atomic<int> registers{0};
  const int st = registers_of(kernel, registers);
  if (st != DMF_ATTN_OK) return st;
  // one wave: as many blocks as the SMs hold at a time, cut at the samples' ends
  const int64_t samples = kOp == kRowLn ? p.batch : 1, per_sample = kOp == kRowLn ? p.seqlen : p.rows, unit = kWarp ? kRowThreads / 32 : 1;
  const int64_t resident = static_cast<int64_t>(sms) * blocks_per_sm(registers.load(std::memory_order_relaxed), threads, smem);
  const int64_t splits = resident / samples > 1 ? resident / samples : 1;
  const int64_t units = (per_sample + unit - 1) / unit;
  const int rpb = static_cast<int>((units + splits - 1) / splits * unit);
  const dim3 grid(static_cast<unsigned>((per_sample + rpb - 1) / rpb), static_cast<unsigned>(samples));
  return launch_dependent(kernel, grid, threads, smem, 1, stream, p, rpb);
}

template <int kOp, typename TX, typename TA>
int launch_vectors(const Int8RowParams& p, int sms, cudaStream_t stream) {
  const int eights = p.channels / 8, wide = ((eights + 3) / 4 + 31) / 32 * 32;   // threads, four eights each
  const unsigned rows = static_cast<unsigned>(p.rows);
  if (!many_rows(p, kOp, sms)) {
    return launch_dependent(int8_row_block_kernel<kOp, TX, TA, 1>, dim3(rows), (eights + 31) / 32 * 32, 0, 1, stream, p);
  }
  if (eights <= 64) return launch_group<kOp, TX, TA, 2, true>(p, kRowThreads, sms, stream);
  if (eights <= kWarpRowEights) return launch_group<kOp, TX, TA, 5, true>(p, kRowThreads, sms, stream);
  if constexpr (kOp == kRowLn) return launch_group<kOp, TX, TA, 4, false>(p, wide, sms, stream);
  return launch_dependent(int8_row_block_kernel<kOp, TX, TA, 4>, dim3(rows), wide, 0, 1, stream, p);
}

constexpr int kNoKernel = -1;   // of launch_types: a pair of types without a kernel of its own

template <int kOp, typename TX>
int launch_types(const Int8RowParams& p, int sms, cudaStream_t stream) {
  if constexpr (kIsNorm<kOp>) {
    if (p.add != nullptr) {
      constexpr bool kF32 = std::is_same<TX, float>::value;
      if (p.add_dtype == DMF_INT8_F32) return launch_vectors<kOp, TX, float>(p, sms, stream);
      if (p.add_dtype == DMF_INT8_BF16) {
        if constexpr (kF32 || std::is_same<TX, __nv_bfloat16>::value) return launch_vectors<kOp, TX, __nv_bfloat16>(p, sms, stream);
      } else {
        if constexpr (kF32 || std::is_same<TX, __half>::value) return launch_vectors<kOp, TX, __half>(p, sms, stream);
      }
      return kNoKernel;
    }
  }
  return launch_vectors<kOp, TX, void>(p, sms, stream);
}

template <int kOp>
int launch_rows(const Int8RowParams& p, cudaStream_t stream) {
  int sms = 0, st = sm_count_of_current_device(&sms);
  if (st != DMF_ATTN_OK) return st;
  if (p.rows == 0) return DMF_ATTN_OK;
  // (65535: samples are a grid dimension of the kernel that a LayerNorm of more than 8192 channels takes whatever its rows)
  if (reads_vectors(p, kOp) && p.channels / 8 <= kMaxEights && (kOp != kRowLn || p.channels <= 8192 || p.batch <= 65535)) {
    switch (p.x_dtype) {
      case DMF_INT8_BF16: st = launch_types<kOp, __nv_bfloat16>(p, sms, stream); break;
      case DMF_INT8_FP16: st = launch_types<kOp, __half>(p, sms, stream); break;
      default: st = launch_types<kOp, float>(p, sms, stream);
    }
    if (st != kNoKernel) return st;
  }
  auto singles = [&](auto kernel, int warps) {
    return launch_dependent(kernel, dim3(static_cast<unsigned>((p.rows * warps + 7) / 8)), kRowThreads, 0, 1, stream, p);
  };
  if (p.channels <= 512) return singles(int8_row_single_kernel<kOp, 16, 1>, 1);
  if (p.channels <= 1024) return singles(int8_row_single_kernel<kOp, 32, 1>, 1);
  if (p.channels <= 1536) return singles(int8_row_single_kernel<kOp, 24, 2>, 2);
  if (p.channels <= 2048) return singles(int8_row_single_kernel<kOp, 32, 2>, 2);
  if (p.channels <= 4096) return singles(int8_row_single_kernel<kOp, 32, 4>, 4);
  if (p.channels <= 8192) return singles(int8_row_single_kernel<kOp, 32, 8>, 8);
  return launch_dependent(int8_row_any_kernel<kOp>, dim3(static_cast<unsigned>(p.rows)), kRowThreads, 0, 1, stream, p);
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
  p.rows = rows; p.batch = a->batch; p.seqlen = a->seqlen; p.channels = a->channels;
  set_out(&p, a->out);
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  switch (a->act) {
    case DMF_INT8_ACT_GELU: return launch_rows<kRowGelu>(p, stream);
    case DMF_INT8_ACT_SILU: return launch_rows<kRowSilu>(p, stream);
    default: return launch_rows<kRowQuantize>(p, stream);
  }
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
  p.rows = rows; p.batch = a->batch; p.seqlen = a->seqlen; p.channels = a->channels; p.eps = a->eps;
  set_out(&p, a->out);
  return launch_rows<kRowRms>(p, static_cast<cudaStream_t>(a->stream));
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
  p.rows = rows; p.batch = a->batch; p.seqlen = a->seqlen; p.channels = a->channels; p.eps = a->eps;
  set_out(&p, a->out);
  return launch_rows<kRowLn>(p, static_cast<cudaStream_t>(a->stream));
}

int run_dequantize(const dmf_int8_dequantize_args* a) {
  if (a == nullptr) return DMF_ATTN_ERR_NULL;
  if (!known_dtype(a->out_dtype)) return DMF_ATTN_ERR_DTYPE;
  if (a->rows < 0 || a->rows > 0x7fffffff || a->channels < 1 || a->channels > kMaxChannels) return DMF_ATTN_ERR_SHAPE;
  int sms = 0, st = DMF_ATTN_OK;
  if (a->rows > 0) {
    if ((st = check_matrix(a->x, a->channels, false)) != DMF_ATTN_OK) return st;
    if (a->out_stride < a->channels) return DMF_ATTN_ERR_STRIDE;
    if ((st = check_pointer(a->out, element_bytes(a->out_dtype))) != DMF_ATTN_OK) return st;
  }
  if ((st = sm_count_of_current_device(&sms)) != DMF_ATTN_OK) return st;
  if (a->rows == 0) return DMF_ATTN_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  const bool vectors = a->channels % 8 == 0 && reinterpret_cast<uintptr_t>(a->x.values) % 8 == 0 && (a->rows == 1 || a->x.stride % 8 == 0) &&
                       whole_vectors(a->out, a->out_dtype, 0, 1, a->out_stride, a->rows == 1 ? 1 : 2);
  const int per_piece = vectors ? 8 * kDequantizeEights : kDequantizeSingles, pieces = (a->channels + per_piece - 1) / per_piece;
  const int64_t blocks = (a->rows * pieces + kRowThreads / 32 - 1) / (kRowThreads / 32);
  if (blocks > 0x7fffffff) return DMF_ATTN_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(blocks));
  const int8_t* values = a->x.values;
  const float* scale = a->x.scale;
  if (!vectors)
    return launch_dependent(int8_dequantize_any_kernel, grid, kRowThreads, 0, 1, stream, values, a->x.stride, scale, a->out, a->out_stride,
                            a->out_dtype, a->rows, a->channels, pieces);
  auto launch = [&](auto kernel) {
    return launch_dependent(kernel, grid, kRowThreads, 0, 1, stream, values, a->x.stride, scale, a->out, a->out_stride, a->rows,
                            a->channels / 8, pieces);
  };
  switch (a->out_dtype) {
    case DMF_INT8_BF16: return launch(int8_dequantize_kernel<__nv_bfloat16>);
    case DMF_INT8_FP16: return launch(int8_dequantize_kernel<__half>);
    default: return launch(int8_dequantize_kernel<float>);
  }
}

}  // namespace

#define DMF_API extern "C" __attribute__((visibility("default")))
DMF_API int dmf_int8_quantize(const dmf_int8_quantize_args* args) { return run_quantize(args); }
DMF_API int dmf_int8_rmsnorm(const dmf_int8_rmsnorm_args* args) { return run_rmsnorm(args); }
DMF_API int dmf_int8_ln_modulate(const dmf_int8_ln_modulate_args* args) { return run_ln_modulate(args); }
DMF_API int dmf_int8_dequantize(const dmf_int8_dequantize_args* args) { return run_dequantize(args); }
