// C ABI of inference in 8-bit integers (include/dmf_int8.h), the product: validation, choice of kernel and launches.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>

#include "attn_launch.h"
#include "dmf_attn.h"
#include "dmf_int8.h"
#include "int8_gemm_few.cuh"
#include "int8_gemm_pair.cuh"
#include "int8_launch.h"
#include "int8_linear.cuh"
#include "tensor_map.h"

namespace {

using namespace dmf;

constexpr int kMaxK = 131071;  // 128 * 128 * K stays below 2^31
constexpr int kMaxN = 1 << 30;  // the columns of a last tile stay in int

// ---- the product on the tensor cores ----

// rows that TMA can read: base and pitch in whole 16-byte units, rows that do not overlap
bool tma_can_read(const dmf_int8_matrix& t, int rows, int k) {
  return reinterpret_cast<uintptr_t>(t.values) % 16 == 0 && (rows == 1 || (t.stride % 16 == 0 && t.stride >= k));
}

// map of `rows` rows of k bytes, boxes of 128 bytes x box_rows; what a box has beyond the matrix reads as zeros
int make_map8(CUtensorMap* map, const dmf_int8_matrix& t, int rows, int k, int box_rows) {
  const EncodeTiledFn encode = get_encode_fn();
  if (encode == nullptr) return DMF_ATTN_ERR_DEVICE;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {rows == 1 ? (static_cast<cuuint64_t>(k) + 15) / 16 * 16 : static_cast<cuuint64_t>(t.stride)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
  const CUresult r = encode_in_context([&] {
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, t.values, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
  return r == CUDA_SUCCESS ? DMF_ATTN_OK : DMF_ATTN_ERR_TENSOR_MAP;
}

// map of the result for TMA stores of 128 bytes x 32 rows
int make_out_map(CUtensorMap* map, const dmf_int8_linear_args* a) {
  const EncodeTiledFn encode = get_encode_fn();
  if (encode == nullptr) return DMF_ATTN_ERR_DEVICE;
  const int bytes = element_bytes(a->out_dtype);
  const CUtensorMapDataType dt = a->out_dtype == DMF_INT8_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                 : a->out_dtype == DMF_INT8_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a->n), static_cast<cuuint64_t>(a->m)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a->out_stride) * bytes};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / bytes), 32}, steps[2] = {1, 1};
  const CUresult r = encode_in_context([&] {
    return encode(map, dt, 2, a->out, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
  return r == CUDA_SUCCESS ? DMF_ATTN_OK : DMF_ATTN_ERR_TENSOR_MAP;
}

template <int BN, typename T>
int launch_pair_gemm(const Int8GemmParams& p, int sms, cudaStream_t stream) {
  static bool allowed[64];
  const auto kernel = int8_gemm_pair_kernel<BN, T>;
  if (!allow_smem(kernel, Int8PairTraits<BN>::kSmemBytes, allowed)) return DMF_ATTN_ERR_LAUNCH;
  const int tiles = p.tiles_m * (p.tiles_n + p.narrow), clusters = tiles < sms / 2 ? tiles : sms / 2;
  return launch_dependent(kernel, dim3(2u * clusters), Int8PairTraits<BN>::kThreads, Int8PairTraits<BN>::kSmemBytes, 2, stream, p);
}

template <int TB, typename T>
int launch_few_gemm(const Int8GemmParams& p, int splits, cudaStream_t stream) {
  static bool allowed[64];
  const auto kernel = int8_gemm_few_kernel<TB, T>;
  if (!allow_smem(kernel, Int8FewTraits<TB>::kSmemBytes, allowed)) return DMF_ATTN_ERR_LAUNCH;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(p.tiles_m * p.tiles_n * splits)), kInt8FewThreads, Int8FewTraits<TB>::kSmemBytes,
                        splits, stream, p, splits);
}

// Whether the columns of a product on CTA pairs end in tiles of half the width.
bool narrow_end(int n, int bn) { return bn == 256 && n % 256 != 0 && n % 256 <= 128; }

// How a product is cut up: on CTA pairs with tiles of 256 x bn, or (few) tiles of tb tokens x 128 channels, k over `splits` CTAs.
struct GemmPlan {
  bool few;
  int tile;    // bn or tb
  int splits;
};

// The cut with the shortest time by a model of it in microseconds, fitted to measurements of all of them at 38 shapes of 1 to
// 16384 rows (K 128 to 8192, N 100 to 8192), where its choice is 1 % above the best on average and 11 % at most.  A step of k costs
// what its loads take: their latency over the stages in flight for a CTA alone, the 100 to 115 GB/s that the L2 gives an SM for
// several; the rest is start and end of a tile, and the exchange of the sums of a split k, as it is with the bank conflicts of its layout
// (int8_gemm_few.cuh).  Measured in bursts, short of the power limit, at the turning points:
// 512 x 1152 x 3456 pairs of 128 6.6 us, of 256 7.7, few rows of 64 9.7; 16384 x 1152 x 3456 pairs of 256 51, of 192 56, of 128 66;
// 1024 x 1152 x 1152 few rows of 64 5.7, pairs of 128 6.1; 16 x 4608 x 1152 few rows of 16 in one piece 10.0, in eight 4.6.
//   pair: rounds of tiles over the SM pairs, each c(bn) + steps * t(bn); a last round that is partly empty runs faster, so the
//         rounds are halfway between the whole and the fractional number
//   few:  n tiles per SM, two at a time, each e(tb) and its steps; splits only where every CTA has an SM of its own, for 1.1 + 0.0007
//         per CTA and column sent
GemmPlan plan_gemm(int m, int n, int k, int sms) {
  const double steps = (k + 127) / 128;
  auto tiles = [&](int tm, int tn) { return static_cast<double>((static_cast<int64_t>(m) + tm - 1) / tm) * static_cast<double>((static_cast<int64_t>(n) + tn - 1) / tn); };
  GemmPlan best = {false, 256, 1};
  double least = 1e30;
  auto consider = [&](bool few, int tile, int splits, double us) {
    if (us < least) {
      least = us;
      best = {few, tile, splits};
    }
  };
  struct { int bn; double c, t; } pairs[] = {{128, 0.35, 0.256}, {192, 0.77, 0.279}, {256, 0.95, 0.33}};
  for (const auto& g : pairs) {
    const double rounds = (tiles(256, g.bn) - (narrow_end(n, g.bn) ? 0.4 * tiles(256, n) : 0.0)) / (sms / 2);
    consider(false, g.bn, 1, 3.4 + (std::fmax(rounds, 1.0) + std::ceil(rounds)) / 2 * (g.c + steps * g.t));
  }
  struct { int tb; double e; } fews[] = {{16, 0.1}, {32, 0.25}, {64, 0.9}};
  for (const auto& g : fews)
    for (int s = 1; s <= 8 && s <= steps; s *= 2) {
      const double count = tiles(g.tb, 128) * s, n = std::ceil(count / sms), waves = std::ceil(n / 2), own = std::ceil(steps / s);
      if (s > 1 && count > sms) break;
      consider(true, g.tb, s, 2.3 + n * g.e + std::fmax(waves * own * 0.213, n * own * (128 + g.tb) * 128 / 115e3) + 2.0 * (waves - 1) +
                                  (s > 1 ? 1.1 + 0.0007 * count * g.tb * (s - 1) / s : 0.0));
    }
  return best;
}

template <typename T>
int launch_gemm(const GemmPlan& g, const Int8GemmParams& p, int sms, cudaStream_t stream) {
  if (g.few) {
    switch (g.tile) {
      case 16: return launch_few_gemm<16, T>(p, g.splits, stream);
      case 32: return launch_few_gemm<32, T>(p, g.splits, stream);
      default: return launch_few_gemm<64, T>(p, g.splits, stream);
    }
  }
  switch (g.tile) {
    case 128: return launch_pair_gemm<128, T>(p, sms, stream);
    case 192: return launch_pair_gemm<192, T>(p, sms, stream);
    default: return launch_pair_gemm<256, T>(p, sms, stream);
  }
}

int run_plan(const GemmPlan& g, const dmf_int8_linear_args* a, int sms) {
  Int8GemmParams p;
  std::memset(&p, 0, sizeof(p));
  int st = make_map8(&p.x_map, a->x, a->m, a->k, g.few ? g.tile : 128);
  if (st != DMF_ATTN_OK) return st;
  if ((st = make_map8(&p.w_map, a->w, a->n, a->k, g.few ? 128 : g.tile / 2)) != DMF_ATTN_OK) return st;
  p.x_scale = a->x.scale; p.w_scale = a->w.scale;
  p.bias = a->bias; p.bias_dtype = a->bias_dtype;
  p.out = a->out; p.out_stride = a->out_stride; p.out_dtype = a->out_dtype;
  p.out_vec = reinterpret_cast<uintptr_t>(a->out) % 16 == 0 && a->out_stride * element_bytes(a->out_dtype) % 16 == 0;
  if (p.out_vec && !g.few && (st = make_out_map(&p.out_map, a)) != DMF_ATTN_OK) return st;
  p.status_word = a->status_word;
  p.m = a->m; p.n = a->n; p.k = a->k;
  const int64_t tiles_m = (static_cast<int64_t>(a->m) + (g.few ? g.tile : 256) - 1) / (g.few ? g.tile : 256);
  const int64_t tiles_n = (static_cast<int64_t>(a->n) + (g.few ? 128 : g.tile) - 1) / (g.few ? 128 : g.tile);
  if (tiles_m * tiles_n * g.splits > 0x7fffffff) return DMF_ATTN_ERR_SHAPE;
  p.narrow = !g.few && narrow_end(a->n, g.tile);
  if (p.narrow && (st = make_map8(&p.w_half_map, a->w, a->n, a->k, 64)) != DMF_ATTN_OK) return st;
  p.tiles_m = static_cast<int>(tiles_m);
  p.tiles_n = static_cast<int>(tiles_n) - p.narrow;
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  switch (a->out_dtype) {
    case DMF_INT8_BF16: return launch_gemm<__nv_bfloat16>(g, p, sms, stream);
    case DMF_INT8_FP16: return launch_gemm<__half>(g, p, sms, stream);
    default: return launch_gemm<float>(g, p, sms, stream);
  }
}

int run_gemm(const dmf_int8_linear_args* a, int sms) { return run_plan(plan_gemm(a->m, a->n, a->k, sms), a, sms); }

// ---- the product of rows that TMA cannot read ----

int run_linear_any(const dmf_int8_linear_args* a) {
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
    const int st = launch_dependent(int8_linear_any_kernel, grid, 256, 0, 1, stream, p);
    if (st != DMF_ATTN_OK) return st;
  }
  return DMF_ATTN_OK;
}

int run_linear(const dmf_int8_linear_args* a) {
  if (a == nullptr) return DMF_ATTN_ERR_NULL;
  if (!known_dtype(a->out_dtype) || (a->bias != nullptr && !known_dtype(a->bias_dtype))) return DMF_ATTN_ERR_DTYPE;
  if (a->m < 0 || a->n < 1 || a->n > kMaxN || a->k < 1 || a->k > kMaxK) return DMF_ATTN_ERR_SHAPE;
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
  return tma_can_read(a->x, a->m, a->k) && tma_can_read(a->w, a->n, a->k) ? run_gemm(a, sms) : run_linear_any(a);
}

int linear_kernel_name(int m, int n, int k, char* buf, size_t len) {
  if (buf == nullptr || len == 0) return DMF_ATTN_ERR_NULL;
  if (m < 1 || n < 1 || n > kMaxN || k < 1 || k > kMaxK) return DMF_ATTN_ERR_SHAPE;
  int sms = 0;
  if (sm_count_of_current_device(&sms) != DMF_ATTN_OK) sms = 148;
  const GemmPlan g = plan_gemm(m, n, k, sms);
  if (!g.few) std::snprintf(buf, len, "int8_gemm_pair_kernel<%d>%s", g.tile, narrow_end(n, g.tile) ? ", narrow end" : "");
  else if (g.splits == 1) std::snprintf(buf, len, "int8_gemm_few_kernel<%d>", g.tile);
  else std::snprintf(buf, len, "int8_gemm_few_kernel<%d>, k over %d CTAs", g.tile, g.splits);
  return DMF_ATTN_OK;
}

}  // namespace

#define DMF_API extern "C" __attribute__((visibility("default")))
DMF_API int dmf_int8_linear(const dmf_int8_linear_args* args) { return run_linear(args); }
DMF_API int dmf_int8_linear_kernel_name(int32_t m, int32_t n, int32_t k, char* buf, size_t len) {
  return linear_kernel_name(m, n, k, buf, len);
}
