// Tensor maps for TMA: the driver's encoder, found at run time (no link-time libcuda dependency).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

namespace dmf {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode_fn() {
  static std::atomic<EncodeTiledFn> cached{nullptr};
  EncodeTiledFn fn = cached.load(std::memory_order_acquire);
  if (fn != nullptr) return fn;
  void* sym = nullptr;
  cudaDriverEntryPointQueryResult qres;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) != cudaSuccess ||
      qres != cudaDriverEntryPointSuccess || sym == nullptr) {
    (void)cudaGetLastError();
    return nullptr;
  }
  fn = reinterpret_cast<EncodeTiledFn>(sym);
  cached.store(fn, std::memory_order_release);
  return fn;
}

// The encoder is a driver call: it needs the device's context current to this thread, and on a thread without a runtime call
// so far (an autograd worker whose memory all comes from a cache) nothing has bound it yet; cudaSetDevice does.
template <typename Encode>
inline CUresult encode_in_context(Encode&& encode) {
  CUresult r = encode();
  if (r != CUDA_SUCCESS) {
    int dev = -1;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
    (void)cudaGetLastError();
  }
  return r;
}

}  // namespace dmf
