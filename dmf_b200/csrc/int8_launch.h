// What the host code of the 8-bit entry points (include/dmf_int8.h) shares: the device's properties and checks of arguments.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "dmf_attn.h"
#include "dmf_int8.h"

namespace dmf {

inline int sm_count_of_current_device(int* sm_count) {
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

inline int element_bytes(int dtype) { return dtype == DMF_INT8_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == DMF_INT8_BF16 || dtype == DMF_INT8_FP16 || dtype == DMF_INT8_F32; }

inline int check_pointer(const void* p, int bytes) {
  if (p == nullptr) return DMF_ATTN_ERR_NULL;
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 ? DMF_ATTN_OK : DMF_ATTN_ERR_ALIGN;
}

// `written`: rows that are written must not overlap
inline int check_matrix(const dmf_int8_matrix& t, int columns, bool written) {
  if (t.values == nullptr) return DMF_ATTN_ERR_NULL;
  if (t.stride < (written ? columns : 0)) return DMF_ATTN_ERR_STRIDE;
  return check_pointer(t.scale, 4);
}

// Launches a kernel that begins with grid_dependency_wait, so that its blocks may be set up while the grid before it ends.
template <typename Kernel, typename... Args>
inline int launch_dependent(Kernel kernel, dim3 grid, unsigned threads, int smem, int cluster, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    (void)cudaGetLastError();
    return DMF_ATTN_ERR_LAUNCH;
  }
  return DMF_ATTN_OK;
}

}  // namespace dmf
