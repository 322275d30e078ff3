// host_util.cuh -- what the entry points of every translation unit share on the
// host: the driver's tensor-map encoder, checks and launches.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "canvas_attn.h"

namespace ca {

constexpr int kMaxDevices = 64;
constexpr int kSms = 148;

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A launch that may overlap the end of the kernel before it (dependency_wait),
// in clusters of `cluster` CTAs along x.
template <class... P, class... A>
int launch_cluster_after(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster,
                         cudaStream_t st, A... args) {
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return CA_ERR_CUDA;
  }
  return CA_OK;
}

template <class... P, class... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                 A... args) {
  return launch_cluster_after(kernel, grid, threads, smem, 1, st, args...);
}

// Every translation unit with waits has a device-wide error word of its own
// (sm100.cuh). Reads and clears that of layer.cu on the current device:
// ca_device_status asks it too.
int layer_device_error();

}  // namespace ca
