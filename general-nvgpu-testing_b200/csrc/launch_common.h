// What the launchers of feedforward_launch.cu and mxfp4_launch.cu share: kernel set-up per device and dependent launches.
#pragma once

#include <cstdint>
#include <mutex>

#include "host_common.h"

namespace beam {

inline int ceil_div(int a, int b) { return a / b + (a % b != 0); }

// Whether two tensors share any byte (a null one shares none).
inline bool overlap(const void* p, size_t pb, const void* q, size_t qb) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return p && q && a < b + qb && b < a + pb;
}

// How many clusters of `ctas` CTAs of `kernel` the device holds at once, one CTA per SM; the first call
// on a device opts in to the large shared memory and asks.  `known` is the launcher's own table for this kernel.
struct ResidentTable {
  std::mutex mutex;
  int count[64] = {};
};

template <typename Kernel>
int resident_grid(ResidentTable* known, Kernel kernel, DeviceCtx* ctx, int threads, int smem_bytes, int ctas, int* out) {
  std::lock_guard<std::mutex> lock(known->mutex);
  int& n = known->count[ctx->device];
  if (n == 0) {
    if (smem_bytes > ctx->max_smem_optin) return BEAM_ERR_UNSUPPORTED;
    BEAM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes),
                  "cudaFuncSetAttribute(smem)");
    int fit = ctx->sm_count / ctas;
    if (ctas > 1) {
      cudaLaunchConfig_t probe = {};
      probe.gridDim = dim3(static_cast<unsigned>(ctx->sm_count / ctas * ctas), 1, 1);
      probe.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
      probe.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      probe.attrs = attr;
      probe.numAttrs = 1;
      int clusters = 0;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, kernel, &probe);
      if (e == cudaSuccess && clusters > 0 && clusters < fit) fit = clusters;
      (void)cudaGetLastError();
    }
    n = fit > 0 ? fit : 1;
  }
  *out = n;
  return BEAM_OK;
}

// A launch in clusters of `ctas`, a programmatic dependent of the kernel before it on the stream: its set-up overlaps that
// kernel's tail, and it waits for that kernel's completion before its first global access.
template <typename... Params, typename... Args>
int launch_dependent(void (*kernel)(Params...), int grid, int threads, int smem_bytes, int ctas, cudaStream_t stream,
                     const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  BEAM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...), what);
  return BEAM_OK;
}

}  // namespace beam
