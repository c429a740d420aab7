// What the host sides of the GEMM files share: the tensor-map encoder and per-device state.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <utility>

namespace smoe {

inline PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
inline std::once_flag g_encode_once;

// The encoder wants a current context, which a thread that has launched nothing yet (autograd's, whose first call is a product) lacks
inline void bind_context() {
  static thread_local int bound = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev != bound && cudaSetDevice(dev) == cudaSuccess) bound = dev;
}

inline bool load_encode() {
  bind_context();
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &qres) ==
            cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  return g_encode != nullptr;
}

// Per-device state: the SM count and the "large dynamic shared memory" function attribute belong to a device,
// not to the process, so both are kept per device ordinal.
constexpr int kMaxDevices = 64;
inline int g_sm_count[kMaxDevices] = {};

inline int current_device() {
  int dev = 0;
  cudaGetDevice(&dev);
  return (dev >= 0 && dev < kMaxDevices) ? dev : 0;
}

inline int sm_count() {
  const int dev = current_device();
  if (g_sm_count[dev] == 0) cudaDeviceGetAttribute(&g_sm_count[dev], cudaDevAttrMultiProcessorCount, dev);
  return g_sm_count[dev];
}

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) once per (kernel instantiation, device)
template <typename Kern>
inline bool ensure_smem_attr(Kern kern, int bytes, bool (&done)[kMaxDevices]) {
  const int dev = current_device();
  if (done[dev]) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done[dev] = true;
  return true;
}

// A launch that may be made ready while the kernel before it in the stream ends; the kernel waits for that one's end (and so for
// everything before it) before it touches memory.  cluster: CTAs of a cluster, 0 where the kernel names them itself or has none.
template <typename... P, typename... A>
inline cudaError_t launch_early(void (*kern)(P...), unsigned blocks, unsigned threads, size_t smem, unsigned cluster, cudaStream_t stream,
                                A&&... args) {
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  const cudaError_t rc = cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
  return rc == cudaSuccess ? cudaGetLastError() : rc;
}

}  // namespace smoe
