// What the host sides of the GEMM files share: the tensor-map encoder and per-device state.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <mutex>

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

}  // namespace smoe
