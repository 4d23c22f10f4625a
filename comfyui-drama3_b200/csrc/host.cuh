// Host helpers of the C ABI shared by the library's translation units: status codes, device properties, launches with
// programmatic dependent launch, the tensor-map encoder.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

#include <cudaTypedefs.h>

#include "../../include/drama3_b200.h"

namespace d3host {

inline thread_local int g_last_cuda = 0;

inline int cuda_status(cudaError_t e) {
  if (e == cudaSuccess) return D3_OK;
  g_last_cuda = (int)e;
  return D3_ERR_CUDA;
}

inline int launch_status() { return cuda_status(cudaGetLastError()); }

inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

constexpr int kMaxDevices = 64;

struct DeviceInfo {
  int sms = 0;
  int smem_optin = 0;
  int cc = 0;
};

inline std::mutex g_mu;
inline DeviceInfo g_dev[kMaxDevices];

inline int device_info(DeviceInfo* out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return D3_ERR_DEVICE;
  std::lock_guard<std::mutex> lock(g_mu);
  DeviceInfo& d = g_dev[dev];
  if (d.sms == 0) {
    int major = 0, minor = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
    cudaDeviceGetAttribute(&d.smem_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    d.cc = major * 10 + minor;
  }
  *out = d;
  if (d.cc != 100) return D3_ERR_DEVICE;
  return D3_OK;
}

// Raise a kernel's dynamic shared-memory ceiling (once per device and kernel).
template <class K>
int allow_smem(K kernel, int bytes) {
  if (bytes <= 48 * 1024) return D3_OK;
  return cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

// The same, asked for once per device: `done` has a bit for each device on which it was.
template <class K>
int allow_smem_once(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (int st = cuda_status(cudaGetDevice(&dev))) return st;
  const uint64_t bit = 1ull << (dev & 63);  // kMaxDevices
  if (done.load(std::memory_order_relaxed) & bit) return D3_OK;
  if (int st = allow_smem(kernel, bytes)) return st;
  done.fetch_or(bit, std::memory_order_relaxed);
  return D3_OK;
}

template <class K, class... Args>
int launch(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  if (pdl) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args...));
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link against libcuda).
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
  });
  return fn;
}

// A tiled tensor map of `rank` dimensions (strides: of all but the first), elements next to one another, not interleaved,
// zeros outside. Encoding wants a current context, which a thread has only once it has made a runtime call that needs
// one; where there is none yet, the current device's is made current and the map encoded again.
inline bool encode_tiled(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                         const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
  auto encode = [&] {
    return fn(map, type, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  int dev = 0;
  return encode() || (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess && encode());
}

}  // namespace d3host
