// Host-side launch helpers shared by the kernel files and the C ABI layer.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

namespace exf {

// Blocks that fill every SM of the current device at the kernel's occupancy (cached per
// device and kernel); 0 if the query fails.
int persistent_grid(const void* kernel, int threads, size_t dynamic_smem);
int sm_count();

// Raises a kernel's shared-memory limit once per device.
template <typename K>
static cudaError_t allow_smem(K* kern, size_t bytes, std::mutex& mu, bool (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  done[dev] = e == cudaSuccess;
  return e;
}

// Launch as a programmatic dependent of the previous kernel in the stream (the kernel calls
// griddepcontrol.wait before reading anything that kernel wrote).
template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                              cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace exf
