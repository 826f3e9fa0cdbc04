// A projection with low-rank adapters: parameter block and host entries (internal).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exf {

struct AdapterArgs {
  const void* x;          // [tokens][inner]
  const void* w;          // [outer][inner]
  const void* a;          // [adapters][rank][inner]
  const void* b;          // [adapters][outer][rank]
  const int32_t* ids;     // [tokens], none outside [0, adapters)
  const float* scaling;   // [adapters] or null: 1
  bool bf16;              // else fp16
  int64_t tokens;
  int inner, outer, adapters, rank;
  void* y;                // [tokens][outer]
  int32_t* status;
};

int64_t adapters_workspace(int64_t tokens, int rank);
cudaError_t launch_adapters(const AdapterArgs& a, void* workspace, cudaStream_t s);

}  // namespace exf
