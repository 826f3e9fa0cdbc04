// Gated feed-forward block: parameter block and host entries (internal).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exf {

enum GatedActivation { kSilu = 0, kGeluTanh = 1 };

struct GatedArgs {
  const void* x;     // [tokens][hidden]
  const void* w13;   // [2 * inter][hidden]: gate rows, then up rows
  bool bf16;         // operand and result type: bf16, else fp16
  int64_t tokens;
  int hidden;
  int inter;
  int activation;
  int32_t* status;   // set to 1 if a pipeline wait timed out (may be null)
};

// h [tokens][inter]; pre fp32 [tokens][2 * inter] or null: gate and up projections for backward
int64_t gated_forward_workspace(int64_t tokens, int hidden, int inter);
cudaError_t launch_gated_forward(const GatedArgs& a, void* h, float* pre, void* workspace,
                                 cudaStream_t s);
// dx [tokens][hidden] or null, dw13 [2 * inter][hidden] or null
int64_t gated_backward_workspace(int64_t tokens, int hidden, int inter);
cudaError_t launch_gated_backward(const GatedArgs& a, const void* dh, const float* pre,
                                  void* workspace, void* dx, void* dw13, cudaStream_t s);

}  // namespace exf
