// Balance loss of a router: parameter block and host entries (internal).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exf {

struct BalanceArgs {
  const void* logits;  // [groups][tokens][experts], EXF_F32 / EXF_BF16 / EXF_F16
  int dtype;
  const uint8_t* mask;  // [groups][tokens], 0: left out; or null
  int groups;
  int64_t tokens;
  int experts;
  int top_k;
  bool sigmoid;
};

int64_t balance_workspace(int groups, int64_t tokens, int experts);
// loss [groups], counts [groups][experts], valid [groups]
cudaError_t launch_balance_loss(const BalanceArgs& a, const void* ids, bool ids64, void* workspace,
                                float* loss, int32_t* counts, int32_t* valid, cudaStream_t s);
cudaError_t launch_balance_loss_backward(const BalanceArgs& a, const float* dloss,
                                         const int32_t* counts, const int32_t* valid, void* dlogits,
                                         cudaStream_t s);

}  // namespace exf
