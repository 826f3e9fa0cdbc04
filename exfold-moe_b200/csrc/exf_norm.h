// Root-mean-square norm: parameter block and host entries (internal).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exf {

struct NormArgs {
  const void* x;         // [rows][cols], rows x_stride elements apart
  int64_t x_stride;
  const void* residual;  // the same, or null
  int64_t r_stride;
  const void* weight;    // [cols], fp32 or of x's type
  int dtype;             // EXF_F32 / EXF_BF16 / EXF_F16
  bool weight_f32;
  int64_t rows;
  int cols;
  float eps;
  void* sum;             // [rows][cols]: x + residual rounded (null without a residual)
};

cudaError_t launch_rms_norm(const NormArgs& a, void* y, cudaStream_t s);

// codes e4m3 (or int8) [rows][cols], scales fp32 [rows][ceil(cols / group)]
cudaError_t launch_rms_norm_8bit(const NormArgs& a, bool int8, int group, uint8_t* codes,
                                 float* scales, cudaStream_t s);
cudaError_t launch_dequantize_8bit(const uint8_t* codes, bool int8, const float* scales,
                                   int64_t rows, int cols, int group, void* out, int dtype,
                                   cudaStream_t s);

// dy, ds (or null) [rows][cols]; x: the normed rows (a.residual and a.sum unused); dx [rows][cols] or
// null, dw [cols] of the weight's type or null
int64_t norm_backward_workspace(int64_t rows, int cols);
cudaError_t launch_rms_norm_backward(const NormArgs& a, const void* dy, const void* ds, void* dx,
                                     void* dw, void* workspace, cudaStream_t s);

}  // namespace exf
