// MXFP4 (microscaled 4-bit floating point): host entries (internal).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exf {

// x [rows][cols] (EXF_F32 / EXF_BF16 / EXF_F16, rows row_stride elements apart) <-> codes
// [rows][ceil(cols / 32)][16], scales [rows][ceil(cols / 32)].
cudaError_t launch_mxfp4_quantize(const void* x, int dtype, int64_t rows, int64_t cols,
                                  int64_t row_stride, uint8_t* codes, uint8_t* scales,
                                  cudaStream_t s);
cudaError_t launch_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                    int64_t cols, void* out, int dtype, cudaStream_t s);

}  // namespace exf
