// MXFP4 quantisation and reading back (sm_100a).
//
// A block is 32 consecutive values of a row sharing one power of two: with a = max |x|,
//   e = max(floor(log2 a) - 2, -127), scale byte e + 127 (E8M0),
//   code = the e2m1 value nearest to x 2^-e (ties to the even code, saturating at +-6),
// two codes a byte, the even column in the low half.  A block that holds an infinity or a NaN
// gets the scale byte 255 (NaN) and codes 0.  x 2^-e is exact (a power of two, and what becomes
// subnormal rounds to code 0 either way), so the one rounding is the conversion's.
//
// Both kernels are bound by HBM: 4 lanes share a block, 8 values a lane, so a warp's loads and
// stores are contiguous; each warp takes kUnits x 8 blocks at a time and issues all its loads
// first.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "exf_common.cuh"
#include "exf_launch.h"
#include "exf_mxfp4.h"

namespace exf {

constexpr int kMxThreads = 256;
constexpr int kUnits = 4;  // 8-block units a warp has in flight

template <typename T>
struct Vec8 {  // 8 values of T as loaded
  static constexpr int kWords = (int)sizeof(T) * 2;
  uint32_t w[kWords];
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, Vec8<T>& v) {
  const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int i = 0; i < Vec8<T>::kWords / 4; ++i) {
    const uint4 a = __ldg(q + i);
    v.w[4 * i] = a.x;
    v.w[4 * i + 1] = a.y;
    v.w[4 * i + 2] = a.z;
    v.w[4 * i + 3] = a.w;
  }
}
__device__ __forceinline__ void unpack8(const Vec8<float>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v.w[i]);
}
__device__ __forceinline__ void unpack8(const Vec8<__nv_bfloat16>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(v.w[i] << 16);
    f[2 * i + 1] = __uint_as_float(v.w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const Vec8<__half>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }

// 8 values -> 8 e2m1 codes, the first in the low half of the low byte
__device__ __forceinline__ uint32_t codes8(const float (&f)[8], float inv) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = f[i] * inv;
  uint32_t out;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(out)
      : "f"(s[0]), "f"(s[1]), "f"(s[2]), "f"(s[3]), "f"(s[4]), "f"(s[5]), "f"(s[6]), "f"(s[7]));
  return out;
}
// 8 codes -> their values (exact in fp16)
__device__ __forceinline__ void values8(uint32_t codes, float (&f)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
// 2^(byte - 127), NaN for 255
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fffffffu : byte == 0u ? 0x00400000u : byte << 23);
}

// FLAT: cols a multiple of 32, rows contiguous, x 16-byte aligned: the matrix is one row of
// rows * cols values.  Otherwise a unit stays in one row, and its 8-value groups are read with
// vector loads where the row pitch keeps them aligned (vec) and they are whole, else one by one.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(kMxThreads)
    mxfp4_quantize_kernel(const T* x, int64_t rows, int64_t cols, int64_t row_stride, bool vec,
                          uint8_t* codes, uint8_t* scales) {
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (cols + 31) / 32;       // of one row
  const int64_t strips = (blocks + 8 * kUnits - 1) / (8 * kUnits);
  const int64_t warps = (int64_t)gridDim.x * (kMxThreads / 32);
  for (int64_t u = (int64_t)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5);
       u < rows * strips; u += warps) {
    const int64_t row = FLAT ? 0 : u / strips;
    const int64_t b0 = (FLAT ? u : u - row * strips) * (8 * kUnits) + (lane >> 2);
    const T* xr = x + row * row_stride;
    Vec8<T> v[kUnits];
    float f[kUnits][8];
    if (FLAT || vec) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int64_t c = (b0 + 8 * i) * 32 + 8 * (lane & 3);
        if (c + 8 <= cols)
          load8(xr + c, v[i]);
        else
#pragma unroll
          for (int j = 0; j < Vec8<T>::kWords; ++j) v[i].w[j] = 0;
      }
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t c = (b0 + 8 * i) * 32 + 8 * (lane & 3);
      if (FLAT || (vec && (c + 8 <= cols || c >= cols))) {
        unpack8(v[i], f[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] = c + j < cols ? to_f(xr[c + j]) : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      uint32_t top = 0;  // magnitudes order like their bits; a NaN ranks above infinity
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[i][j]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int b = (int)(top >> 23) > 2 ? (int)(top >> 23) - 2 : 0;  // scale byte
      const bool bad = top >= 0x7f800000u;
      const float inv = __uint_as_float((uint32_t)(254 - b) << 23);
      const uint32_t q = bad ? 0u : codes8(f[i], inv);
      const int64_t blk = b0 + 8 * i;
      if (blk < blocks) {
        reinterpret_cast<uint32_t*>(codes)[(row * blocks + blk) * 4 + (lane & 3)] = q;
        if ((lane & 3) == 0) scales[row * blocks + blk] = bad ? 255 : (uint8_t)b;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]);
template <>
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
template <>
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ void store8(__half* p, const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store1(__half* p, float v) { *p = __float2half_rn(v); }

// out [rows][cols]; FLAT and vec as above (out 16-byte aligned)
template <typename T, bool FLAT>
__global__ void __launch_bounds__(kMxThreads)
    mxfp4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                            int64_t cols, bool vec, T* out) {
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (cols + 31) / 32;
  const int64_t strips = (blocks + 8 * kUnits - 1) / (8 * kUnits);
  const int64_t warps = (int64_t)gridDim.x * (kMxThreads / 32);
  for (int64_t u = (int64_t)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5);
       u < rows * strips; u += warps) {
    const int64_t row = FLAT ? 0 : u / strips;
    const int64_t b0 = (FLAT ? u : u - row * strips) * (8 * kUnits) + (lane >> 2);
    uint32_t q[kUnits], sb[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t blk = b0 + 8 * i;
      q[i] = blk < blocks ? __ldg(reinterpret_cast<const uint32_t*>(codes) +
                                  (row * blocks + blk) * 4 + (lane & 3))
                          : 0u;
      sb[i] = blk < blocks ? __ldg(scales + row * blocks + blk) : 0u;
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t c = (b0 + 8 * i) * 32 + 8 * (lane & 3);
      float f[8];
      values8(q[i], f);
      const float s = scale_value(sb[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= s;
      T* o = out + row * cols + c;
      if ((FLAT || vec) && c + 8 <= cols) {
        store8<T>(o, f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < cols) store1(o + j, f[j]);
      }
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------
static unsigned mx_grid(const void* kernel, int64_t rows, int64_t cols) {
  const int64_t strips = ((cols + 31) / 32 + 8 * kUnits - 1) / (8 * kUnits);
  const int64_t need = (rows * strips + kMxThreads / 32 - 1) / (kMxThreads / 32);
  const int64_t most = persistent_grid(kernel, kMxThreads, 0);
  return (unsigned)(most > 0 && need > most ? most : need);
}
static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
static cudaError_t quantize_t(const void* xv, int64_t rows, int64_t cols, int64_t stride,
                              uint8_t* codes, uint8_t* scales, cudaStream_t s) {
  const T* x = static_cast<const T*>(xv);
  if (cols % 32 == 0 && (stride == cols || rows == 1) && al16(x)) {
    auto* k = mxfp4_quantize_kernel<T, true>;
    const int64_t n = rows * cols;
    k<<<mx_grid((const void*)k, 1, n), kMxThreads, 0, s>>>(x, 1, n, n, true, codes, scales);
  } else {
    auto* k = mxfp4_quantize_kernel<T, false>;
    const bool vec = al16(x) && (rows == 1 || stride * (int64_t)sizeof(T) % 16 == 0);
    k<<<mx_grid((const void*)k, rows, cols), kMxThreads, 0, s>>>(x, rows, cols, stride, vec, codes,
                                                              scales);
  }
  return cudaGetLastError();
}

template <typename T>
static cudaError_t dequantize_t(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                int64_t cols, void* ov, cudaStream_t s) {
  T* out = static_cast<T*>(ov);
  if (cols % 32 == 0 && al16(out)) {
    auto* k = mxfp4_dequantize_kernel<T, true>;
    const int64_t n = rows * cols;
    k<<<mx_grid((const void*)k, 1, n), kMxThreads, 0, s>>>(codes, scales, 1, n, true, out);
  } else {
    auto* k = mxfp4_dequantize_kernel<T, false>;
    const bool vec = al16(out) && cols * (int64_t)sizeof(T) % 16 == 0;
    k<<<mx_grid((const void*)k, rows, cols), kMxThreads, 0, s>>>(codes, scales, rows, cols, vec,
                                                              out);
  }
  return cudaGetLastError();
}

cudaError_t launch_mxfp4_quantize(const void* x, int dtype, int64_t rows, int64_t cols,
                                  int64_t row_stride, uint8_t* codes, uint8_t* scales,
                                  cudaStream_t s) {
  switch (dtype) {
    case EXF_F32: return quantize_t<float>(x, rows, cols, row_stride, codes, scales, s);
    case EXF_BF16: return quantize_t<__nv_bfloat16>(x, rows, cols, row_stride, codes, scales, s);
    case EXF_F16: return quantize_t<__half>(x, rows, cols, row_stride, codes, scales, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                    int64_t cols, void* out, int dtype, cudaStream_t s) {
  switch (dtype) {
    case EXF_F32: return dequantize_t<float>(codes, scales, rows, cols, out, s);
    case EXF_BF16: return dequantize_t<__nv_bfloat16>(codes, scales, rows, cols, out, s);
    case EXF_F16: return dequantize_t<__half>(codes, scales, rows, cols, out, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace exf
