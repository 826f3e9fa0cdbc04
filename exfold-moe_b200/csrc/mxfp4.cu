// MXFP4 quantisation and reading back (sm_100a).
//
// A block is 32 consecutive values of a row sharing one power of two: with a = max |x|,
//   e = max(floor(log2 a) - 2, -127), scale byte e + 127 (E8M0),
//   code = the e2m1 value nearest to x 2^-e (ties to the even code, saturating at +-6),
// two codes a byte, the even column in the low half.  A block that holds an infinity or a NaN
// gets the scale byte 255 (NaN) and codes 0.  x 2^-e is exact (a power of two, and what becomes
// subnormal rounds to code 0 either way), so the one rounding is the conversion's.
//
// Both kernels are bound by HBM.  Quantising, 4 lanes share a block, 8 values a lane, so a warp's
// loads and stores are contiguous; each warp takes kUnits x 8 blocks at a time and issues all its
// loads first.  Reading back, a lane writes 16 values in whole 32-byte sectors.  Rows that no
// 16-byte vector divides are read through aligned vectors shifted into place, and written in the
// pieces that share aligned places of the result.  403 M bf16 values (196608 x 2048): 155 us to quantise,
// 185 to read back (6.6 and 5.5 TB/s; four fifths of the latter's bytes are writes, and a fill alone
// runs at 3.9); with 2044 columns 309 and 283, bound by the shifting and the row arithmetic.
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

// One vector, element by element, of what lies in [lo, hi); the rest zero.
template <typename T>
__device__ __noinline__ uint4 load_edge(const char* a, const T* lo, const T* hi) {
  uint32_t e[4] = {0, 0, 0, 0};
  constexpr int kPer = 16 / (int)sizeof(T);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const T* t = reinterpret_cast<const T*>(a) + j;
    if (t < lo || t >= hi) continue;
    if (sizeof(T) == 4)
      e[j] = *reinterpret_cast<const uint32_t*>(t);
    else
      e[j / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(t) << (16 * (j & 1));
  }
  return make_uint4(e[0], e[1], e[2], e[3]);
}

// The 8 (n < 8: the first n) values at p, which need not be aligned to 16 bytes, the rest zero:
// aligned vectors shifted into place.  [lo, hi) is the memory that may be read; the vectors at its
// ends are read element by element.
template <typename T>
__device__ __forceinline__ void load8_any(const T* p, int n, const T* lo, const T* hi, Vec8<T>& v) {
  constexpr int W = Vec8<T>::kWords;
  const uint32_t sh = reinterpret_cast<uintptr_t>(p) & 15u;
  const char* at = reinterpret_cast<const char*>(p) - sh;
  uint32_t w[W + 4];
  if (p - lo >= 8 && hi - p >= 16) {
#pragma unroll
    for (int k = 0; k < W / 4 + 1; ++k) {
      uint4 q = make_uint4(0, 0, 0, 0);
      if (k < W / 4 || sh) q = __ldg(reinterpret_cast<const uint4*>(at) + k);
      w[4 * k] = q.x;
      w[4 * k + 1] = q.y;
      w[4 * k + 2] = q.z;
      w[4 * k + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < W / 4 + 1; ++k) {
      uint4 q = make_uint4(0, 0, 0, 0);
      if (16 * k < (int)sh + n * (int)sizeof(T)) q = load_edge(at + 16 * k, lo, hi);
      w[4 * k] = q.x;
      w[4 * k + 1] = q.y;
      w[4 * k + 2] = q.z;
      w[4 * k + 3] = q.w;
    }
  }
  if (sh) {
#pragma unroll
    for (int d = 1; d <= 2; d *= 2)  // whole words: 1, then 2
      if ((sh >> 2) & d) {
#pragma unroll
        for (int i = 0; i + d < W + 4; ++i) w[i] = w[i + d];
      }
    if (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (sh & 2u) * 8);
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) v.w[i] = w[i];
  if (n < 8) {  // the values past the n-th
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (sizeof(T) == 4) {
        if (i >= n) v.w[i] = 0;
      } else if (2 * i + 1 >= n) {
        v.w[i] = 2 * i >= n ? 0u : v.w[i] & 0xffffu;
      }
    }
  }
}

// FLAT: cols a multiple of 32, rows contiguous, x 16-byte aligned: the matrix is one run of rows *
// cols values.  Otherwise every 4 lanes find the row of their block.  I: the type of a block's number
// (a 64-bit division costs several times a 32-bit one).
template <typename T, bool FLAT, typename I>
__global__ void __launch_bounds__(kMxThreads)
    mxfp4_quantize_kernel(const T* x, int64_t rows, int64_t cols, int64_t row_stride,
                          uint8_t* codes, uint8_t* scales) {
  const int lane = threadIdx.x & 31;
  const I blocks = (I)((cols + 31) / 32);        // of one row
  const int64_t total = rows * (int64_t)blocks;
  const int64_t strips = (total + 8 * kUnits - 1) / (8 * kUnits);
  const int64_t warps = (int64_t)gridDim.x * (kMxThreads / 32);
  const T* hi = x + (rows - 1) * row_stride + cols;
  for (int64_t u = (int64_t)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); u < strips;
       u += warps) {
    const int64_t q0 = u * (8 * kUnits) + (lane >> 2);
    Vec8<T> v[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t q = q0 + 8 * i;
      if (FLAT) {
        if (q < total)
          load8(x + q * 32 + 8 * (lane & 3), v[i]);
        else
#pragma unroll
          for (int j = 0; j < Vec8<T>::kWords; ++j) v[i].w[j] = 0;
      } else {
        const I row = (I)q / blocks;
        const int64_t c = (int64_t)((I)q - row * blocks) * 32 + 8 * (lane & 3);
        if (q < total && c < cols) {
          load8_any(x + (int64_t)row * row_stride + c, cols - c < 8 ? (int)(cols - c) : 8, x, hi,
                    v[i]);
        } else {
#pragma unroll
          for (int j = 0; j < Vec8<T>::kWords; ++j) v[i].w[j] = 0;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      float f[8];
      unpack8(v[i], f);
      uint32_t top = 0;  // magnitudes order like their bits; a NaN ranks above infinity
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int b = (int)(top >> 23) > 2 ? (int)(top >> 23) - 2 : 0;  // scale byte
      const bool bad = top >= 0x7f800000u;
      const float inv = __uint_as_float((uint32_t)(254 - b) << 23);
      const uint32_t code = bad ? 0u : codes8(f, bad ? 0.0f : inv);
      const int64_t q = q0 + 8 * i;
      if (q < total) {
        reinterpret_cast<uint32_t*>(codes)[q * 4 + (lane & 3)] = code;
        if ((lane & 3) == 0) scales[q] = bad ? 255 : (uint8_t)b;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[8], bool wide) {
  if (wide) {  // a 32-byte sector
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
// 16 values at p, 16-byte aligned (32-byte if wide)
__device__ __forceinline__ void store16(float* p, const float (&f)[16], bool wide) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(f[8 * h + j]);
    store_words(p + 8 * h, w, wide);
  }
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const float (&f)[16], bool wide) {
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = pack2<T>(f[2 * j], f[2 * j + 1]);
  store_words(p, w, wide);
}
// 8 values at p, 16-byte aligned; fewer one by one
__device__ __forceinline__ void store8(float* p, const float (&f)[8], int n) {
  if (n == 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) p[j] = f[j];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8], int n) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
  if (n == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < n) reinterpret_cast<uint16_t*>(p)[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
}

// cols a multiple of 32: 16 values, half a block, a thread and step; out [halves][16]
template <typename T>
__global__ void __launch_bounds__(kMxThreads)
    mxfp4_dequantize_flat_kernel(const uint2* __restrict__ codes,
                                 const uint8_t* __restrict__ scales, int64_t halves, bool wide,
                                 T* out) {
  const int64_t stride = (int64_t)gridDim.x * kMxThreads;
  for (int64_t g0 = (int64_t)blockIdx.x * kMxThreads + threadIdx.x; g0 < halves;
       g0 += kUnits * stride) {
    uint2 q[kUnits];
    uint32_t sb[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t g = g0 + i * stride;
      if (g >= halves) continue;
      q[i] = __ldg(codes + g);
      sb[i] = __ldg(scales + (g >> 1));
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t g = g0 + i * stride;
      if (g >= halves) continue;
      float a[8], b[8], f[16];
      values8(q[i].x, a);
      values8(q[i].y, b);
      const float s = scale_value(sb[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = a[j] * s;
        f[8 + j] = b[j] * s;
      }
      store16(out + 16 * g, f, wide);
    }
  }
}

// Any cols: a thread takes the values of a row that share 8 aligned places of the result (the row's
// first and last may be fewer): a codes word and its neighbour shifted into place, two scales.  I: the
// type of values' numbers.
template <typename T, typename I>
__global__ void __launch_bounds__(kMxThreads)
    mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                            int64_t rows, int64_t cols64, T* out) {
  const I cols = (I)cols64;
  const I blocks = (cols + 31) / 32;
  const I per_row = (cols + 14) / 8;
  const int64_t total = rows * (int64_t)per_row;
  const int64_t stride = (int64_t)gridDim.x * kMxThreads;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(codes);
  for (int64_t g0 = (int64_t)blockIdx.x * kMxThreads + threadIdx.x; g0 < total;
       g0 += kUnits * stride) {
    uint32_t q[kUnits], sb[kUnits];
    I at[kUnits];
    int n[kUnits], in[kUnits];  // values, and how many of them are of the first block
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t g = g0 + i * stride;
      n[i] = 0;
      if (g >= total) continue;
      const I row = (I)g / per_row;
      const I k8 = ((I)g - row * per_row) * 8;
      const I before = (row * cols) & 7;  // places of the first 8 that belong to earlier rows
      const I c = k8 > before ? k8 - before : 0;
      const I end = k8 + 8 - before < cols ? k8 + 8 - before : cols;
      if (c >= end) continue;
      n[i] = (int)(end - c);
      in[i] = 32 - (int)(c & 31);
      at[i] = row * cols + c;
      const I w = row * blocks * 4 + (c >> 3);
      const int k = (int)c & 7;
      q[i] = __ldg(words + w);
      // (the neighbour is of this row where the values reach into it)
      if (k + n[i] > 8) q[i] = __funnelshift_r(q[i], __ldg(words + w + 1), 4 * k);
      else q[i] >>= 4 * k;
      const I s = row * blocks;
      sb[i] = __ldg(scales + s + (c >> 5)) | (uint32_t)__ldg(scales + s + ((end - 1) >> 5)) << 8;
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      if (n[i] == 0) continue;
      float f[8];
      values8(q[i], f);
      const float a = scale_value(sb[i] & 255u), b = scale_value(sb[i] >> 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= j < in[i] ? a : b;
      store8(out + at[i], f, n[i]);
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------
static unsigned mx_grid(const void* kernel, int64_t warps) {
  const int64_t need = (warps + kMxThreads / 32 - 1) / (kMxThreads / 32);
  const int64_t most = persistent_grid(kernel, kMxThreads, 0);
  return (unsigned)(most > 0 && need > most ? most : need);
}
// every number of a value, padding and a grid's overshoot included, fits 32 bits
static bool narrow(int64_t rows, int64_t cols) { return rows * (cols + 64) < ((int64_t)1 << 31); }
static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
static cudaError_t quantize_t(const void* xv, int64_t rows, int64_t cols, int64_t stride,
                              uint8_t* codes, uint8_t* scales, cudaStream_t s) {
  const T* x = static_cast<const T*>(xv);
  if (rows == 1) stride = cols;
  const bool flat = cols % 32 == 0 && stride == cols && al16(x);
  auto* k = flat              ? mxfp4_quantize_kernel<T, true, int64_t>
            : narrow(rows, cols) ? mxfp4_quantize_kernel<T, false, uint32_t>
                                 : mxfp4_quantize_kernel<T, false, int64_t>;
  const int64_t strips = (rows * ((cols + 31) / 32) + 8 * kUnits - 1) / (8 * kUnits);
  k<<<mx_grid((const void*)k, strips), kMxThreads, 0, s>>>(x, rows, cols, stride, codes, scales);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t dequantize_t(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                int64_t cols, void* ov, cudaStream_t s) {
  T* out = static_cast<T*>(ov);
  if (cols % 32 == 0) {
    auto* k = mxfp4_dequantize_flat_kernel<T>;
    const int64_t halves = rows * cols / 16;
    k<<<mx_grid((const void*)k, (halves + 32 * kUnits - 1) / (32 * kUnits)), kMxThreads, 0, s>>>(
        reinterpret_cast<const uint2*>(codes), scales, halves,
        (reinterpret_cast<uintptr_t>(out) & 31u) == 0, out);
  } else {
    auto* k = narrow(rows, cols) ? mxfp4_dequantize_kernel<T, uint32_t>
                                 : mxfp4_dequantize_kernel<T, int64_t>;
    const int64_t groups = rows * ((cols + 14) / 8);
    k<<<mx_grid((const void*)k, (groups + 32 * kUnits - 1) / (32 * kUnits)), kMxThreads, 0, s>>>(
        codes, scales, rows, cols, out);
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
