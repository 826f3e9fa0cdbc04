// Device helpers of the norm kernels: rows as vectors of 16 bytes or single elements, sums and maxima over
// the threads of a row.
#pragma once

#include "exf_common.cuh"
#include "exf_norm.h"

namespace exf {

// V elements of a row of type T, one access (V = 1, or 16 bytes where base and stride allow it)
template <typename T, int V>
struct Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&out)[V]) {
  if constexpr (V == 1) {
    out[0] = to_f32<T>(*p);
  } else {
    static_assert(V * sizeof(T) == 16, "one 16-byte vector");
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = to_f32<T>(k.v[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&in)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<T>(in[0]);
  } else {
    Pack<T, V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) k.v[i] = from_f32<T>(in[i]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&k);
  }
}
// V weights from column c on, fp32 or of type T (16-byte aligned where V > 1)
template <typename T, int V>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int c, float (&out)[V]) {
  if (f32) {
    const float* p = static_cast<const float*>(w) + c;
    if constexpr (V == 1) {
      out[0] = *p;
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 q = *reinterpret_cast<const float4*>(p + i);
        out[i] = q.x;
        out[i + 1] = q.y;
        out[i + 2] = q.z;
        out[i + 3] = q.w;
      }
    }
  } else {
    load_pack<T, V>(static_cast<const T*>(w) + c, out);
  }
}

// x (+ residual), rounded to T: what the norm is taken of
template <typename T, int V>
__device__ __forceinline__ void load_sum(const T* x, const T* r, float (&out)[V]) {
  load_pack<T, V>(x, out);
  if (r) {
    float b[V];
    load_pack<T, V>(r, b);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = to_f32<T>(from_f32<T>(out[i] + b[i]));
  }
}

// The sum over the G threads of a row (in a fixed order), for all of them.  G <= 32: lanes of a warp; else
// the whole block, through 32 words of shared memory that a barrier frees for the next use.
template <typename A>
__device__ __forceinline__ A row_sum(A v, int g, A* shared) {
  const int w = g < 32 ? g : 32;
  for (int d = w / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (g <= 32) return v;
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = g >> 5, lane = threadIdx.x & 31;
  v = lane < warps ? shared[lane] : A(0);
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  __syncthreads();
  return v;
}
template <typename A>
__device__ __forceinline__ A row_max(A v, int g, A* shared) {
  const int w = g < 32 ? g : 32;
  for (int d = w / 2; d > 0; d >>= 1) {
    const A o = __shfl_xor_sync(0xffffffffu, v, d);
    v = o > v ? o : v;
  }
  if (g <= 32) return v;
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = g >> 5, lane = threadIdx.x & 31;
  v = lane < warps ? shared[lane] : A(0);
  for (int d = 16; d > 0; d >>= 1) {
    const A o = __shfl_xor_sync(0xffffffffu, v, d);
    v = o > v ? o : v;
  }
  __syncthreads();
  return v;
}

// Whether a sum of squares has left the range in which fp32 holds it to its last bits: it overflowed (or
// holds an infinity or a NaN), or it is so small that its terms were cut off.  Then it is summed again in
// 64 bits.  (Small sums count only where eps does not hide them.)
__device__ __forceinline__ bool out_of_range(float sum, float eps) {
  return !(sum < 3.0e38f) || (sum < 1.0e-28f && eps < 1.0e-26f);
}

// 1 / sqrt(mean square + eps) of a row from its threads' sums q; sum64 gives a thread's sum in 64 bits.  Every
// thread of the block calls it.
template <typename F>
__device__ __forceinline__ float inverse_norm(float q, const NormArgs& a, int g, float* part,
                                              double* part64, F sum64) {
  q = row_sum(q, g, part);
  float v = rsqrtf(q / (float)a.cols + a.eps);
  const bool again = out_of_range(q, a.eps);
  // (the same for the block where a row is a block; else the warp's other rows go along)
  if (g > 32 ? again : __any_sync(0xffffffffu, again)) {
    const double d = row_sum(sum64(), g, part64);
    if (again) v = (float)(1.0 / sqrt(d / a.cols + (double)a.eps));
  }
  return v;
}

// ---- layout, host side --------------------------------------------------------------------------------
static inline bool norm_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Threads a row: a power of two, so that each holds about `per` units of the row's `units`; from `least`.
static inline int norm_threads(int64_t units, int per, int least) {
  int g = least;
  while (g < 1024 && (int64_t)g * per < units) g *= 2;
  return g;
}

// Whether rows can be read and written as 16-byte vectors.
template <typename T>
static bool norm_vectors(const NormArgs& a) {
  constexpr int V = 16 / sizeof(T);
  return a.cols % V == 0 &&
         (a.rows == 1 || (a.x_stride % V == 0 && (!a.residual || a.r_stride % V == 0))) &&
         norm_aligned(a.x) && norm_aligned(a.residual) && norm_aligned(a.weight) &&
         norm_aligned(a.sum);
}

}  // namespace exf
