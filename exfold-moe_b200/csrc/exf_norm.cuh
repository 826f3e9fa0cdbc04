// Device helpers of the norm kernels: rows as vectors of 16 bytes or single elements, sums and maxima over
// the threads of a row.
#pragma once

#include "exf_common.cuh"
#include "exf_launch.h"
#include "exf_norm.h"

#include <string.h>

#include <type_traits>

namespace exf {

// V elements of type T as they lie in memory: one element, or 16 bytes (fp32 weights beside 16-bit values: 32).
// Kept as words and taken apart where they are used: as elements, the compiler gives each 16-bit one a
// register of its own.
template <typename T, int V>
struct Pack {
  static constexpr int kWords = V * sizeof(T) > 4 ? V * sizeof(T) / 4 : 1;
  static_assert(V == 1 || V == 2 || kWords % 4 == 0, "one element, two, or whole 16-byte vectors");
  uint32_t w[kWords];

  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[j]);
    } else {
      const uint32_t two = w[j >> 1];
      if constexpr (std::is_same<T, __half>::value)
        return __half2float(__ushort_as_half((unsigned short)(j & 1 ? two >> 16 : two & 0xffffu)));
      else
        return __uint_as_float(j & 1 ? two & 0xffff0000u : two << 16);
    }
  }
  __device__ __forceinline__ void set(const float (&e)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = __float_as_uint(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const float hi = j + 1 < V ? e[j + 1 < V ? j + 1 : j] : 0.0f;
        if constexpr (std::is_same<T, __half>::value) {
          const __half2 h = __floats2half2_rn(e[j], hi);
          memcpy(&w[j >> 1], &h, 4);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(e[j], hi);
          memcpy(&w[j >> 1], &h, 4);
        }
      }
    }
  }
  __device__ __forceinline__ void read(const T* p) {
    if constexpr (V == 1) {
      if constexpr (sizeof(T) == 4)
        w[0] = *reinterpret_cast<const uint32_t*>(p);
      else
        w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else if constexpr (kWords < 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i / 4];
        w[i] = u.x;
        w[i + 1] = u.y;
        w[i + 2] = u.z;
        w[i + 3] = u.w;
      }
    }
  }
  __device__ __forceinline__ void write(T* p) const {
    if constexpr (V == 1) {
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<uint32_t*>(p) = w[0];
      else
        *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    } else if constexpr (kWords < 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4)
        reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
  }
  // the words as if newly read: what was taken from them before is not kept for later
  __device__ __forceinline__ void anew() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) asm volatile("" : "+r"(w[i]));
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
};
template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&out)[V]) {
  Pack<T, V> k;
  k.read(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = k.get(i);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&in)[V]) {
  Pack<T, V> k;
  k.set(in);
  k.write(p);
}
// V weights from column c on as fp32, of type T or fp32 (16-byte aligned where V > 1)
template <typename T, int V>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int c, float (&out)[V]) {
  if (f32)
    load_pack<float, V>(static_cast<const float*>(w) + c, out);
  else
    load_pack<T, V>(static_cast<const T*>(w) + c, out);
}

// x (+ residual), rounded to T: what the norm is taken of
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> rounded_sum(const Pack<T, V>& x, const Pack<T, V>& r) {
  float e[V];
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = x.get(i) + r.get(i);
  Pack<T, V> k;
  k.set(e);
  return k;
}
template <typename T, int V>
__device__ __forceinline__ void load_sum(const T* x, const T* r, float (&out)[V]) {
  Pack<T, V> k;
  k.read(x);
  if (r) {
    Pack<T, V> b;
    b.read(r);
    k = rounded_sum<T, V>(k, b);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = k.get(i);
}

// The sum over the G threads of a row (in a fixed order), for all of them.  G <= 32: lanes of a warp; else
// the whole block, through 32 words of shared memory; the next use of the same words needs a barrier of
// all threads in between (another row_sum over other words is one).
__device__ __forceinline__ float plus_lane(float v, int d) { return v + __shfl_xor_sync(0xffffffffu, v, d); }
__device__ __forceinline__ double plus_lane(double v, int d) {
  return v + __shfl_xor_sync(0xffffffffu, v, d);
}
__device__ __forceinline__ float2 plus_lane(float2 v, int d) {
  return make_float2(plus_lane(v.x, d), plus_lane(v.y, d));
}
template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = plus_lane(v, d);
  return v;
}
template <typename A>
__device__ __forceinline__ A row_sum(A v, int g, A* shared) {
  if (g < 32) {
    for (int d = g / 2; d > 0; d >>= 1) v = plus_lane(v, d);
    return v;
  }
  v = warp_sum(v);
  if (g == 32) return v;
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum(lane < (g >> 5) ? shared[lane] : A{});
}
// Whether a sum of squares has left the range in which fp32 holds it to its last bits: it overflowed (or
// holds an infinity or a NaN), or it is so small that its terms were cut off.  Then it is summed again in
// 64 bits.  (Small sums count only where eps does not hide them.)
__device__ __forceinline__ bool out_of_range(float sum, float eps) {
  return !(sum < 3.0e38f) || (sum < 1.0e-28f && eps < 1.0e-26f);
}

// A thread's sums of a row's squares, and of w dy s where dy is given, in 64 bits (read again from memory;
// out of line, so that its registers cost the usual path nothing).
template <typename T>
__device__ __noinline__ double2 sums_64(const T* x, const T* r, const T* dy, const void* weight,
                                        bool weight_f32, int cols, int t, int g) {
  double2 d = make_double2(0.0, 0.0);
  for (int c = t; c < cols; c += g) {
    float s[1], e[1], w[1];
    load_sum<T, 1>(x + c, r ? r + c : nullptr, s);
    d.x = fma((double)s[0], (double)s[0], d.x);
    if (dy) {
      load_pack<T, 1>(dy + c, e);
      load_weight<T, 1>(weight, weight_f32, c, w);
      d.y = fma((double)e[0] * (double)w[0], (double)s[0], d.y);
    }
  }
  return d;
}

// 1 / sqrt(mean square + eps) of a row from its threads' sums q; mean: 1 / cols (a product, one rounding
// of 2^-24 more than a quotient, and no division per row); x, r: the row.  Every thread of the block
// calls it.
template <typename T>
__device__ __forceinline__ float inverse_norm(float q, float mean, const NormArgs& a, int g, int t,
                                              const T* x, const T* r, float* part, double* part64) {
  q = row_sum(q, g, part);
  float v = rsqrtf(q * mean + a.eps);
  const bool again = out_of_range(q, a.eps);
  // (the same for the block where a row is a block; else the warp's other rows go along)
  if (g > 32 ? again : __any_sync(0xffffffffu, again)) {
    const double2 d = sums_64<T>(x, r, nullptr, nullptr, false, a.cols, t, g);
    const double sum = row_sum(d.x, g, part64);
    if (g > 32) __syncthreads();
    if (again) v = (float)(1.0 / sqrt(sum / a.cols + (double)a.eps));
  }
  return v;
}

// ---- rows in units -----------------------------------------------------------------------------------
// A row is taken in units of V elements, a unit being one aligned access: 16 bytes where base, stride and
// length allow it; else 4 bytes (two 16-bit elements, V = 2), else one element.  Units of two: a row that
// begins on an odd element has its units one element on (shift 1), and a row of odd length leaves one
// element, its first (shift 1) or last, to thread 0 of the row.  Unit u holds the columns V u + shift +
// [0, V).  A thread's rows all have one shift: the blocks' stride is even (even_grid).
// Vectors: the units of a row's g threads are strided by g.  Smaller units, of which a row has more: a
// thread's unit i lies 32 behind its unit i - 1, so that all of a row's accesses are one address and
// constants, and a warp's units lie behind one another, as many on each warp of the row (fewer threads than
// a warp have one unit each).  Strided by g, 65536 x 1001 fp16 takes 131 us for 102; vectors the other way,
// 32768 x 4096 bf16 180 for 175, its 8-bit form 221 for 213.
template <int V>
struct Units {
  static constexpr bool kSmall = V <= 2;
  int count, shift, odd;  // odd: the column of the element left over, or -1
  int g, first, left;     // the thread's first unit; units from that to the row's (its warp's) last
  __device__ __forceinline__ Units(int64_t row, int cols, int t, int g) : g(g) {
    count = cols / V;
    shift = V == 2 ? (int)row & cols & 1 : 0;
    odd = V == 2 && (cols & 1) ? (shift ? 0 : cols - 1) : -1;
    first = t;
    left = count - t;
    if (kSmall && g >= 32) {
      const int each = (count + g - 1) / g * 32;  // of a warp
      const int base = (t >> 5) * each;
      first = base + (t & 31);
      left = min(count, base + each) - first;
    }
  }
  __device__ __forceinline__ int step(int i) const { return (kSmall ? 32 : g) * i; }
  __device__ __forceinline__ bool has(int i) const { return step(i) < left; }
  __device__ __forceinline__ int column(int i) const { return (first + step(i)) * V + shift; }
};

// A thread's weights, kept from row to row, and the element left over's.
template <typename W, int V, int NU>
struct Weights {
  Pack<W, V> w[NU];
  float single;
  __device__ __forceinline__ void init(const void* weight, int t, const Units<V>& n) {
    const W* p = static_cast<const W*>(weight);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      w[i].clear();
      if (n.has(i)) {
        const int c = n.column(i);
        if constexpr (V == 2) {  // (the weights themselves do not move)
          const float e[2] = {to_f32<W>(p[c]), to_f32<W>(p[c + 1])};
          w[i].set(e);
        } else {
          w[i].read(p + c);
        }
      }
    }
    single = 0.0f;
    if (V == 2 && n.odd >= 0 && t == 0) single = to_f32<W>(p[n.odd]);
  }
};

// ---- layout, host side --------------------------------------------------------------------------------
static inline bool norm_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Threads a row: a power of two, so that each holds about `per` units of V of the row's `units` (fewer than
// a warp with small units: one); from `least`.
template <int V>
static inline int norm_threads(int64_t units, int per, int least) {
  int g = least;
  while (g < 1024 && (int64_t)g * (V <= 2 && g < 32 ? 1 : per) < units) g *= 2;
  return g;
}

// Blocks that fill the card once, at most one for each of `need`.
static inline unsigned stay_grid(const void* kernel, int block, size_t smem, int64_t need) {
  const int64_t most = persistent_grid(kernel, block, smem);
  return (unsigned)(most > 0 && most < need ? most : need);
}

// The same for rows in units of two: an even stride between a block's rows.
static inline unsigned even_grid(unsigned grid, int64_t need) {
  return grid < need && grid > 1 ? grid & ~1u : grid;
}

// The widest unit that every row of the call allows: 16 bytes, two 16-bit elements (base aligned to 4
// bytes; rows of the inputs and the results then begin on odd elements together), or one element.
enum NormUnit { kVector, kPair, kSingle };
template <typename T, typename... P>
static NormUnit norm_unit(const NormArgs& a, P... others) {
  constexpr int V = 16 / sizeof(T);
  const void* all[] = {a.x, a.residual, a.sum, others...};
  uintptr_t bits = 0;
  for (const void* p : all) bits |= reinterpret_cast<uintptr_t>(p);
  const int64_t xs = a.rows > 1 ? a.x_stride : a.cols;
  const int64_t rs = a.rows > 1 && a.residual ? a.r_stride : a.cols;
  if (a.cols % V == 0 && xs % V == 0 && rs % V == 0 && bits % 16 == 0 && norm_aligned(a.weight))
    return kVector;
  if (sizeof(T) == 2 && bits % 4 == 0 && (xs - a.cols) % 2 == 0 && (rs - a.cols) % 2 == 0 &&
      (a.weight_f32 || reinterpret_cast<uintptr_t>(a.weight) % 4 == 0))
    return kPair;
  return kSingle;
}

// f(weight type, V) for the call's unit and weight
template <typename T, typename F>
static cudaError_t norm_dispatch(const NormArgs& a, NormUnit unit, F f) {
  using std::integral_constant;
  auto by_weight = [&](auto v) {
    if constexpr (!std::is_same<T, float>::value)
      if (!a.weight_f32) return f(T(), v);
    return f(float(), v);
  };
  if (unit == kVector) return by_weight(integral_constant<int, 16 / sizeof(T)>());
  if constexpr (sizeof(T) == 2)
    if (unit == kPair) return by_weight(integral_constant<int, 2>());
  return by_weight(integral_constant<int, 1>());
}

}  // namespace exf
