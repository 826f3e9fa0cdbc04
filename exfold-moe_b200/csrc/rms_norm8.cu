// Root-mean-square norm with its output in 8 bits and scales, and reading it back (sm_100a).
//
//   s = round(x + residual) (or x),  v = 1 / sqrt(mean s^2 + eps),  p_j = s_j w_j
//   a group of 32, 64 or 128 columns (or the row) has top = max |p_j|
//   code_j = p_j M / top, rounded to the nearest e4m3 (M = 448) or integer (M = 127), ties to even
//   scale = top v / M, so that code scale is the norm's s_j v w_j
//
// v is the same for the row, so the codes do not depend on its rounding: equal inputs give the codes of the
// definition (products of fp32 values with fp32 weights to 2^-48).  Products are held in fp32, those with fp32
// values or weights as two fp32 terms: exact, but that what lies below fp32's smallest value, 2^-149, is rounded
// to it, in a group's largest as in its other products.  A group with a product that is not
// finite in fp32 gets codes 0 and a NaN scale, a group of zeros codes 0 and scale 0.
//
// Bound by memory (x, residual in, sum and codes out, once each) and, beside it, by the instructions of the
// codes: 32768 x 4096 bf16 with a residual, a scale a row, 167 us = 0.86 of a copy's rate; e4m3 in groups of
// 128 199 us = 0.72.
#include <mutex>

#include "exf_launch.h"
#include "exf_norm.cuh"

namespace exf {

// ---- the largest product of a group ----------------------------------------------------------------
// Products of 16-bit values are exact in fp32 (EXACT; to 2^-149): the value.  Others: an integer that compares
// as the magnitudes do, the rounded product's bits and, below them, what the rounding left (to 2^-149), its order
// made that of unsigned integers.  Infinities and NaN come out above all.
template <bool EXACT>
struct Top;
template <>
struct Top<true> {
  using Key = float;
  using Shared = uint32_t;
  static __device__ __forceinline__ Key of(float s, float w, float p) { return fabsf(p); }
  static __device__ __forceinline__ Key larger(Key a, Key b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
  }
  static __device__ __forceinline__ Shared shared(Key k) { return __float_as_uint(k); }
  static __device__ __forceinline__ Key back(Shared k) { return __uint_as_float(k); }
  static __device__ __forceinline__ float rounded(Key k) { return k; }
  static __device__ __forceinline__ double value(Key k) { return (double)k; }
};
template <>
struct Top<false> {
  using Key = unsigned long long;
  using Shared = unsigned long long;
  static __device__ __forceinline__ Key of(float s, float w, float p) {
    const float a = fabsf(p);
    const uint32_t rest = __float_as_uint(fmaf(fabsf(s), fabsf(w), -a));
    const uint32_t order = rest ^ ((uint32_t)((int32_t)rest >> 31) | 0x80000000u);
    return (Key)__float_as_uint(a) << 32 | order;
  }
  static __device__ __forceinline__ Key larger(Key a, Key b) { return a > b ? a : b; }
  static __device__ __forceinline__ Shared shared(Key k) { return k; }
  static __device__ __forceinline__ Key back(Shared k) { return k; }
  static __device__ __forceinline__ float rounded(Key k) { return __uint_as_float((uint32_t)(k >> 32)); }
  static __device__ __forceinline__ double value(Key k) {
    const uint32_t order = (uint32_t)k;
    const uint32_t rest = order & 0x80000000u ? order ^ 0x80000000u : ~order;
    return k ? (double)rounded(k) + (double)__uint_as_float(rest) : 0.0;
  }
};
// The largest of `lanes` neighbouring lanes (4 to 32).  A whole warp's, or a half's: the integer maximum of
// the lanes in one instruction.
__device__ __forceinline__ uint32_t top_bits(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ float top_warp(float k) { return __uint_as_float(top_bits(__float_as_uint(k))); }
__device__ __forceinline__ unsigned long long top_warp(unsigned long long k) {
  const uint32_t hi = (uint32_t)(k >> 32), top = top_bits(hi);
  return (unsigned long long)top << 32 | top_bits(hi == top ? (uint32_t)k : 0u);
}
template <bool EXACT>
__device__ __forceinline__ typename Top<EXACT>::Key top_over(typename Top<EXACT>::Key k, int lanes) {
  using Key = typename Top<EXACT>::Key;
  if (lanes == 32) return top_warp(k);
  if (lanes == 16) {
    const bool upper = threadIdx.x & 16;
    const Key lo = top_warp(upper ? Key(0) : k), hi = top_warp(upper ? k : Key(0));
    return upper ? hi : lo;
  }
#pragma unroll
  for (int d = 4; d > 0; d >>= 1)
    if (2 * d <= lanes) k = Top<EXACT>::larger(k, __shfl_xor_sync(0xffffffffu, k, d));
  return k;
}

// ---- codes --------------------------------------------------------------------------------------------
// A group's factors: quotients p M / top are taken with M / top a little too small and a little too large.
// Where both give the same code it is the definition's (2^-20 to either side; the rounded top, the division
// (2 units in the last place) and the products are off by 8 steps of 2^-24 together).  Else, one value in
// 2^15, and for all values of a group whose top is far from 1, the quotient is taken in 64 bits, where its
// distance from a border shows.
struct Quantum {
  float low, high, scale;
  bool all;  // in 64 bits
};
template <bool INT8>
__device__ __forceinline__ Quantum quantum_of(float top, float v) {
  Quantum z;
  const float m = __fdividef(INT8 ? 127.0f : 448.0f, top);
  z.low = m * (1.0f - 0x1p-20f);
  z.high = m * (1.0f + 0x1p-20f);
  z.scale = top * v * (1.0f / (INT8 ? 127.0f : 448.0f));
  z.all = !(top > 0x1p-100f) || !(top < 0x1p100f);
  return z;
}
// the scale of a group whose top is far from 1: NaN for one that is not finite
__device__ __forceinline__ float top_scale(float top, const Quantum& z) {
  return top < __int_as_float(0x7f800000) ? z.scale : __int_as_float(0x7fc00000);
}
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {  // a in the low byte
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// the distance of e4m3's values about q: three bits behind the leading one, multiples of 2^-9 below 2^-6
__device__ __forceinline__ float unit_of(float q) {
  const uint32_t e = __float_as_uint(q) >> 23;
  return __uint_as_float(((e < 121u ? 121u : e) - 3u) << 23);
}
// The code of one value, in 64 bits, read again from memory; top is its group's.  (Out of line: its
// registers cost the usual path nothing.)
template <typename T, typename W, bool INT8>
__device__ __noinline__ uint8_t code_64(const T* x, const T* r, const W* w, double top) {
  if (!(top > 0.0) || !(top < 3.4028235677973366e38)) return 0;
  float s[1];
  load_sum<T, 1>(x, r, s);
  const float f = to_f32<W>(*w), m = INT8 ? 127.0f : 448.0f;
  // (as the group's largest is held, so that no product is above it)
  using K = Top<sizeof(T) == 2 && sizeof(W) == 2>;
  const double p = K::value(K::of(s[0], f, s[0] * f)) * (double)m;
  float c;
  if (top > 0x1p-100 && top < 0x1p100) {
    // the border beside the quotient, and the side of it on which p lies
    const float q = __fdividef((float)p, (float)top);
    float unit = 1.0f;
    if (!INT8) unit = unit_of(q);
    const float h = rintf(q / unit - 0.5f);
    const double side = p - (double)((h + 0.5f) * unit) * top;
    c = (h + (side > 0.0 || (side == 0.0 && ((int)h & 1)) ? 1.0f : 0.0f)) * unit;
  } else {
    const double q = p / top;
    const double unit = INT8 ? 1.0 : (double)unit_of((float)q);
    c = (float)(rint(q / unit) * unit);
  }
  c = copysignf(c, s[0] * f);
  return (uint8_t)(INT8 ? (uint32_t)(int)c : e4m3_pair(c, 0.0f));
}
// The codes of up to four products, the first in the low byte.  Integers: rounded by adding 1.5 2^23, whose
// low byte they become.
template <bool INT8, int N>
__device__ __forceinline__ uint32_t code_word(const float* p, float m) {
  if (INT8) {
    uint32_t b[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < N; ++j) b[j] = __float_as_uint(fmaf(p[j], m, 12582912.0f));
    const uint32_t lo = N > 1 ? __byte_perm(b[0], b[1], 0x0040) : b[0];
    if (N > 2) return __byte_perm(lo, __byte_perm(b[2], b[3], 0x0040), 0x5410);
    return N > 1 ? lo & 0xffffu : lo & 0xffu;
  }
  if (N == 1) return e4m3_pair(p[0] * m, 0.0f) & 0xffu;
  uint32_t lo = e4m3_pair(p[0] * m, p[N > 1 ? 1 : 0] * m);
  if (N > 2) lo |= e4m3_pair(p[N > 2 ? 2 : 0] * m, p[N > 2 ? 3 : 0] * m) << 16;
  return lo;
}

// The codes of N products beside one another; doubt gets a bit, from the given one on, for each whose code
// is to be taken again in 64 bits.
template <bool INT8, int N>
__device__ __forceinline__ uint32_t sure_word(const float* p, const Quantum& z, int bit, uint32_t& doubt) {
  const uint32_t low = code_word<INT8, N>(p, z.low), other = low ^ code_word<INT8, N>(p, z.high);
  if (other || z.all) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (z.all || (other >> (8 * j) & 255u)) doubt |= 1u << (bit + j);
  }
  return low;
}

// ---- rows of whole vectors ---------------------------------------------------------------------------------
// Blocks that stay, as rms_norm_kernel's, with at least a warp a row.  The largest products are taken with
// the loads' results; a group lies on 32 / V to 128 / V neighbouring lanes, which find its largest among
// them.  group 0: the row, reduced beside the sum of squares.
template <typename T, typename W, int NU, int THREADS, bool INT8>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1)
    rms_norm_8bit_kernel(const NormArgs a, int g, int group, uint8_t* codes, float* scales) {
  constexpr bool EXACT = sizeof(T) == 2 && sizeof(W) == 2;
  constexpr int V = 16 / sizeof(T);
  using K = Top<EXACT>;
  using Key = typename K::Key;
  __shared__ float part[2][32];
  __shared__ double part64[32];
  __shared__ Key part_top[2][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_block = blockDim.x / g;
  const int sub = threadIdx.x / g, t = threadIdx.x % g;
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.residual);
  const W* weight = static_cast<const W*>(a.weight);
  T* sum = static_cast<T*>(a.sum);
  const int64_t step = (int64_t)gridDim.x * per_block;
  const int64_t first = (int64_t)blockIdx.x * per_block;
  int64_t row = first + sub;
  const Units<V> n(row, a.cols, t, g);
  const int shift = group == 32 ? 5 : group == 64 ? 6 : 7;  // columns to groups
  const int groups = group ? (a.cols + group - 1) >> shift : 1;

  Pack<T, V> nx[NU], nr[NU];
  Weights<W, V, NU> w;
  auto fetch = [&](int64_t at) {
    const T* xr = x + at * a.x_stride + n.column(0);
    const T* rr = r + at * a.r_stride + n.column(0);
    const bool live = at < a.rows;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (n.has(i) && live) {
        nx[i].read(xr + n.step(i) * V);
        if (r) nr[i].read(rr + n.step(i) * V);
      } else {
        nx[i].clear();
        nr[i].clear();
      }
    }
  };
  fetch(row);
  w.init(a.weight, t, n);
  const float mean = 1.0f / (float)a.cols;
  int b = 0;
  for (int64_t base = first; base < a.rows; base += step, row += step, b ^= 1) {
    const bool live = row < a.rows;
    const int64_t at = row * a.cols;
    float q = 0.0f;
    Key top[NU], all = Key(0);
    float p[NU][V];
    T* to = sum + at + n.column(0);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const Pack<T, V> s = r ? rounded_sum<T, V>(nx[i], nr[i]) : nx[i];
      if (r && live && n.has(i)) s.write(to + n.step(i) * V);
      w.w[i].anew();
      top[i] = Key(0);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float e = s.get(j);
        q = fmaf(e, e, q);
        p[i][j] = e * w.w[i].get(j);
        top[i] = K::larger(top[i], K::of(e, w.w[i].get(j), p[i][j]));
      }
      all = K::larger(all, top[i]);
    }
    fetch(row + step);
    const int64_t mine = live ? row : 0;
    const T* xr = x + mine * a.x_stride;
    const T* rr = r ? r + mine * a.r_stride : nullptr;
    if (group == 0) {
      // (its barrier is the sum's: the partial maxima are written before it and read after it)
      all = top_over<EXACT>(all, 32);
      if (g > 32 && (threadIdx.x & 31) == 0) part_top[b][threadIdx.x >> 5] = all;
    }
    const float v = inverse_norm<T>(q, mean, a, g, t, xr, rr, part[b], part64);
    if (group == 0 && g > 32) {
      const int lane = threadIdx.x & 31;
      all = top_over<EXACT>(lane < (g >> 5) ? part_top[b][lane] : Key(0), 32);
    }
    float* row_scales = scales + row * groups;
    uint8_t* out = codes + at;
    Quantum z = quantum_of<INT8>(K::rounded(all), v);  // (of the row; of groups below)
    if (group == 0 && live && t == 0) row_scales[0] = z.all ? top_scale(K::rounded(all), z) : z.scale;
    uint32_t doubt = 0;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int c = n.column(i);
      if (group != 0) {
        top[i] = top_over<EXACT>(top[i], group / V);
        z = quantum_of<INT8>(K::rounded(top[i]), v);
      }
      if (n.has(i) && live) {
        if (group != 0 && (c & (group - 1)) == 0)
          row_scales[c >> shift] = z.all ? top_scale(K::rounded(top[i]), z) : z.scale;
        if constexpr (V == 8)
          *reinterpret_cast<uint2*>(out + c) =
              make_uint2(sure_word<INT8, 4>(p[i], z, i * V, doubt),
                         sure_word<INT8, 4>(p[i] + V / 2, z, i * V + 4, doubt));
        else
          *reinterpret_cast<uint32_t*>(out + c) = sure_word<INT8, 4>(p[i], z, i * V, doubt);
      }
    }
#pragma unroll 1
    for (; doubt; doubt &= doubt - 1) {
      const int j = __ffs(doubt) - 1;
      const int c = n.column(j / V) + j % V;
      Key k = all;
      if (group != 0) {
#pragma unroll
        for (int h = 0; h < NU; ++h) k = h == j / V ? top[h] : k;
      }
      out[c] = code_64<T, W, INT8>(xr + c, rr ? rr + c : nullptr, weight + c, K::value(k));
    }
  }
}

// ---- other rows ----------------------------------------------------------------------------------------
// Rows that begin or end inside a vector pass through shared memory: read in units of V <= 2 elements, they
// lie there with column 0 at element 0 or, where the units are one column on, 1; then a thread takes 8
// columns, as above, from there; its codes go back to shared memory and from there to memory in aligned
// words.  The block's weights stay in shared memory.  g threads a row; g = 32: blockDim.x / 32 rows beside
// one another, and nothing waits but lanes for lanes.  (Groups of units of two by atomic maxima instead:
// 65536 x 1001 bf16 in e4m3 435 us for 142.)
template <typename T>
__host__ __device__ constexpr int staged_bytes(int cols) {  // of a row: elements, then codes
  return ((cols + 7) / 8 * 8 + 8) * (int)(sizeof(T) + 1) + 15 & ~15;
}
template <typename T, typename W, int V, bool INT8>
__global__ void __launch_bounds__(512, 2)
    rms_norm_8bit_staged_kernel(const NormArgs a, int g, int group, uint8_t* codes, float* scales) {
  constexpr bool EXACT = sizeof(T) == 2 && sizeof(W) == 2;
  using K = Top<EXACT>;
  using Key = typename K::Key;
  constexpr int NU = 4;  // units of V in flight
  __shared__ float part[32];
  __shared__ double part64[32];
  __shared__ Key part_top[32];
  extern __shared__ __align__(16) unsigned char staged[];
  const int padded = (a.cols + 7) / 8 * 8;
  const int per_block = blockDim.x / g;
  const int sub = threadIdx.x / g, t = threadIdx.x % g, lane = threadIdx.x & 31;
  W* weight = reinterpret_cast<W*>(staged);
  T* s = reinterpret_cast<T*>(staged + padded * sizeof(W) + sub * staged_bytes<T>(a.cols));
  uint8_t* here = reinterpret_cast<uint8_t*>(s + padded + 8);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const W* given = static_cast<const W*>(a.weight);
  for (int c = threadIdx.x; c < padded; c += blockDim.x) weight[c] = c < a.cols ? given[c] : from_f32<W>(0.0f);
  __syncthreads();
  auto wait = [&] {
    if (g > 32)
      __syncthreads();
    else
      __syncwarp();
  };
  const int shift = group == 32 ? 5 : group == 64 ? 6 : 7;  // columns to groups
  const int groups = group ? (a.cols + group - 1) >> shift : 1;
  const float mean = 1.0f / (float)a.cols;
  const int64_t step = (int64_t)gridDim.x * per_block;
  // (rows of a block end together, or a warp's alone)
  for (int64_t row = (int64_t)blockIdx.x * per_block + sub; row < a.rows; row += step) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.r_stride : nullptr;
    T* sum = static_cast<T*>(a.sum) + row * a.cols;
    const int on = V == 2 ? (int)row & a.cols & 1 : 0;
    const int count = a.cols / V;
    float q = 0.0f;
    // (a warp's units behind one another: a step's accesses are one address and constants)
#pragma unroll 1
    for (int u = (t >> 5) * 32 * NU + lane; u - lane < count; u += g * NU) {
      Pack<T, V> e[NU], f[NU];
      const int c = u * V + on;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        e[i].clear();
        f[i].clear();
        if (u + 32 * i < count) {
          e[i].read(x + c + 32 * i * V);
          if (r) f[i].read(r + c + 32 * i * V);
        }
      }
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        if (r) e[i] = rounded_sum<T, V>(e[i], f[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) q = fmaf(e[i].get(j), e[i].get(j), q);
        if (u + 32 * i < count) {
          e[i].write(s + c + on + 32 * i * V);
          if (r) e[i].write(sum + c + 32 * i * V);
        }
      }
    }
    if (V == 2 && (a.cols & 1) && t == 0) {
      const int c = on ? 0 : a.cols - 1;
      float e[1];
      load_sum<T, 1>(x + c, r ? r + c : nullptr, e);
      q = fmaf(e[0], e[0], q);
      store_pack<T, 1>(s + c + on, e);
      if (r) store_pack<T, 1>(sum + c, e);
    }
    if (t < padded + 1 - a.cols) s[a.cols + on + t] = from_f32<T>(0.0f);  // (as far as is read)
    // (the row is complete behind the barrier of its sum)
    const float v = inverse_norm<T>(q, mean, a, g, t, x, r, part, part64);
    if (g == 32) __syncwarp();

    float p[8];
    auto products = [&](int c) {  // of 8 columns; their largest
      Pack<T, 8> e;
      e.read(s + c);
      if constexpr (V == 2) {
        const uint32_t next = *reinterpret_cast<const uint32_t*>(s + c + 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) e.w[i] = __funnelshift_r(e.w[i], i < 3 ? e.w[i + 1] : next, 16 * on);
      }
      Pack<W, 8> w;
      w.read(weight + c);
      Key k = Key(0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = e.get(j) * w.get(j);
        k = K::larger(k, K::of(e.get(j), w.get(j), p[j]));
      }
      return k;
    };
    float* row_scales = scales + row * groups;
    Key top = Key(0);
    Quantum z;
    if (group == 0) {
      for (int c = t * 8; c < padded; c += g * 8) top = K::larger(top, products(c));
      top = top_over<EXACT>(top, 32);
      if (g > 32) {
        if (lane == 0) part_top[t >> 5] = top;
        __syncthreads();
        top = top_over<EXACT>(lane < (g >> 5) ? part_top[lane] : Key(0), 32);
      }
      z = quantum_of<INT8>(K::rounded(top), v);
      if (t == 0) row_scales[0] = z.all ? top_scale(K::rounded(top), z) : z.scale;
    }
#pragma unroll 1
    for (int c = t * 8; c - 8 * lane < padded; c += g * 8) {
      const bool mine = c < padded;
      if (group != 0) {
        top = top_over<EXACT>(mine ? products(c) : Key(0), group / 8);
        z = quantum_of<INT8>(K::rounded(top), v);
        if (mine && (c & (group - 1)) == 0)
          row_scales[c >> shift] = z.all ? top_scale(K::rounded(top), z) : z.scale;
      } else if (mine) {
        products(c);
      }
      if (mine) {
        uint32_t doubt = 0;
        *reinterpret_cast<uint2*>(here + c) = make_uint2(sure_word<INT8, 4>(p, z, 0, doubt),
                                                         sure_word<INT8, 4>(p + 4, z, 4, doubt));
#pragma unroll 1
        for (; doubt; doubt &= doubt - 1) {
          const int h = c + __ffs(doubt) - 1;
          here[h] = code_64<T, W, INT8>(s + h + on, nullptr, weight + h, K::value(top));
        }
      }
    }
    wait();
    uint8_t* out = codes + row * a.cols;
    const int head = min((int)(-reinterpret_cast<uintptr_t>(out) & 3), a.cols);
    const int whole = (a.cols - head) >> 2, tail = (a.cols - head) & 3;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(here);
    for (int i = t; i < whole; i += g)
      *reinterpret_cast<uint32_t*>(out + head + 4 * i) =
          __funnelshift_r(words[i], words[i + 1], 8 * head);
    if (t < head) out[t] = here[t];
    if (t < tail) out[a.cols - tail + t] = here[a.cols - tail + t];
    if (g == 32) __syncwarp();
  }
}

// Rows of any length, read again after the reduction; a block a row.  The groups' largest products in shared
// memory.
template <typename T, typename W, bool INT8>
__global__ void __launch_bounds__(1024)
    rms_norm_8bit_long_kernel(const NormArgs a, int group, uint8_t* codes, float* scales) {
  constexpr bool EXACT = sizeof(T) == 2 && sizeof(W) == 2;
  using K = Top<EXACT>;
  using Key = typename K::Key;
  __shared__ float part[32];
  __shared__ double part64[32];
  extern __shared__ unsigned long long words[];
  auto* tops = reinterpret_cast<typename K::Shared*>(words);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.r_stride : nullptr;
  const W* w = static_cast<const W*>(a.weight);
  const int groups = group ? (a.cols + group - 1) / group : 1;
  for (int i = threadIdx.x; i < groups; i += 1024) tops[i] = 0;
  __syncthreads();
  float q = 0.0f;
  Key all = Key(0);
  for (int c0 = 0; c0 < a.cols; c0 += 1024) {  // a warp's 32 columns lie in one group
    const int c = c0 + threadIdx.x;
    Key k = Key(0);
    if (c < a.cols) {
      float s[1];
      load_sum<T, 1>(x + c, r ? r + c : nullptr, s);
      if (r) store_pack<T, 1>(static_cast<T*>(a.sum) + row * a.cols + c, s);
      q = fmaf(s[0], s[0], q);
      const float e = to_f32<W>(w[c]);
      k = K::of(s[0], e, s[0] * e);
    }
    if (group) {
      k = top_over<EXACT>(k, 32);
      if ((threadIdx.x & 31) == 0 && c < a.cols) atomicMax(tops + c / group, K::shared(k));
    } else {
      all = K::larger(all, k);
    }
  }
  if (!group) {
    all = top_over<EXACT>(all, 32);
    if ((threadIdx.x & 31) == 0) atomicMax(tops, K::shared(all));
  }
  // (behind a barrier of its own: the maxima are complete)
  const float mean = 1.0f / (float)a.cols;
  const float v = inverse_norm<T>(q, mean, a, 1024, threadIdx.x, x, r, part, part64);
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    float s[1];
    load_sum<T, 1>(x + c, r ? r + c : nullptr, s);
    const float p = s[0] * to_f32<W>(w[c]);
    const Key k = K::back(tops[group ? c / group : 0]);
    const Quantum z = quantum_of<INT8>(K::rounded(k), v);
    if (group == 0 ? c == 0 : c % group == 0)
      scales[row * groups + (group ? c / group : 0)] =
          z.all ? top_scale(K::rounded(k), z) : z.scale;
    uint32_t code = code_word<INT8, 1>(&p, z.low);
    if (code != code_word<INT8, 1>(&p, z.high) || z.all)
      code = code_64<T, W, INT8>(x + c, r ? r + c : nullptr, w + c, K::value(k));
    codes[row * a.cols + c] = (uint8_t)code;
  }
}

// ---- reading back -------------------------------------------------------------------------------
// out = code * scale, rounded.  A thread takes 16 values that lie together, whichever rows they belong to,
// so every access is a whole vector whatever the row's length; most lie in one group, and need one scale.
// 32768 x 4096 to bf16: 72 us, 0.85 of a copy's rate.
template <typename T, bool INT8>
__global__ void __launch_bounds__(256)
    dequantize_8bit_kernel(const uint8_t* codes, const float* scales, int64_t total, int cols,
                           int shift, int groups, T* out) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  auto pair = [](uint32_t code) {  // two codes' values
    if (INT8) return make_float2((float)(int8_t)(uint8_t)code, (float)(int8_t)(uint8_t)(code >> 8));
    uint32_t two;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"((uint16_t)code));
    return __half22float2(*reinterpret_cast<const __half2*>(&two));
  };
  const int inside = (int)((1ll << shift) - 1);
  const int64_t step = (int64_t)gridDim.x * blockDim.x * 16;
  for (int64_t f = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 16; f < total; f += step) {
    int64_t row;
    if (total <= 0xffffffffll)
      row = (uint32_t)f / (uint32_t)cols;
    else
      row = f / cols;
    int c = (int)(f - row * cols);
    if (total - f < 16) {
      for (int64_t i = f; i < total; ++i, ++c) {
        if (c == cols) {
          c = 0;
          ++row;
        }
        out[i] = from_f32<T>(pair(codes[i]).x * scales[row * groups + (c >> shift)]);
      }
      break;
    }
    const uint4 k = *reinterpret_cast<const uint4*>(codes + f);
    const uint32_t word[4] = {k.x, k.y, k.z, k.w};
    float e[16];
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float2 p = pair(word[j >> 2] >> (8 * (j & 2)) & 0xffffu);
      e[j] = p.x;
      e[j + 1] = p.y;
    }
    float scale = scales[row * groups + (c >> shift)];
    if (c + 16 <= cols && (c & inside) + 15 <= inside) {
#pragma unroll
      for (int j = 0; j < 16; ++j) e[j] *= scale;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (c == cols) {
          c = 0;
          ++row;
        }
        if (j > 0 && (c & inside) == 0) scale = scales[row * groups + (c >> shift)];
        e[j] *= scale;
        ++c;
      }
    }
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 16 / V; ++h) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = e[h * V + j];
      store_pack<T, V>(out + f + h * V, o);
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------
template <typename T, typename W, int V, bool INT8>
static cudaError_t quantize_v(const NormArgs& a, int group, uint8_t* codes, float* scales,
                              cudaStream_t s) {
  const bool few = a.rows <= 148;
  auto go = [&](auto* kern, int g, int block, size_t smem) {
    const int64_t need = (a.rows + block / g - 1) / (block / g);
    const unsigned grid = stay_grid(reinterpret_cast<const void*>(kern), block, smem, need);
    return launch_pdl(kern, dim3(grid), dim3(block), smem, s, a, g, group, codes, scales);
  };
  if constexpr (V > 2) {
    constexpr int NU = 2;
    const int64_t units = a.cols / V;
    if (units > 1024 * NU)
      return quantize_v<T, W, sizeof(T) == 2 ? 2 : 1, INT8>(a, group, codes, scales, s);
    const int g = norm_threads<V>(units, few ? NU / 2 : NU, 32), block = g <= 32 ? 128 : g;
    if (block <= 256) return go(rms_norm_8bit_kernel<T, W, NU, 256, INT8>, g, block, 0);
    return go(rms_norm_8bit_kernel<T, W, NU, 1024, INT8>, g, block, 0);
  } else {
    const int units = (a.cols + 7) / 8;
    int g = norm_threads<8>(units, few ? 1 : 2, 32);
    if (g > 512) g = 512;
    const int block = g <= 32 ? 128 : g;
    const size_t smem = (size_t)units * 8 * sizeof(W) + (size_t)(block / g) * staged_bytes<T>(a.cols);
    constexpr size_t kMost = 200 * 1024;
    if (smem <= kMost) {
      static std::mutex mu;
      static bool done[64];
      auto* kern = rms_norm_8bit_staged_kernel<T, W, V, INT8>;
      if (const cudaError_t e = allow_smem(kern, kMost, mu, done); e != cudaSuccess) return e;
      return go(kern, g, block, smem);
    }
    const int groups = group ? (a.cols + group - 1) / group : 1;
    const size_t key = sizeof(T) == 2 && sizeof(W) == 2 ? 4 : 8;
    return launch_pdl(rms_norm_8bit_long_kernel<T, W, INT8>, dim3((unsigned)a.rows), dim3(1024),
                      groups * key, s, a, group, codes, scales);
  }
}

template <typename T>
static cudaError_t quantize_t(const NormArgs& a, bool int8, int group, uint8_t* codes,
                              float* scales, cudaStream_t s) {
  // (vectors' codes are written 8 bytes at a time)
  NormUnit unit = norm_unit<T>(a);
  if (unit == kVector && reinterpret_cast<uintptr_t>(codes) % 8 != 0)
    unit = sizeof(T) == 2 ? kPair : kSingle;
  return norm_dispatch<T>(a, unit, [&](auto w, auto v) {
    return int8 ? quantize_v<T, decltype(w), decltype(v)::value, true>(a, group, codes, scales, s)
                : quantize_v<T, decltype(w), decltype(v)::value, false>(a, group, codes, scales, s);
  });
}

cudaError_t launch_rms_norm_8bit(const NormArgs& a, bool int8, int group, uint8_t* codes,
                                 float* scales, cudaStream_t s) {
  if (a.dtype == EXF_F32) return quantize_t<float>(a, int8, group, codes, scales, s);
  if (a.dtype == EXF_BF16) return quantize_t<__nv_bfloat16>(a, int8, group, codes, scales, s);
  return quantize_t<__half>(a, int8, group, codes, scales, s);
}

cudaError_t launch_dequantize_8bit(const uint8_t* codes, bool int8, const float* scales,
                                   int64_t rows, int cols, int group, void* out, int dtype,
                                   cudaStream_t s) {
  const int64_t total = rows * cols;
  const int shift = group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 31;
  const int groups = group ? (cols + group - 1) / group : 1;
  auto run = [&](auto* kern, auto* o) {
    const unsigned grid = stay_grid(reinterpret_cast<const void*>(kern), 256, 0, (total + 4095) / 4096);
    return launch_pdl(kern, dim3(grid), dim3(256), 0, s, codes, scales, total, cols, shift, groups,
                      o);
  };
  auto go = [&](auto* o) {
    using T = std::remove_pointer_t<decltype(o)>;
    return int8 ? run(dequantize_8bit_kernel<T, true>, o) : run(dequantize_8bit_kernel<T, false>, o);
  };
  if (dtype == EXF_F32) return go(static_cast<float*>(out));
  if (dtype == EXF_BF16) return go(static_cast<__nv_bfloat16*>(out));
  return go(static_cast<__half*>(out));
}

}  // namespace exf
