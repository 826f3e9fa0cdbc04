// Root-mean-square norm with its output in 8 bits and scales, and reading it back (sm_100a).
//
//   s = round(x + residual) (or x),  v = 1 / sqrt(mean s^2 + eps),  p_j = s_j w_j
//   a group of 32, 64 or 128 columns (or the row) has top = max |p_j|
//   code_j = p_j M / top, rounded to the nearest e4m3 (M = 448) or integer (M = 127), ties to even
//   scale = top v / M, so that code scale is the norm's s_j v w_j
//
// v is the same for the row, so the codes do not depend on its rounding: equal inputs give the codes of the
// definition (products of fp32 values with fp32 weights to 2^-53).  A group with a product that is not
// finite in fp32 gets codes 0 and a NaN scale, a group of zeros codes 0 and scale 0.
//
// Bound by memory: x, residual in, sum and codes out, once each.
#include <mutex>

#include "exf_launch.h"
#include "exf_norm.cuh"

namespace exf {

// ---- the largest product of a group ----------------------------------------------------------------
// Kept as an integer that compares as the magnitudes do, infinities and NaN above all.  Products of 16-bit
// values are exact in fp32 (EXACT): the bits.  Others: the rounded product's bits and, below them, what the
// rounding left, its order made that of unsigned integers.
template <bool EXACT>
struct Top;
template <>
struct Top<true> {
  using Key = uint32_t;
  static __device__ __forceinline__ Key of(float s, float w) {
    return __float_as_uint(s * w) & 0x7fffffffu;
  }
  static __device__ __forceinline__ float rounded(Key k) { return __uint_as_float(k); }
  static __device__ __forceinline__ double value(Key k) { return (double)__uint_as_float(k); }
};
template <>
struct Top<false> {
  using Key = unsigned long long;
  static __device__ __forceinline__ Key of(float s, float w) {
    const float a = fabsf(s), b = fabsf(w), p = a * b;
    const uint32_t rest = __float_as_uint(fmaf(a, b, -p));
    const uint32_t order = rest ^ ((uint32_t)((int32_t)rest >> 31) | 0x80000000u);
    return (Key)(__float_as_uint(p) & 0x7fffffffu) << 32 | order;
  }
  static __device__ __forceinline__ float rounded(Key k) { return __uint_as_float((uint32_t)(k >> 32)); }
  static __device__ __forceinline__ double value(Key k) {
    const uint32_t order = (uint32_t)k;
    const uint32_t rest = order & 0x80000000u ? order ^ 0x80000000u : ~order;
    return k ? (double)rounded(k) + (double)__uint_as_float(rest) : 0.0;
  }
};

// ---- codes --------------------------------------------------------------------------------------------
// A group's factors: quotients p M / top are taken with M / top a little too small and a little too large.
// Where both give the same code it is the definition's (2^-21 to either side; the rounded top, the division
// and the product are off by 4 steps of 2^-24 together).  Else, one value in 2^16, and for all values of a
// group below 2^-100, the quotient is taken in 64 bits, where its distance from a border shows.
struct Quantum {
  float low, high, scale;
  bool all;  // in 64 bits
};
__device__ __forceinline__ Quantum quantum_of(float top, float v, float most) {
  Quantum z;
  const float m = top > 0.0f ? most / top : 0.0f;
  z.low = m * (1.0f - 0x1p-21f);
  z.high = m * (1.0f + 0x1p-21f);
  z.scale = top * v / most;
  z.all = top < 0x1p-100f && top > 0.0f;
  if (!(top < __int_as_float(0x7f800000))) {
    z.low = z.high = 0.0f;
    z.scale = __int_as_float(0x7fc00000);
  }
  return z;
}
// the value of the code of p = s w, in 64 bits
template <bool INT8>
__device__ __noinline__ float code_64(float s, float w, double top) {
  const double q = fabs((double)s * (double)w) * (INT8 ? 127.0 : 448.0) / top;
  double unit = 1.0;
  if (!INT8) {  // three bits behind the leading one, multiples of 2^-9 below 2^-6
    int e = (int)((unsigned long long)__double_as_longlong(q) >> 52) - 1023;
    e = e < -6 ? -6 : e;
    unit = __longlong_as_double((long long)(e - 3 + 1023) << 52);
  }
  return copysignf((float)(rint(q / unit) * unit), s * w);
}
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {  // a in the low byte
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// The codes of up to four products, the first in the low byte.  Integers: rounded by adding 1.5 2^23, whose
// low byte they become.
template <bool INT8, int N>
__device__ __forceinline__ uint32_t code_word(const float (&p)[N], float m) {
  uint32_t b[4] = {0, 0, 0, 0};
  if (INT8) {
#pragma unroll
    for (int j = 0; j < N; ++j) b[j] = __float_as_uint(fmaf(p[j], m, 12582912.0f));
    uint32_t lo = b[0], hi = b[2];
    if (N > 1) lo = __byte_perm(b[0], b[1], 0x0040);
    if (N > 2) hi = __byte_perm(b[2], b[3], 0x0040);
    return N > 2 ? __byte_perm(lo, hi, 0x5410) : N > 1 ? lo & 0xffffu : lo & 0xffu;
  }
  uint32_t lo = e4m3_pair(p[0] * m, N > 1 ? p[N > 1 ? 1 : 0] * m : 0.0f), hi = 0;
  if (N > 2) hi = e4m3_pair(p[N > 2 ? 2 : 0] * m, p[N > 2 ? 3 : 0] * m);
  return lo | hi << 16;
}
template <bool INT8, bool EXACT, int N, typename S, typename W>
__device__ __forceinline__ uint32_t codes_of(S s, W w, const Quantum& z,
                                             typename Top<EXACT>::Key top) {
  if (z.scale != z.scale) return 0;
  float p[N];
#pragma unroll
  for (int j = 0; j < N; ++j) p[j] = s(j) * w(j);
  uint32_t low = code_word<INT8, N>(p, z.low);
  const uint32_t high = code_word<INT8, N>(p, z.high);
  if (low != high || z.all) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (!z.all && ((low ^ high) >> (8 * j) & 255u) == 0) continue;
      const float q = code_64<INT8>(s(j), w(j), Top<EXACT>::value(top));
      const uint32_t c = (INT8 ? (uint32_t)(int)q : e4m3_pair(q, 0.0f)) & 255u;
      low = (low & ~(255u << (8 * j))) | c << (8 * j);
    }
  }
  return low;
}

// ---- the kernel -----------------------------------------------------------------------------------------
// Blocks that stay, as rms_norm_kernel's, with at least a warp a row.  The largest products are taken with
// the loads' results; 32 columns lie on 32 / V neighbouring lanes.  Vectors: a group is 1 to 4 such runs, so
// its lanes find its largest among them.  Else (V <= 2) a run's largest goes to the group's word in shared
// memory (three sets of words: one is filled, one read, one zeroed), and where an odd row's units begin one
// column early, the run's first element goes to its own group.  group 0: the row, reduced beside the sum
// of squares.
template <typename T, typename W, int V, int NU, int THREADS, bool INT8>
__global__ void __launch_bounds__(THREADS)
    rms_norm_8bit_kernel(const NormArgs a, int g, int group, uint8_t* codes, float* scales) {
  constexpr bool EXACT = sizeof(T) == 2 && sizeof(W) == 2;
  using Key = typename Top<EXACT>::Key;
  constexpr int kRun = 32 / V;
  __shared__ float part[2][32];
  __shared__ double part64[32];
  __shared__ Key part_top[2][32];
  extern __shared__ unsigned long long words[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_block = blockDim.x / g;
  const int sub = threadIdx.x / g, t = threadIdx.x % g;
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.residual);
  T* sum = static_cast<T*>(a.sum);
  const int64_t step = (int64_t)gridDim.x * per_block;
  const int64_t first = (int64_t)blockIdx.x * per_block;
  int64_t row = first + sub;
  const int groups = group ? (a.cols + group - 1) / group : 1;
  constexpr float kMost = INT8 ? 127.0f : 448.0f;
  Key* tops = reinterpret_cast<Key*>(words) + (size_t)sub * 3 * groups;
  const bool shared_tops = V <= 2 && group != 0;

  Pack<T, V> nx[NU], nr[NU], s[NU];
  Weights<W, V, NU> w;
  auto shift_of = [&](int64_t at) { return V == 2 ? (int)at & a.cols & 1 : 0; };
  auto fetch = [&](int64_t at) {
    const int shift = shift_of(at), units = units_of<V>(a.cols, shift);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = t + g * i;
      if (u < units && at < a.rows) {
        read_unit<T, V>(nx[i], x + at * a.x_stride, u, a.cols, shift);
        if (r) read_unit<T, V>(nr[i], r + at * a.r_stride, u, a.cols, shift);
      } else {
        nx[i].clear();
        nr[i].clear();
      }
    }
  };
  fetch(row);
  w.init(a.weight, t, g, a.cols);
  if (shared_tops) {
    for (int i = t; i < groups; i += g) tops[i] = 0;
    if (g > 32)
      __syncthreads();
    else
      __syncwarp();
  }
  int b = 0, set = 0;
  for (int64_t base = first; base < a.rows; base += step, row += step, b ^= 1) {
    const bool live = row < a.rows;
    const int64_t at = row * a.cols;
    const int shift = shift_of(row), units = units_of<V>(a.cols, shift);
    Key* here = tops + set * groups;
    set = set == 2 ? 0 : set + 1;
    if (shared_tops)
      for (int i = t; i < groups; i += g) tops[set * groups + i] = 0;
    float q = 0.0f;
    Key top[NU], all = 0;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = t + g * i;
      s[i] = r ? rounded_sum<T, V>(nx[i], nr[i]) : nx[i];
      const Pack<W, V> k = w.of(a.weight, i, u, a.cols, shift);
      Key one[V], most = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        q = fmaf(s[i].get(j), s[i].get(j), q);
        one[j] = u < units ? Top<EXACT>::of(s[i].get(j), k.get(j)) : 0;
        if (j > 0 || !shared_tops || !shift || t % kRun != 0)
          most = one[j] > most ? one[j] : most;
      }
      if (shared_tops) {
#pragma unroll
        for (int d = kRun / 2; d > 0; d >>= 1) {
          const Key o = __shfl_xor_sync(0xffffffffu, most, d);
          most = o > most ? o : most;
        }
        if (t % kRun == 0 && u < units) {
          const int c = u * V;
          if (c < a.cols) atomicMax(here + c / group, most);
          if (shift && c > 0) atomicMax(here + (c - 1) / group, one[0]);
        }
      }
      top[i] = most;
      all = most > all ? most : all;
    }
    fetch(row + step);
    if (r && live) {
#pragma unroll
      for (int i = 0; i < NU; ++i)
        if (t + g * i < units) write_unit<T, V>(s[i], sum + at, t + g * i, a.cols, shift);
    }
    const int64_t mine = live ? row : 0;
    if (group == 0) {
      // (its barrier is the sum's: the partial maxima are written before it and read after it)
      all = warp_max(all, g < 32 ? g : 32);
      if (g > 32 && (threadIdx.x & 31) == 0) part_top[b][threadIdx.x >> 5] = all;
    }
    const float v = inverse_norm<T>(q, a, g, t, x + mine * a.x_stride,
                                    r ? r + mine * a.r_stride : nullptr, part[b], part64);
    if (group == 0 && g > 32) {
      const int lane = threadIdx.x & 31;
      all = warp_max(lane < (g >> 5) ? part_top[b][lane] : Key(0), 32);
    }
    if (g <= 32 && shared_tops) __syncwarp();
    float* row_scales = scales + row * groups;
    uint8_t* out = codes + at;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = t + g * i;
      s[i].anew();
      if constexpr (V > 2) {
        Key k = top[i];
        if (group == 0) {
          k = all;
        } else {
          for (int d = group / V / 2; d > 0; d >>= 1) {
            const Key o = __shfl_xor_sync(0xffffffffu, k, d);
            k = o > k ? o : k;
          }
        }
        if (u < units && live) {
          const Quantum z = quantum_of(Top<EXACT>::rounded(k), v, kMost);
          const Pack<W, V> e = w.of(a.weight, i, u, a.cols, shift);
          const int c = u * V;
          if (group == 0 ? c == 0 : c % group == 0) row_scales[group ? c / group : 0] = z.scale;
          uint32_t word[V / 4];
#pragma unroll
          for (int h = 0; h < V / 4; ++h)
            word[h] = codes_of<INT8, EXACT, 4>([&](int j) { return s[i].get(4 * h + j); },
                                               [&](int j) { return e.get(4 * h + j); }, z, k);
          if constexpr (V == 8)
            *reinterpret_cast<uint2*>(out + c) = make_uint2(word[0], word[V / 4 - 1]);
          else
            *reinterpret_cast<uint32_t*>(out + c) = word[0];
        }
      } else if (u < units && live) {
        const Pack<W, V> e = w.of(a.weight, i, u, a.cols, shift);
        const int c0 = u * V - shift;
        uint32_t code[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = c0 + j;
          code[j] = 0;
          if (c >= 0 && c < a.cols) {
            const Key k = group == 0 ? all : here[c / group];
            const Quantum z = quantum_of(Top<EXACT>::rounded(k), v, kMost);
            if (group == 0 ? c == 0 : c % group == 0) row_scales[group ? c / group : 0] = z.scale;
            code[j] = codes_of<INT8, EXACT, 1>([&](int) { return s[i].get(j); },
                                               [&](int) { return e.get(j); }, z, k);
          }
        }
        // (an odd row's units begin on even places of the codes too)
        if (V == 2 && c0 >= 0 && c0 + 1 < a.cols && reinterpret_cast<uintptr_t>(codes) % 2 == 0) {
          *reinterpret_cast<uint16_t*>(out + c0) = (uint16_t)(code[0] | code[V - 1] << 8);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (c0 + j >= 0 && c0 + j < a.cols) out[c0 + j] = (uint8_t)code[j];
        }
      }
    }
  }
}

// Rows of any length, read again after the reduction; a block a row.  The groups' largest products in shared
// memory.
template <typename T, typename W, bool INT8>
__global__ void __launch_bounds__(1024)
    rms_norm_8bit_long_kernel(const NormArgs a, int group, uint8_t* codes, float* scales) {
  constexpr bool EXACT = sizeof(T) == 2 && sizeof(W) == 2;
  using Key = typename Top<EXACT>::Key;
  __shared__ float part[32];
  __shared__ double part64[32];
  extern __shared__ unsigned long long words[];
  Key* tops = reinterpret_cast<Key*>(words);
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
  Key all = 0;
  for (int c0 = 0; c0 < a.cols; c0 += 1024) {  // a warp's 32 columns lie in one group
    const int c = c0 + threadIdx.x;
    Key k = 0;
    if (c < a.cols) {
      float s[1];
      load_sum<T, 1>(x + c, r ? r + c : nullptr, s);
      if (r) store_pack<T, 1>(static_cast<T*>(a.sum) + row * a.cols + c, s);
      q = fmaf(s[0], s[0], q);
      k = Top<EXACT>::of(s[0], to_f32<W>(w[c]));
    }
    if (group) {
      k = warp_max(k, 32);
      if ((threadIdx.x & 31) == 0 && c < a.cols) atomicMax(tops + c / group, k);
    } else {
      all = k > all ? k : all;
    }
  }
  if (!group) {
    all = warp_max(all, 32);
    if ((threadIdx.x & 31) == 0) atomicMax(tops, all);
  }
  // (behind a barrier of its own: the maxima are complete)
  const float v = inverse_norm<T>(q, a, 1024, threadIdx.x, x, r, part, part64);
  for (int c = threadIdx.x; c < a.cols; c += 1024) {
    float s[1];
    load_sum<T, 1>(x + c, r ? r + c : nullptr, s);
    const float e = to_f32<W>(w[c]);
    const Key k = tops[group ? c / group : 0];
    const Quantum z = quantum_of(Top<EXACT>::rounded(k), v, INT8 ? 127.0f : 448.0f);
    if (group == 0 ? c == 0 : c % group == 0) scales[row * groups + (group ? c / group : 0)] = z.scale;
    codes[row * a.cols + c] = (uint8_t)codes_of<INT8, EXACT, 1>(
        [&](int) { return s[0]; }, [&](int) { return e; }, z, k);
  }
}

// ---- reading back -------------------------------------------------------------------------------
// out = code * scale, rounded.  A thread takes 16 values that lie together, whichever rows they belong to,
// so every access is a whole vector whatever the row's length; most lie in one group, and need one scale.
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
  constexpr int NU = V > 2 ? 2 : 8;
  const size_t key = sizeof(T) == 2 && sizeof(W) == 2 ? 4 : 8;
  const int64_t units = V == 2 ? a.cols / 2 + 1 : a.cols / V;
  const int groups = group ? (a.cols + group - 1) / group : 1;
  if (units > 1024 * NU)
    return launch_pdl(rms_norm_8bit_long_kernel<T, W, INT8>, dim3((unsigned)a.rows), dim3(1024),
                      groups * key, s, a, group, codes, scales);
  const int g = norm_threads(units, a.rows <= 148 ? NU / 2 : NU, 32);
  const int block = g <= 32 ? 128 : g;
  const int per_block = block / g;
  const size_t smem = V <= 2 && group ? per_block * 3 * groups * key : 0;
  auto go = [&](auto* kern) {
    const unsigned grid = stay_grid(reinterpret_cast<const void*>(kern), block, smem,
                                    (a.rows + per_block - 1) / per_block);
    return launch_pdl(kern, dim3(grid), dim3(block), smem, s, a, g, group, codes, scales);
  };
  if (block <= 256) return go(rms_norm_8bit_kernel<T, W, V, NU, 256, INT8>);
  return go(rms_norm_8bit_kernel<T, W, V, NU, 1024, INT8>);
}

template <typename T>
static cudaError_t quantize_t(const NormArgs& a, bool int8, int group, uint8_t* codes,
                              float* scales, cudaStream_t s) {
  // (the codes need half the vectors' alignment at most)
  const NormUnit unit = norm_unit<T>(a);
  const bool whole = reinterpret_cast<uintptr_t>(codes) % 8 == 0;
  return norm_dispatch<T>(a, unit == kVector && !whole ? kSingle : unit, [&](auto w, auto v) {
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
