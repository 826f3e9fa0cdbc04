// Root-mean-square norm with its output in 8 bits and scales, and reading it back (sm_100a).
//
//   s = round(x + residual) (or x),  v = 1 / sqrt(mean s^2 + eps),  p_j = s_j w_j
//   a group of 32, 64 or 128 columns (or the row) has top = max |p_j|
//   code_j = p_j M / top, rounded to the nearest e4m3 (M = 448) or integer (M = 127), ties to even
//   scale = top v / M, so that code scale is the norm's s_j v w_j
//
// v is the same for the row, so the codes do not depend on its rounding.  A code is decided in fp32 unless
// the quotient lies within its rounding of a border between two codes; there p M and border top are
// compared in 64 bits, where the products are exact (fp32 inputs with fp32 weights: to 2^-53), so equal
// inputs give the codes of the definition.  fp32 inputs or weights have products of more than 24 bits:
// their largest is taken in 64 bits.  A group with a product that is not finite in fp32 gets codes 0 and
// a NaN scale, a group of zeros codes 0 and scale 0.
//
// Bound by memory: x, residual in, sum and codes out, once each.
#include <mutex>

#include "exf_launch.h"
#include "exf_norm.cuh"

namespace exf {

// the largest magnitude as bits: integers compare as the values do, infinities and NaN above all
template <bool EXACT>
struct TopOf {
  using Bits = uint32_t;
};
template <>
struct TopOf<false> {
  using Bits = unsigned long long;
};
template <bool EXACT>
__device__ __forceinline__ typename TopOf<EXACT>::Bits product_bits(float s, float w) {
  if constexpr (EXACT)
    return __float_as_uint(s * w) & 0x7fffffffu;
  else
    return (unsigned long long)__double_as_longlong((double)s * (double)w) & 0x7fffffffffffffffull;
}
template <bool EXACT>
__device__ __forceinline__ double top_value(typename TopOf<EXACT>::Bits b) {
  if constexpr (EXACT)
    return (double)__uint_as_float(b);
  else
    return __longlong_as_double((long long)b);
}

struct Quantum {
  float m;     // M / top, or 0
  float f;     // a power of two that keeps small groups inside fp32's range
  float scale;
  double top;
};

template <bool EXACT>
__device__ __forceinline__ Quantum quantum_of(typename TopOf<EXACT>::Bits bits, float v, bool int8) {
  Quantum z;
  z.top = top_value<EXACT>(bits);
  const float most = int8 ? 127.0f : 448.0f;
  const float top = (float)z.top;
  z.f = top < 0x1p-100f ? 0x1p64f : 1.0f;
  const float scaled = (float)(z.top * (double)z.f);
  z.m = scaled > 0.0f ? most / scaled : 0.0f;
  z.scale = top * v / most;
  if (!(top < __int_as_float(0x7f800000))) {
    z.m = 0.0f;
    z.scale = __int_as_float(0x7fc00000);
  }
  return z;
}

// The quotient p m, its value moved to the right code where it lies at a border.  It is off by up to 4
// steps of 2^-24 relative (top, M / top, p and the product, each rounded once), 5 in the last place with
// the shift of small values; product() is p in 64 bits.
template <typename F>
__device__ __forceinline__ float to_code(float p, const Quantum& z, bool int8, F product) {
  float q = p * z.f * z.m;
  const float a = fabsf(q);
  if (int8) {
    const float t = rintf(a);
    if (fabsf(fabsf(a - t) - 0.5f) < 4e-5f) {
      const float low = floorf(a);
      const double side = fabs(product()) * 127.0 - (double)(low + 0.5f) * z.top;
      const bool up = side > 0.0 || (side == 0.0 && ((int)low & 1));
      return copysignf(low + (up ? 1.0f : 0.0f), q);
    }
    return copysignf(t, q);
  }
  // e4m3: three bits behind the leading one, multiples of 2^-9 below 2^-6
  const float shift = a < 0x1p-6f ? 0x1p-6f : 0.0f;
  const uint32_t b = __float_as_uint(a + shift);
  if (((b - 0x7fff8u) & 0xfffffu) < 16u) {
    const float low = __uint_as_float(b & 0xfff00000u);
    const float high = __uint_as_float((b & 0xfff00000u) + 0x100000u);
    const float mid = __uint_as_float((b & 0xfff00000u) + 0x80000u);
    const double side = fabs(product()) * 448.0 - (double)(mid - shift) * z.top;
    const bool up = side > 0.0 || (side == 0.0 && (b & 0x100000u));
    q = copysignf((up ? high : low) - shift, q);
  }
  return q;
}

__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {  // a in the low byte
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

template <int V>
__device__ __forceinline__ void store_codes(uint8_t* at, const float (&q)[V], bool int8) {
  uint32_t word[(V + 3) / 4];
#pragma unroll
  for (int i = 0; i < (V + 3) / 4; ++i) {
    word[i] = 0;
#pragma unroll
    for (int j = 0; j < 4 && 4 * i + j < V; j += 2) {
      const float a = q[4 * i + j], b = 4 * i + j + 1 < V ? q[4 * i + j + 1 < V ? 4 * i + j + 1 : 0] : 0.0f;
      const uint32_t two = int8 ? ((uint32_t)(int)a & 255u) | ((uint32_t)(int)b & 255u) << 8
                                : e4m3_pair(a, b);
      word[i] |= two << (8 * j);
    }
  }
  if constexpr (V == 8)
    *reinterpret_cast<uint2*>(at) = make_uint2(word[0], word[1]);
  else if constexpr (V == 4)
    *reinterpret_cast<uint32_t*>(at) = word[0];
  else
    *at = (uint8_t)word[0];
}

// Layout as rms_norm_kernel, with at least a warp a row.  group 0: the row.  With vectors, a group's units
// lie in neighbouring lanes (4 to 32 of them); with single elements the groups' largest are kept in shared
// memory ([rows of the block][groups]).
template <typename T, int V, int NV, bool EXACT>
__global__ void __launch_bounds__(1024)
    rms_norm_8bit_kernel(const NormArgs a, int g, bool int8, int group, uint8_t* codes,
                         float* scales) {
  using Bits = typename TopOf<EXACT>::Bits;
  __shared__ float part[32];
  __shared__ double part64[32];
  __shared__ Bits part_top[32];
  extern __shared__ unsigned long long group_raw[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_block = blockDim.x / g;
  const int sub = threadIdx.x / g, t = threadIdx.x % g;
  const int64_t row = (int64_t)blockIdx.x * per_block + sub;
  const bool live = row < a.rows;
  const int64_t at = live ? row : 0;
  const T* x = static_cast<const T*>(a.x) + at * a.x_stride;
  const T* r = a.residual ? static_cast<const T*>(a.residual) + at * a.r_stride : nullptr;
  T* sum_out = a.residual && live ? static_cast<T*>(a.sum) + row * a.cols : nullptr;
  const int units = a.cols / V;
  const int groups = group ? (a.cols + group - 1) / group : 1;
  Bits* tops = reinterpret_cast<Bits*>(group_raw) + (size_t)sub * groups;
  const bool shared_tops = V == 1 && group != 0;
  if (shared_tops) {
    for (int i = t; i < groups; i += g) tops[i] = 0;
    __syncthreads();
  }

  // p = s w of a unit, in p; the unit's largest, and (first time) its squares
  float q = 0.0f;
  auto take = [&](int u, float (&p)[V], bool first) {
    float w[V];
    Bits top = 0;
    if (u < units) {
      load_sum<T, V>(x + u * V, r ? r + u * V : nullptr, p);
      load_weight<T, V>(a.weight, a.weight_f32, u * V, w);
      if (first && sum_out) store_pack<T, V>(sum_out + u * V, p);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (first) q = fmaf(p[j], p[j], q);
        const Bits b = product_bits<EXACT>(p[j], w[j]);
        top = b > top ? b : top;
        p[j] = p[j] * w[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) p[j] = 0.0f;
    }
    return top;
  };
  // the largest of a unit's group: V > 1, by the lanes that share it
  auto of_group = [&](Bits top) {
    for (int d = group / V / 2; d > 0; d >>= 1) {
      const Bits o = __shfl_xor_sync(0xffffffffu, top, d);
      top = o > top ? o : top;
    }
    return top;
  };

  constexpr int N = NV > 0 ? NV : 1;
  float p[N][V];
  Bits top[N];
  Bits all = 0;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) top[i] = take(t + g * i, p[i], true);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      all = top[i] > all ? top[i] : all;
      if (shared_tops && t + g * i < units) atomicMax(tops + (t + g * i) / group, top[i]);
    }
  } else {
    for (int u = t; u < units; u += g) {
      const Bits b = take(u, p[0], true);
      all = b > all ? b : all;
      if (shared_tops) atomicMax(tops + u / group, b);
    }
  }
  // (the shared maxima are complete behind one of its barriers where a row has several warps)
  const float v = inverse_norm(q, a, g, part, part64, [&] {
    double d = 0.0;
    for (int u = t; u < units; u += g) {
      float e[V];
      load_sum<T, V>(x + u * V, r ? r + u * V : nullptr, e);
#pragma unroll
      for (int j = 0; j < V; ++j) d = fma((double)e[j], (double)e[j], d);
    }
    return d;
  });
  if (group == 0) {
    all = row_max(all, g, part_top);
  } else if (shared_tops) {
    __syncthreads();
  }

  auto finish = [&](int u, float (&e)[V], Bits b) {
    const bool in = u < units;
    if (group == 0)
      b = all;
    else if (V > 1)
      b = of_group(b);
    else if (in)
      b = tops[u / group];
    if (!in || !live) return;
    const Quantum z = quantum_of<EXACT>(b, v, int8);
    const int c = u * V;
    if (group == 0 ? c == 0 : c % group == 0) scales[row * groups + (group ? c / group : 0)] = z.scale;
#pragma unroll
    for (int j = 0; j < V; ++j)
      e[j] = to_code(e[j], z, int8, [&] {
        if constexpr (EXACT) return (double)e[j];
        float one[1], w[1];
        load_sum<T, 1>(x + c + j, r ? r + c + j : nullptr, one);
        load_weight<T, 1>(a.weight, a.weight_f32, c + j, w);
        return (double)one[0] * (double)w[0];
      });
    store_codes<V>(codes + row * a.cols + c, e, int8);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) finish(t + g * i, p[i], top[i]);
  } else {
    for (int u0 = 0; u0 < units; u0 += g) {  // (every lane goes along: lanes share their maxima)
      const Bits b = take(u0 + t, p[0], false);
      finish(u0 + t, p[0], b);
    }
  }
}

// ---- reading back -------------------------------------------------------------------------------
// out = code * scale, rounded.  A thread takes 8 values that lie together, whichever rows they belong to,
// so every access is a whole vector whatever the row's length.
template <typename T>
__global__ void __launch_bounds__(256)
    dequantize_8bit_kernel(const uint8_t* codes, bool int8, const float* scales, int64_t total,
                           int cols, int shift, int groups, T* out) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  auto value = [&](uint32_t code) {
    if (int8) return (float)(int8_t)(uint8_t)code;
    uint32_t two;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"((uint16_t)code));
    return __half2float(__ushort_as_half((unsigned short)two));
  };
  const int64_t step = (int64_t)gridDim.x * blockDim.x * 8;
  for (int64_t f = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8; f < total; f += step) {
    int64_t row;
    if (total <= 0xffffffffll)
      row = (uint32_t)f / (uint32_t)cols;
    else
      row = f / cols;
    int c = (int)(f - row * cols);
    const int n = total - f < 8 ? (int)(total - f) : 8;
    uint32_t word[2] = {0, 0};
    if (n == 8) {
      const uint2 k = *reinterpret_cast<const uint2*>(codes + f);
      word[0] = k.x;
      word[1] = k.y;
    } else {
      for (int j = 0; j < n; ++j) word[j >> 2] |= (uint32_t)codes[f + j] << (8 * (j & 3));
    }
    float e[8];
    float scale = scales[row * groups + (c >> shift)];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < n) {
        if (c == cols) {
          c = 0;
          ++row;
        }
        if (j > 0 && (c & ((1ll << shift) - 1)) == 0) scale = scales[row * groups + (c >> shift)];
        e[j] = value(word[j >> 2] >> (8 * (j & 3)) & 255u) * scale;
        ++c;
      }
    }
    if (n == 8) {
      if constexpr (sizeof(T) == 2) {
        store_pack<T, 8>(out + f, e);
      } else {
        const float lo[4] = {e[0], e[1], e[2], e[3]}, hi[4] = {e[4], e[5], e[6], e[7]};
        store_pack<T, 4>(out + f, lo);
        store_pack<T, 4>(out + f + 4, hi);
      }
    } else {
      for (int j = 0; j < n; ++j) out[f + j] = from_f32<T>(e[j]);
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------
template <typename T, int V, bool EXACT>
static cudaError_t quantize_v(const NormArgs& a, bool int8, int group, uint8_t* codes,
                              float* scales, cudaStream_t s) {
  const int64_t units = a.cols / V;
  const int per = a.rows < 296 ? 1 : V > 1 ? 2 : 4;
  const int g = norm_threads(units, per, 32);
  const int block = g <= 32 ? 128 : g;
  const int per_block = block / g;
  const int64_t grid = (a.rows + per_block - 1) / per_block;
  const int need = (int)((units + g - 1) / g);
  const int groups = group ? (a.cols + group - 1) / group : 1;
  const size_t smem = V == 1 && group ? (size_t)per_block * groups * (EXACT ? 4 : 8) : 0;
  auto go = [&](auto* kern) {
    return launch_pdl(kern, dim3((unsigned)grid), dim3(block), smem, s, a, g, int8, group, codes,
                      scales);
  };
  if (need <= 1) return go(rms_norm_8bit_kernel<T, V, 1, EXACT>);
  if (V > 1 && need <= 2) return go(rms_norm_8bit_kernel<T, V, 2, EXACT>);
  if (V == 1 && need <= 4) return go(rms_norm_8bit_kernel<T, V, (V > 1 ? 1 : 4), EXACT>);
  return go(rms_norm_8bit_kernel<T, V, 0, EXACT>);
}

template <typename T>
static cudaError_t quantize_t(const NormArgs& a, bool int8, int group, uint8_t* codes,
                              float* scales, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool vectors = norm_vectors<T>(a) && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
  if (sizeof(T) == 2 && !a.weight_f32)  // products of 22 bits at most
    return vectors ? quantize_v<T, V, sizeof(T) == 2>(a, int8, group, codes, scales, s)
                   : quantize_v<T, 1, sizeof(T) == 2>(a, int8, group, codes, scales, s);
  return vectors ? quantize_v<T, V, false>(a, int8, group, codes, scales, s)
                 : quantize_v<T, 1, false>(a, int8, group, codes, scales, s);
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
  int64_t blocks = (total + 2047) / 2048;
  const int64_t most = 16 * (int64_t)(sm_count() > 0 ? sm_count() : 1);
  if (blocks > most) blocks = most;
  const int shift = group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 31;
  const int groups = group ? (cols + group - 1) / group : 1;
  auto go = [&](auto* o) {
    return launch_pdl(dequantize_8bit_kernel<std::remove_pointer_t<decltype(o)>>,
                      dim3((unsigned)blocks), dim3(256), 0, s, codes, int8, scales, total, cols,
                      shift, groups, o);
  };
  if (dtype == EXF_F32) return go(static_cast<float*>(out));
  if (dtype == EXF_BF16) return go(static_cast<__nv_bfloat16*>(out));
  return go(static_cast<__half*>(out));
}

}  // namespace exf
