// 16-bit operands of the tensor-core kernels (bf16 or fp16): packing, the epilogues' stores, two-term splits.
// Used by gated_mlp.cu and adapters.cu.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "exf_tc.cuh"

namespace exf {
using tc::pack_bf16;

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) return pack_bf16(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ void store_16b(void* base, int64_t at, const float* v) {
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) =
      make_uint4(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]), pack2<BF16>(v[4], v[5]),
                 pack2<BF16>(v[6], v[7]));
}

// 16 results, 32 bytes: one store of a whole sector where `wide` says that rows keep its alignment
// (a row a thread, two 16-byte stores cost L2 a partial write each), the last 8 columns only if n1
template <bool BF16>
__device__ __forceinline__ void store_32b(void* base, int64_t at, const float* v, bool wide,
                                          bool n1) {
  if (wide && n1) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = pack2<BF16>(v[2 * j], v[2 * j + 1]);
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                     static_cast<uint16_t*>(base) + at),
                 "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]),
                 "r"(w[7])
                 : "memory");
  } else {
    store_16b<BF16>(base, at, v);
    if (n1) store_16b<BF16>(base, at + 8, v + 8);
  }
}
// 8 fp32 sums, 32-byte aligned
__device__ __forceinline__ void store_sums(float* at, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "f"(v[0]),
               "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// what rounding v to the operand type leaves; 0 where it overflows to an infinity or is one
template <bool BF16>
__device__ __forceinline__ float remainder_of(float v) {
  const float2 r = unpack2<BF16>(pack2<BF16>(v, 0.0f));
  return fabsf(r.x) < __int_as_float(0x7f800000) ? v - r.x : 0.0f;
}

}  // namespace exf
