// The two-term 8-bit form of activations for the MXFP4 expert layer, and where its rows lie.
//
// An activation is the sum of two e4m3 terms with scales 2^-5 apart: over a block of 32 with the
// largest magnitude in [2^m, 2^(m+1)) and s = 2^(m-7),
//   hi = e4m3(v / s),  lo = e4m3(32 (v / s - hi)),  v = s hi + (s / 32) lo.
// hi keeps 4 significant bits and the remainder, below 2^-4 of v, keeps 4 more: a bf16 activation
// (8 bits) is represented exactly unless it is smaller than 2^-13 of its block's largest, where the
// error stays below 2^-22 of that; an fp32 value is rounded by at most 2^-9 of itself (half as much as by
// bf16).  s is at least 2^-122 (lo's scale byte is 5 below hi's), so that lo's smallest step is 2^-136:
// in blocks whose largest is below 2^-115 either may be off by 2^-137 instead.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace exf {

constexpr int kMxK = 128;          // k values of a scale table: 4 MMA steps, one 32-bit scale word
constexpr int kMxPrefillBlock = 128; // routes of a block at prefill; 16 or 32 at decode

// scale byte of a block from the bits of its largest magnitude: s = 2^(byte - 127); at least 5, so
// that lo's byte (5 less) exists; 255 (NaN) if the block holds an infinity or NaN
__device__ __forceinline__ uint32_t split_scale(uint32_t top_bits) {
  const int e = (int)(top_bits >> 23) - 7;
  return top_bits >= 0x7f800000u ? 255u : (uint32_t)(e > 5 ? e : 5);
}
__device__ __forceinline__ float split_inverse(uint32_t byte) {
  return __uint_as_float((254u - (byte == 255u ? 127u : byte)) << 23);
}
__device__ __forceinline__ uint32_t split_lo_byte(uint32_t byte) {
  return byte == 255u ? 255u : byte - 5u;
}
// two values -> hi and lo terms, the first in the low byte
__device__ __forceinline__ void split2(float a, float b, float inv, uint32_t& hi, uint32_t& lo) {
  const float2 v = make_float2(a * inv, b * inv);
  const __nv_fp8x2_storage_t h = __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
  const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
  hi = h;
  lo = __nv_cvt_float2_to_fp8x2(make_float2((v.x - f.x) * 32.0f, (v.y - f.y) * 32.0f),
                                __NV_SATFINITE, __NV_E4M3);
}

// Rows of a route block (of the two-term tensor and of the MMA's M side alike).  A block of 128: the
// hi rows, then the lo rows, an MMA tile each.  A smaller one is (part of) one tile: each 32-row
// quarter (the TMEM lanes of an epilogue warp) holds the hi rows of 16 routes, then their lo rows.
__device__ __forceinline__ int mx_row(int block, int r) {
  return block == kMxPrefillBlock ? r : 32 * (r >> 4) + (r & 15);
}
__host__ __device__ constexpr int mx_lo(int block) { return block == kMxPrefillBlock ? 128 : 16; }

// Scales of a route block: tables [k / 128][512], one per 128 MMA rows (two for a block of 128).
// Byte of row n and scale block kb; `table` is the route block's first.
__device__ __forceinline__ int64_t scale_at(int64_t table, int kblocks, int kb, int n) {
  return ((table + (n >> 7)) * kblocks + (kb >> 2)) * 512 + (n & 31) * 16 + ((n >> 5) & 3) * 4 +
         (kb & 3);
}
__host__ __device__ constexpr int scale_tables(int block) {
  return block == kMxPrefillBlock ? 2 : 1;
}

// 8 bf16 values (vector c of a row, c = the lane modulo 32) in the two-term form; the 4 lanes of a block
// of 32 together.  scales, lo_scales: the terms' scale bytes of the half warp's 4 blocks.
struct MxTerms {
  uint2 hi, lo;
  uint32_t scales, lo_scales;
};
__device__ __forceinline__ MxTerms split8(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    top = max(top, max((w[j] << 16) & 0x7fff0000u, w[j] & 0x7fff0000u));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  MxTerms t;
  const uint32_t scale = split_scale(top);
  const float inv = split_inverse(scale);
  t.scales = t.lo_scales = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = __shfl_sync(0xffffffffu, scale, (threadIdx.x & 16) + 4 * j);
    t.scales |= b << (8 * j);
    t.lo_scales |= split_lo_byte(b) << (8 * j);
  }
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    split2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u), inv, hi[j], lo[j]);
  t.hi = make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
  t.lo = make_uint2(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
  return t;
}
struct MxRows {
  uint8_t* xq;   // [blocks][2 * block][hidden]
  uint8_t* xs;   // [blocks][tables][hidden / 128][512]
  int hidden;
  int block;
};
// the hi row of a slot
__device__ __forceinline__ int mx_slot_row(int block, int slot) {
  const int blk = slot / block;
  return blk * 2 * block + mx_row(block, slot - blk * block);
}
// writes vector c of a token to the slot with that hi row
__device__ __forceinline__ void put8(const MxRows& o, int row, int c, const MxTerms& t) {
  uint8_t* hi = o.xq + (int64_t)row * o.hidden + 8 * c;
  *reinterpret_cast<uint2*>(hi) = t.hi;
  *reinterpret_cast<uint2*>(hi + mx_lo(o.block) * o.hidden) = t.lo;
  if ((c & 15) < 2) {  // a word of 4 blocks' scales: hi's, lo's
    const bool lo = c & 1;
    const int blk = row / (2 * o.block);
    const int n = row - blk * 2 * o.block + (lo ? mx_lo(o.block) : 0);
    *reinterpret_cast<uint32_t*>(o.xs + scale_at((int64_t)blk * scale_tables(o.block),
                                                 o.hidden / kMxK, (c >> 4) * 4, n)) =
        lo ? t.lo_scales : t.scales;
  }
}

}  // namespace exf
