// The MXFP4 expert layer for a few routes (single tokens): FMA kernels over the routes as they come, no
// moe_align, no two-term form, no combine.  Two launches:
//   gate: h[r][f] = silu(W1[e] x) * (W3[e] x), a warp a route and feature (a gate and an up row);
//   down: y[t][c] = sum_j w[t, j] W2[e][c] h[r], a warp a token and column, over all its routes.
// A lane takes one scale block (32 codes, 16 bytes) at a time: the codes become fp32 values (e2m1 to
// fp16 by conversion, exact), the dot product with 32 activations is taken in fp32 and multiplied by
// the block's power of two.  h is fp32.  Every SM streams weights from the first microsecond; the tensor
// path has 48 tiles for one token and spends 10 us in moe_align and the combine.  Bound by latency, then
// by the FMA pipe (about 2.5 instructions a weight), so it serves up to kMxFewRoutes routes: EXF_FEW.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "exf_common.cuh"
#include "exf_launch.h"
#include "exf_mx.cuh"
#include "exf_mxmoe.h"

namespace exf {

constexpr int kFewWarps = 8;

// 8 codes -> their values (exact in fp16)
__device__ __forceinline__ void code_values(uint32_t codes, float (&f)[8]) {
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
__device__ __forceinline__ float block_scale(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fffffffu : byte == 0u ? 0x00400000u : byte << 23);
}
// the scale byte of a weight row's block b: tiles of 128 rows x 4 blocks
__device__ __forceinline__ uint32_t tiled_scale(const uint8_t* s, int row, int kblocks, int b) {
  return __ldg(s + ((int64_t)(row >> 7) * kblocks + (b >> 2)) * 512 + (row & 31) * 16 +
               ((row >> 5) & 3) * 4 + (b & 3));
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__global__ void __launch_bounds__(32 * kFewWarps)
    mx_few_gate_kernel(const __nv_bfloat16* __restrict__ x, const int32_t* ids,
                       const uint8_t* __restrict__ w13, const uint8_t* __restrict__ s13,
                       int experts, int top_k, int hidden, int inter, float* h) {
  // waits for the launches before it, then lets the down kernel start (which may therefore read
  // what those wrote before it waits for this one)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int route = blockIdx.y;
  const int f = blockIdx.x * kFewWarps + (threadIdx.x >> 5);
  const int e = ids[route];
  if (e < 0 || e >= experts || f >= inter) return;
  const int gate = e * 2 * inter + f, up = gate + inter;
  const uint4* cg = reinterpret_cast<const uint4*>(w13 + (int64_t)gate * (hidden / 2));
  const uint4* cu = reinterpret_cast<const uint4*>(w13 + (int64_t)up * (hidden / 2));
  const uint4* xr = reinterpret_cast<const uint4*>(x + (int64_t)(route / top_k) * hidden);
  const int kblocks = hidden / kMxK;
  float g = 0.0f, u = 0.0f;
#pragma unroll 2
  for (int b = lane; b < hidden / 32; b += 32) {
    const uint4 a = __ldg(cg + b), c = __ldg(cu + b);
    const uint32_t sg = tiled_scale(s13, gate, kblocks, b), su = tiled_scale(s13, up, kblocks, b);
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, cw[4] = {c.x, c.y, c.z, c.w};
    float dg = 0.0f, du = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = __ldg(xr + 4 * b + i);
      const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
      float fg[8], fu[8];
      code_values(aw[i], fg);
      code_values(cw[i], fu);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float xv = __uint_as_float((j & 1) ? vw[j >> 1] & 0xffff0000u : vw[j >> 1] << 16);
        dg = fmaf(xv, fg[j], dg);
        du = fmaf(xv, fu[j], du);
      }
    }
    g = fmaf(dg, block_scale(sg), g);
    u = fmaf(du, block_scale(su), u);
  }
  g = warp_sum(g);
  u = warp_sum(u);
  if (lane == 0) h[(int64_t)route * inter + f] = __fdividef(g, 1.0f + __expf(-g)) * u;
}

__global__ void __launch_bounds__(32 * kFewWarps)
    mx_few_down_kernel(const float* h, const float* route_w, const int32_t* ids,
                       const uint8_t* __restrict__ w2, const uint8_t* __restrict__ s2, int experts,
                       int top_k, int hidden, int inter, __nv_bfloat16* y) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t t = blockIdx.y;
  const int col = blockIdx.x * kFewWarps + (threadIdx.x >> 5);
  // routes and weights were there before the gate kernel started: they are read while it runs
  const int mine = lane < top_k ? __ldcg(ids + t * top_k + lane) : -1;
  const uint32_t use = __ballot_sync(0xffffffffu, mine >= 0 && mine < experts);
  const int kblocks = inter / kMxK;
  const int blocks = inter / 32;
  float acc = 0.0f;
  for (int b0 = 0; b0 < blocks; b0 += 32) {
    const int b = b0 + lane;
    uint4 c[8];
    uint32_t s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!((use >> j) & 1)) continue;
      const int row = __shfl_sync(0xffffffffu, mine, j) * hidden + col;
      if (b < blocks) {
        c[j] = __ldg(reinterpret_cast<const uint4*>(w2 + (int64_t)row * (inter / 2)) + b);
        s[j] = tiled_scale(s2, row, kblocks, b);
      }
    }
    if (b0 == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!((use >> j) & 1) || b >= blocks) continue;
      const int64_t route = t * top_k + j;
      const float4* hr = reinterpret_cast<const float4*>(h + route * inter + 32 * b);
      const uint32_t cw[4] = {c[j].x, c[j].y, c[j].z, c[j].w};
      float d = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 p = __ldcg(hr + 2 * i), q = __ldcg(hr + 2 * i + 1);
        float fv[8];
        code_values(cw[i], fv);
        d = fmaf(p.x, fv[0], d);
        d = fmaf(p.y, fv[1], d);
        d = fmaf(p.z, fv[2], d);
        d = fmaf(p.w, fv[3], d);
        d = fmaf(q.x, fv[4], d);
        d = fmaf(q.y, fv[5], d);
        d = fmaf(q.z, fv[6], d);
        d = fmaf(q.w, fv[7], d);
      }
      acc = fmaf(d * block_scale(s[j]), route_w[route], acc);
    }
  }
  acc = warp_sum(acc);
  if (lane == 0) y[t * hidden + col] = __float2bfloat16_rn(acc);
}

cudaError_t launch_mx_few(const MxArgs& a, float* h, cudaStream_t s) {
  const int numel = (int)(a.tokens * a.top_k);
  const unsigned fx = (unsigned)((a.inter + kFewWarps - 1) / kFewWarps);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(32 * kFewWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(fx, (unsigned)numel);
  cudaError_t e = cudaLaunchKernelEx(&cfg, mx_few_gate_kernel,
                                     static_cast<const __nv_bfloat16*>(a.x), a.topk_ids, a.w13,
                                     a.s13, a.experts, a.top_k, a.hidden, a.inter, h);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3((unsigned)(a.hidden / kFewWarps), (unsigned)a.tokens);
  e = cudaLaunchKernelEx(&cfg, mx_few_down_kernel, static_cast<const float*>(h), a.topk_w,
                         a.topk_ids, a.w2, a.s2, a.experts, a.top_k, a.hidden, a.inter,
                         static_cast<__nv_bfloat16*>(a.y));
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace exf
