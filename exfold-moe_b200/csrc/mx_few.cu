// The MXFP4 expert layer for a few routes (single tokens): matrix-vector products of the routes as
// they come, with no moe_align, no two-term activations and no combine.  Two launches:
//   gate: h[r][f] = silu(W1[e] x) * (W3[e] x), 16 features of a route a block, its warps over hidden;
//   down: y[t][c] = sum_j w[t, j] W2[e_j] h[t, j], 16 columns of a token a block, its warps over the
//         routes (and inter where there are fewer than 8 routes).
// Warp matrix instructions (m16n8k16, fp16 in, fp32 out) take the products: tcgen05 wants 128 rows of
// weights staged in shared memory and their scales in tensor memory, which is the latency that a
// single token waits for.  A lane loads 32 codes, one scale block, of each of its two rows with one
// 16-byte load: the four lanes of a row hold four neighbouring blocks.  The activations of block b
// stand in column b alone, with zeros in the other lanes' places, so that column b of the product is
// block b's sum, which the powers of two of weights and activations then scale in fp32.
// What bounds them: from cold weights latency (one token: 39 and 19 % of the issue slots; 24 routes: 47
// and 37), from weights in L2 the warps' instructions (32 routes to 8 experts: 63 and 55 %): one conversion
// a pair of codes, then one matrix instruction for 256 weights; the same kernels with an FMA a weight
// took 18.4 us where these take 16.4 (one token, 128 experts of 2048 x 768, cold: 20 MB, 3 us of
// the memory's time), and 88 where these take 75 for 8 tokens.  Moving the codes' bits into fp16
// fields instead of the conversion: 22.5.  Three blocks an SM with one group of 128 in flight a warp
// beat two blocks with twice the loads in flight at many routes (39 and 45 us for 32).  Persistent
// blocks with a ring of asynchronous copies three and four groups deep: the same (4 tokens 36.8 us).
// Blocks over several steps, with the activations prepared once: 20.5 and 40.7 us for 1 and 4 tokens
// (16.4 and 36.8 here), and 34.8 for 32 routes to 8 experts (38.9 here).
// Activations are fp16 times a power of two per 32, with the largest in [2^14, 2^15): bf16 is exact
// down to 2^-31 of the largest and off by at most 2^-39 of it below; h (fp32) is the sum of two such
// terms, the second in columns 4 to 7, with error 2^-22.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "exf_common.cuh"
#include "exf_launch.h"
#include "exf_mx.cuh"
#include "exf_mxmoe.h"

namespace exf {

constexpr int kFewWarps = 8;
constexpr int kFewTiles = 2;   // tiles of 8 features (8 gate rows, 8 up rows) of a gate block
constexpr int kFewDownK = 2;   // groups of 128 whose codes a warp of the down kernel loads at once
constexpr int kFewCols = 16;   // columns of a down block

// 8 codes -> their values in fp16 (exact), in pairs
__device__ __forceinline__ void code_pairs(uint32_t codes, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the powers of two of two scale bytes (NaN for 255)
__device__ __forceinline__ float2 block_scales(uint32_t bytes) {
  uint32_t p;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, a;\n\t}"
      : "=r"(p)
      : "r"(bytes));
  return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}
// byte offset of a weight row's four scale bytes of group 0 (tiles of 128 rows x 4 blocks; group k is
// 512 k further, the row 8 below within a 16-row tile 128, and a whole tile of rows 512 * groups)
__device__ __forceinline__ int64_t scale_offset(int row, int groups) {
  return (int64_t)(row >> 7) * groups * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// The warp's 128 activations of a group, four a lane, to fp16 terms in buf ([term][128]); returns
// the power of two of this lane's block (lanes 8 b to 8 b + 7 hold block b).
template <int TERMS>
__device__ __forceinline__ float put_group(const float (&v)[4], uint2* buf, int lane) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  const int k = min(14 + 127 - (int)(m >> 23), 126);
  const float up = __uint_as_float((uint32_t)(127 + k) << 23);
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = v[i] * up;
  __syncwarp();
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    const __half2 a = __floats2half2_rn(r[0], r[1]), b = __floats2half2_rn(r[2], r[3]);
    buf[32 * t + lane] = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                    *reinterpret_cast<const uint32_t*>(&b));
    if (t + 1 < TERMS) {
      const float2 fa = __half22float2(a), fb = __half22float2(b);
      r[0] -= fa.x;
      r[1] -= fa.y;
      r[2] -= fb.x;
      r[3] -= fb.y;
    }
  }
  __syncwarp();
  return __uint_as_float((uint32_t)(127 - k) << 23);
}

// (buf ends with 64 zero bytes, which the lanes without a block's activations read.)
// acc[tile][half] += this lane's share (two blocks) of rows g and g + 8 of each tile
template <int TILES, int TERMS>
__device__ __forceinline__ void group_product(const uint4 (&c)[TILES][2],
                                              const uint32_t (&s)[TILES][2], const uint2* buf,
                                              float power, int lane, float (&acc)[TILES][2]) {
  const int g = lane >> 2, t = lane & 3;
  uint32_t b[16];
  const bool mine = g == t || (TERMS == 2 && g == t + 4);
  const uint4* src =
      reinterpret_cast<const uint4*>(buf) + (mine ? (g >> 2) * 16 + t * 4 : TERMS * 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 q = src[i];
    b[4 * i] = q.x;
    b[4 * i + 1] = q.y;
    b[4 * i + 2] = q.z;
    b[4 * i + 3] = q.w;
  }
  const int blk = 2 * (t & 1);
  const float p0 = __shfl_sync(0xffffffffu, power, 8 * blk);
  const float p1 = __shfl_sync(0xffffffffu, power, 8 * blk + 8);
#pragma unroll
  for (int i = 0; i < TILES; ++i) {
    float d[2][4] = {};
    const uint32_t lo[4] = {c[i][0].x, c[i][0].y, c[i][0].z, c[i][0].w};
    const uint32_t hi[4] = {c[i][1].x, c[i][1].y, c[i][1].z, c[i][1].w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t a[4], e[4];
      code_pairs(lo[w], a);
      code_pairs(hi[w], e);
      mma_16816(d[0], a[0], e[0], a[1], e[1], b[4 * w], b[4 * w + 1]);
      mma_16816(d[1], a[2], e[2], a[3], e[3], b[4 * w + 2], b[4 * w + 3]);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float2 w = block_scales(s[i][r] >> (8 * blk));
      const float q0 = (d[0][2 * r] + d[1][2 * r]) * p0;
      const float q1 = (d[0][2 * r + 1] + d[1][2 * r + 1]) * p1;
      acc[i][r] = fmaf(q0, w.x, acc[i][r]);
      acc[i][r] = fmaf(q1, w.y, acc[i][r]);
    }
  }
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

__global__ void __launch_bounds__(32 * kFewWarps, 3)
    mx_few_gate_kernel(const __nv_bfloat16* x, const int32_t* ids,
                       const uint8_t* __restrict__ w13, const uint8_t* __restrict__ s13,
                       int experts, int top_k, int hidden, int inter, float* h) {
  constexpr int T = kFewTiles;
  __shared__ __align__(16) uint2 buf[kFewWarps][32 + 8];
  __shared__ float part[kFewWarps][T][16];
  // waits for the launches before it, then lets the down kernel start (which may therefore read
  // what those wrote before it waits for this one)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int route = blockIdx.y;
  const int f = blockIdx.x * 8 * T;
  const int e = ids[route];
  if (e < 0 || e >= experts) return;
  if (lane < 8) buf[warp][32 + lane] = make_uint2(0, 0);
  const int groups = hidden / 128;
  const int row0 = e * 2 * inter + f + g;
  const uint2* xr = reinterpret_cast<const uint2*>(x + (int64_t)(route / top_k) * hidden) + lane;
  const uint4* codes = reinterpret_cast<const uint4*>(w13 + (int64_t)row0 * (hidden / 2)) + t;
  const uint8_t* scales = s13 + scale_offset(row0, groups);
  const int64_t up_codes = (int64_t)inter * (hidden / 32);
  const int64_t up_scales = (int64_t)(inter / 128) * groups * 512;
  float acc[T][2] = {};
  for (int k = warp; k < groups; k += kFewWarps) {
    const uint2 xv = xr[32 * k];
    uint4 c[T][2];
    uint32_t s[T][2];
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        c[i][r] = __ldg(codes + 4 * k + r * up_codes + i * (hidden / 4));
        s[i][r] = __ldg(reinterpret_cast<const uint32_t*>(scales + 512 * k + r * up_scales +
                                                          128 * i));
      }
    const float v[4] = {__uint_as_float(xv.x << 16), __uint_as_float(xv.x & 0xffff0000u),
                        __uint_as_float(xv.y << 16), __uint_as_float(xv.y & 0xffff0000u)};
    const float power = put_group<1>(v, buf[warp], lane);
    group_product<T, 1>(c, s, buf[warp], power, lane, acc);
  }
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float v = quad_sum(acc[i][r]);
      if (t == 0) part[warp][i][8 * r + g] = v;
    }
  __syncthreads();
  if (threadIdx.x < 8 * T) {
    const int i = threadIdx.x >> 3, n = threadIdx.x & 7;
    float gate = 0.0f, up = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      gate += part[w][i][n];
      up += part[w][i][8 + n];
    }
    h[(int64_t)route * inter + f + threadIdx.x] = gate * logistic(gate) * up;
  }
}

__global__ void __launch_bounds__(32 * kFewWarps, 3)
    mx_few_down_kernel(const float* h, const float* route_w, const int32_t* ids,
                       const uint8_t* __restrict__ w2, const uint8_t* __restrict__ s2, int experts,
                       int top_k, int split, int hidden, int inter, __nv_bfloat16* y) {
  constexpr int K = kFewDownK;
  __shared__ __align__(16) uint2 buf[kFewWarps][64 + 8];
  __shared__ float part[kFewWarps][16];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int64_t token = blockIdx.y;
  const int col = blockIdx.x * kFewCols;
  const int64_t route = token * top_k + warp / split;
  // routes and weights were there before the gate kernel started: they are read while it runs
  const int e = __ldcg(ids + route);
  const bool use = e >= 0 && e < experts;
  const int groups = inter / 128;
  const int last = use ? groups : 0;
  if (lane < 8) buf[warp][64 + lane] = make_uint2(0, 0);
  const int row0 = (use ? e : 0) * hidden + col + g;
  const uint4* codes = reinterpret_cast<const uint4*>(w2 + (int64_t)row0 * (inter / 2)) + t;
  const uint8_t* scales = s2 + scale_offset(row0, groups);
  float acc[1][2] = {};
  bool waited = false;
  for (int k0 = warp % split; k0 < last; k0 += split * K) {
    uint4 c[K][1][2];
    uint32_t s[K][1][2];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int k = k0 + j * split;
      if (k >= groups) break;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        c[j][0][r] = __ldg(codes + 4 * k + r * (inter / 4));
        s[j][0][r] =
            __ldg(reinterpret_cast<const uint32_t*>(scales + 512 * k + 128 * r));
      }
    }
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    waited = true;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int k = k0 + j * split;
      if (k >= groups) break;
      const float4 q = *(reinterpret_cast<const float4*>(h + route * inter + 128 * k) + lane);
      const float v[4] = {q.x, q.y, q.z, q.w};
      const float power = put_group<2>(v, buf[warp], lane);
      group_product<1, 2>(c[j], s[j], buf[warp], power, lane, acc);
    }
  }
  if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
  const float w = use ? route_w[route] : 0.0f;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float v = quad_sum(acc[0][r]);
    if (t == 0) part[warp][8 * r + g] = use ? v * w : 0.0f;
  }
  __syncthreads();
  if (threadIdx.x < kFewCols) {
    float sum = 0.0f;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) sum += part[i][threadIdx.x];
    y[token * hidden + col + threadIdx.x] = __float2bfloat16_rn(sum);
  }
}

// The tensor-core layer starts at about 20 us (moe_align and the combine cost 10) and reads an
// expert's weights once for all its routes; these kernels start at 8 us and read and convert them once
// a route, 5 million weights a us.  Times of the two in us, cold weights, by routes x hidden x inter:
//   8 x 2048 x 768  16.4 / 26.6     16 x 2048 x 768  22.5 / 32.7    24 x 2048 x 768  26.6 / 34.7
//   32 x 2048 x 768 36.6 / 38.3 (128 experts), 36.6 / 34.8 (32)     24 x 2048 x 1024 32.7 / 29.1
//   8 x 4096 x 2048 40.9 / 40.7     64 x 1024 x 512  26.6 / 26.6    128 x 512 x 256  22.5 / 22.4
//   256 x 512 x 256 33.9 / 24.4
bool mx_few(int64_t routes, int hidden, int inter) {
  return routes <= 128 && routes * hidden * inter <= ((int64_t)5 << 23);
}

cudaError_t launch_mx_few(const MxArgs& a, float* h, cudaStream_t s) {
  const int numel = (int)(a.tokens * a.top_k);
  const int split = kFewWarps / a.top_k;
  cudaError_t e = launch_pdl(mx_few_gate_kernel,
                             dim3((unsigned)(a.inter / (8 * kFewTiles)), (unsigned)numel),
                             dim3(32 * kFewWarps), 0, s, static_cast<const __nv_bfloat16*>(a.x),
                             a.topk_ids, a.w13, a.s13, a.experts, a.top_k, a.hidden, a.inter, h);
  if (e != cudaSuccess) return e;
  return launch_pdl(mx_few_down_kernel,
                    dim3((unsigned)(a.hidden / kFewCols), (unsigned)a.tokens),
                    dim3(32 * split * a.top_k), 0, s, static_cast<const float*>(h), a.topk_w,
                    a.topk_ids, a.w2, a.s2, a.experts, a.top_k, split, a.hidden, a.inter,
                    static_cast<__nv_bfloat16*>(a.y));
}

}  // namespace exf
