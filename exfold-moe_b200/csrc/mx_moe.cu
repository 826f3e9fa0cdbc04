// The SwiGLU expert layer with MXFP4 weights (sm_100a: tcgen05 block-scaled MMA + TMA):
//   y[t] = sum_j w[t, j] W2[e] (silu(W1[e] x[t]) * (W3[e] x[t])),  e = ids[t, j].
//
// The weights go to the tensor cores as they are: TMA pads 16 packed codes to 16 bytes, and
// tcgen05.mma kind::mxf8f6f4 takes e2m1 codes with their E8M0 scales (one per row and 32 k) against
// 8-bit activations.  An activation is the sum of two e4m3 terms with scales 2^-5 apart: over a
// block of 32 with the largest magnitude in [2^m, 2^(m+1)) and s = 2^(m-7),
//   hi = e4m3(v / s),  lo = e4m3(32 (v / s - hi)),  v = s hi + (s / 32) lo.
// hi keeps 4 significant bits and the remainder, below 2^-4 of v, keeps 4 more: a bf16 activation
// (8 bits) is represented exactly unless it is smaller than 2^-13 of its block's largest, where
// the error stays below 2^-22 of that; the fp32 intermediate h is rounded by at most 2^-9 of its
// value (as bf16 would).  hi and lo are the two halves of the N side, so the weights are read once for
// both, and the epilogue adds the two accumulators.  The products are exact, the sums fp32.
//
// Launches: moe_align -> split (token rows into hi / lo rows in route order) -> the layer (both
// GEMMs, persistent) -> combine (each token's routes summed in fp32, in order).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <mutex>

#include "exf_common.cuh"
#include "exf_launch.h"
#include "exf_mxmoe.h"
#include "exf_tc.cuh"

namespace exf {
using namespace tc;

constexpr int kMxLayerThreads = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
constexpr int kMxK = 128;             // k values of a stage: 4 MMA steps, one scale word

// ---- the two-term form ------------------------------------------------------------------------
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
// byte of row n, block kb of a [tile][k / 128][512] scale table
__device__ __forceinline__ int64_t scale_at(int64_t tile, int kblocks, int kb, int n) {
  return (tile * kblocks + (kb >> 2)) * 512 + (n & 31) * 16 + (n >> 5) * 4 + (kb & 3);
}

// ---- split: token rows in route order ------------------------------------------------------------
// For every real slot m (block m / BT, row r = m % BT): rows r and BT + r of the block in xq hold
// the hi and lo terms of x[token], xs their scales.  4 lanes share a block of 32.  Padding rows
// keep whatever the workspace holds: a row feeds its own accumulator column only, and a padding
// column is never stored.  Also zeroes the layer's counters.
__global__ void __launch_bounds__(256) mx_split_kernel(const __nv_bfloat16* x, MxRoutes r,
                                                       int64_t rows, int numel, int top_k,
                                                       int hidden, int bt, uint8_t* xq, uint8_t* xs,
                                                       int32_t* zero, int zero_n) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < zero_n; i += gridDim.x * blockDim.x)
    zero[i] = 0;
  const int vec = hidden / 8;  // a multiple of 32: a warp stays in one row
  const int64_t used = *r.num_post_pad < rows ? *r.num_post_pad : rows;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < used * vec;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t m = i / vec;
    const int c = (int)(i - m * vec);
    const int route = r.sorted_ids[m];
    if (route >= numel) continue;
    const uint4 v = reinterpret_cast<const uint4*>(x + (int64_t)(route / top_k) * hidden)[c];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      top = max(top, max((w[j] << 16) & 0x7fff0000u, w[j] & 0x7fff0000u));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t sb = split_scale(top);
    const float inv = split_inverse(sb);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      split2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u), inv, hi[j], lo[j]);
    const int64_t blk = m / bt;
    const int n = (int)(m - blk * bt);
    uint8_t* q = xq + (blk * 2 * bt + n) * hidden + 8 * c;
    *reinterpret_cast<uint2*>(q) = make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
    *reinterpret_cast<uint2*>(q + (int64_t)bt * hidden) =
        make_uint2(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16);
    if ((c & 3) == 0) {
      xs[scale_at(blk, hidden / kMxK, c >> 2, n)] = (uint8_t)sb;
      xs[scale_at(blk, hidden / kMxK, c >> 2, bt + n)] = (uint8_t)split_lo_byte(sb);
    }
  }
}

// ---- the layer ------------------------------------------------------------------------------------
// As the bf16 decode layer: a tile is 256 weight rows of one expert (two 128-row MMA tiles on the M
// side) times a block of BT of its routes (N = 2 BT: hi rows, lo rows).
//   GEMM-1 tile (block, f): gate rows [128 f, +128) and up rows [I + 128 f, +128) of W13[e], K = H;
//     the epilogue forms h = silu(gate) * up, a lane per feature, and writes its two-term form
//     (a warp's 32 features are one scale block);
//   GEMM-2 tile (block, f): rows [256 f, +256) of W2[e], K = I; out[route][256 f + i] = w_route D.
// One persistent launch: warp 0 takes tiles from a counter (every GEMM-1 tile, then the GEMM-2
// tiles) and, before the first load of a GEMM-2 tile, waits until the epilogue warps of the block's
// GEMM-1 tiles have counted themselves off.  A GEMM-1 tile waits only for earlier tiles of its own
// CTA and was handed out before every GEMM-2 tile, so the wait ends; it is bounded all the same.
template <int BT>
struct MxCfg {
  static constexpr int kN = 2 * BT;
  static constexpr int kWTile = 128 * kMxK;              // padded codes of 128 rows
  static constexpr int kTTile = kN * kMxK;
  static constexpr int kScales = 3 * 512;                // two weight tiles, one token tile
  static constexpr int kTiles = 2 * kWTile + kTTile;
  static constexpr int kTxBytes = kWTile + kTTile + kScales;  // weights count packed
  static constexpr int kStages = (210 * 1024) / (kTiles + kScales);
  static constexpr int kAccCols = 2 * kN;
  static constexpr int kAccs = kAccCols * 2 + 64 <= 512 ? 2 : 1;
  static constexpr int kScaleCol = kAccs * kAccCols;     // 4 sets of 16 columns
  static constexpr int kTmemCols = kScaleCol + 64 <= 128 ? 128 : kScaleCol + 64 <= 256 ? 256 : 512;
  static constexpr int kRing = 8;
};
template <int BT>
struct MxSmem {
  alignas(1024) uint8_t tiles[MxCfg<BT>::kStages][MxCfg<BT>::kTiles];
  alignas(128) uint8_t scales[MxCfg<BT>::kStages][MxCfg<BT>::kScales];
  alignas(8) uint64_t full[MxCfg<BT>::kStages];
  alignas(8) uint64_t empty[MxCfg<BT>::kStages];
  alignas(8) uint64_t acc_full[2];
  alignas(8) uint64_t acc_empty[2];
  alignas(8) uint64_t ring_full[MxCfg<BT>::kRing];
  alignas(8) uint64_t ring_empty[MxCfg<BT>::kRing];
  alignas(8) uint64_t drain;
  int ring[MxCfg<BT>::kRing];
  uint32_t tmem_base;
  int failed;
};
template <int BT>
constexpr size_t mx_smem_bytes() { return sizeof(MxSmem<BT>) + 1024; }
static_assert(mx_smem_bytes<16>() <= 232448 && mx_smem_bytes<32>() <= 232448 &&
                  mx_smem_bytes<64>() <= 232448,
              "expert layer shared memory");

struct MxTile {
  bool down;
  int blk;
  int ft;
};
__device__ __forceinline__ MxTile mx_tile(int t, int blocks, int n1, int n2) {
  MxTile r;
  r.down = t >= blocks * n1;
  if (r.down) t -= blocks * n1;
  const int n = r.down ? n2 : n1;
  r.blk = t / n;
  r.ft = t - r.blk * n;
  return r;
}

template <int BT>
__global__ void __launch_bounds__(kMxLayerThreads, 1)
    mx_layer_kernel(const __grid_constant__ CUtensorMap map_w13,
                    const __grid_constant__ CUtensorMap map_xq,
                    const __grid_constant__ CUtensorMap map_w2,
                    const __grid_constant__ CUtensorMap map_hq, const MxLayerParams p) {
  using C = MxCfg<BT>;
  constexpr int kStages = C::kStages;
  constexpr int kRing = C::kRing;
  extern __shared__ uint8_t smem_raw[];
  MxSmem<BT>& sm = *reinterpret_cast<MxSmem<BT>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 4);
    }
    for (int j = 0; j < kRing; ++j) {
      mbar_init(&sm.ring_full[j], 1);
      mbar_init(&sm.ring_empty[j], 5);  // the MMA thread and the four epilogue warps
    }
    mbar_init(&sm.drain, 1);
    sm.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, C::kTmemCols);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int post = *p.routes.num_post_pad;
  const int blocks = (post + BT - 1) / BT < p.m_blocks ? (post + BT - 1) / BT : p.m_blocks;
  const int n1 = p.inter / 128;
  const int n2 = p.hidden / 256;
  const int total = blocks * (n1 + n2);
  const uint32_t tmem = sm.tmem_base;
  volatile int* failed = &sm.failed;
  auto expert_of = [&](const MxTile& lt) {
    const int e = p.routes.expert_ids[lt.blk];
    return (e >= 0 && e < p.experts) ? e : -1;
  };

  if (warp == 0) {
    // ---- scheduler + producer (one thread)
    if (lane == 0) {
      uint32_t g = 0;
      bool ok = true;
      int t = atomicAdd(p.sync, 1);
      for (int j = 0; ok; ++j) {
        const int tile = t < total ? t : -1;
        const int slot = j % kRing;
        ok = mbar_wait(&sm.ring_empty[slot], ((j / kRing) & 1) ^ 1, failed);
        if (!ok) break;
        sm.ring[slot] = tile;
        mbar_arrive(&sm.ring_full[slot]);
        if (tile < 0) break;
        t = atomicAdd(p.sync, 1);
        const MxTile lt = mx_tile(tile, blocks, n1, n2);
        const int expert = expert_of(lt);
        if (expert < 0) continue;
        if (lt.down) {
          const int32_t* flag = p.sync + 1 + lt.blk;
          uint32_t it = 0;
          while (ld_acquire_gpu(flag) < 4 * n1) {
            if (*failed || ++it >= kWaitLimit) {
              *failed = 1;
              ok = false;
              break;
            }
            __nanosleep(128);
          }
          if (!ok) break;
          asm volatile("fence.proxy.async.global;" ::: "memory");
        }
        const int kblocks = (lt.down ? p.inter : p.hidden) / kMxK;
        const CUtensorMap* mw = lt.down ? &map_w2 : &map_w13;
        const CUtensorMap* mt = lt.down ? &map_hq : &map_xq;
        // both weight tiles: gate and up rows of W13[e], or 256 rows of W2[e]
        const int row0 =
            lt.down ? expert * p.hidden + lt.ft * 256 : expert * 2 * p.inter + lt.ft * 128;
        const int row1 = lt.down ? row0 + 128 : row0 + p.inter;
        const uint8_t* ws = lt.down ? p.s2 : p.s13;
        const uint8_t* ws0 = ws + (int64_t)(row0 / 128) * kblocks * 512;
        const uint8_t* ws1 = ws + (int64_t)(row1 / 128) * kblocks * 512;
        const uint8_t* ts = (lt.down ? p.hs : p.xs) + (int64_t)lt.blk * kblocks * 512;
        for (int kb = 0; kb < kblocks; ++kb, ++g) {
          const int s = g % kStages;
          ok = mbar_wait(&sm.empty[s], ((g / kStages) & 1) ^ 1, failed);
          if (!ok) break;
          uint8_t* st = sm.tiles[s];
          uint64_t* bar = &sm.full[s];
          mbar_expect_tx(bar, C::kTxBytes);
          tma_load_2d(st, mw, bar, kb * kMxK, row0);
          tma_load_2d(st + C::kWTile, mw, bar, kb * kMxK, row1);
          tma_load_2d(st + 2 * C::kWTile, mt, bar, kb * kMxK, lt.blk * C::kN);
          bulk_load(sm.scales[s], ws0 + kb * 512, 512, bar);
          bulk_load(sm.scales[s] + 512, ws1 + kb * 512, 512, bar);
          bulk_load(sm.scales[s] + 1024, ts + kb * 512, 512, bar);
        }
      }
      for (uint32_t j = g > kStages ? g - kStages : 0; j < g; ++j)
        mbar_wait_drain(&sm.full[j % kStages], (j / kStages) & 1);
    }
  } else if (warp == 1) {
    // ---- MMA issuer; scale sets rotate over 4 groups of 16 TMEM columns
    if (lane == 0) {
      uint32_t g = 0;
      int i = 0;
      bool ok = true;
      for (int j = 0; ok; ++j) {
        const int slot = j % kRing;
        ok = mbar_wait(&sm.ring_full[slot], (j / kRing) & 1, failed);
        if (!ok) break;
        const int tile = sm.ring[slot];
        mbar_arrive(&sm.ring_empty[slot]);
        if (tile < 0) break;
        const MxTile lt = mx_tile(tile, blocks, n1, n2);
        if (expert_of(lt) < 0) continue;
        const int kblocks = (lt.down ? p.inter : p.hidden) / kMxK;
        const int b = i % C::kAccs;
        ok = mbar_wait(&sm.acc_empty[b], ((i / C::kAccs) & 1) ^ 1, failed);
        if (!ok) break;
        fence_after_sync();
        const uint32_t acc = tmem + static_cast<uint32_t>(b * C::kAccCols);
        for (int kb = 0; kb < kblocks; ++kb, ++g) {
          const int s = g % kStages;
          ok = mbar_wait(&sm.full[s], (g / kStages) & 1, failed);
          if (!ok) break;
          fence_after_sync();
          const uint32_t w_base = smem_addr(sm.tiles[s]);
          const uint32_t t_base = w_base + 2 * C::kWTile;
          const uint32_t sc = smem_addr(sm.scales[s]);
          const uint32_t sf = tmem + C::kScaleCol + (g & 3) * 16;
          tmem_copy_scales(sf, sc);
          tmem_copy_scales(sf + 4, sc + 512);
          tmem_copy_scales(sf + 8, sc + 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t on = (kb > 0 || k > 0) ? 1u : 0u;
            const uint32_t id = idesc_mx(128, C::kN, kMxE2M1, kMxE4M3, k);
            mma_mx(acc, smem_desc(w_base + k * 32), smem_desc(t_base + k * 32), id, sf, sf + 8,
                   on);
            mma_mx(acc + C::kN, smem_desc(w_base + C::kWTile + k * 32),
                   smem_desc(t_base + k * 32), id, sf + 4, sf + 8, on);
          }
          mma_commit(&sm.empty[s]);
        }
        if (!ok) break;
        mma_commit(&sm.acc_full[b]);
        ++i;
      }
      mma_commit(&sm.drain);
      mbar_wait_drain(&sm.drain, 0);
    }
  } else {
    // ---- epilogue: warp q owns TMEM lanes 32 q .. +31, i.e. 32 weight rows of each M tile;
    // columns are routes (hi, then lo), 16 at a time
    const int q = warp & 3;
    int i = 0;
    for (int j = 0;; ++j) {
      const int slot = j % kRing;
      int tile = -2;
      if (lane == 0 && mbar_wait(&sm.ring_full[slot], (j / kRing) & 1, failed)) {
        tile = sm.ring[slot];
        mbar_arrive(&sm.ring_empty[slot]);
      }
      tile = __shfl_sync(0xffffffffu, tile, 0);
      if (tile < 0) break;
      const MxTile lt = mx_tile(tile, blocks, n1, n2);
      if (expert_of(lt) < 0) continue;
      const int b = i % C::kAccs;
      const bool ok = mbar_wait(&sm.acc_full[b], (i / C::kAccs) & 1, failed);
      fence_after_sync();
      if (!__all_sync(0xffffffffu, ok && !*failed)) break;
      const uint32_t taddr =
          tmem + static_cast<uint32_t>(b * C::kAccCols) + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < BT; c += 16) {
        const int route_l =
            lane < 16 ? p.routes.sorted_ids[lt.blk * BT + c + lane] : p.numel;
        const uint32_t real = __ballot_sync(0xffffffffu, route_l < p.numel);
        if (real == 0) continue;
        uint32_t a0[16], a1[16], b0[16], b1[16];
        tmem_load16(taddr + c, a0);
        tmem_load16(taddr + BT + c, a1);
        tmem_load16(taddr + C::kN + c, b0);
        tmem_load16(taddr + C::kN + BT + c, b1);
        tmem_wait();
        if (!lt.down) {
          const int feat = lt.ft * 128 + q * 32 + lane;
          uint8_t* hq = p.hq + ((int64_t)lt.blk * C::kN + c) * p.inter + feat;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if (!((real >> r) & 1)) continue;
            const float gt = __uint_as_float(a0[r]) + __uint_as_float(a1[r]);
            const float up = __uint_as_float(b0[r]) + __uint_as_float(b1[r]);
            const float h = gt / (1.0f + __expf(-gt)) * up;
            const uint32_t top =
                __reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7fffffffu);
            const uint32_t sb = split_scale(top);
            uint32_t hi, lo;
            split2(h, 0.0f, split_inverse(sb), hi, lo);
            hq[(int64_t)r * p.inter] = (uint8_t)hi;
            hq[(int64_t)(BT + r) * p.inter] = (uint8_t)lo;
            if (lane < 2)
              p.hs[scale_at(lt.blk, p.inter / kMxK, lt.ft * 4 + q, c + r + (lane ? BT : 0))] =
                  (uint8_t)(lane ? split_lo_byte(sb) : sb);
          }
        } else {
          const int feat = lt.ft * 256 + q * 32 + lane;
          const float w_l = route_l < p.numel ? p.route_w[route_l] : 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int route = __shfl_sync(0xffffffffu, route_l, r);
            const float wr = __shfl_sync(0xffffffffu, w_l, r);
            if (!((real >> r) & 1)) continue;
            float* o = p.out + (int64_t)route * p.hidden + feat;
            o[0] = (__uint_as_float(a0[r]) + __uint_as_float(a1[r])) * wr;
            o[128] = (__uint_as_float(b0[r]) + __uint_as_float(b1[r])) * wr;
          }
        }
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[b]);
      ++i;
      if (!lt.down) {
        // visible to the TMA loads of the block's GEMM-2 tiles, in any CTA; then count the warp off
        asm volatile("fence.proxy.async.global;" ::: "memory");
        __threadfence();
        __syncwarp();
        if (lane == 0) red_release_gpu_add(p.sync + 1 + lt.blk, 1);
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    fence_after_sync();
    tmem_free(tmem, C::kTmemCols);
  }
  if (threadIdx.x == 0 && sm.failed && p.status) atomicExch(p.status, 1);
}

// ---- combine ---------------------------------------------------------------------------------------
// y[t] = sum_j out[t * top_k + j] in fp32, in route order; routes out of range were never placed.
// The route outputs are fp32: rounding each to bf16 would add as much error as the result's own.
__global__ void __launch_bounds__(256, 4)
    mx_combine_kernel(const float* __restrict__ out, const int32_t* __restrict__ ids, int experts,
                      int64_t tokens, int top_k, int hidden, __nv_bfloat16* y) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int vec = hidden / 4;
  const float4* out4 = reinterpret_cast<const float4*>(out);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < tokens * vec;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / vec;
    const int c = (int)(i - t * vec);
    float4 v[8];
    bool use[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = j < top_k ? __ldg(ids + t * top_k + j) : -1;
      use[j] = e >= 0 && e < experts;
      if (use[j]) v[j] = __ldg(out4 + (t * top_k + j) * vec + c);
    }
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!use[j]) continue;
      acc.x += v[j].x;
      acc.y += v[j].y;
      acc.z += v[j].z;
      acc.w += v[j].w;
    }
    reinterpret_cast<uint2*>(y)[i] = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
  }
}

// ---- host side ---------------------------------------------------------------------------------
// The route block: the smallest of 16, 32 and 64 that holds the average expert's routes.
static int mx_block(int64_t numel, int experts) {
  return numel <= (int64_t)experts * 16 ? 16 : numel <= (int64_t)experts * 32 ? 32 : 64;
}

static int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

MxWorkspace mx_workspace(int64_t tokens, int top_k, int experts, int hidden, int inter,
                         void* base) {
  MxWorkspace w{};
  const int64_t numel = tokens * top_k;
  w.block = mx_block(numel, experts);
  int64_t cap = numel + (int64_t)experts * (w.block - 1);
  cap = (cap + w.block - 1) / w.block * w.block;
  if (numel < experts && numel * w.block < cap) cap = numel * w.block;
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = off;
    off += up256(bytes);
    return base ? static_cast<uint8_t*>(base) + o : nullptr;
  };
  w.capacity = cap;
  const int64_t blocks = cap / w.block;
  w.sorted_ids = reinterpret_cast<int32_t*>(take(cap * 4));
  w.expert_ids = reinterpret_cast<int32_t*>(take(blocks * 4));
  w.num_post_pad = reinterpret_cast<int32_t*>(take(4));
  const int64_t align_bytes = align_workspace_bytes(numel, experts);
  w.align_ws = take(align_bytes > 0 ? align_bytes : 4);
  w.xq = take(2 * cap * hidden);
  w.xs = take(blocks * (hidden / kMxK) * 512);
  w.hq = take(2 * cap * inter);
  w.hs = take(blocks * (inter / kMxK) * 512);
  w.out = reinterpret_cast<float*>(take(numel * hidden * 4));
  w.sync_ints = (int)(1 + blocks);
  w.sync = reinterpret_cast<int32_t*>(take(w.sync_ints * 4));
  w.bytes = off;
  return w;
}

template <int BT>
static cudaError_t launch_mx_layer(const MxArgs& a, const MxWorkspace& w, cudaStream_t s) {
  auto* kern = mx_layer_kernel<BT>;
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!done[dev]) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)mx_smem_bytes<BT>());
      if (e != cudaSuccess) return e;
      done[dev] = true;
    }
  }
  const int64_t blocks = w.capacity / BT;
  CUtensorMap m13, mx, m2, mh;
  if (!make_map_4bit(&m13, a.w13, (uint64_t)a.experts * 2 * a.inter, a.hidden, 128) ||
      !make_map_8bit(&mx, w.xq, blocks * 2 * BT, a.hidden, 2 * BT) ||
      !make_map_4bit(&m2, a.w2, (uint64_t)a.experts * a.hidden, a.inter, 128) ||
      !make_map_8bit(&mh, w.hq, blocks * 2 * BT, a.inter, 2 * BT))
    return cudaErrorInvalidValue;
  MxLayerParams p{};
  p.routes = {w.num_post_pad, w.expert_ids, w.sorted_ids};
  p.experts = a.experts;
  p.numel = (int)(a.tokens * a.top_k);
  p.hidden = a.hidden;
  p.inter = a.inter;
  p.m_blocks = (int)blocks;
  p.status = a.status;
  p.s13 = a.s13;
  p.s2 = a.s2;
  p.xs = w.xs;
  p.hq = w.hq;
  p.hs = w.hs;
  p.route_w = a.topk_w;
  p.out = w.out;
  p.sync = w.sync;
  const int sms = sm_count();
  return launch_pdl(kern, sms > 0 ? (unsigned)sms : 1u, kMxLayerThreads, mx_smem_bytes<BT>(), s,
                    m13, mx, m2, mh, p);
}

static unsigned stream_grid(int64_t threads) {
  int64_t blocks = (threads + 255) / 256;
  const int lim = 8 * sm_count();
  if (lim > 0 && blocks > lim) blocks = lim;
  return (unsigned)(blocks > 0 ? blocks : 1);
}

cudaError_t launch_mx_experts(const MxArgs& a, const MxWorkspace& w, cudaStream_t s) {
  const int64_t numel = a.tokens * a.top_k;
  AlignParams ap{a.topk_ids, numel, a.experts, w.block, w.capacity, w.sorted_ids, w.expert_ids,
                 w.num_post_pad, static_cast<int32_t*>(w.align_ws), 0};
  cudaError_t e = launch_align(EXF_I32, ap, s);
  if (e != cudaSuccess) return e;
  const MxRoutes routes{w.num_post_pad, w.expert_ids, w.sorted_ids};
  e = launch_pdl(mx_split_kernel, stream_grid(w.capacity * (a.hidden / 8)), 256, 0, s,
                 static_cast<const __nv_bfloat16*>(a.x), routes, w.capacity, (int)numel, a.top_k,
                 a.hidden, w.block, w.xq, w.xs, w.sync, w.sync_ints);
  if (e != cudaSuccess) return e;
  e = w.block == 16   ? launch_mx_layer<16>(a, w, s)
      : w.block == 32 ? launch_mx_layer<32>(a, w, s)
                      : launch_mx_layer<64>(a, w, s);
  if (e != cudaSuccess) return e;
  return launch_pdl(mx_combine_kernel, stream_grid(a.tokens * (a.hidden / 4)), 256, 0, s,
                    static_cast<const float*>(w.out), a.topk_ids, a.experts, a.tokens, a.top_k,
                    a.hidden, static_cast<__nv_bfloat16*>(a.y));
}

}  // namespace exf
