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

constexpr int kMxLayerThreads = 256;  // warps 0, 6, 7 TMA, warp 1 MMA, warps 2-5 epilogue
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
// Scales of a route block's rows [0, 2 BT): tables [k / 128][512], one per 128 rows.  Byte of row n,
// scale block kb, in the tables of the route block's first one.
__device__ __forceinline__ int64_t scale_at(int64_t table, int kblocks, int kb, int n) {
  return ((table + (n >> 7)) * kblocks + (kb >> 2)) * 512 + (n & 31) * 16 + ((n >> 5) & 3) * 4 +
         (kb & 3);
}
// tables of a route block
__host__ __device__ constexpr int scale_tables(int bt) { return bt > 64 ? 2 : 1; }

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
      const int64_t table = blk * scale_tables(bt);
      xs[scale_at(table, hidden / kMxK, c >> 2, n)] = (uint8_t)sb;
      xs[scale_at(table, hidden / kMxK, c >> 2, bt + n)] = (uint8_t)split_lo_byte(sb);
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
// tiles) and passes them on through a ring.  Three warps load: the first weight tile, the second,
// and the token tile, each with its scales (one thread issuing every copy of a stage held the
// weight stream at 4.0 TB/s: a row of packed codes is a 64-byte request; alone, 16-byte padded
// tiles stream at 5.3 TB/s from one issuing thread and at 6.6 from two).  The warp that loads
// tokens waits, before the first load of a GEMM-2 tile, until the epilogue warps of the block's
// GEMM-1 tiles have counted themselves off; the weights of such a tile do not wait.  A GEMM-1 tile
// waits only for earlier tiles of its own CTA and was handed out before every GEMM-2 tile, so the
// wait ends; it is bounded all the same.
template <int BT>
struct MxCfg {
  static constexpr int kN = 2 * BT;
  static constexpr int kWTile = 128 * kMxK;              // padded codes of 128 rows
  static constexpr int kTTile = kN * kMxK;
  static constexpr int kScales = 3 * 512;                // two weight tiles, one token tile
  static constexpr int kTiles = 2 * kWTile + kTTile;
  static constexpr int kWTx = kWTile / 2 + 512;          // a copy of codes counts them packed
  static constexpr int kTTx = kTTile + 512;
  static constexpr int kStages = (210 * 1024) / (kTiles + kScales);
  static constexpr int kAccCols = 2 * kN;
  static constexpr int kAccs = kAccCols * 2 + 64 <= 512 ? 2 : 1;
  static constexpr int kScaleCol = kAccs * kAccCols;     // 4 sets of 16 columns
  static constexpr int kTmemCols = 512;
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
static_assert(mx_smem_bytes<32>() <= 232448 && mx_smem_bytes<64>() <= 232448,
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

// After a time-out (else every load has been consumed): copies still in flight land before shared
// memory is released.  The other loading warps may never arrive on a stage, so that its barrier
// does not complete: the wait is bounded.
template <int STAGES>
__device__ __forceinline__ void drain_loads(uint64_t* full, uint32_t g) {
  for (uint32_t j = g > STAGES ? g - STAGES : 0; j < g; ++j) {
    for (int i = 0; i < 4096; ++i) {
      if (mbar_try_wait(&full[j % STAGES], (j / STAGES) & 1)) break;
      __nanosleep(256);
    }
  }
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
      mbar_init(&sm.full[s], 3);  // one arrival per loading warp
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 4);
    }
    for (int j = 0; j < kRing; ++j) {
      mbar_init(&sm.ring_full[j], 1);
      mbar_init(&sm.ring_empty[j], 7);  // two loading warps, the MMA thread, four epilogue warps
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

  uint32_t issued = 0;  // stages this thread has loaded into
  if (warp == 0 || warp >= 6) {
    // ---- loads: warp 0 (which also hands out the tiles) and warp 6 a weight tile each, warp 7 the
    // token tile; one thread each
    if (lane == 0) {
      uint32_t g = 0;
      bool ok = true;
      int t = warp == 0 ? atomicAdd(p.sync, 1) : 0;
      for (int j = 0; ok; ++j) {
        const int slot = j % kRing;
        int tile;
        if (warp == 0) {
          tile = t < total ? t : -1;
          ok = mbar_wait(&sm.ring_empty[slot], ((j / kRing) & 1) ^ 1, failed);
          if (!ok) break;
          sm.ring[slot] = tile;
          mbar_arrive(&sm.ring_full[slot]);
          if (tile >= 0) t = atomicAdd(p.sync, 1);  // its latency overlaps this tile's loads
        } else {
          ok = mbar_wait(&sm.ring_full[slot], (j / kRing) & 1, failed);
          if (!ok) break;
          tile = sm.ring[slot];
          mbar_arrive(&sm.ring_empty[slot]);
        }
        if (tile < 0) break;
        const MxTile lt = mx_tile(tile, blocks, n1, n2);
        const int expert = expert_of(lt);
        if (expert < 0) continue;
        const int kblocks = (lt.down ? p.inter : p.hidden) / kMxK;
        if (warp == 7) {
          if (lt.down) {
            const int32_t* flag = p.sync + 1 + lt.blk;
            uint32_t it = 0;
            while (ld_acquire_gpu(flag) < 4 * n1) {
              if (*failed || ++it >= kWaitLimit) {
                *failed = 1;
                ok = false;
                break;
              }
              __nanosleep(64);
            }
            if (!ok) break;
            asm volatile("fence.proxy.async.global;" ::: "memory");
          }
          const CUtensorMap* map = lt.down ? &map_hq : &map_xq;
          const uint8_t* sc = (lt.down ? p.hs : p.xs) + (int64_t)lt.blk * kblocks * 512;
          for (int kb = 0; kb < kblocks; ++kb, ++g) {
            const int s = g % kStages;
            ok = mbar_wait(&sm.empty[s], ((g / kStages) & 1) ^ 1, failed);
            if (!ok) break;
            mbar_expect_tx(&sm.full[s], C::kTTx);
            tma_load_2d(sm.tiles[s] + 2 * C::kWTile, map, &sm.full[s], kb * kMxK, lt.blk * C::kN);
            bulk_load(sm.scales[s] + 1024, sc + kb * 512, 512, &sm.full[s]);
          }
        } else {
          // gate (warp 0) and up (warp 6) rows of W13[e], or the halves of 256 rows of W2[e]
          const int half = warp == 0 ? 0 : 1;
          const int row = lt.down
                              ? expert * p.hidden + lt.ft * 256 + half * 128
                              : expert * 2 * p.inter + lt.ft * 128 + half * p.inter;
          const CUtensorMap* map = lt.down ? &map_w2 : &map_w13;
          const uint8_t* sc = (lt.down ? p.s2 : p.s13) + (int64_t)(row / 128) * kblocks * 512;
          for (int kb = 0; kb < kblocks; ++kb, ++g) {
            const int s = g % kStages;
            ok = mbar_wait(&sm.empty[s], ((g / kStages) & 1) ^ 1, failed);
            if (!ok) break;
            mbar_expect_tx(&sm.full[s], C::kWTx);
            tma_load_2d(sm.tiles[s] + half * C::kWTile, map, &sm.full[s], kb * kMxK, row);
            bulk_load(sm.scales[s] + half * 512, sc + kb * 512, 512, &sm.full[s]);
          }
        }
      }
      issued = g;
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
  if (sm.failed) {
    drain_loads<kStages>(sm.full, issued);
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 1);
  }
}

// ---- prefill ------------------------------------------------------------------------------------
// Experts with many routes: 128 routes on the M side (hi rows, then lo rows of a route block, both
// added into one accumulator), 256 weight rows on the N side, so that the MMA (128 x 256 x 32, 128
// cycles) is not held up by its operand reads and the epilogue has a row a thread.
//   GEMM-1 tile: gate rows [128 f, +128) and up rows of W13[e]; GEMM-2 tile: 256 rows of W2[e].
// The accumulator takes 256 TMEM columns and the scales 64, which leaves no room for a second one:
// 8 epilogue warps copy it to registers at once and give it back before they compute, so the
// tensor cores wait for the copy only.  A persistent launch per GEMM, tiles of one route block side
// by side (its rows and the expert's weights are reused from L2).
constexpr int kMxGemmThreads = 384;  // warps 0, 2, 3 TMA, warp 1 MMA, warps 4-11 epilogue
constexpr int kMxGemmStages = 3;
struct MxGemmSmem {
  // a stage: 128 hi rows, 128 lo rows, 256 rows of padded codes
  alignas(1024) uint8_t tiles[kMxGemmStages][4 * 128 * kMxK];
  alignas(128) uint8_t scales[kMxGemmStages][4 * 512];
  alignas(8) uint64_t full[kMxGemmStages];
  alignas(8) uint64_t empty[kMxGemmStages];
  alignas(8) uint64_t acc_full;
  alignas(8) uint64_t acc_empty;
  alignas(8) uint64_t drain;
  uint32_t tmem_base;
  int failed;
};
constexpr size_t mx_gemm_smem_bytes() { return sizeof(MxGemmSmem) + 1024; }
static_assert(mx_gemm_smem_bytes() <= 232448, "prefill expert GEMM shared memory");

template <bool DOWN>
__global__ void __launch_bounds__(kMxGemmThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_t, const MxLayerParams p) {
  constexpr int kTile = 128 * kMxK;
  extern __shared__ uint8_t smem_raw[];
  MxGemmSmem& sm = *reinterpret_cast<MxGemmSmem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kMxGemmStages; ++s) {
      mbar_init(&sm.full[s], 3);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.acc_full, 1);
    mbar_init(&sm.acc_empty, 8);
    mbar_init(&sm.drain, 1);
    sm.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, 512);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int post = *p.routes.num_post_pad;
  const int blocks = (post + 127) / 128 < p.m_blocks ? (post + 127) / 128 : p.m_blocks;
  const int n_tiles = DOWN ? p.hidden / 256 : p.inter / 128;
  const int kblocks = (DOWN ? p.inter : p.hidden) / kMxK;
  const int total = blocks * n_tiles;
  const uint32_t tmem = sm.tmem_base;
  volatile int* failed = &sm.failed;
  auto expert_of = [&](int blk) {
    const int e = p.routes.expert_ids[blk];
    return (e >= 0 && e < p.experts) ? e : -1;
  };

  uint32_t issued = 0;
  if (warp == 0 || warp == 2 || warp == 3) {
    // ---- loads: warp 0 the hi and lo rows, warps 2 and 3 a weight tile each
    if (lane == 0) {
      uint32_t g = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const int blk = t / n_tiles, ft = t - blk * n_tiles;
        const int expert = expert_of(blk);
        if (expert < 0) continue;
        const int half = warp - 2;
        const int row = DOWN ? expert * p.hidden + ft * 256 + half * 128
                             : expert * 2 * p.inter + ft * 128 + half * p.inter;
        const uint8_t* sc =
            warp == 0 ? (DOWN ? p.hs : p.xs) + (int64_t)blk * 2 * kblocks * 512
                      : (DOWN ? p.s2 : p.s13) + (int64_t)(row / 128) * kblocks * 512;
        for (int kb = 0; kb < kblocks; ++kb, ++g) {
          const int s = g % kMxGemmStages;
          ok = mbar_wait(&sm.empty[s], ((g / kMxGemmStages) & 1) ^ 1, failed);
          if (!ok) break;
          uint64_t* bar = &sm.full[s];
          if (warp == 0) {
            mbar_expect_tx(bar, 2 * kTile + 1024);
            tma_load_2d(sm.tiles[s], &map_t, bar, kb * kMxK, blk * 256);
            bulk_load(sm.scales[s], sc + kb * 512, 512, bar);
            bulk_load(sm.scales[s] + 512, sc + (kblocks + kb) * 512, 512, bar);
          } else {
            mbar_expect_tx(bar, kTile / 2 + 512);
            tma_load_2d(sm.tiles[s] + (2 + half) * kTile, &map_w, bar, kb * kMxK, row);
            bulk_load(sm.scales[s] + 1024 + half * 512, sc + kb * 512, 512, bar);
          }
        }
      }
      issued = g;
    }
  } else if (warp == 1) {
    // ---- MMA issuer
    if (lane == 0) {
      uint32_t g = 0;
      int i = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        if (expert_of(t / n_tiles) < 0) continue;
        ok = mbar_wait(&sm.acc_empty, (i & 1) ^ 1, failed);
        if (!ok) break;
        fence_after_sync();
        for (int kb = 0; kb < kblocks; ++kb, ++g) {
          const int s = g % kMxGemmStages;
          ok = mbar_wait(&sm.full[s], (g / kMxGemmStages) & 1, failed);
          if (!ok) break;
          fence_after_sync();
          const uint32_t a = smem_addr(sm.tiles[s]);
          const uint32_t b = a + 2 * kTile;
          const uint32_t sc = smem_addr(sm.scales[s]);
          const uint32_t sf = tmem + 256 + (g & 3) * 16;
#pragma unroll
          for (int j = 0; j < 4; ++j) tmem_copy_scales(sf + 4 * j, sc + 512 * j);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t id = idesc_mx(128, 256, kMxE4M3, kMxE2M1, k);
            mma_mx(tmem, smem_desc(a + k * 32), smem_desc(b + k * 32), id, sf, sf + 8,
                   (kb > 0 || k > 0) ? 1u : 0u);
            mma_mx(tmem, smem_desc(a + kTile + k * 32), smem_desc(b + k * 32), id, sf + 4, sf + 8,
                   1u);
          }
          mma_commit(&sm.empty[s]);
        }
        if (!ok) break;
        mma_commit(&sm.acc_full);
        ++i;
      }
      mma_commit(&sm.drain);
      mbar_wait_drain(&sm.drain, 0);
    }
  } else {
    // ---- epilogue: warp w has TMEM lanes 32 (w % 4) .. +31 and half the columns; a row a thread
    const int q = warp & 3;
    const int hf = (warp - 4) >> 2;
    int i = 0;
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const int blk = t / n_tiles, ft = t - blk * n_tiles;
      if (expert_of(blk) < 0) continue;
      const int r = q * 32 + lane;
      const int route = p.routes.sorted_ids[blk * 128 + r];
      const bool real = route < p.numel;
      const bool ok = mbar_wait(&sm.acc_full, i & 1, failed);
      fence_after_sync();
      if (!__all_sync(0xffffffffu, ok && !*failed)) break;
      const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
      // columns [64 hf, +64) and [128 + 64 hf, +64): 64 features' gate and up, or two runs of 64
      // output columns
      uint32_t v[8][16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        tmem_load16(taddr + 64 * hf + 16 * j, v[j]);
        tmem_load16(taddr + 128 + 64 * hf + 16 * j, v[4 + j]);
      }
      tmem_wait();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty);
      ++i;
      if (DOWN) {
        if (real) {
          const float wr = p.route_w[route];
          float* o = p.out + (int64_t)route * p.hidden + ft * 256 + 64 * hf;
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < 16; c += 4)
              *reinterpret_cast<float4*>(o + (j >> 2) * 128 + (j & 3) * 16 + c) = make_float4(
                  __uint_as_float(v[j][c]) * wr, __uint_as_float(v[j][c + 1]) * wr,
                  __uint_as_float(v[j][c + 2]) * wr, __uint_as_float(v[j][c + 3]) * wr);
        }
      } else if (real) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {  // two scale blocks of 32 features
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float gt = __uint_as_float(v[2 * b + j][c]);
              const float h = gt / (1.0f + __expf(-gt)) * __uint_as_float(v[4 + 2 * b + j][c]);
              v[2 * b + j][c] = __float_as_uint(h);
              top = max(top, __float_as_uint(h) & 0x7fffffffu);
            }
          const uint32_t sb = split_scale(top);
          const float inv = split_inverse(sb);
          const int feat = ft * 128 + 64 * hf + 32 * b;
          uint8_t* hi_row = p.hq + ((int64_t)blk * 256 + r) * p.inter + feat;
          uint8_t* lo_row = hi_row + (int64_t)128 * p.inter;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t h0, l0, h1, l1;
              split2(__uint_as_float(v[2 * b + j][4 * c]),
                     __uint_as_float(v[2 * b + j][4 * c + 1]), inv, h0, l0);
              split2(__uint_as_float(v[2 * b + j][4 * c + 2]),
                     __uint_as_float(v[2 * b + j][4 * c + 3]), inv, h1, l1);
              hi[c] = h0 | h1 << 16;
              lo[c] = l0 | l1 << 16;
            }
            reinterpret_cast<uint4*>(hi_row)[j] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            reinterpret_cast<uint4*>(lo_row)[j] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
          p.hs[scale_at(2 * blk, p.inter / kMxK, feat / 32, r)] = (uint8_t)sb;
          p.hs[scale_at(2 * blk, p.inter / kMxK, feat / 32, 128 + r)] =
              (uint8_t)split_lo_byte(sb);
        }
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    fence_after_sync();
    tmem_free(tmem, 512);
  }
  if (sm.failed) {
    drain_loads<kMxGemmStages>(sm.full, issued);
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 1);
  }
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
// The route block, which also picks the kernels: 32 or 64 routes on the N side (decode) while the
// average expert's routes fit with room for the fuller ones (an expert's second block reads its
// weights again), else 128 on the M side (prefill).
static int mx_block(int64_t numel, int experts) {
  return numel <= (int64_t)experts * 18 ? 32 : numel <= (int64_t)experts * 44 ? 64 : 128;
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
  const int tables = scale_tables(w.block);
  w.xs = take(blocks * tables * (hidden / kMxK) * 512);
  w.hq = take(2 * cap * inter);
  w.hs = take(blocks * tables * (inter / kMxK) * 512);
  w.out = reinterpret_cast<float*>(take(numel * hidden * 4));
  w.sync_ints = (int)(1 + blocks);
  w.sync = reinterpret_cast<int32_t*>(take(w.sync_ints * 4));
  w.bytes = off;
  return w;
}

// Raises a kernel's shared-memory limit once per device.
template <typename K>
static cudaError_t allow_smem(K* kern, size_t bytes, std::mutex& mu, bool (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  if (done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  done[dev] = e == cudaSuccess;
  return e;
}

static MxLayerParams layer_params(const MxArgs& a, const MxWorkspace& w) {
  MxLayerParams p{};
  p.routes = {w.num_post_pad, w.expert_ids, w.sorted_ids};
  p.experts = a.experts;
  p.numel = (int)(a.tokens * a.top_k);
  p.hidden = a.hidden;
  p.inter = a.inter;
  p.m_blocks = (int)(w.capacity / w.block);
  p.status = a.status;
  p.s13 = a.s13;
  p.s2 = a.s2;
  p.xs = w.xs;
  p.hq = w.hq;
  p.hs = w.hs;
  p.route_w = a.topk_w;
  p.out = w.out;
  p.sync = w.sync;
  return p;
}

template <int BT>
static cudaError_t launch_mx_layer(const MxArgs& a, const MxWorkspace& w, cudaStream_t s) {
  auto* kern = mx_layer_kernel<BT>;
  static std::mutex mu;
  static bool done[64] = {};
  const cudaError_t e = allow_smem(kern, mx_smem_bytes<BT>(), mu, done);
  if (e != cudaSuccess) return e;
  const int64_t rows = w.capacity / BT * 2 * BT;
  CUtensorMap m13, mx, m2, mh;
  if (!make_map_4bit(&m13, a.w13, (uint64_t)a.experts * 2 * a.inter, a.hidden, 128) ||
      !make_map_8bit(&mx, w.xq, rows, a.hidden, 2 * BT) ||
      !make_map_4bit(&m2, a.w2, (uint64_t)a.experts * a.hidden, a.inter, 128) ||
      !make_map_8bit(&mh, w.hq, rows, a.inter, 2 * BT))
    return cudaErrorInvalidValue;
  const int sms = sm_count();
  return launch_pdl(kern, sms > 0 ? (unsigned)sms : 1u, kMxLayerThreads, mx_smem_bytes<BT>(), s,
                    m13, mx, m2, mh, layer_params(a, w));
}

template <bool DOWN>
static cudaError_t launch_mx_gemm(const MxArgs& a, const MxWorkspace& w, cudaStream_t s) {
  auto* kern = mx_gemm_kernel<DOWN>;
  static std::mutex mu;
  static bool done[64] = {};
  const cudaError_t e = allow_smem(kern, mx_gemm_smem_bytes(), mu, done);
  if (e != cudaSuccess) return e;
  CUtensorMap mw, mt;
  const int k = DOWN ? a.inter : a.hidden;
  if (!make_map_4bit(&mw, DOWN ? a.w2 : a.w13,
                     (uint64_t)a.experts * (DOWN ? a.hidden : 2 * a.inter), k, 128) ||
      !make_map_8bit(&mt, DOWN ? w.hq : w.xq, 2 * w.capacity, k, 256))
    return cudaErrorInvalidValue;
  const int64_t tiles = w.capacity / 128 * (DOWN ? a.hidden / 256 : a.inter / 128);
  const int sms = sm_count();
  return launch_pdl(kern, (unsigned)(sms > 0 && tiles > sms ? sms : tiles), kMxGemmThreads,
                    mx_gemm_smem_bytes(), s, mw, mt, layer_params(a, w));
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
  if (w.block == 128) {
    e = launch_mx_gemm<false>(a, w, s);
    if (e == cudaSuccess) e = launch_mx_gemm<true>(a, w, s);
  } else {
    e = w.block == 32 ? launch_mx_layer<32>(a, w, s) : launch_mx_layer<64>(a, w, s);
  }
  if (e != cudaSuccess) return e;
  return launch_pdl(mx_combine_kernel, stream_grid(a.tokens * (a.hidden / 4)), 256, 0, s,
                    static_cast<const float*>(w.out), a.topk_ids, a.experts, a.tokens, a.top_k,
                    a.hidden, static_cast<__nv_bfloat16*>(a.y));
}

}  // namespace exf
