// The SwiGLU expert layer with MXFP4 weights (sm_100a: tcgen05 block-scaled MMA + TMA):
//   y[t] = sum_j w[t, j] W2[e] (silu(W1[e] x[t]) * (W3[e] x[t])),  e = ids[t, j].
//
// The weights go to the tensor cores as they are: TMA pads 16 packed codes to 16 bytes, and
// tcgen05.mma kind::mxf8f6f4 takes e2m1 codes with their E8M0 scales (one per row and 32 k) against
// 8-bit activations, which enter as the sum of two e4m3 terms (exf_mx.cuh).  The products are exact,
// the sums fp32.
//
// A few routes take kernels of their own (mx_few.cu).  Else the launches are: moe_align and the token
// rows' two-term form in route order (one launch up to 8192 routes) -> the layer (decode: both GEMMs
// in one persistent launch; prefill: a launch each) -> combine (each token's routes summed in fp32,
// in order).
#include <cuda.h>
#include <cuda_bf16.h>

#include <mutex>

#include "exf_common.cuh"
#include "exf_launch.h"
#include "exf_mx.cuh"
#include "exf_mxmoe.h"
#include "exf_tc.cuh"

namespace exf {
using namespace tc;

constexpr int kMxLayerThreads = 416;  // warps 0, 2, 3 TMA, 1 MMA, 4-11 epilogue, 12 schedule

// ---- token rows in route order (more than align_gather_max_numel() routes) -----------------------
// A warp takes 1024 columns of a token: they are split once and written to the slots of its routes.
__global__ void __launch_bounds__(256) mx_split_kernel(const __nv_bfloat16* x, const int32_t* slots,
                                                       int64_t tokens, int top_k, MxRows rows,
                                                       int32_t* zero, int zero_n) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < zero_n; i += gridDim.x * blockDim.x)
    zero[i] = 0;
  const int lane = threadIdx.x & 31;
  const int vecs = rows.hidden / 8;          // a multiple of 32
  const int pieces = (vecs + 127) / 128;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t u = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
       u < tokens * pieces; u += warps) {
    const int64_t t = u / pieces;
    const int c0 = (int)(u - t * pieces) * 128;
    int mine = lane < top_k ? slots[t * top_k + lane] : -1;
    if (mine >= 0) mine = mx_slot_row(rows.block, mine);
    if (__ballot_sync(0xffffffffu, mine >= 0) == 0) continue;
    const uint4* row = reinterpret_cast<const uint4*>(x + t * rows.hidden);
    uint4 raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      raw[j] = c0 + 32 * j < vecs ? __ldcg(row + c0 + 32 * j + lane) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 32 * j + lane;
      if (c0 + 32 * j >= vecs) break;
      const MxTerms v = split8(raw[j]);
      for (int r = 0; r < top_k; ++r) {
        const int to = __shfl_sync(0xffffffffu, mine, r);
        if (to >= 0) put8(rows, to, c, v);
      }
    }
  }
}

// ---- decode ---------------------------------------------------------------------------------------
// A tile is 256 weight rows of one expert (two MMA tiles of 128 rows on the M side) times a block of
// BT = 16 or 32 of its routes (the N side: 2 BT hi and lo rows).
//   GEMM-1 tile (block, f): gate rows [128 f, +128) and up rows [I + 128 f, +128) of W13[e], K = H;
//     the epilogue forms h = silu(gate) * up and writes its two-term form;
//   GEMM-2 tile (block, f): rows [256 f, +256) of W2[e], K = I; out[route][256 f + i] = w_route D.
// One persistent launch: a scheduler warp takes tiles from a counter (every GEMM-1 tile, then the
// GEMM-2 tiles) and passes them on through a ring.  Three warps load: the first 128 weight rows, the
// second, and the token rows, each with its scales (a row of packed codes is a 64-byte request:
// padded tiles stream at 5.3 TB/s from one issuing thread and at 6.6 from two).  The warp that
// loads tokens waits, before the first load of a GEMM-2 tile, until the epilogue warps of the
// block's GEMM-1 tiles have counted themselves off; the weights of such a tile do not wait.  A
// GEMM-1 tile waits only for earlier GEMM-1 tiles of its own CTA and was handed out before every
// GEMM-2 tile, so the wait ends; it is bounded all the same.
//
// 8 epilogue warps sum the two terms into registers and give the accumulator back before they
// compute; there are two accumulators.
//
// What bounds the layer is the bytes in flight: padded, a stage's 17 KB of codes and scales take
// 32 KB of shared memory and its token rows 4 or 8.  us of a 742 MB layer with blocks of 16: 149 with
// four stages, 141 with five, 139 with six.
template <int BT>
struct MxCfg {
  static constexpr int kN = 2 * BT;
  static constexpr int kTTile = kN * kMxK;
  static constexpr int kWTile = 128 * kMxK;              // padded codes of 128 rows
  static constexpr int kStages = BT == 16 ? 6 : 5;
  static constexpr int kRing = 4;                        // tiles handed out ahead
  static constexpr int kAccCols = 2 * kN;
  static constexpr int kScaleCol = 2 * kAccCols;         // 4 sets of 16 columns
  static constexpr int kTmemCols = kScaleCol + 64 <= 256 ? 256 : 512;
};
struct MxTile {
  int kind;      // kGate, kDown, or kEnd: no more tiles
  int blk, ft;
  int expert;
  int quarters;  // 32-row quarters of the block that hold routes
};
enum { kEnd = -1, kGate = 0, kDown = 1 };
template <int BT>
struct MxSmem {
  using C = MxCfg<BT>;
  // a stage: 256 rows of codes, token rows
  alignas(1024) uint8_t tiles[C::kStages][2 * C::kWTile + C::kTTile];
  alignas(128) uint8_t scales[C::kStages][3][512];  // token rows, first and second weight rows
  alignas(8) uint64_t full[C::kStages];
  alignas(8) uint64_t empty[C::kStages];
  alignas(8) uint64_t acc_full[2];
  alignas(8) uint64_t acc_empty[2];
  alignas(8) uint64_t ring_full[C::kRing];
  alignas(8) uint64_t ring_empty[C::kRing];
  alignas(8) uint64_t drain;
  MxTile ring[C::kRing];
  uint32_t tmem_base;
  int failed;
};
template <int BT>
constexpr size_t mx_smem_bytes() { return sizeof(MxSmem<BT>) + 1024; }
static_assert(mx_smem_bytes<16>() <= 232448 && mx_smem_bytes<32>() <= 232448,
              "decode expert layer shared memory");

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

__device__ __forceinline__ float silu_up(float g, float u) { return g * logistic(g) * u; }

// N consecutive fp32 columns of this thread's TMEM lane, N = 8 or 16
template <int N>
__device__ __forceinline__ void tmem_load_cols(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 8)
    tmem_load8(taddr, r);
  else
    tmem_load16(taddr, r);
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
  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 3);  // one arrival per loading warp
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 8);
    }
    for (int j = 0; j < kRing; ++j) {
      mbar_init(&sm.ring_full[j], 1);
      mbar_init(&sm.ring_empty[j], 12);  // three loading warps, the MMA thread, 8 epilogue warps
    }
    mbar_init(&sm.drain, 1);
    sm.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 32) {
    prefetch_map(&map_w13);
    prefetch_map(&map_xq);
    prefetch_map(&map_w2);
    prefetch_map(&map_hq);
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
  const uint32_t tmem = uniform(sm.tmem_base);
  volatile int* failed = &sm.failed;
  // the next tile from the ring, for a whole warp
  auto next_tile = [&](int j, MxTile& lt) {
    const int slot = j % kRing;
    if (!warp_wait(&sm.ring_full[slot], (j / kRing) & 1, failed)) return false;
    const MxTile& t = sm.ring[slot];
    lt = {uniform(t.kind), uniform(t.blk), uniform(t.ft), uniform(t.expert), uniform(t.quarters)};
    if (lane == 0) mbar_arrive(&sm.ring_empty[slot]);
    return lt.kind != kEnd;
  };

  uint32_t issued = 0;  // stages this thread has loaded into
  if (warp == 12) {
    // ---- scheduler: takes tiles from the counter and looks up what the other roles need to know of
    // them (each of them doing so for itself lost a memory latency or two at every tile)
    for (int j = 0;; ++j) {
      int t = lane == 0 ? atomicAdd(p.sync, 1) : 0;
      t = __shfl_sync(0xffffffffu, t, 0);
      MxTile lt{kEnd, 0, 0, 0, 0};
      if (t < total) {
        lt.kind = t < blocks * n1 ? kGate : kDown;
        if (lt.kind == kDown) t -= blocks * n1;
        const int n = lt.kind == kDown ? n2 : n1;
        lt.blk = t / n;
        lt.ft = t - lt.blk * n;
        lt.expert = p.routes.expert_ids[lt.blk];
        const int32_t* ids = p.routes.sorted_ids + (int64_t)lt.blk * BT;
        const int real = __popc(__ballot_sync(0xffffffffu, lane < BT && ids[lane] < p.numel));
        lt.quarters = (real + 15) >> 4;
        if (lt.expert < 0 || lt.expert >= p.experts) {
          --j;
          continue;
        }
      }
      const int slot = j % kRing;
      if (!warp_wait(&sm.ring_empty[slot], ((j / kRing) & 1) ^ 1, failed)) break;
      if (lane == 0) {
        sm.ring[slot] = lt;
        mbar_arrive(&sm.ring_full[slot]);
      }
      if (lt.kind == kEnd) break;
    }
  } else if (warp == 0 || warp == 2) {
    // ---- weight loads: gate (warp 0) and up (warp 2) rows of W13[e], or the halves of 256 rows of
    // W2[e]
    const int half = warp == 0 ? 0 : 1;
    uint32_t g = 0;
    bool ok = true;
    MxTile lt;
    for (int j = 0; ok && next_tile(j, lt); ++j) {
      const bool down = lt.kind == kDown;
      const int kblocks = (down ? p.inter : p.hidden) / kMxK;
      const int row = down ? lt.expert * p.hidden + lt.ft * 256 + half * 128
                           : lt.expert * 2 * p.inter + lt.ft * 128 + half * p.inter;
      const CUtensorMap* map = down ? &map_w2 : &map_w13;
      const uint8_t* sc = (down ? p.s2 : p.s13) + (int64_t)(row / 128) * kblocks * 512;
      for (int kb = 0; kb < kblocks; ++kb, ++g) {
        const int s = g % kStages;
        ok = warp_wait(&sm.empty[s], ((g / kStages) & 1) ^ 1, failed);
        if (!ok) break;
        if (elect_one()) {
          mbar_expect_tx(&sm.full[s], C::kWTile / 2 + 512);  // codes count as they lie in memory
          tma_load_2d(sm.tiles[s] + half * C::kWTile, map, &sm.full[s], kb * kMxK, row);
          bulk_load(sm.scales[s][1 + half], sc + kb * 512, 512, &sm.full[s]);
        }
      }
    }
    issued = g;
  } else if (warp == 3) {
    // ---- token loads: the quarters of the block that hold routes
    uint32_t g = 0;
    bool ok = true;
    MxTile lt;
    for (int j = 0; ok && next_tile(j, lt); ++j) {
      const bool down = lt.kind == kDown;
      if (down) {
        const int32_t* flag = p.sync + 1 + lt.blk;
        for (uint32_t it = 0; ok && !__all_sync(0xffffffffu, ld_acquire_gpu(flag) >= 8 * n1);) {
          ok = !__any_sync(0xffffffffu, *failed || ++it >= kWaitLimit);
          if (!ok) *failed = 1;
          __nanosleep(32);
        }
        if (!ok) break;
        asm volatile("fence.proxy.async.global;" ::: "memory");
      }
      const int kblocks = (down ? p.inter : p.hidden) / kMxK;
      const CUtensorMap* map = down ? &map_hq : &map_xq;
      const uint8_t* sc = (down ? p.hs : p.xs) + (int64_t)lt.blk * kblocks * 512;
      for (int kb = 0; kb < kblocks; ++kb, ++g) {
        const int s = g % kStages;
        ok = warp_wait(&sm.empty[s], ((g / kStages) & 1) ^ 1, failed);
        if (!ok) break;
        if (elect_one()) {
          mbar_expect_tx(&sm.full[s], lt.quarters * 32 * kMxK + 512);
          for (int q = 0; q < lt.quarters; ++q)
            tma_load_2d(sm.tiles[s] + 2 * C::kWTile + q * 32 * kMxK, map, &sm.full[s],
                        kb * kMxK, lt.blk * 2 * BT + 32 * q);
          bulk_load(sm.scales[s][0], sc + kb * 512, 512, &sm.full[s]);
        }
      }
    }
    issued = g;
  } else if (warp == 1) {
    // ---- MMA issuer; scale sets rotate over 4 groups of 16 TMEM columns
    uint32_t g = 0;
    int i = 0;
    bool ok = true;
    MxTile lt;
    for (int j = 0; ok && next_tile(j, lt); ++j) {
      const int kblocks = (lt.kind == kDown ? p.inter : p.hidden) / kMxK;
      const int b = i % 2;
      ok = warp_wait(&sm.acc_empty[b], ((i / 2) & 1) ^ 1, failed);
      if (!ok) break;
      fence_after_sync();
      const uint32_t acc = tmem + static_cast<uint32_t>(b * C::kAccCols);
      for (int kb = 0; kb < kblocks; ++kb, ++g) {
        const int s = g % kStages;
        ok = warp_wait(&sm.full[s], (g / kStages) & 1, failed);
        if (!ok) break;
        fence_after_sync();
        const uint64_t w0 = smem_desc(smem_addr(sm.tiles[s]));
        const uint64_t w1 = w0 + C::kWTile / 16, t0 = w0 + 2 * C::kWTile / 16;
        const uint32_t sc = smem_addr(sm.scales[s][0]);
        const uint32_t sf = tmem + C::kScaleCol + (g & 3) * 16;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 3; ++k) tmem_copy_scales(sf + 4 * k, sc + k * 512);
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // a K step is 32 bytes further on: 2 in the descriptor
            const uint32_t on = (kb > 0 || k > 0) ? 1u : 0u;
            const uint32_t id = idesc_mx(128, C::kN, kMxE2M1, kMxE4M3, k);
            mma_mx(acc, w0 + 2 * k, t0 + 2 * k, id, sf + 4, sf, on);
            mma_mx(acc + C::kN, w1 + 2 * k, t0 + 2 * k, id, sf + 8, sf, on);
          }
          mma_commit(&sm.empty[s]);
        }
      }
      if (!ok) break;
      if (elect_one()) mma_commit(&sm.acc_full[b]);
      ++i;
    }
    if (elect_one()) mma_commit(&sm.drain);
    mbar_wait_drain(&sm.drain, 0);
  } else {
    // ---- epilogue: a warp has 32 weight rows of each MMA tile (TMEM lanes 32 q .. +31) and half of
    // the block's routes; in the columns of 16 routes the hi rows come first, then the lo rows
    constexpr int kHalf = BT / 2;
    const int q = warp & 3, hf = (warp - 4) >> 2;
    int i = 0;
    MxTile lt;
    for (int j = 0; next_tile(j, lt); ++j) {
      const bool down = lt.kind == kDown;
      // lane l looks after route l of the warp's half
      const int r0 = hf * kHalf;
      const int route_l = lane < kHalf ? p.routes.sorted_ids[lt.blk * BT + r0 + lane] : p.numel;
      const float w_l = down && route_l < p.numel ? p.route_w[route_l] : 0.0f;
      const int real = __popc(__ballot_sync(0xffffffffu, route_l < p.numel));  // they come first
      const int b = i % 2;
      if (!warp_wait(&sm.acc_full[b], (i / 2) & 1, failed)) break;
      fence_after_sync();
      float v0[kHalf], v1[kHalf];  // gate and up, or rows r and r + 128
      if (real > 0) {
        const uint32_t col = tmem + static_cast<uint32_t>(b * C::kAccCols) +
                             ((uint32_t)(q * 32) << 16) + 32 * (r0 >> 4) + (r0 & 15);
        uint32_t a0[kHalf], a1[kHalf], b0[kHalf], b1[kHalf];
        tmem_load_cols<kHalf>(col, a0);
        tmem_load_cols<kHalf>(col + 16, a1);
        tmem_load_cols<kHalf>(col + C::kN, b0);
        tmem_load_cols<kHalf>(col + C::kN + 16, b1);
        tmem_wait();
#pragma unroll
        for (int n = 0; n < kHalf; ++n) {
          v0[n] = __uint_as_float(a0[n]) + __uint_as_float(a1[n]);
          v1[n] = __uint_as_float(b0[n]) + __uint_as_float(b1[n]);
        }
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[b]);
      ++i;
      if (!down) {
        const int feat = lt.ft * 128 + q * 32 + lane;  // the warp's features: one scale block
#pragma unroll
        for (int n = 0; n < kHalf; ++n) {
          if (n >= real) break;
          const float h = silu_up(v0[n], v1[n]);
          const uint32_t sb =
              split_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7fffffffu));
          uint32_t hi, lo;
          split2(h, 0.0f, split_inverse(sb), hi, lo);
          const int row = mx_row(BT, r0 + n);
          uint8_t* at = p.hq + ((int64_t)lt.blk * C::kN + row) * p.inter + feat;
          at[0] = (uint8_t)hi;
          at[(int64_t)mx_lo(BT) * p.inter] = (uint8_t)lo;
          if (lane < 2)
            p.hs[scale_at(lt.blk, p.inter / kMxK, feat >> 5, lane ? row + mx_lo(BT) : row)] =
                (uint8_t)(lane ? split_lo_byte(sb) : sb);
        }
      } else {
        float* o = p.out + lt.ft * 256 + q * 32 + lane;
#pragma unroll
        for (int n = 0; n < kHalf; ++n) {
          if (n >= real) break;
          const int64_t route = __shfl_sync(0xffffffffu, route_l, n);
          const float wr = __shfl_sync(0xffffffffu, w_l, n);
          o[route * p.hidden] = v0[n] * wr;
          o[route * p.hidden + 128] = v1[n] * wr;
        }
      }
      if (!down) {
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

// The route outputs at prefill, 16-bit: 32 columns share u = 2^(byte - 127), the largest magnitude
// being in [2^13 u, 2^14 u); a value is a signed 16-bit multiple of u, within 2^-14 of that magnitude.
// (bf16 route outputs would add as much error as the result's own rounding, fp32 ones twice the
// traffic.)  Values that are not finite leave the other 31 as they are: they have multiples beyond
// +-2^14, which no finite value reaches.
constexpr int kHalfNan = -32768, kHalfInf = 32767;  // and -32767
__device__ __forceinline__ uint32_t half_scale(uint32_t top_bits) {
  const uint32_t e = top_bits >> 23;
  return e < 14 ? 1u : e - 13u;
}
// 32 columns with a value that is not finite, or of which the largest before its weight is below
// 2^-113 (the factor of store_halves would overflow); returns their byte
__device__ __forceinline__ uint32_t store_by_value(int16_t* at, const uint32_t* v0,
                                                     const uint32_t* v1, float wr) {
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const uint32_t x =
        __float_as_uint(__uint_as_float(c < 16 ? v0[c] : v1[c - 16]) * wr) & 0x7fffffffu;
    if (x < 0x7f800000u) top = max(top, x);
  }
  const uint32_t sb = half_scale(top);
  const float inv = __uint_as_float((254u - sb) << 23);
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const float x = __uint_as_float(c < 16 ? v0[c] : v1[c - 16]) * wr;
    const int q = x != x                  ? kHalfNan
                  : isinf(x)              ? (x > 0.0f ? kHalfInf : -kHalfInf)
                                          : __float2int_rn(x * inv);
    at[c] = (int16_t)q;
  }
  return sb;
}
// the value of a multiple
__device__ __forceinline__ float half_value(int q, float s) {
  return q == kHalfNan    ? __uint_as_float(0x7fffffffu)
         : q == kHalfInf  ? __uint_as_float(0x7f800000u)
         : q == -kHalfInf ? __uint_as_float(0xff800000u)
                          : (float)q * s;
}
// 16 values times w -> 16 multiples, one 32-byte sector.  Adding 1.5 2^23 rounds to an integer, whose
// low 16 bits are its two's complement.
__device__ __forceinline__ void store_halves(int16_t* at, const uint32_t* v, float w) {
  uint32_t o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    o[j] = __byte_perm(__float_as_uint(fmaf(__uint_as_float(v[2 * j]), w, 12582912.0f)),
                       __float_as_uint(fmaf(__uint_as_float(v[2 * j + 1]), w, 12582912.0f)), 0x5410);
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(o[0]),
               "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
               : "memory");
}

template <bool DOWN>
__global__ void __launch_bounds__(kMxGemmThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_t, const MxLayerParams p) {
  constexpr int kTile = 128 * kMxK;
  extern __shared__ uint8_t smem_raw[];
  MxGemmSmem& sm = *reinterpret_cast<MxGemmSmem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = uniform(threadIdx.x >> 5);
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
  const uint32_t tmem = uniform(sm.tmem_base);
  volatile int* failed = &sm.failed;
  auto expert_of = [&](int blk) {
    const int e = p.routes.expert_ids[blk];
    return uniform((e >= 0 && e < p.experts) ? e : -1);
  };

  uint32_t issued = 0;
  if (warp == 0 || warp == 2 || warp == 3) {
    // ---- loads: warp 0 the hi and lo rows, warps 2 and 3 a weight tile each
    uint32_t g = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const int blk = t / n_tiles, ft = t - blk * n_tiles;
      const int expert = expert_of(blk);
      if (expert < 0) continue;
      const int half = warp - 2;
      const int row = DOWN ? expert * p.hidden + ft * 256 + half * 128
                           : expert * 2 * p.inter + ft * 128 + half * p.inter;
      // quarters of 32 routes that hold any (routes fill their block from its first row)
      const int first = p.routes.sorted_ids[blk * 128 + 32 * (lane & 3)];
      const int quarters = __popc(__ballot_sync(0xffffffffu, lane < 4 && first < p.numel));
      const uint8_t* sc = warp == 0
                              ? (DOWN ? p.hs : p.xs) + (int64_t)blk * 2 * kblocks * 512
                              : (DOWN ? p.s2 : p.s13) + (int64_t)(row / 128) * kblocks * 512;
      for (int kb = 0; kb < kblocks; ++kb, ++g) {
        const int s = g % kMxGemmStages;
        ok = warp_wait(&sm.empty[s], ((g / kMxGemmStages) & 1) ^ 1, failed);
        if (!ok) break;
        uint64_t* bar = &sm.full[s];
        if (elect_one()) {
          if (warp == 0) {
            mbar_expect_tx(bar, quarters * (2 * kTile / 4) + 1024);
            for (int q = 0; q < quarters; ++q) {
              tma_load_2d(sm.tiles[s] + q * (kTile / 4), &map_t, bar, kb * kMxK,
                          blk * 256 + 32 * q);
              tma_load_2d(sm.tiles[s] + kTile + q * (kTile / 4), &map_t, bar, kb * kMxK,
                          blk * 256 + 128 + 32 * q);
            }
            bulk_load(sm.scales[s], sc + kb * 512, 512, bar);
            bulk_load(sm.scales[s] + 512, sc + (int64_t)(kblocks + kb) * 512, 512, bar);
          } else {
            mbar_expect_tx(bar, kTile / 2 + 512);
            tma_load_2d(sm.tiles[s] + (2 + half) * kTile, &map_w, bar, kb * kMxK, row);
            bulk_load(sm.scales[s] + 1024 + half * 512, sc + kb * 512, 512, bar);
          }
        }
      }
    }
    issued = g;
  } else if (warp == 1) {
    // ---- MMA issuer
    uint32_t g = 0;
    int i = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      if (expert_of(t / n_tiles) < 0) continue;
      ok = warp_wait(&sm.acc_empty, (i & 1) ^ 1, failed);
      if (!ok) break;
      fence_after_sync();
      for (int kb = 0; kb < kblocks; ++kb, ++g) {
        const int s = g % kMxGemmStages;
        ok = warp_wait(&sm.full[s], (g / kMxGemmStages) & 1, failed);
        if (!ok) break;
        fence_after_sync();
        const uint64_t hi = smem_desc(smem_addr(sm.tiles[s]));
        const uint64_t lo = hi + kTile / 16, w = hi + 2 * kTile / 16;
        const uint32_t sc = smem_addr(sm.scales[s]);
        const uint32_t sf = tmem + 256 + (g & 3) * 16;
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j) tmem_copy_scales(sf + 4 * j, sc + 512 * j);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t id = idesc_mx(128, 256, kMxE4M3, kMxE2M1, k);
            mma_mx(tmem, hi + 2 * k, w + 2 * k, id, sf, sf + 8, (kb > 0 || k > 0) ? 1u : 0u);
            mma_mx(tmem, lo + 2 * k, w + 2 * k, id, sf + 4, sf + 8, 1u);
          }
          mma_commit(&sm.empty[s]);
        }
      }
      if (!ok) break;
      if (elect_one()) mma_commit(&sm.acc_full);
      ++i;
    }
    if (elect_one()) mma_commit(&sm.drain);
    mbar_wait_drain(&sm.drain, 0);
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
      if (!warp_wait(&sm.acc_full, i & 1, failed)) break;
      fence_after_sync();
      const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
      // 64 features' gate and up: columns [64 hf, +64) and [128 + 64 hf, +64); or 128 output columns
      uint32_t v[8][16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        tmem_load16(taddr + (DOWN ? 128 : 64) * hf + 16 * j, v[j]);
        tmem_load16(taddr + (DOWN ? 64 + 128 * hf : 128 + 64 * hf) + 16 * j, v[4 + j]);
      }
      tmem_wait();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty);
      ++i;
      if (DOWN) {
        if (real) {
          const float wr = p.route_w[route];
          const int64_t at = (int64_t)route * p.hidden + ft * 256 + 128 * hf;
          int16_t* o = reinterpret_cast<int16_t*>(p.out);
          uint32_t bytes = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {  // runs of 32 columns
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int c = 0; c < 16; ++c) top = max(top, v[2 * b + j][c] & 0x7fffffffu);
            top = __float_as_uint(__uint_as_float(top) * wr) & 0x7fffffffu;
            uint32_t sb = half_scale(top);
            const float w = wr * __uint_as_float((254u - sb) << 23);
            if (top >= 0x7f800000u || isinf(w)) {
              sb = store_by_value(o + at + 32 * b, v[2 * b], v[2 * b + 1], wr);
            } else {
              store_halves(o + at + 32 * b, v[2 * b], w);
              store_halves(o + at + 32 * b + 16, v[2 * b + 1], w);
            }
            bytes |= sb << (8 * b);
          }
          *reinterpret_cast<uint32_t*>(p.out_scale + at / 32) = bytes;
        }
      } else if (real) {
        uint32_t hi_bytes = 0, lo_bytes = 0;
#pragma unroll
        for (int b = 0; b < 2; ++b) {  // two scale blocks of 32 features
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float h = silu_up(__uint_as_float(v[2 * b + j][c]),
                                      __uint_as_float(v[4 + 2 * b + j][c]));
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
          hi_bytes |= sb << (8 * b);
          lo_bytes |= split_lo_byte(sb) << (8 * b);
        }
        // the two blocks' scales are neighbouring bytes
        const int kb = ft * 4 + 2 * hf;
        *reinterpret_cast<uint16_t*>(p.hs + scale_at(2 * blk, p.inter / kMxK, kb, r)) =
            (uint16_t)hi_bytes;
        *reinterpret_cast<uint16_t*>(p.hs + scale_at(2 * blk, p.inter / kMxK, kb, 128 + r)) =
            (uint16_t)lo_bytes;
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
// y[t] = sum_j out[t * top_k + j] in fp32, in route order; routes out of range were never placed.  (These
// kernels may be resident while the one before still writes what they read after their wait: no load
// through the read-only path, here and wherever a kernel reads a predecessor's results.)
// The 16-bit form of the route outputs (prefill).
__global__ void __launch_bounds__(256)
    mx_combine16_kernel(const int16_t* out, const uint8_t* out_scale, const int32_t* ids, int experts,
                        int64_t tokens, int top_k, int hidden, __nv_bfloat16* y) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // a warp takes 1024 columns of a token, 256 at a time, the loads of all its routes together
  const int lane = threadIdx.x & 31;
  const int vecs = hidden / 8;  // a multiple of 32
  const int pieces = (vecs + 127) / 128;
  const uint4* out4 = reinterpret_cast<const uint4*>(out);
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t u = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
       u < tokens * pieces; u += warps) {
    const int64_t t = u / pieces;
    const int c0 = (int)(u - t * pieces) * 128;
    const int e = lane < top_k ? ids[t * top_k + lane] : -1;
    const uint32_t use = __ballot_sync(0xffffffffu, e >= 0 && e < experts);
    for (int c1 = c0; c1 < c0 + 128 && c1 < vecs; c1 += 32) {
      const int c = c1 + lane;
      uint4 v[8];
      uint32_t b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if ((use >> j) & 1) {
          v[j] = __ldcg(out4 + (t * top_k + j) * vecs + c);
          b[j] = __ldcg(out_scale + (t * top_k + j) * (vecs / 4) + (c >> 2));
        }
      }
      float acc[8] = {};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!((use >> j) & 1)) continue;
        const float s = __uint_as_float(b[j] << 23);
        const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
        // multiples outside [-2^14, 2^14) differ in their two highest bits
        uint32_t far = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) far |= w[k] ^ (w[k] << 1);
        if (far & 0x80008000u) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            acc[2 * k] += half_value((int16_t)(w[k] & 0xffffu), s);
            acc[2 * k + 1] += half_value((int32_t)w[k] >> 16, s);
          }
          continue;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          // a signed 16-bit q, its sign bit flipped, in the low bits of 2^23: 2^23 + 2^15 + q
          const uint32_t f = w[k] ^ 0x80008000u;
          acc[2 * k] = fmaf(__uint_as_float(__byte_perm(f, 0x4b000000u, 0x7610)) - 8421376.0f, s,
                            acc[2 * k]);
          acc[2 * k + 1] = fmaf(__uint_as_float(__byte_perm(f, 0x4b000000u, 0x7632)) - 8421376.0f,
                                s, acc[2 * k + 1]);
        }
      }
      reinterpret_cast<uint4*>(y)[t * vecs + c] =
          make_uint4(pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3]),
                     pack_bf16(acc[4], acc[5]), pack_bf16(acc[6], acc[7]));
    }
  }
}

// fp32 route outputs (decode): a warp takes 256 columns of a token.
__global__ void __launch_bounds__(256)
    mx_combine_kernel(const float* out, const int32_t* ids, int experts, int64_t tokens,
                      int top_k, int hidden, __nv_bfloat16* y) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int pieces = hidden / 256;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
  for (int64_t u = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
       u < tokens * pieces; u += warps) {
    const int64_t t = u / pieces;
    const int c = (int)(u - t * pieces) * 256 + 4 * lane;
    const int e = lane < top_k ? ids[t * top_k + lane] : -1;
    const uint32_t use = __ballot_sync(0xffffffffu, e >= 0 && e < experts);
    float4 v[8][2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!((use >> j) & 1)) continue;
      const float* o = out + (t * top_k + j) * hidden + c;
      v[j][0] = __ldcg(reinterpret_cast<const float4*>(o));
      v[j][1] = __ldcg(reinterpret_cast<const float4*>(o + 128));
    }
    float4 acc[2] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (!((use >> j) & 1)) continue;
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        acc[z].x += v[j][z].x;
        acc[z].y += v[j][z].y;
        acc[z].z += v[j][z].z;
        acc[z].w += v[j][z].w;
      }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z)
      *reinterpret_cast<uint2*>(y + t * hidden + c + 128 * z) =
          make_uint2(pack_bf16(acc[z].x, acc[z].y), pack_bf16(acc[z].z, acc[z].w));
  }
}

// ---- host side ---------------------------------------------------------------------------------
// The route block, which also picks the kernels, by the average expert's routes: 16, 32 (decode) or
// 128 (prefill).  An expert's second block reads its weights again, from L2.  128 experts of 2048 x
// 768, us with blocks of 16 / 32 / 128: 84 / 86 / 127 at 2 routes an expert, 96 / 98 / 139 at 12,
// 129 / 108 / 143 at 20, - / 156 / 162 at 39, - / 168 / 168 at 47.
static int mx_block(int64_t numel, int experts) {
  return numel <= (int64_t)experts * 12   ? 16
         : numel <= (int64_t)experts * 44 ? 32
                                          : kMxPrefillBlock;
}

static int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

MxWorkspace mx_workspace(int64_t tokens, int top_k, int experts, int hidden, int inter,
                         void* base) {
  MxWorkspace w{};
  const int64_t numel = tokens * top_k;
  if (mx_few(numel, hidden, inter)) {
    w.out = static_cast<float*>(base);
    w.bytes = up256(numel * inter * 4);
    return w;
  }
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
  w.slots = reinterpret_cast<int32_t*>(take(numel > align_gather_max_numel() ? numel * 4 : 4));
  w.xq = take(2 * cap * hidden);
  const int tables = scale_tables(w.block);
  w.xs = take(blocks * tables * (hidden / kMxK) * 512);
  w.hq = take(2 * cap * inter);
  w.hs = take(blocks * tables * (inter / kMxK) * 512);
  // fp32, or 16-bit with a scale byte per 32 columns
  w.out = reinterpret_cast<float*>(take(numel * hidden * (w.block == kMxPrefillBlock ? 2 : 4)));
  w.out_scale = take(w.block == kMxPrefillBlock ? numel * (hidden / 32) : 4);
  w.sync_ints = (int)(1 + blocks);
  w.sync = reinterpret_cast<int32_t*>(take(w.sync_ints * 4));
  w.bytes = off;
  return w;
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
  p.w13 = a.w13;
  p.s13 = a.s13;
  p.w2 = a.w2;
  p.s2 = a.s2;
  p.xs = w.xs;
  p.hq = w.hq;
  p.hs = w.hs;
  p.route_w = a.topk_w;
  p.out = w.out;
  p.out_scale = w.out_scale;
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
  CUtensorMap m13, mx, m2, mh;
  if (!make_map_4bit(&m13, a.w13, (uint64_t)a.experts * 2 * a.inter, a.hidden, 128) ||
      !make_map_8bit(&mx, w.xq, 2 * w.capacity, a.hidden, 32) ||
      !make_map_4bit(&m2, a.w2, (uint64_t)a.experts * a.hidden, a.inter, 128) ||
      !make_map_8bit(&mh, w.hq, 2 * w.capacity, a.inter, 32))
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
      !make_map_8bit(&mt, DOWN ? w.hq : w.xq, 2 * w.capacity, k, 32))
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
  if (mx_few(numel, a.hidden, a.inter)) return launch_mx_few(a, w.out, s);
  AlignParams ap{a.topk_ids, numel, a.experts, w.block, w.capacity, w.sorted_ids, w.expert_ids,
                 w.num_post_pad, static_cast<int32_t*>(w.align_ws), 0};
  cudaError_t e;
  if (numel <= align_gather_max_numel()) {
    e = launch_align_split(ap, a.x, a.top_k, a.hidden, w.xq, w.xs, w.sync, w.sync_ints, s);
  } else {
    ap.slots = w.slots;
    e = launch_align(EXF_I32, ap, s);
    if (e == cudaSuccess)
      e = launch_pdl(mx_split_kernel, stream_grid(a.tokens * 32 * ((a.hidden + 1023) / 1024)), 256,
                     0, s,
                     static_cast<const __nv_bfloat16*>(a.x),
                     static_cast<const int32_t*>(w.slots), a.tokens, a.top_k,
                     MxRows{w.xq, w.xs, a.hidden, w.block}, w.sync, w.sync_ints);
  }
  if (e != cudaSuccess) return e;
  if (w.block == kMxPrefillBlock) {
    e = launch_mx_gemm<false>(a, w, s);
    if (e == cudaSuccess) e = launch_mx_gemm<true>(a, w, s);
    if (e != cudaSuccess) return e;
    return launch_pdl(mx_combine16_kernel,
                      stream_grid(a.tokens * 32 * ((a.hidden + 1023) / 1024)), 256, 0, s,
                      reinterpret_cast<const int16_t*>(w.out),
                      static_cast<const uint8_t*>(w.out_scale), a.topk_ids, a.experts, a.tokens,
                      a.top_k, a.hidden, static_cast<__nv_bfloat16*>(a.y));
  } else {
    e = w.block == 16 ? launch_mx_layer<16>(a, w, s) : launch_mx_layer<32>(a, w, s);
  }
  if (e != cudaSuccess) return e;
  return launch_pdl(mx_combine_kernel, stream_grid(a.tokens * (a.hidden / 8)), 256, 0, s,
                    static_cast<const float*>(w.out), a.topk_ids, a.experts, a.tokens, a.top_k,
                    a.hidden, static_cast<__nv_bfloat16*>(a.y));
}

}  // namespace exf
