// The gated feed-forward block h = act(x Wg^T) * (x Wu^T) and its gradients (sm_100a: tcgen05 +
// TMA), bf16 or fp16 operands, fp32 accumulation.
//
//   forward   G = x Wg^T, U = x Wu^T                 one GEMM over W13 = [Wg; Wu]
//             h = act(G) * U                         its epilogue
//   backward  dG = dh * U * act'(G), dU = dh * act(G) elementwise, from G and U kept in fp32
//             dx = [dG dU] W13                       reduction over the 2 * inter columns
//             dW13 = [dG dU]^T x                     reduction over the tokens
//   act(g) = g s(c(g)) with the logistic s: c(g) = g (silu) or 2 sqrt(2 / pi) (g + 0.044715 g^3)
//   (the tanh form of gelu); act'(g) = s + g s (1 - s) c'(g).
//
// Every product is D[m][n] = sum_k A[m][k] B[n][k] on tcgen05.mma (M = 128, K = 16), both operands
// in 128-byte-swizzled shared memory loaded by TMA.  The forward reads both operands along k
// (K-major tiles).  The gradients need W13, x and [dG dU] along their other axis: those tiles are
// loaded as they lie in memory, 64 m or n values by 64 k rows, and the MMA reads them MN-major, so
// nothing is transposed in memory.  Sizes that are no multiple of a tile are filled with zeros by
// TMA and masked on the store.
//
// G and U are kept in fp32 because the gradients already round twice (dG / dU to the operand type
// for the tensor cores, and the result): rounding G and U too would add as much again.  Over many
// values the two roundings make sqrt(2) of one; over few (up to 65536 tokens x inter) a few large ones
// can weigh more, and there dG and dU go in as the sum of two terms of the operand type, the reduction
// running over both (gradient_terms).
//
// fp16 holds 2^-14 to 2^16 at full precision, and dG, dU of a scaled loss or of a mean over many tokens
// lie outside.  Their fp16 form is therefore multiplied by a power of two that brings the largest finite
// one to [2^14, 2^15), and the product's row by its inverse in fp32: a power per token for dx, per
// feature for dW13, so that a token far above the others takes nothing from them.  An element is then
// off by 2^-11 of itself or 2^-39 of that largest.  It costs fp16 a pass that finds the largest and a
// second form of dG and dU (8192 tokens, 4096 x 2048, forward and gradients: 627 -> 705 us; 777 tokens,
// 1000 x 520: 115 -> 121); bf16 has fp32's range and needs none.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "exf_common.cuh"
#include "exf_gated.h"
#include "exf_launch.h"
#include "exf_tc.cuh"

namespace exf {
using namespace tc;

constexpr int kGatedThreads = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
constexpr int kGBM = 128;
constexpr int kGBK = 64;            // 16-bit elements of a 128-byte row

enum GatedKind { kForward = 0, kGradX = 1, kGradW = 2 };

struct GatedGemm {
  int m, n, k;       // n: inter (forward) or hidden
  int m_tiles, n_tiles;
  int kblocks;
  int activation;
  void* out;         // [m][n]
  float* pre;        // forward: [m][2 * n] or null
  int32_t* status;
  int k_term;        // k blocks of one term of A; the second term's rows lie term_rows further on,
  int term_rows;     // and take B's k blocks again
  int splits;        // the reduction is split over this many tiles, whose fp32 sums go to
  float* part;       // [splits][m][n] (forward: [splits][m][2 * n]) when there are several
  bool wide;         // rows of out are 32-byte aligned
  const uint32_t* top;  // fp16 gradients: the bits of the largest finite magnitude in each row of A
};

// ---- activation -----------------------------------------------------------------------------
template <int ACT>
__device__ __forceinline__ float gate_sigmoid(float g) {
  float c = g;
  if (ACT == kGeluTanh) c = 1.5957691216057308f * fmaf(0.044715f * g, g * g, g);
  return logistic(c);
}
template <int ACT>
__device__ __forceinline__ float gate_slope(float g, float s) {
  float dc = 1.0f;
  if (ACT == kGeluTanh) {
    // s (1 - s) is 0 long before |g| = 100, and the clamp keeps 0 * inf away
    const float b = fminf(fmaxf(g, -100.0f), 100.0f);
    dc = 1.5957691216057308f * fmaf(0.134145f * b, b, 1.0f);
    return fmaf(b * s * (1.0f - s), dc, s);
  }
  return fmaf(g * s, 1.0f - s, s);
}

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

// ---- the powers of two of fp16 gradients ----------------------------------------------------------
// From the bits of a finite magnitude: the power that brings it to [2^14, 2^15) (at most 2^126, for 0 and
// what is below 2^-112), and the inverse.
__device__ __forceinline__ int top_power(uint32_t top) {
  const int k = 14 + 127 - (int)(top >> 23);
  return k < 126 ? k : 126;
}
__device__ __forceinline__ float scale_up(uint32_t top) {
  return __uint_as_float((uint32_t)(127 + top_power(top)) << 23);
}
__device__ __forceinline__ float scale_back(uint32_t top) {
  return __uint_as_float((uint32_t)(127 - top_power(top)) << 23);
}

// ---- the GEMM ---------------------------------------------------------------------------------
template <int NT>
struct GatedCfg {
  static constexpr int kATile = kGBM * kGBK * 2;
  static constexpr int kBTile = NT * kGBK * 2;
  static constexpr int kStage = kATile + kBTile;
  static constexpr int kStages = (196 * 1024) / kStage;
  static constexpr int kTmem = 2 * NT;                 // two accumulators, a power of two
};
template <int NT>
struct GatedSmem {
  alignas(1024) uint8_t tiles[GatedCfg<NT>::kStages][GatedCfg<NT>::kStage];
  alignas(8) uint64_t full[GatedCfg<NT>::kStages];
  alignas(8) uint64_t empty[GatedCfg<NT>::kStages];
  alignas(8) uint64_t acc_full[2];
  alignas(8) uint64_t acc_empty[2];
  alignas(8) uint64_t drain;
  uint32_t tmem_base;
  int failed;
};
template <int NT>
constexpr size_t gated_smem_bytes() { return sizeof(GatedSmem<NT>) + 1024; }

// Shared-memory matrix descriptor of an MN-major tile: 64 mn values (128 bytes, swizzled) a row, 64
// k rows a box; 8-row groups along k 1024 bytes apart (SBO), boxes along mn 8192 bytes apart (LBO).
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(8192 >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// The epilogue of a tile: row `row` of D, columns from TMEM address taddr on (NT of them, a thread a
// row); every lane of the warp takes part in the TMEM loads.
template <int KIND, int NT, bool BF16>
__device__ __forceinline__ void write_tile(const GatedGemm& p, uint32_t taddr, int row, int nt,
                                           int part) {
        if (p.splits > 1) {  // fp32 sums of this part of the reduction
          constexpr int kRuns = KIND == kForward ? 2 : 1;  // gate and up columns
          float* at = p.part + ((int64_t)part * p.m + row) * kRuns * p.n;
  #pragma unroll 1
          for (int c = 0; c < NT; c += 32) {
            float v[32];
            __syncwarp();
            tmem_load32(taddr + c, v);
            const int run = c / (NT / kRuns);
            const int col = nt * (NT / kRuns) + c % (NT / kRuns);
            if (row < p.m) {
  #pragma unroll
              for (int j = 0; j < 32; j += 8)
                if (col + j < p.n) store_sums(at + run * p.n + col + j, v + j);
            }
          }
        } else if (KIND == kForward) {
  #pragma unroll 1
          for (int c = 0; c < NT / 2; c += 32) {
            float gt[32], up[32];
            __syncwarp();
            tmem_load32(taddr + c, gt);
            tmem_load32(taddr + NT / 2 + c, up);
            const int col = nt * (NT / 2) + c;
            if (row < p.m) {
              if (p.pre) {
                float* pg = p.pre + (int64_t)row * 2 * p.n + col;
  #pragma unroll
                for (int j = 0; j < 32; j += 8)
                  if (col + j < p.n) {
                    store_sums(pg + j, gt + j);
                    store_sums(pg + p.n + j, up + j);
                  }
              }
              if (p.activation == kSilu) {
  #pragma unroll
                for (int j = 0; j < 32; ++j) gt[j] = gt[j] * gate_sigmoid<kSilu>(gt[j]) * up[j];
              } else {
  #pragma unroll
                for (int j = 0; j < 32; ++j)
                  gt[j] = gt[j] * gate_sigmoid<kGeluTanh>(gt[j]) * up[j];
              }
  #pragma unroll
              for (int j = 0; j < 32; j += 16)
                if (col + j < p.n)
                  store_32b<BF16>(p.out, (int64_t)row * p.n + col + j, gt + j, p.wide,
                                  col + j + 8 < p.n);
            }
          }
        } else {
          const float back = !BF16 && row < p.m ? scale_back(p.top[row]) : 1.0f;
  #pragma unroll 1
          for (int c = 0; c < NT; c += 32) {
            float v[32];
            __syncwarp();
            tmem_load32(taddr + c, v);
            const int col = nt * NT + c;
            if (row < p.m) {
              if (!BF16) {
  #pragma unroll
                for (int j = 0; j < 32; ++j) v[j] *= back;
              }
  #pragma unroll
              for (int j = 0; j < 32; j += 16)
                if (col + j < p.n)
                  store_32b<BF16>(p.out, (int64_t)row * p.n + col + j, v + j, p.wide,
                                  col + j + 8 < p.n);
            }
          }
        }
}

template <int KIND, int NT, bool BF16>
__global__ void __launch_bounds__(kGatedThreads, 1)
    gated_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                      const __grid_constant__ CUtensorMap map_b, const GatedGemm p) {
  using C = GatedCfg<NT>;
  constexpr bool kAMn = KIND == kGradW, kBMn = KIND != kForward;
  constexpr uint32_t kIdesc = idesc_f16(kGBM, NT, BF16) | (kAMn ? 1u << 15 : 0u) |
                              (kBMn ? 1u << 16 : 0u);
  extern __shared__ uint8_t smem_raw[];
  GatedSmem<NT>& sm = *reinterpret_cast<GatedSmem<NT>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 4);
    }
    mbar_init(&sm.drain, 1);
    sm.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, C::kTmem);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int mn_tiles = p.m_tiles * p.n_tiles;
  const int ntiles = mn_tiles * p.splits;
  // tile t: reduction part, M tile, N tile; k blocks [kb0, kb1)
  struct Tile {
    int part, mt, nt, kb0, kb1;
  };
  auto tile_of = [&](int t) {
    Tile r;
    r.part = t / mn_tiles;
    t -= r.part * mn_tiles;
    r.mt = t / p.n_tiles;
    r.nt = t - r.mt * p.n_tiles;
    r.kb0 = (int)((int64_t)p.kblocks * r.part / p.splits);
    r.kb1 = (int)((int64_t)p.kblocks * (r.part + 1) / p.splits);
    return r;
  };
  const uint32_t tmem = uniform(sm.tmem_base);
  volatile int* failed = &sm.failed;

  if (warp == 0) {
    // ---- TMA producer
    uint32_t g = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
      const Tile tl = tile_of(t);
      const int mt = tl.mt, nt = tl.nt;
      for (int kb = tl.kb0; kb < tl.kb1; ++kb, ++g) {
        const int s = g % C::kStages;
        ok = warp_wait(&sm.empty[s], ((g / C::kStages) & 1) ^ 1, failed);
        if (!ok) break;
        uint8_t* a = sm.tiles[s];
        uint8_t* b = a + C::kATile;
        uint64_t* bar = &sm.full[s];
        // (in a term's last k block B's rows or columns past the end are zeros, whatever A has there)
        const int term = KIND != kForward && kb >= p.k_term ? p.term_rows : 0;
        const int k0 = (kb - (term ? p.k_term : 0)) * kGBK;
        if (elect_one()) {
          mbar_expect_tx(bar, C::kStage);
          if (kAMn) {
            tma_load_2d(a, &map_a, bar, mt * kGBM, term + k0);
            tma_load_2d(a + 8192, &map_a, bar, mt * kGBM + 64, term + k0);
          } else {
            tma_load_2d(a, &map_a, bar, k0, term + mt * kGBM);
          }
          if (kBMn) {
#pragma unroll
            for (int j = 0; j < NT / 64; ++j)
              tma_load_2d(b + j * 8192, &map_b, bar, nt * NT + 64 * j, k0);
          } else {  // gate rows, then up rows
            tma_load_2d(b, &map_b, bar, k0, nt * (NT / 2));
            tma_load_2d(b + C::kBTile / 2, &map_b, bar, k0, p.n + nt * (NT / 2));
          }
        }
      }
    }
    for (uint32_t j = g > C::kStages ? g - C::kStages : 0; j < g; ++j)
      mbar_wait_drain(&sm.full[j % C::kStages], (j / C::kStages) & 1);
  } else if (warp == 1) {
    // ---- MMA issuer: tile i accumulates into TMEM columns [NT (i & 1), +NT)
    uint32_t g = 0;
    int i = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x, ++i) {
      const int b = i & 1;
      ok = warp_wait(&sm.acc_empty[b], ((i >> 1) & 1) ^ 1, failed);
      if (!ok) break;
      fence_after_sync();
      const uint32_t acc = tmem + static_cast<uint32_t>(b * NT);
      const Tile tl = tile_of(t);
      for (int kb = tl.kb0; kb < tl.kb1; ++kb, ++g) {
        const int s = g % C::kStages;
        ok = warp_wait(&sm.full[s], (g / C::kStages) & 1, failed);
        if (!ok) break;
        fence_after_sync();
        // a K step of 16 is 32 bytes further on K-major, 16 rows of 128 bytes MN-major (the
        // descriptors count 16 bytes)
        const uint32_t base = smem_addr(sm.tiles[s]);
        const uint64_t da = kAMn ? smem_desc_mn(base) : smem_desc(base);
        const uint64_t db = kBMn ? smem_desc_mn(base + C::kATile) : smem_desc(base + C::kATile);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kGBK / 16; ++k)
            mma_kind_f16(acc, da + k * (kAMn ? 128 : 2), db + k * (kBMn ? 128 : 2), kIdesc,
                         (kb > tl.kb0 || k > 0) ? 1u : 0u);
          mma_commit(&sm.empty[s]);
        }
      }
      if (!ok) break;
      if (elect_one()) mma_commit(&sm.acc_full[b]);
    }
    if (elect_one()) mma_commit(&sm.drain);
    mbar_wait_drain(&sm.drain, 0);
  } else {
    // ---- epilogue: one output row per thread
    const int q = warp & 3;
    int i = 0;
    for (int t = blockIdx.x; t < ntiles; t += gridDim.x, ++i) {
      const Tile tl = tile_of(t);
      const int mt = tl.mt, nt = tl.nt;
      const int b = i & 1;
      if (!warp_wait(&sm.acc_full[b], (i >> 1) & 1, failed)) break;
      fence_after_sync();
      const int row = mt * kGBM + q * 32 + lane;
      const uint32_t taddr = tmem + static_cast<uint32_t>(b * NT) + ((uint32_t)(q * 32) << 16);
      write_tile<KIND, NT, BF16>(p, taddr, row, nt, tl.part);
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[b]);
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    fence_after_sync();
    tmem_free(tmem, C::kTmem);
  }
  if (threadIdx.x == 0 && sm.failed && p.status) atomicExch(p.status, 1);
}

// ---- joining a split reduction --------------------------------------------------------------------
// out [m][n] from the parts' sums, added in order; forward: h and pre from the gate and up sums.  8
// columns a thread.
template <int KIND, bool BF16>
__global__ void __launch_bounds__(256)
    gated_join_kernel(const float* part, int splits, int64_t m, int n, int activation, void* out,
                      float* pre, const uint32_t* top) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kRuns = KIND == kForward ? 2 : 1;
  const int vec = n / 8;
  const int64_t stride = m * kRuns * n;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < m * vec;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / vec;
    const int c = (int)(i - row * vec) * 8;
    float v[kRuns][8] = {};
#pragma unroll 4
    for (int s = 0; s < splits; ++s)
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        const float4* at =
            reinterpret_cast<const float4*>(part + s * stride + (row * kRuns + r) * n + c);
        const float4 a = __ldcg(at), b = __ldcg(at + 1);
        v[r][0] += a.x;
        v[r][1] += a.y;
        v[r][2] += a.z;
        v[r][3] += a.w;
        v[r][4] += b.x;
        v[r][5] += b.y;
        v[r][6] += b.z;
        v[r][7] += b.w;
      }
    if (KIND == kForward) {
      float(&u)[8] = v[kRuns - 1];
      if (pre) {
#pragma unroll
        for (int r = 0; r < kRuns; ++r) {
          float4* at = reinterpret_cast<float4*>(pre + (row * kRuns + r) * n + c);
          at[0] = make_float4(v[r][0], v[r][1], v[r][2], v[r][3]);
          at[1] = make_float4(v[r][4], v[r][5], v[r][6], v[r][7]);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[0][j] *= (activation == kSilu ? gate_sigmoid<kSilu>(v[0][j])
                                        : gate_sigmoid<kGeluTanh>(v[0][j])) *
                   u[j];
    } else if (!BF16) {
      const float back = scale_back(top[row]);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[0][j] *= back;
    }
    store_16b<BF16>(out, row * n + c, v[0]);
  }
}

// ---- a few tokens ------------------------------------------------------------------------------
// Up to 4 tokens: a warp computes one feature (a gate and an up row against every token) with fp32
// FMAs, so that every SM streams weights; an MMA tile would be 1/32 full and 64 features wide.  us of
// this kernel and of the tiles with a split reduction: 8 / 10 (512 x 256), 12 / 14 (2048 x 768) and
// 18 / 20 (4096 x 2048) up to 4 tokens, 31 / 20 at 8 (4096 x 2048).  Bound by the weights' latency and
// bytes.  TT: tokens rounded up to a power of two.
constexpr int kFewTokens = 4;
constexpr int kFewWarps = 4;

template <bool BF16, int TT>
__global__ void __launch_bounds__(32 * kFewWarps)
    gated_few_kernel(const uint16_t* x, const uint16_t* __restrict__ w13, int tokens,
                     int hidden, int inter, int activation, uint16_t* h, float* pre) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int f = blockIdx.x * kFewWarps + (threadIdx.x >> 5);
  if (f >= inter) return;
  const uint4* wg = reinterpret_cast<const uint4*>(w13 + (int64_t)f * hidden);
  const uint4* wu = reinterpret_cast<const uint4*>(w13 + (int64_t)(inter + f) * hidden);
  const int vecs = hidden / 8;
  float g[TT] = {}, u[TT] = {};
#pragma unroll(TT <= 2 ? 8 : 4)
  for (int c = lane; c < vecs; c += 32) {
    const uint4 a = __ldg(wg + c), b = __ldg(wu + c);
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      // (rows past the last token read it again; their sums are not stored)
      const uint4 v = *(reinterpret_cast<const uint4*>(
                            x + (int64_t)(t < tokens ? t : tokens - 1) * hidden) + c);
      const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 xv = unpack2<BF16>(vw[j]), av = unpack2<BF16>(aw[j]),
                     bv = unpack2<BF16>(bw[j]);
        g[t] = fmaf(xv.x, av.x, g[t]);
        g[t] = fmaf(xv.y, av.y, g[t]);
        u[t] = fmaf(xv.x, bv.x, u[t]);
        u[t] = fmaf(xv.y, bv.y, u[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      g[t] += __shfl_xor_sync(0xffffffffu, g[t], d);
      u[t] += __shfl_xor_sync(0xffffffffu, u[t], d);
    }
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    if (lane != t || t >= tokens) continue;
    const float s = activation == kSilu ? gate_sigmoid<kSilu>(g[t]) : gate_sigmoid<kGeluTanh>(g[t]);
    const uint32_t v = pack2<BF16>(g[t] * s * u[t], 0.0f);
    h[(int64_t)t * inter + f] = (uint16_t)v;
    if (pre) {
      pre[(int64_t)t * 2 * inter + f] = g[t];
      pre[(int64_t)t * 2 * inter + inter + f] = u[t];
    }
  }
}

// ---- the GEMM on pairs of SMs -------------------------------------------------------------------
// Large products: a cluster of two CTAs computes a tile of 256 x 256 with tcgen05.mma cta_group::2.
// Each CTA loads 128 rows of A and 128 of B into its own shared memory (32 KB a stage instead of 48)
// and holds 128 rows of D in its TMEM; the MMA, issued by the leader (rank 0), reads both CTAs'
// operands.  A third less traffic from L2 and into shared memory also buys clock under the power
// limit.  Pairs / single SMs, us: 8192 tokens, 4096 x 2048, forward 171 / 188 (1.61 PFLOP/s, 0.97 of the
// measured bf16 burst rate), with gradients 600 / 652; 2048 tokens 53 / 59; 8192 tokens, 256 x 2048
// (the epilogue bounds it) 33 / 29.
// Barriers: `full` of the leader counts both CTAs' copies; `empty` and `acc_full` of each CTA are
// signalled by the leader's commits; `acc_empty` of the leader collects both CTAs' epilogue warps.
constexpr int kPairStages = 6;
struct PairSmem {
  alignas(1024) uint8_t tiles[kPairStages][32768];
  alignas(8) uint64_t full[kPairStages];
  alignas(8) uint64_t empty[kPairStages];
  alignas(8) uint64_t acc_full[2];
  alignas(8) uint64_t acc_empty[2];
  alignas(8) uint64_t drain;
  uint32_t tmem_base;
  int failed;
};
constexpr size_t pair_smem_bytes() { return sizeof(PairSmem) + 1024; }

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// the address of a shared object in the leader's CTA
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_addr(p)));
  return a;
}
// a copy into this CTA's shared memory that completes on a barrier of the pair
__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* map, uint32_t bar, int c0,
                                             int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// arrives on the barrier at this offset in both CTAs once the MMAs issued so far have completed
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}

template <int KIND, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGatedThreads, 1)
    gated_pair_kernel(const __grid_constant__ CUtensorMap map_a,
                      const __grid_constant__ CUtensorMap map_b, const GatedGemm p) {
  constexpr bool kAMn = KIND == kGradW, kBMn = KIND != kForward;
  constexpr uint32_t kIdesc =
      idesc_f16(256, 256, BF16) | (kAMn ? 1u << 15 : 0u) | (kBMn ? 1u << 16 : 0u);
  constexpr int S = kPairStages;
  extern __shared__ uint8_t smem_raw[];
  PairSmem& sm = *reinterpret_cast<PairSmem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 8);
    }
    mbar_init(&sm.drain, 1);
    sm.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&sm.tmem_base)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before_sync();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised
  fence_after_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const int ntiles = p.m_tiles * p.n_tiles;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const uint32_t tmem = uniform(sm.tmem_base);
  volatile int* failed = &sm.failed;

  if (warp == 0) {
    // ---- TMA producer of this CTA's halves
    uint32_t g = 0;
    bool ok = true;
    for (int t = first; t < ntiles && ok; t += step) {
      const int mt = t / p.n_tiles, nt = t - mt * p.n_tiles;
      const int row = mt * 256 + rank * 128;
      for (int kb = 0; kb < p.kblocks; ++kb, ++g) {
        const int s = g % S;
        ok = warp_wait(&sm.empty[s], ((g / S) & 1) ^ 1, failed);
        if (!ok) break;
        uint8_t* a = sm.tiles[s];
        uint8_t* b = a + 16384;
        const uint32_t bar = leader_addr(&sm.full[s]);
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(&sm.full[s], 65536);  // both CTAs' copies
          if (kAMn) {
            pair_load_2d(a, &map_a, bar, row, kb * kGBK);
            pair_load_2d(a + 8192, &map_a, bar, row + 64, kb * kGBK);
          } else {
            pair_load_2d(a, &map_a, bar, kb * kGBK, row);
          }
          if (kBMn) {
            pair_load_2d(b, &map_b, bar, nt * 256 + rank * 128, kb * kGBK);
            pair_load_2d(b + 8192, &map_b, bar, nt * 256 + rank * 128 + 64, kb * kGBK);
          } else {  // the leader has the gate rows, its peer the up rows
            pair_load_2d(b, &map_b, bar, kb * kGBK, rank * p.n + nt * 128);
          }
        }
      }
    }
    // the leader's last commits on this CTA's `empty` barriers arrive before it leaves
    for (uint32_t j = g > S ? g - S : 0; j < g; ++j)
      mbar_wait_drain(&sm.empty[j % S], (j / S) & 1);
  } else if (warp == 1) {
    // ---- MMA issuer, in the leader
    if (rank == 0) {
      uint32_t g = 0;
      int i = 0;
      bool ok = true;
      for (int t = first; t < ntiles && ok; t += step, ++i) {
        const int b = i & 1;
        ok = warp_wait(&sm.acc_empty[b], ((i >> 1) & 1) ^ 1, failed);
        if (!ok) break;
        fence_after_sync();
        const uint32_t acc = tmem + static_cast<uint32_t>(b * 256);
        for (int kb = 0; kb < p.kblocks; ++kb, ++g) {
          const int s = g % S;
          ok = warp_wait(&sm.full[s], (g / S) & 1, failed);
          if (!ok) break;
          fence_after_sync();
          const uint32_t base = smem_addr(sm.tiles[s]);
          const uint64_t da = kAMn ? smem_desc_mn(base) : smem_desc(base);
          const uint64_t db = kBMn ? smem_desc_mn(base + 16384) : smem_desc(base + 16384);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kGBK / 16; ++k)
              pair_mma(acc, da + k * (kAMn ? 128 : 2), db + k * (kBMn ? 128 : 2), kIdesc,
                       (kb > 0 || k > 0) ? 1u : 0u);
            pair_commit(&sm.empty[s]);
          }
        }
        if (!ok) break;
        if (elect_one()) pair_commit(&sm.acc_full[b]);
      }
      if (elect_one()) pair_commit(&sm.drain);
      mbar_wait_drain(&sm.drain, 0);
    }
  } else {
    // ---- epilogue of this CTA's 128 rows
    const int q = warp & 3;
    int i = 0;
    for (int t = first; t < ntiles; t += step, ++i) {
      const int mt = t / p.n_tiles, nt = t - mt * p.n_tiles;
      const int b = i & 1;
      if (!warp_wait(&sm.acc_full[b], (i >> 1) & 1, failed)) break;
      fence_after_sync();
      write_tile<KIND, 256, BF16>(
          p, tmem + static_cast<uint32_t>(b * 256) + ((uint32_t)(q * 32) << 16),
          mt * 256 + rank * 128 + q * 32 + lane, nt, 0);
      fence_before_sync();
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                         leader_addr(&sm.acc_empty[b]))
                     : "memory");
    }
  }
  fence_before_sync();
  __syncthreads();
  // Neither CTA leaves while the other may still read its operands or signal its barriers: all of the
  // leader's commits have arrived here too (`empty` and `acc_full` are waited for above, `drain` is the
  // last), and the threads' own arrivals are ordered by the cluster's barrier.  After a time-out, copies
  // still in flight land first (a load started has at most its memory's latency left).
  if (warp == 1 && rank == 1) mbar_wait_drain(&sm.drain, 0);
  if (sm.failed) {
    for (int j = 0; j < 256; ++j) __nanosleep(1000);
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, 1);
  }
  cluster_sync();
  if (warp == 1) {
    __syncwarp();
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// what rounding v to the operand type leaves; 0 where it overflows to an infinity or is one
template <bool BF16>
__device__ __forceinline__ float remainder_of(float v) {
  const float2 r = unpack2<BF16>(pack2<BF16>(v, 0.0f));
  return fabsf(r.x) < __int_as_float(0x7f800000) ? v - r.x : 0.0f;
}

// ---- the elementwise part of backward -----------------------------------------------------------
// dG = dh * U * act'(G) and dU = dh * act(G) of 8 columns of a token
template <bool BF16, int ACT>
__device__ __forceinline__ void projection_grads(const uint16_t* dh, const float* pre, int64_t t,
                                                 int inter, int c, float (&dg)[8], float (&du)[8]) {
  const float4* gp = reinterpret_cast<const float4*>(pre + t * 2 * inter + c);
  const float4* up = reinterpret_cast<const float4*>(pre + t * 2 * inter + inter + c);
  const float4 g0 = gp[0], g1 = gp[1], u0 = up[0], u1 = up[1];
  const uint4 d = *reinterpret_cast<const uint4*>(dh + t * inter + c);
  const float g[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
  const float u[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
  const uint32_t dw[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 e = unpack2<BF16>(dw[j >> 1]);
    const float dv = (j & 1) ? e.y : e.x;
    const float s = gate_sigmoid<ACT>(g[j]);
    dg[j] = dv * u[j] * gate_slope<ACT>(g[j], s);
    du[j] = dv * (g[j] * s);
  }
}

// fp16: the bits of the largest finite |dG|, |dU| of each feature in top[0, 2 * inter) and of each token in
// top[2 * inter, +tokens), which are 0 before.  A block takes 256 columns of 8 * rows tokens, a warp a
// token at a time; maxima do not depend on the atomics' order.
template <int ACT>
__global__ void __launch_bounds__(256)
    gated_top_kernel(const uint16_t* dh, const float* pre, int64_t tokens, int inter, int rows,
                     uint32_t* top) {
  __shared__ uint32_t part[8][2][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (inter + 255) / 256;
  const int64_t t0 = (int64_t)(blockIdx.x / groups) * rows * 8;
  const int c0 = (int)(blockIdx.x % groups) * 256;
  const int c = c0 + 8 * lane;
  auto finite = [](float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
  };
  uint32_t of[2][8] = {};
#pragma unroll 2
  for (int i = 0; i < rows; ++i) {
    const int64_t t = t0 + 8 * i + warp;
    if (t >= tokens) break;
    uint32_t m = 0;
    if (c < inter) {
      float dg[8], du[8];
      projection_grads<false, ACT>(dh, pre, t, inter, c, dg, du);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = finite(dg[j]), b = finite(du[j]);
        of[0][j] = max(of[0][j], a);
        of[1][j] = max(of[1][j], b);
        m = max(m, max(a, b));
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) atomicMax(top + 2 * inter + t, m);
  }
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int j = 0; j < 8; ++j) part[warp][r][8 * lane + j] = of[r][j];
  __syncthreads();
  const int at = c0 + (int)threadIdx.x;
  if (at >= inter) return;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    uint32_t m = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, part[w][r][threadIdx.x]);
    atomicMax(top + r * inter + at, m);
  }
}

// The 16-bit form of 8 columns of dG and dU, [tokens][2 * inter]; with a second term, the remainders in the
// same form behind it.
template <bool BF16>
__device__ __forceinline__ void store_grads(uint16_t* both, int64_t tokens, int64_t t, int inter,
                                            int c, int terms, float (&dg)[8], float (&du)[8]) {
  store_16b<BF16>(both, t * 2 * inter + c, dg);
  store_16b<BF16>(both, t * 2 * inter + inter + c, du);
  if (terms == 2) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dg[j] = remainder_of<BF16>(dg[j]);
      du[j] = remainder_of<BF16>(du[j]);
    }
    store_16b<BF16>(both, (tokens + t) * 2 * inter + c, dg);
    store_16b<BF16>(both, (tokens + t) * 2 * inter + inter + c, du);
  }
}

// by_token = (dG, dU); 8 columns a thread.  fp16: times the tokens' powers of two, and by_feature the same
// with the features' (either may be null).
template <bool BF16, int ACT>
__global__ void __launch_bounds__(256)
    gated_slope_kernel(const uint16_t* dh, const float* pre, int64_t tokens, int inter, int terms,
                       const uint32_t* top, uint16_t* by_token, uint16_t* by_feature) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int vec = inter / 8;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < tokens * vec;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / vec;
    const int c = (int)(i - t * vec) * 8;
    float dg[8], du[8];
    projection_grads<BF16, ACT>(dh, pre, t, inter, c, dg, du);
    if (BF16) {
      store_grads<BF16>(by_token, tokens, t, inter, c, terms, dg, du);
      continue;
    }
    float a[8], b[8];
    if (by_token) {
      const float up = scale_up(top[2 * inter + t]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] = dg[j] * up;
        b[j] = du[j] * up;
      }
      store_grads<BF16>(by_token, tokens, t, inter, c, terms, a, b);
    }
    if (by_feature) {
      const uint4* tg = reinterpret_cast<const uint4*>(top + c);
      const uint4* tu = reinterpret_cast<const uint4*>(top + inter + c);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 g = tg[h], u = tu[h];
        const uint32_t gw[4] = {g.x, g.y, g.z, g.w}, uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[4 * h + j] = dg[4 * h + j] * scale_up(gw[j]);
          b[4 * h + j] = du[4 * h + j] * scale_up(uw[j]);
        }
      }
      store_grads<BF16>(by_feature, tokens, t, inter, c, terms, a, b);
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------
template <int KIND, int NT, bool BF16>
static cudaError_t launch_gemm(const CUtensorMap& ma, const CUtensorMap& mb, GatedGemm p,
                               cudaStream_t s) {
  auto* kern = gated_gemm_kernel<KIND, NT, BF16>;
  static std::mutex mu;
  static bool done[64] = {};
  const cudaError_t e = allow_smem(kern, gated_smem_bytes<NT>(), mu, done);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles * p.splits;
  const int sms = sm_count();
  const unsigned grid = (unsigned)(sms > 0 && tiles > sms ? sms : tiles);
  return launch_pdl(kern, grid, kGatedThreads, gated_smem_bytes<NT>(), s, ma, mb, p);
}

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

static unsigned stream_grid(int64_t threads) {
  int64_t blocks = (threads + 255) / 256;
  const int lim = 8 * sm_count();
  if (lim > 0 && blocks > lim) blocks = lim;
  return (unsigned)(blocks > 0 ? blocks : 1);
}

// The N tile and the parts of the reduction of a GEMM [m][n] over k.  Tiles of 256 columns (forward:
// 128 gate and 128 up) while they fill more than half of the SMs; else narrower ones, and where the
// reduction is long it is split, at least 8 k blocks a part, until the SMs are full (9 tokens, 4096 x
// 2048: 31 us with 64 whole tiles of 64 columns, 18 with 32 x 4 of 128; 333 tokens, 1000 x 712: 14 and
// 16).  Pairs of SMs where their tiles fill the card and the reduction outlasts the epilogue.
struct GatedPlan {
  int nt, splits;
  bool pair;  // tiles of 256 x 256 on pairs of SMs
};
static GatedPlan plan(int kind, int64_t m, int64_t n, int64_t k, int terms) {
  const int sms = sm_count() > 0 ? sm_count() : 1;
  const int64_t kblocks = terms * ceil_div(k, kGBK);
  auto tiles = [&](int nt) {
    return ceil_div(m, kGBM) * ceil_div(n, kind == kForward ? nt / 2 : nt);
  };
  if (terms == 1 && m >= 1024 && kblocks >= 12 && tiles(256) >= sms) return {256, 1, true};
  if (tiles(256) * 2 > sms) return {256, 1, false};
  if (kblocks < 32) return {tiles(128) * 2 > sms ? 128 : 64, 1, false};
  int64_t s = sms / tiles(128);
  if (s > kblocks / 8) s = kblocks / 8;
  return {128, (int)(s > 1 ? s : 1), false};
}
static int64_t part_bytes(int kind, int64_t m, int64_t n, int64_t k, int terms) {
  const GatedPlan pl = plan(kind, m, n, k, terms);
  return pl.splits > 1 ? pl.splits * m * n * (kind == kForward ? 8 : 4) : 0;
}

template <int KIND, int NT, bool BF16>
static cudaError_t run_gemm(const void* a, int64_t a_rows, int64_t a_cols, const void* b,
                            int64_t b_rows, int64_t b_cols, int terms, GatedGemm p,
                            cudaStream_t s) {
  constexpr auto dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap ma, mb;
  if (!make_map(&ma, a, terms * a_rows, a_cols, KIND == kGradW ? kGBK : kGBM, dt) ||
      !make_map(&mb, b, b_rows, b_cols, KIND == kForward ? NT / 2 : kGBK, dt))
    return cudaErrorInvalidValue;
  p.m_tiles = (int)ceil_div(p.m, kGBM);
  p.n_tiles = (int)ceil_div(p.n, KIND == kForward ? NT / 2 : NT);
  p.k_term = (int)ceil_div(p.k, kGBK);
  p.kblocks = terms * p.k_term;
  p.wide = p.n % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 32 == 0;
  cudaError_t e = launch_gemm<KIND, NT, BF16>(ma, mb, p, s);
  if (e != cudaSuccess || p.splits == 1) return e;
  return launch_pdl(gated_join_kernel<KIND, BF16>, stream_grid((int64_t)p.m * (p.n / 8)), 256, 0, s,
                    static_cast<const float*>(p.part), p.splits, (int64_t)p.m, p.n, p.activation,
                    p.out, p.pre, p.top);
}

template <int KIND, bool BF16>
static cudaError_t run_pair(const void* a, int64_t a_rows, int64_t a_cols, const void* b,
                            int64_t b_rows, int64_t b_cols, GatedGemm p, cudaStream_t s) {
  constexpr auto dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto* kern = gated_pair_kernel<KIND, BF16>;
  static std::mutex mu;
  static bool done[64] = {};
  const cudaError_t e = allow_smem(kern, pair_smem_bytes(), mu, done);
  if (e != cudaSuccess) return e;
  CUtensorMap ma, mb;
  if (!make_map(&ma, a, a_rows, a_cols, KIND == kGradW ? kGBK : 128, dt) ||
      !make_map(&mb, b, b_rows, b_cols, KIND == kForward ? 128 : kGBK, dt))
    return cudaErrorInvalidValue;
  p.m_tiles = (int)ceil_div(p.m, 256);
  p.n_tiles = (int)ceil_div(p.n, KIND == kForward ? 128 : 256);
  p.kblocks = (int)ceil_div(p.k, kGBK);
  p.wide = p.n % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 32 == 0;
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  const int64_t pairs = sm_count() > 1 ? sm_count() / 2 : 1;
  return launch_pdl(kern, (unsigned)(2 * (tiles < pairs ? tiles : pairs)), kGatedThreads,
                    pair_smem_bytes(), s, ma, mb, p);
}

// One product: its A (`terms` of them, one behind the other) and B tensors as they lie in memory, m, n,
// k and outputs in p.
template <int KIND, bool BF16>
static cudaError_t product(const void* a, int64_t a_rows, int64_t a_cols, const void* b,
                           int64_t b_rows, int64_t b_cols, int terms, GatedGemm p,
                           cudaStream_t s) {
  const GatedPlan pl = plan(KIND, p.m, p.n, p.k, terms);
  p.splits = pl.splits;
  p.term_rows = (int)a_rows;
  if (pl.pair) return run_pair<KIND, BF16>(a, a_rows, a_cols, b, b_rows, b_cols, p, s);
  switch (pl.nt) {
    case 256: return run_gemm<KIND, 256, BF16>(a, a_rows, a_cols, b, b_rows, b_cols, terms, p, s);
    case 128: return run_gemm<KIND, 128, BF16>(a, a_rows, a_cols, b, b_rows, b_cols, terms, p, s);
    default: return run_gemm<KIND, 64, BF16>(a, a_rows, a_cols, b, b_rows, b_cols, terms, p, s);
  }
}

template <bool BF16, int TT>
static cudaError_t forward_few(const GatedArgs& a, void* h, float* pre, cudaStream_t s) {
  return launch_pdl(gated_few_kernel<BF16, TT>, (unsigned)ceil_div(a.inter, kFewWarps),
                    32 * kFewWarps, 0, s, static_cast<const uint16_t*>(a.x),
                    static_cast<const uint16_t*>(a.w13), (int)a.tokens, a.hidden, a.inter,
                    a.activation, static_cast<uint16_t*>(h), pre);
}

template <bool BF16>
static cudaError_t forward_t(const GatedArgs& a, void* h, float* pre, float* part,
                             cudaStream_t s) {
  if (a.tokens <= kFewTokens)
    return a.tokens == 1   ? forward_few<BF16, 1>(a, h, pre, s)
           : a.tokens == 2 ? forward_few<BF16, 2>(a, h, pre, s)
                           : forward_few<BF16, 4>(a, h, pre, s);
  GatedGemm p{};
  p.m = (int)a.tokens;
  p.n = a.inter;
  p.k = a.hidden;
  p.activation = a.activation;
  p.out = h;
  p.pre = pre;
  p.status = a.status;
  p.part = part;
  return product<kForward, BF16>(a.x, a.tokens, a.hidden, a.w13, 2 * (int64_t)a.inter, a.hidden, 1,
                                 p, s);
}

// Device time of a forward and backward step in us, bf16, with one term and two: 27 and 31 (32 tokens,
// 2048 x 2048), 22 and 23 (64, 1024 x 1024) at the border, hidden behind a call's host time of over 100;
// 26 and 35 (777, 1000 x 520), 55 and 75 (2048, 2048 x 1024) above it.
static int gradient_terms(int64_t tokens, int inter) { return tokens * inter <= 65536 ? 2 : 1; }

template <int ACT>
static cudaError_t launch_top(const GatedArgs& a, const void* dh, const float* pre, uint32_t* top,
                              cudaStream_t s) {
  const cudaError_t e =
      cudaMemsetAsync(top, 0, (size_t)(a.tokens + 2 * (int64_t)a.inter) * 4, s);
  if (e != cudaSuccess) return e;
  // 8 tokens a warp, fewer where the card would not fill
  const int64_t groups = ceil_div(a.inter, 256);
  int64_t rows = a.tokens * groups / (32 * (int64_t)(sm_count() > 0 ? sm_count() : 1));
  rows = rows < 1 ? 1 : rows > 8 ? 8 : rows;
  gated_top_kernel<ACT><<<(unsigned)(ceil_div(a.tokens, 8 * rows) * groups), 256, 0, s>>>(
      static_cast<const uint16_t*>(dh), pre, a.tokens, a.inter, (int)rows, top);
  return cudaGetLastError();
}

static int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }
static int64_t both_bytes(int64_t tokens, int inter) {
  return up256(gradient_terms(tokens, inter) * tokens * 2 * inter * 2);
}
static int64_t top_bytes(int64_t tokens, int inter) {
  return up256((tokens + 2 * (int64_t)inter) * 4);
}
// fp16: up to 16 MB a form, the two forms of [dG dU] lie side by side and are written at once; above,
// the second takes the first's place, by an elementwise pass of its own.  Forward and gradients of 777
// tokens, 1000 x 520: 121 us at once, 126 in two passes; 8192 tokens, 4096 x 2048: 678 and 706, which
// would cost every caller 67 MB more workspace.
static bool two_forms(int64_t tokens, int inter) { return both_bytes(tokens, inter) <= (16 << 20); }

template <bool BF16>
static cudaError_t backward_t(const GatedArgs& a, const void* dh, const float* pre,
                              uint8_t* workspace, void* dx, void* dw13, cudaStream_t s) {
  const int terms = gradient_terms(a.tokens, a.inter);
  const bool silu = a.activation == kSilu;
  const int64_t wide = 2 * (int64_t)a.inter;
  const int64_t form = both_bytes(a.tokens, a.inter);
  // [dG dU]: by token for dx, by feature for dW13 (bf16: the same); the maxima (fp16); the parts of a
  // split reduction (dx's, then dW13's)
  const bool at_once = !BF16 && two_forms(a.tokens, a.inter);
  uint16_t* by_token = reinterpret_cast<uint16_t*>(workspace);
  uint16_t* by_feature = reinterpret_cast<uint16_t*>(workspace + (at_once ? form : 0));
  uint8_t* at = workspace + (two_forms(a.tokens, a.inter) ? 2 : 1) * form;
  uint32_t* top = reinterpret_cast<uint32_t*>(at);
  GatedGemm p{};
  p.activation = a.activation;
  p.status = a.status;
  p.part = reinterpret_cast<float*>(at + top_bytes(a.tokens, a.inter));
  p.n = a.hidden;
  auto slope = [&](bool tokens, bool features) {
    auto* kern = silu ? gated_slope_kernel<BF16, kSilu> : gated_slope_kernel<BF16, kGeluTanh>;
    return launch_pdl(kern, stream_grid(a.tokens * (a.inter / 8)), 256, 0, s,
                      static_cast<const uint16_t*>(dh), pre, a.tokens, a.inter, terms,
                      static_cast<const uint32_t*>(top), tokens ? by_token : nullptr,
                      features ? by_feature : nullptr);
  };
  cudaError_t e = cudaSuccess;
  if (!BF16)
    e = silu ? launch_top<kSilu>(a, dh, pre, top, s) : launch_top<kGeluTanh>(a, dh, pre, top, s);
  if (e == cudaSuccess && (BF16 || at_once)) e = slope(BF16 || dx, !BF16 && dw13);
  if (e == cudaSuccess && dx) {
    if (!BF16 && !at_once) e = slope(true, false);
    if (e != cudaSuccess) return e;
    p.m = (int)a.tokens;
    p.k = (int)wide;
    p.out = dx;
    p.top = top + wide;
    e = product<kGradX, BF16>(by_token, a.tokens, wide, a.w13, wide, a.hidden, terms, p, s);
  }
  if (e == cudaSuccess && dw13) {
    if (!BF16 && !at_once) e = slope(false, true);
    if (e != cudaSuccess) return e;
    p.m = (int)wide;
    p.k = (int)a.tokens;
    p.out = dw13;
    p.top = top;
    e = product<kGradW, BF16>(by_feature, a.tokens, wide, a.x, a.tokens, a.hidden, terms, p, s);
  }
  return e;
}

int64_t gated_forward_workspace(int64_t tokens, int hidden, int inter) {
  return tokens <= kFewTokens ? 0 : part_bytes(kForward, tokens, inter, hidden, 1);
}

int64_t gated_backward_workspace(int64_t tokens, int hidden, int inter) {
  if (tokens == 0) return 0;  // nothing is launched, and there are no tiles to plan with
  const int terms = gradient_terms(tokens, inter);
  const int64_t x = part_bytes(kGradX, tokens, hidden, 2 * (int64_t)inter, terms);
  const int64_t w = part_bytes(kGradW, 2 * (int64_t)inter, hidden, tokens, terms);
  return (two_forms(tokens, inter) ? 2 : 1) * both_bytes(tokens, inter) +
         top_bytes(tokens, inter) + (x > w ? x : w);
}

cudaError_t launch_gated_forward(const GatedArgs& a, void* h, float* pre, void* workspace,
                                 cudaStream_t s) {
  return a.bf16 ? forward_t<true>(a, h, pre, static_cast<float*>(workspace), s)
                : forward_t<false>(a, h, pre, static_cast<float*>(workspace), s);
}

cudaError_t launch_gated_backward(const GatedArgs& a, const void* dh, const float* pre,
                                  void* workspace, void* dx, void* dw13, cudaStream_t s) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return a.bf16 ? backward_t<true>(a, dh, pre, ws, dx, dw13, s)
                : backward_t<false>(a, dh, pre, ws, dx, dw13, s);
}

}  // namespace exf
