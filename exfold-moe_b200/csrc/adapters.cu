// A shared projection with the low-rank adapters of many requests (sm_100a), bf16 or fp16, fp32 sums:
//
//   y_t = x_t W^T + z_t B_i^T,   z_t = scaling_i x_t A_i^T,   i = ids[t], z_t = 0 for ids outside
//
// Two launches.  adapter_down_kernel computes z in fp32, each token against its own adapter, by warp matrix
// instructions: x and the adapters in use are read once.  Then one GEMM over W whose reduction goes on over
// z and B: a tile of 128 tokens lists its distinct adapters, and for each the reduction gains 2 rank columns,
// z of that adapter's tokens (0 for the others) as the sum of two 16-bit terms (what one would round away is
// in the other: 2^-16 of z in bf16) against B twice.  So the adapters' part costs matrix instructions on
// tiles that are there anyway, and y is written once, rounded once.  The GEMM starts on x and W while z is
// still being computed.  Up to 16 tokens, where W's bytes are all that counts, a kernel of warp matrix
// instructions reads W by every SM and adds z B in fp32.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "exf_adapters.h"
#include "exf_common.cuh"
#include "exf_launch.h"
#include "exf_tc.cuh"
#include "exf_tc16.cuh"

namespace exf {
using namespace tc;

constexpr int kFewAdapted = 16;     // tokens of the kernel without tiles
constexpr int kAdaptedThreads = 320;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue, warps 6-9 adapters
constexpr int kABM = 128;           // tokens of a tile
constexpr int kABK = 64;            // columns of a stage: 128 bytes

struct AdapterPlan {
  int parts;        // z's reduction lies in this many parts, added where it is read
  int block_tokens; // of adapter_down_kernel
  int nt, splits;   // the GEMM's tile and the parts of its reduction
};

// What the kernels hand on: z [parts][tokens][rank]; for each tile of 128 tokens its number of distinct
// adapters and their ids, and for each token its place among them (255: none).
struct AdapterLists {
  float* z;
  int32_t* count;   // [tiles]
  int32_t* list;    // [tiles][128]
  uint8_t* place;   // [tokens]
  float* part;      // split reductions: [splits][tokens][outer]
};

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8), 16-bit operands
template <bool BF16>
__device__ __forceinline__ void warp_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// whether one of two 16-bit values is an infinity or a NaN
template <bool BF16>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  return (w & kExp) == kExp || (w >> 16 & kExp) == kExp;
}
template <bool BF16>
__device__ __forceinline__ bool not_finite(const uint4& v) {
  return not_finite2<BF16>(v.x) || not_finite2<BF16>(v.y) || not_finite2<BF16>(v.z) ||
         not_finite2<BF16>(v.w);
}
// 8 columns of 16 bits, or zeros
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool there) {
  return there ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

// ---- z --------------------------------------------------------------------------------------------------
// A block takes TB = 8 NB tokens and one part of the reduction, its 8 warps an eighth of that each; for each
// distinct adapter among the tokens, 16 MB of its rows against all of them (a token keeps its own adapter's
// column).  A lane loads 8 columns (16 bytes) of a row, and the instruction's 16 columns are taken as words
// 0, 1 and then 2, 3 of each: the order of a sum is free as long as both operands have the same.  Blocks
// before them (one for each tile of 128 tokens; none where no tiles follow) list the tiles' adapters.
template <bool BF16, int MB, int NB>
__global__ void __launch_bounds__(256)
    adapter_down_kernel(const AdapterArgs p, const AdapterLists l, int list_blocks, int parts) {
  constexpr int TB = 8 * NB, R = 16 * MB;
  extern __shared__ float sums[];  // [8 warps][TB tokens][R ranks]
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // (only now: the GEMM reads x before it waits for this kernel)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tokens = (int)p.tokens;

  if ((int)blockIdx.x < list_blocks) {
    __shared__ int id[128], first[128];
    const int t = blockIdx.x * 128 + threadIdx.x;
    if (threadIdx.x < 128) {
      const int i = t < tokens ? p.ids[t] : -1;
      id[threadIdx.x] = i >= 0 && i < p.adapters ? i : -1;
    }
    __syncthreads();
    int lead = 0;
    if (threadIdx.x < 128) {
      while (id[lead] != id[threadIdx.x]) ++lead;
      first[threadIdx.x] = lead == (int)threadIdx.x && id[threadIdx.x] >= 0;
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      int before = 0;
      for (int j = 0; j < lead; ++j) before += first[j];
      if (first[threadIdx.x]) l.list[blockIdx.x * 128 + before] = id[threadIdx.x];
      if (t < tokens) l.place[t] = id[threadIdx.x] >= 0 ? (uint8_t)before : 255;
      if (threadIdx.x == 127) {
        int all = 0;
        for (int j = 0; j < 128; ++j) all += first[j];
        l.count[blockIdx.x] = all;
      }
    }
    return;
  }

  const int block = blockIdx.x - list_blocks;
  const int part = block % parts, t0 = block / parts * TB;
  // this warp's columns, in units of 32
  const int units = (p.inner + 31) / 32, slices = parts * 8, slice = part * 8 + warp;
  const int k0 = (int)((int64_t)units * slice / slices) * 32;
  const int k1 = (int)((int64_t)units * (slice + 1) / slices) * 32;
  int mine = lane < TB && t0 + lane < tokens ? p.ids[t0 + lane] : -1;
  if (mine < 0 || mine >= p.adapters) mine = -1;
  const uint32_t same = __match_any_sync(0xffffffffu, mine);
  const uint32_t leaders = __ballot_sync(0xffffffffu, mine >= 0 && __ffs(same) - 1 == lane);

  const uint16_t* x = static_cast<const uint16_t*>(p.x);
  const int g = lane >> 2, c = lane & 3;
  float* own = sums + warp * TB * R;
  for (int r0 = 0; r0 < p.rank; r0 += R) {
    for (uint32_t left = leaders; left; left &= left - 1) {
      const int lead = __ffs(left) - 1;
      const int id = __shfl_sync(0xffffffffu, mine, lead);
      const uint32_t members = __shfl_sync(0xffffffffu, same, lead);
      const uint16_t* a = static_cast<const uint16_t*>(p.a) + ((int64_t)id * p.rank + r0) * p.inner;
      float d[MB][NB][4] = {};
#pragma unroll 2
      for (int k = k0 + 8 * c; k < k1 + 8 * c; k += 32) {
        const bool in = k < p.inner;
        uint4 xv[NB], av[MB][2];
#pragma unroll
        for (int n = 0; n < NB; ++n)
          xv[n] = load8(x + (int64_t)(t0 + 8 * n + g) * p.inner + k, in && t0 + 8 * n + g < tokens);
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            av[m][h] = load8(a + (int64_t)(16 * m + 8 * h + g) * p.inner + k,
                             in && r0 + 16 * m + 8 * h + g < p.rank);
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            warp_mma<BF16>(d[m][n], av[m][0].x, av[m][1].x, av[m][0].y, av[m][1].y, xv[n].x, xv[n].y);
            warp_mma<BF16>(d[m][n], av[m][0].z, av[m][1].z, av[m][0].w, av[m][1].w, xv[n].z, xv[n].w);
          }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int t = 8 * n + 2 * c + j;
          if (members >> t & 1) {
#pragma unroll
            for (int m = 0; m < MB; ++m) {
              own[t * R + 16 * m + g] = d[m][n][j];
              own[t * R + 16 * m + 8 + g] = d[m][n][2 + j];
            }
          }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TB * R; i += 256) {
      const int t = i / R, r = r0 + i % R;
      if (t0 + t < tokens && r < p.rank) {
        const int id = p.ids[t0 + t];
        float z = 0.0f;
        if (id >= 0 && id < p.adapters) {
#pragma unroll
          for (int w = 0; w < 8; ++w) z += sums[w * TB * R + i];
          if (p.scaling) z *= p.scaling[id];
        }
        l.z[((int64_t)part * tokens + t0 + t) * p.rank + r] = z;
      }
    }
    __syncthreads();
  }
}

// ---- a few tokens -----------------------------------------------------------------------------------------
// A block computes 16 features of up to 8 NB tokens, its 8 warps an eighth of the reduction each; then a
// thread adds a feature's z B.  W is read ahead of the wait for z.
template <bool BF16, int NB>
__global__ void __launch_bounds__(256)
    adapted_few_kernel(const AdapterArgs p, const AdapterLists l, int parts) {
  constexpr int TB = 8 * NB;
  __shared__ float sums[8][TB][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * 16, tokens = (int)p.tokens;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint16_t* x = static_cast<const uint16_t*>(p.x);
  const uint16_t* w = static_cast<const uint16_t*>(p.w);
  const int units = (p.inner + 31) / 32;
  const int k0 = units * warp / 8 * 32, k1 = units * (warp + 1) / 8 * 32;
  float d[NB][4] = {};
#pragma unroll 4
  for (int k = k0 + 8 * c; k < k1 + 8 * c; k += 32) {
    const bool in = k < p.inner;
    const uint4 lo = load8(w + (int64_t)(n0 + g) * p.inner + k, in && n0 + g < p.outer);
    const uint4 hi = load8(w + (int64_t)(n0 + 8 + g) * p.inner + k, in && n0 + 8 + g < p.outer);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const uint4 v = load8(x + (int64_t)(8 * n + g) * p.inner + k, in && 8 * n + g < tokens);
      warp_mma<BF16>(d[n], lo.x, hi.x, lo.y, hi.y, v.x, v.y);
      warp_mma<BF16>(d[n], lo.z, hi.z, lo.w, hi.w, v.z, v.w);
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sums[warp][8 * n + 2 * c + j][g] = d[n][j];
      sums[warp][8 * n + 2 * c + j][8 + g] = d[n][2 + j];
    }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = threadIdx.x; i < TB * 16; i += 256) {
    const int t = i / 16, f = i % 16, n = n0 + f;
    if (t >= tokens || n >= p.outer) continue;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) y += sums[k][t][f];
    const int id = p.ids[t];
    if (id >= 0 && id < p.adapters) {
      const uint16_t* b = static_cast<const uint16_t*>(p.b) + ((int64_t)id * p.outer + n) * p.rank;
      for (int r = 0; r < p.rank; r += 8) {
        const uint4 v = load8(b + r, true);
        float z[8] = {};
        for (int q = 0; q < parts; ++q) {
          const float4* at = reinterpret_cast<const float4*>(l.z + ((int64_t)q * tokens + t) * p.rank + r);
          const float4 u0 = at[0], u1 = at[1];
          z[0] += u0.x;
          z[1] += u0.y;
          z[2] += u0.z;
          z[3] += u0.w;
          z[4] += u1.x;
          z[5] += u1.y;
          z[6] += u1.z;
          z[7] += u1.w;
        }
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 e = unpack2<BF16>(words[j]);
          y = fmaf(z[2 * j], e.x, y);
          y = fmaf(z[2 * j + 1], e.y, y);
        }
      }
    }
    static_cast<uint16_t*>(p.y)[(int64_t)t * p.outer + n] = (uint16_t)pack2<BF16>(y, 0.0f);
  }
}

// ---- tiles ----------------------------------------------------------------------------------------------
// Stages of 64 columns of x and W come by TMA (128-byte swizzle).  The adapters' columns come in stages of
// 32 (64-byte swizzle) of their own, written by four warps while the main stages are multiplied, and are
// taken in between them, spread over the tile: a sum's order is free, and nothing waits for loads that could
// have been under way.  (The first tile takes them last: z may still be on its way.)
// A tile's tokens meet all of its adapters, all but their own times 0, and 0 times an infinity is a NaN.  So
// eight columns of B with one that is not finite go in as zeros, and the epilogue adds them to their own
// adapter's tokens: one request's broken adapter does not reach another's.
template <int NT>
struct AdaptedCfg {
  static constexpr int kATile = kABM * kABK * 2;
  static constexpr int kBTile = NT * kABK * 2;
  static constexpr int kStage = kATile + kBTile;
  static constexpr int kExtra = (kABM + NT) * 64;
  static constexpr int kExtras = NT == 256 ? 1 : 2;
  static constexpr int kStages = (220 * 1024 - kExtras * kExtra) / kStage;
  static constexpr int kTmem = 2 * NT;  // two accumulators, a power of two
};
template <int NT>
struct AdaptedSmem {
  alignas(1024) uint8_t tiles[AdaptedCfg<NT>::kStages][AdaptedCfg<NT>::kStage];
  alignas(1024) uint8_t extra[AdaptedCfg<NT>::kExtras][AdaptedCfg<NT>::kExtra];
  alignas(8) uint64_t full[AdaptedCfg<NT>::kStages];
  alignas(8) uint64_t empty[AdaptedCfg<NT>::kStages];
  alignas(8) uint64_t extra_full[AdaptedCfg<NT>::kExtras];
  alignas(8) uint64_t extra_empty[AdaptedCfg<NT>::kExtras];
  alignas(8) uint64_t acc_full[2];
  alignas(8) uint64_t acc_empty[2];
  alignas(8) uint64_t drain;
  uint32_t tmem_base;
  int failed;
  int broken[2];  // by accumulator: 1 + the last tile that left columns of B out
};
template <int NT>
constexpr size_t adapted_smem_bytes() { return sizeof(AdaptedSmem<NT>) + 1024; }

// Shared-memory matrix descriptor: K-major tile with 64-byte rows, 64-byte swizzle (16-byte piece j of row m
// at piece j ^ (m / 2 % 4)); 8-row groups 512 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_64(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(512 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)4 << 61);
}

struct AdaptedGemm {
  AdapterArgs a;
  AdapterLists l;
  int m_tiles, n_tiles, kblocks, splits, parts;
  bool wide;  // y's rows are 32-byte aligned
};

// The columns of B that stages [q0, q1) of M tile mt left out, for 32 of a token's features.
template <bool BF16>
__device__ __noinline__ void add_broken(const AdaptedGemm& p, int token, int mt, int col, int q0, int q1,
                                        float (&v)[32]) {
  const int slot = p.l.place[token], rank = p.a.rank, width = 2 * rank;
  if (slot == 255) return;
  const int id = p.l.list[mt * 128 + slot];
  for (int r0 = 0; r0 < rank; r0 += 8) {
    const int q = (slot * width + r0) / 32;  // the stage of their first terms
    if (q < q0 || q >= q1) continue;
#pragma unroll 1
    for (int j = 0; j < 32 && col + j < p.a.outer; ++j) {
      const uint16_t* b =
          static_cast<const uint16_t*>(p.a.b) + ((int64_t)id * p.a.outer + col + j) * rank + r0;
      if (!not_finite<BF16>(load8(b, true))) continue;
      for (int r = 0; r < 8; ++r) {
        float z = 0.0f;
        for (int k = 0; k < p.parts; ++k) z += p.l.z[((int64_t)k * p.a.tokens + token) * rank + r0 + r];
        v[j] = fmaf(z, unpack2<BF16>(b[r]).x, v[j]);
      }
    }
  }
}

template <int NT, bool BF16>
__global__ void __launch_bounds__(kAdaptedThreads, 1)
    adapted_gemm_kernel(const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_w, const AdaptedGemm p) {
  using C = AdaptedCfg<NT>;
  constexpr uint32_t kIdesc = idesc_f16(kABM, NT, BF16);
  extern __shared__ uint8_t smem_raw[];
  AdaptedSmem<NT>& sm = *reinterpret_cast<AdaptedSmem<NT>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int s = 0; s < C::kExtras; ++s) {
      mbar_init(&sm.extra_full[s], 4);
      mbar_init(&sm.extra_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.acc_full[b], 1);
      mbar_init(&sm.acc_empty[b], 4);
    }
    mbar_init(&sm.drain, 1);
    sm.failed = 0;
    sm.broken[0] = sm.broken[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, C::kTmem);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int mn_tiles = p.m_tiles * p.n_tiles;
  const int ntiles = mn_tiles * p.splits;
  const int width = 2 * p.a.rank;  // columns that an adapter adds
  // tile t: reduction part, M tile, N tile, k blocks [kb0, kb1)
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
  // its adapters' stages [q0, q1), read behind the wait for adapter_down_kernel
  auto extra_of = [&](const Tile& tl, int& q0, int& q1) {
    const int chunks = (uniform(p.l.count[tl.mt]) * width + 31) / 32;
    q0 = chunks * tl.part / p.splits;
    q1 = chunks * (tl.part + 1) / p.splits;
  };
  const uint32_t tmem = uniform(sm.tmem_base);
  volatile int* failed = &sm.failed;

  if (warp == 0) {
    // ---- TMA producer of x and W
    uint32_t g = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
      const Tile tl = tile_of(t);
      for (int kb = tl.kb0; kb < tl.kb1; ++kb, ++g) {
        const int s = g % C::kStages;
        ok = warp_wait(&sm.empty[s], ((g / C::kStages) & 1) ^ 1, failed);
        if (!ok) break;
        uint8_t* a = sm.tiles[s];
        uint64_t* bar = &sm.full[s];
        if (elect_one()) {
          mbar_expect_tx(bar, C::kStage);
          tma_load_2d(a, &map_x, bar, kb * kABK, tl.mt * kABM);
          tma_load_2d(a + C::kATile, &map_w, bar, kb * kABK, tl.nt * NT);
        }
      }
    }
    for (uint32_t j = g > C::kStages ? g - C::kStages : 0; j < g; ++j)
      mbar_wait_drain(&sm.full[j % C::kStages], (j / C::kStages) & 1);
  } else if (warp == 1) {
    // ---- MMA issuer: tile i accumulates into TMEM columns [NT (i & 1), +NT)
    uint32_t g = 0, h = 0;
    int i = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x, ++i) {
      const int b = i & 1;
      ok = warp_wait(&sm.acc_empty[b], ((i >> 1) & 1) ^ 1, failed);
      if (!ok) break;
      fence_after_sync();
      const uint32_t acc = tmem + static_cast<uint32_t>(b * NT);
      const Tile tl = tile_of(t);
      const int n = tl.kb1 - tl.kb0;
      int q0 = 0, q1 = 0, j = 0;
      if (i > 0) extra_of(tl, q0, q1);
      // stage j of the adapters comes behind main stage due of n
      int due = n / (q1 - q0 + 1);
      auto extras = [&](int done) {
        while (ok && j < q1 - q0 && due <= done) {
          const int s = h % C::kExtras;
          ok = warp_wait(&sm.extra_full[s], (h / C::kExtras) & 1, failed);
          if (!ok) break;
          fence_after_sync();
          const uint32_t base = smem_addr(sm.extra[s]);
          const uint64_t da = smem_desc_64(base), db = smem_desc_64(base + kABM * 64);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 2; ++k) mma_kind_f16(acc, da + 2 * k, db + 2 * k, kIdesc, 1u);
            mma_commit(&sm.extra_empty[s]);
          }
          ++h;
          ++j;
          due = (int)((int64_t)(j + 1) * n / (q1 - q0 + 1));
        }
      };
      for (int k = 0; k < n && ok; ++k, ++g) {
        const int s = g % C::kStages;
        ok = warp_wait(&sm.full[s], (g / C::kStages) & 1, failed);
        if (!ok) break;
        fence_after_sync();
        const uint32_t base = smem_addr(sm.tiles[s]);
        const uint64_t da = smem_desc(base), db = smem_desc(base + C::kATile);
        if (elect_one()) {
#pragma unroll
          for (int e = 0; e < kABK / 16; ++e)
            mma_kind_f16(acc, da + 2 * e, db + 2 * e, kIdesc, k > 0 || e > 0 ? 1u : 0u);
          mma_commit(&sm.empty[s]);
        }
        extras(k + 1);
      }
      if (ok && i == 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        extra_of(tl, q0, q1);
        due = 0;
        extras(1 << 30);
      }
      if (!ok) break;
      if (elect_one()) mma_commit(&sm.acc_full[b]);
    }
    if (elect_one()) mma_commit(&sm.drain);
    mbar_wait_drain(&sm.drain, 0);
  } else if (warp < 6) {
    // ---- epilogue: one token per thread
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int q = warp & 3;
    const int outer = p.a.outer;
    int i = 0;
    for (int t = blockIdx.x; t < ntiles; t += gridDim.x, ++i) {
      const Tile tl = tile_of(t);
      const int b = i & 1;
      if (!warp_wait(&sm.acc_full[b], (i >> 1) & 1, failed)) break;
      fence_after_sync();
      const int row = tl.mt * kABM + q * 32 + lane;
      const uint32_t taddr = tmem + static_cast<uint32_t>(b * NT) + ((uint32_t)(q * 32) << 16);
      const bool broken = *const_cast<volatile int*>(&sm.broken[b]) == t + 1;
      int q0 = 0, q1 = 0;
      extra_of(tl, q0, q1);  // (by whole warps)
#pragma unroll 1
      for (int c = 0; c < NT; c += 32) {
        float v[32];
        __syncwarp();
        tmem_load32(taddr + c, v);
        const int col = tl.nt * NT + c;
        if (row < p.a.tokens) {
          if (broken) add_broken<BF16>(p, row, tl.mt, col, q0, q1, v);
          if (p.splits > 1) {
            float* at = p.l.part + ((int64_t)tl.part * p.a.tokens + row) * outer + col;
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              if (col + j < outer) store_sums(at + j, v + j);
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 16)
              if (col + j < outer)
                store_32b<BF16>(p.a.y, (int64_t)row * outer + col + j, v + j, p.wide,
                                col + j + 8 < outer);
          }
        }
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[b]);
    }
  } else {
    // ---- the adapters' stages.  Column v of a tile's adapters belongs to adapter v / width, its first rank
    // columns the first terms of z, the others the second.  Eight columns (16 bytes) lie in one adapter and
    // one term; a thread writes the same eight of every 32nd row.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x - 192;
    const int piece = tid & 3, row0 = tid >> 2;
    const int tokens = (int)p.a.tokens, rank = p.a.rank, outer = p.a.outer;
    uint32_t h = 0;
    bool ok = true;
    int i = 0;
    for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x, ++i) {
      const Tile tl = tile_of(t);
      int q0, q1;
      extra_of(tl, q0, q1);
      const int columns = uniform(p.l.count[tl.mt]) * width;
      for (int q = q0; q < q1; ++q, ++h) {
        const int s = h % C::kExtras;
        const int v = q * 32 + 8 * piece;
        const int slot = v / width, w = v - slot * width;
        const bool in = v < columns, second = w >= rank;
        const int r0 = second ? w - rank : w;
        const int id = in ? p.l.list[tl.mt * 128 + slot] : 0;
        // loaded before the stage is free
        uint4 bv[NT / 32], av[kABM / 32];
#pragma unroll
        for (int j = 0; j < NT / 32; ++j) {
          const int col = tl.nt * NT + row0 + 32 * j;
          bv[j] = load8(static_cast<const uint16_t*>(p.a.b) + ((int64_t)id * outer + col) * rank + r0,
                        in && col < outer);
          if (not_finite<BF16>(bv[j])) {
            bv[j] = make_uint4(0, 0, 0, 0);
            *const_cast<volatile int*>(&sm.broken[i & 1]) = t + 1;
          }
        }
#pragma unroll
        for (int j = 0; j < kABM / 32; ++j) {
          const int token = tl.mt * kABM + row0 + 32 * j;
          av[j] = make_uint4(0, 0, 0, 0);
          if (in && token < tokens && p.l.place[token] == slot) {
            float z[8] = {};
            for (int k = 0; k < p.parts; ++k) {
              const float4* at =
                  reinterpret_cast<const float4*>(p.l.z + ((int64_t)k * tokens + token) * rank + r0);
              const float4 u0 = at[0], u1 = at[1];
              z[0] += u0.x;
              z[1] += u0.y;
              z[2] += u0.z;
              z[3] += u0.w;
              z[4] += u1.x;
              z[5] += u1.y;
              z[6] += u1.z;
              z[7] += u1.w;
            }
            if (second) {
#pragma unroll
              for (int k = 0; k < 8; ++k) z[k] = remainder_of<BF16>(z[k]);
            }
            av[j] = make_uint4(pack2<BF16>(z[0], z[1]), pack2<BF16>(z[2], z[3]),
                               pack2<BF16>(z[4], z[5]), pack2<BF16>(z[6], z[7]));
          }
        }
        ok = warp_wait(&sm.extra_empty[s], ((h / C::kExtras) & 1) ^ 1, failed);
        if (!ok) break;
        uint8_t* a = sm.extra[s];
        uint8_t* b = a + kABM * 64;
#pragma unroll
        for (int j = 0; j < NT / 32; ++j) {
          const int n = row0 + 32 * j;
          *reinterpret_cast<uint4*>(b + n * 64 + ((piece ^ (n >> 1 & 3)) << 4)) = bv[j];
        }
#pragma unroll
        for (int j = 0; j < kABM / 32; ++j) {
          const int m = row0 + 32 * j;
          *reinterpret_cast<uint4*>(a + m * 64 + ((piece ^ (m >> 1 & 3)) << 4)) = av[j];
        }
        // written by threads, read by the MMA: to the other proxy, then one arrival a warp
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.extra_full[s]);
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    fence_after_sync();
    tmem_free(tmem, C::kTmem);
  }
  if (threadIdx.x == 0 && sm.failed && p.a.status) atomicExch(p.a.status, 1);
}

// y from the parts of a split reduction, added in order; 8 columns a thread.
template <bool BF16>
__global__ void __launch_bounds__(256)
    adapted_join_kernel(const float* part, int splits, int64_t count, void* y) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8; i < count;
       i += (int64_t)gridDim.x * blockDim.x * 8) {
    float v[8] = {};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float4* at = reinterpret_cast<const float4*>(part + s * count + i);
      const float4 a = __ldcg(at), b = __ldcg(at + 1);
      v[0] += a.x;
      v[1] += a.y;
      v[2] += a.z;
      v[3] += a.w;
      v[4] += b.x;
      v[5] += b.y;
      v[6] += b.z;
      v[7] += b.w;
    }
    store_16b<BF16>(y, i, v);
  }
}

// ---- host side ----------------------------------------------------------------------------------
static int64_t ceil_of(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t up_256(int64_t b) { return (b + 255) / 256 * 256; }

// z: blocks of 8 tokens up to 256 tokens, of 32 above; the reduction in parts until the card is full, at
// least 32 columns a warp.  The GEMM: as the gated block's, tiles of 256 columns while they fill more than
// half of the SMs, else narrower ones, and long reductions split, at least 8 stages a part.
static AdapterPlan plan_of(int64_t tokens, int inner, int outer) {
  const int64_t sms = sm_count() > 0 ? sm_count() : 1;
  AdapterPlan pl;
  pl.block_tokens = tokens <= 256 ? 8 : 32;
  const int64_t blocks = ceil_of(tokens, pl.block_tokens);
  int64_t parts = 2 * sms / blocks;
  if (parts > ceil_of(inner, 256)) parts = ceil_of(inner, 256);
  pl.parts = (int)(parts < 1 ? 1 : parts > 8 ? 8 : parts);
  pl.nt = 256;
  pl.splits = 1;
  auto tiles = [&](int nt) { return ceil_of(tokens, kABM) * ceil_of(outer, nt); };
  const int64_t kblocks = ceil_of(inner, kABK);
  if (tiles(256) * 2 <= sms) {
    if (kblocks < 16) {
      pl.nt = tiles(128) * 2 > sms ? 128 : 64;
    } else {
      pl.nt = 128;
      int64_t s = sms / tiles(128);
      if (s > kblocks / 8) s = kblocks / 8;
      pl.splits = (int)(s > 1 ? s : 1);
    }
  }
  return pl;
}

struct AdapterBytes {
  int64_t z, count, list, place, part, all;
};
static AdapterBytes bytes_of(int64_t tokens, int outer, int rank, const AdapterPlan& pl) {
  AdapterBytes b;
  const int64_t tiles = ceil_of(tokens, kABM);
  const bool few = tokens <= kFewAdapted;
  b.z = up_256(pl.parts * tokens * rank * 4);
  b.count = few ? 0 : up_256(tiles * 4);
  b.list = few ? 0 : up_256(tiles * 128 * 4);
  b.place = few ? 0 : up_256(tokens);
  b.part = !few && pl.splits > 1 ? pl.splits * tokens * outer * 4 : 0;
  b.all = b.z + b.count + b.list + b.place + b.part;
  return b;
}

int64_t adapters_workspace(int64_t tokens, int inner, int outer, int rank) {
  if (tokens == 0) return 0;
  return bytes_of(tokens, outer, rank, plan_of(tokens, inner, outer)).all;
}

template <bool BF16, int MB, int NB>
static cudaError_t down(const AdapterArgs& a, const AdapterLists& l, const AdapterPlan& pl,
                        int list_blocks, cudaStream_t s) {
  auto* kern = adapter_down_kernel<BF16, MB, NB>;
  constexpr size_t smem = 8 * 8 * NB * 16 * MB * sizeof(float);
  static std::mutex mu;
  static bool done[64] = {};
  const cudaError_t e = allow_smem(kern, smem, mu, done);
  if (e != cudaSuccess) return e;
  const int64_t blocks = list_blocks + ceil_of(a.tokens, 8 * NB) * pl.parts;
  return launch_pdl(kern, dim3((unsigned)blocks), dim3(256), smem, s, a, l, list_blocks, pl.parts);
}
template <bool BF16, int NB>
static cudaError_t down_by_rank(const AdapterArgs& a, const AdapterLists& l, const AdapterPlan& pl,
                                int list_blocks, cudaStream_t s) {
  if (a.rank <= 16) return down<BF16, 1, NB>(a, l, pl, list_blocks, s);
  if (a.rank <= 32) return down<BF16, 2, NB>(a, l, pl, list_blocks, s);
  return down<BF16, 4, NB>(a, l, pl, list_blocks, s);
}

template <int NT, bool BF16>
static cudaError_t tiles(const AdapterArgs& a, const AdapterLists& l, const AdapterPlan& pl,
                         cudaStream_t s) {
  constexpr auto dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto* kern = adapted_gemm_kernel<NT, BF16>;
  static std::mutex mu;
  static bool done[64] = {};
  cudaError_t e = allow_smem(kern, adapted_smem_bytes<NT>(), mu, done);
  if (e != cudaSuccess) return e;
  CUtensorMap mx, mw;
  if (!make_map(&mx, a.x, a.tokens, a.inner, kABM, dt) ||
      !make_map(&mw, a.w, a.outer, a.inner, NT, dt))
    return cudaErrorInvalidValue;
  AdaptedGemm p{};
  p.a = a;
  p.l = l;
  p.m_tiles = (int)ceil_of(a.tokens, kABM);
  p.n_tiles = (int)ceil_of(a.outer, NT);
  p.kblocks = (int)ceil_of(a.inner, kABK);
  p.splits = pl.splits;
  p.parts = pl.parts;
  p.wide = a.outer % 16 == 0 && reinterpret_cast<uintptr_t>(a.y) % 32 == 0;
  const int64_t all = (int64_t)p.m_tiles * p.n_tiles * p.splits;
  const int64_t sms = sm_count() > 0 ? sm_count() : all;
  e = launch_pdl(kern, dim3((unsigned)(all < sms ? all : sms)), dim3(kAdaptedThreads),
                 adapted_smem_bytes<NT>(), s, mx, mw, p);
  if (e != cudaSuccess || pl.splits == 1) return e;
  const int64_t count = a.tokens * a.outer;
  const int64_t blocks = ceil_of(count, 2048);
  return launch_pdl(adapted_join_kernel<BF16>, dim3((unsigned)(blocks < 8 * sms ? blocks : 8 * sms)),
                    dim3(256), 0, s, static_cast<const float*>(l.part), pl.splits, count, a.y);
}

template <bool BF16>
static cudaError_t adapted(const AdapterArgs& a, uint8_t* ws, cudaStream_t s) {
  const AdapterPlan pl = plan_of(a.tokens, a.inner, a.outer);
  const AdapterBytes by = bytes_of(a.tokens, a.outer, a.rank, pl);
  AdapterLists l;
  l.z = reinterpret_cast<float*>(ws);
  l.count = reinterpret_cast<int32_t*>(ws + by.z);
  l.list = reinterpret_cast<int32_t*>(ws + by.z + by.count);
  l.place = ws + by.z + by.count + by.list;
  l.part = reinterpret_cast<float*>(ws + by.z + by.count + by.list + by.place);
  const bool few = a.tokens <= kFewAdapted;
  const int lists = few ? 0 : (int)ceil_of(a.tokens, kABM);
  cudaError_t e = pl.block_tokens == 8 ? down_by_rank<BF16, 1>(a, l, pl, lists, s)
                                       : down_by_rank<BF16, 4>(a, l, pl, lists, s);
  if (e != cudaSuccess) return e;
  if (few) {
    const dim3 grid((unsigned)ceil_of(a.outer, 16));
    return a.tokens <= 8 ? launch_pdl(adapted_few_kernel<BF16, 1>, grid, dim3(256), 0, s, a, l, pl.parts)
                         : launch_pdl(adapted_few_kernel<BF16, 2>, grid, dim3(256), 0, s, a, l, pl.parts);
  }
  switch (pl.nt) {
    case 256: return tiles<256, BF16>(a, l, pl, s);
    case 128: return tiles<128, BF16>(a, l, pl, s);
    default: return tiles<64, BF16>(a, l, pl, s);
  }
}

cudaError_t launch_adapters(const AdapterArgs& a, void* workspace, cudaStream_t s) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return a.bf16 ? adapted<true>(a, ws, s) : adapted<false>(a, ws, s);
}

}  // namespace exf
