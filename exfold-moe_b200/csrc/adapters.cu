// A shared projection with the low-rank adapters of many requests (sm_100a), bf16 or fp16, fp32 sums:
//
//   y_t = x_t W^T + z_t B_i^T,   z_t = scaling_i x_t A_i^T,   i = ids[t], z_t = 0 for ids outside
//
// Two launches.  adapter_down_kernel computes z in fp32, each token against its own adapter, by warp matrix
// instructions: x and the adapters in use are read once.  Then one GEMM over W whose reduction goes on over
// z and B: a tile of 128 tokens lists its distinct adapters, and for each the reduction gains columns for z of
// that adapter's tokens (0 for the others) as the sum of three bf16 terms, which hold an fp32 value's 24 bits and
// its range, against B (fp16: against the two bf16 terms that hold B).  So the adapters' part costs matrix
// instructions on tiles that are there anyway, z keeps what fp32 holds whatever the number of tokens, and y is
// written once, rounded once.  The GEMM starts on x and W while z is still being computed.  Up to 128 tokens, where every token may have an adapter of its own, the GEMM's threads
// add z B to its sums instead, a token's row from its own adapter, in fp32 (64 tokens of 32 adapters, rank 16:
// as columns of the reduction 23.8 us, so 17); up to 32 tokens that follows a kernel of warp matrix
// instructions.  8192 tokens in 12 runs of 8 adapters, rank 64, 2048 -> 4096: 138 us
// in bf16 (149 in fp16), of which z 22; 0.62 of a dense product's rate, the adapters' columns included.  Bound by what
// tiles of 128 x 256 bring into single SMs' shared memory: the tensor pipe is active 59 % of the time.
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

// The tokens up to which a form is taken; us of this form and of the next, 2048 -> 4096 bf16.
// The kernel without tiles (it holds no more): 16 tokens of 32 adapters, rank 16: 7.3 and 15.4; 32: 11.2, 14.7.
constexpr int kFewAdapted = 32;
// Adapters added row by row, z in fp32: 65 tokens of 32 adapters, rank 16: 17.4 and 22.4; 128: 25.7, 25.8, of 8
// adapters, rank 64: 38, 33, of 64: 42, 74; 256 of 32, rank 16: 32.7, 33.7, of 64, rank 64: 55, 127, in 4 runs of rank
// 64: 41, 27.
constexpr int kRowTokens = 128;
// z by adapter_down_kernel: 512 tokens of 32 adapters, rank 16: 50 and 78; 1024: 73, 96, in 4 runs of rank 64: 40,
// 39; 2048: 127, 165, in 8 runs of rank 64: 61, 59.
constexpr int kDownTokens = 1024;
constexpr int kAdaptedThreads = 320;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue, warps 6-9 adapters
constexpr int kABM = 128;           // tokens of a tile
constexpr int kABK = 64;            // columns of a stage: 128 bytes

struct AdapterPlan {
  int take;        // tokens a block of adapter_down_kernel
  int parts;       // blocks (a cluster) among which z's reduction is divided
  int nt, splits;  // the GEMM's tile, and the blocks (a cluster) that share its reduction
};

// What the kernels hand on: z, up to kRowTokens tokens fp32 [tokens][rank], else [tokens][ceil(rank / 16)][3][16], the
// three bf16 terms of 16 ranks (zeros past the last); for each tile of 128 tokens its number of distinct
// adapters and their ids, and for each token its place among them (255: none).
struct AdapterLists {
  float* z;
  uint16_t* z16;
  int32_t* count;   // [tiles]
  int32_t* list;    // [tiles][128]
  uint8_t* place;   // [tokens]
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
constexpr int kMostParts = 8;  // blocks of a cluster
// eight sums of the cluster's blocks, added in order
__device__ __forceinline__ void add_peers(const float* at, int parts, float (&z)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = 0.0f;
#pragma unroll
  for (int k = 0; k < kMostParts; ++k)
    if (k < parts) {
      const float4 a = load_peer4(at, k), b = load_peer4(at + 4, k);
      z[0] += a.x;
      z[1] += a.y;
      z[2] += a.z;
      z[3] += a.w;
      z[4] += b.x;
      z[5] += b.y;
      z[6] += b.z;
      z[7] += b.w;
    }
}
// The three bf16 terms of ranks r0 to r0 + 7 of a token, largest first: each the nearest to what is left, and
// the last exactly that (to 2^-133, bf16's smallest).  The first is cut off where rounding it would overflow.
// What is not finite is the last term: of B's two terms in fp16 the second, which is 0 for most values, meets
// only the first two.
constexpr int kTerms = 3;
__device__ __forceinline__ void store_terms(const AdapterLists& l, int token, int rank, int r0,
                                            const float (&z)[8]) {
  const float inf = __int_as_float(0x7f800000);
  float t[kTerms][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float first = unpack2<true>(pack2<true>(z[j], 0.0f)).x;
    if (!(fabsf(first) < inf)) first = __uint_as_float(__float_as_uint(z[j]) & 0xffff0000u);
    if (!(fabsf(z[j]) < inf)) first = 0.0f;
    const float rest = z[j] - first, second = unpack2<true>(pack2<true>(rest, 0.0f)).x;
    t[0][j] = first;
    t[1][j] = fabsf(z[j]) < inf ? second : 0.0f;
    t[2][j] = rest - t[1][j];
  }
  const int64_t at = ((int64_t)token * ((rank + 15) / 16) + r0 / 16) * (16 * kTerms) + r0 % 16;
#pragma unroll
  for (int k = 0; k < kTerms; ++k) store_16b<true>(l.z16, at + 16 * k, t[k]);
}
// 8 columns of 16 bits, or zeros
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool there) {
  return there ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}

// ---- the adapters of a tile --------------------------------------------------------------------------------
// The distinct adapters among 128 tokens in the order of their first token, and each token's place among them
// (255: none), by the first 128 threads of a block that all call it.
struct TileAdapters {
  int id[128], list[128];
  uint32_t first[4];
  int count;
};
__device__ __forceinline__ int list_adapters(const AdapterArgs& p, int tile, TileAdapters& sm) {
  const int t = tile * 128 + (int)threadIdx.x;
  if (threadIdx.x < 128) {
    const int i = t < p.tokens ? p.ids[t] : -1;
    sm.id[threadIdx.x] = i >= 0 && i < p.adapters ? i : -1;
  }
  __syncthreads();
  int lead = 0, mine = -1;
  if (threadIdx.x < 128) {
    mine = sm.id[threadIdx.x];
    while (sm.id[lead] != mine) ++lead;
    const uint32_t word = __ballot_sync(0xffffffffu, mine >= 0 && lead == (int)threadIdx.x);
    if ((threadIdx.x & 31) == 0) sm.first[threadIdx.x >> 5] = word;
  }
  __syncthreads();
  int place = 255;
  if (threadIdx.x < 128) {
    if (mine >= 0) {
      place = __popc(sm.first[lead >> 5] & ((1u << (lead & 31)) - 1u));
      for (int w = 0; w < lead >> 5; ++w) place += __popc(sm.first[w]);
      if (lead == (int)threadIdx.x) sm.list[place] = mine;
    }
    if (threadIdx.x == 0) {
      sm.count = 0;
      for (int w = 0; w < 4; ++w) sm.count += __popc(sm.first[w]);
    }
  }
  __syncthreads();
  return place;
}
__device__ __forceinline__ void write_list(const AdapterArgs& p, const AdapterLists& l, int tile,
                                           const TileAdapters& sm, int place) {
  const int t = tile * 128 + (int)threadIdx.x;
  if (threadIdx.x >= 128) return;
  if (t < p.tokens) l.place[t] = (uint8_t)place;
  if ((int)threadIdx.x < sm.count) l.list[tile * 128 + threadIdx.x] = sm.list[threadIdx.x];
  if (threadIdx.x == 0) l.count[tile] = sm.count;
}

// ---- z of up to 1024 tokens ----------------------------------------------------------------------------------
// A block takes up to 8 tokens and one part of the reduction.  Its work is each distinct adapter's rows, R at a
// time, against all of them (a token keeps its own adapter's column), in units of 32 columns, dealt out to
// the 8 warps in equal runs: where every token has an adapter of its own, each warp streams one of them.  A
// lane loads 8 columns (16 bytes) of a row, and the instruction's 16 columns are taken as words 0, 1 and then
// 2, 3 of each: the order of a sum is free as long as both operands have the same.  (All warps on one
// adapter after another: 64 tokens of 32 adapters, 2048 columns, rank 16: 10 us, a load's latency each.)
// The parts are a cluster, which adds its sums.  The first block of each tile of 128 tokens lists the tile's
// adapters for the GEMM.
template <bool BF16, int MB>
__global__ void __launch_bounds__(256)
    adapter_down_kernel(const AdapterArgs p, const AdapterLists l, bool rows, int parts, int take) {
  constexpr int TB = 8, R = 16 * MB;
  __shared__ float sums[8][TB][R + 1];
  __shared__ __align__(16) float joined[TB][R];
  __shared__ TileAdapters tile;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // (only now: the GEMM reads x before it waits for this kernel)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int part = parts > 1 ? cluster_rank() : 0, t0 = blockIdx.x / parts * take;
  const int tokens = (int)p.tokens < t0 + take ? (int)p.tokens : t0 + take;  // (up to here)
  const int all = (p.inner + 31) / 32;
  const int u0 = all * part / parts, units = all * (part + 1) / parts - u0;
  int mine = lane < TB && t0 + lane < tokens ? p.ids[t0 + lane] : -1;
  if (mine < 0 || mine >= p.adapters) mine = -1;
  const uint32_t same = __match_any_sync(0xffffffffu, mine);
  const uint32_t leaders = __ballot_sync(0xffffffffu, mine >= 0 && __ffs(same) - 1 == lane);
  const int items = __popc(leaders) * units;
  const int i0 = items * warp / 8, i1 = items * (warp + 1) / 8;  // this warp's
  const int first = units ? i0 / units : 0, last = units ? (i1 + units - 1) / units : 0;

  const uint16_t* x = static_cast<const uint16_t*>(p.x);
  const int g = lane >> 2, c = lane & 3;
  for (int r0 = 0; r0 < p.rank; r0 += R) {
    for (int i = lane; i < TB * (R + 1); i += 32) (&sums[warp][0][0])[i] = 0.0f;
    __syncwarp();
    uint32_t left = leaders;
    for (int n = 0; n < last; ++n, left &= left - 1) {
      if (n < first) continue;
      const int lead = __ffs(left) - 1;
      const int id = __shfl_sync(0xffffffffu, mine, lead);
      const uint32_t members = __shfl_sync(0xffffffffu, same, lead);
      const uint16_t* a = static_cast<const uint16_t*>(p.a) + ((int64_t)id * p.rank + r0) * p.inner;
      const int b0 = n == first ? i0 - n * units : 0, b1 = n == last - 1 ? i1 - n * units : units;
      float d[MB][4] = {};
#pragma unroll(MB == 4 ? 3 : 4)
      for (int u = b0; u < b1; ++u) {
        const int k = (u0 + u) * 32 + 8 * c;
        const bool in = k < p.inner;
        uint4 av[MB][2];
        const uint4 xv = load8(x + (int64_t)(t0 + g) * p.inner + k, in && t0 + g < tokens);
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            av[m][h] = load8(a + (int64_t)(16 * m + 8 * h + g) * p.inner + k,
                             in && r0 + 16 * m + 8 * h + g < p.rank);
#pragma unroll
        for (int m = 0; m < MB; ++m) {
          warp_mma<BF16>(d[m], av[m][0].x, av[m][1].x, av[m][0].y, av[m][1].y, xv.x, xv.y);
          warp_mma<BF16>(d[m], av[m][0].z, av[m][1].z, av[m][0].w, av[m][1].w, xv.z, xv.w);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = 2 * c + j;
        if (members >> t & 1) {
#pragma unroll
          for (int m = 0; m < MB; ++m) {
            sums[warp][t][16 * m + g] = d[m][j];
            sums[warp][t][16 * m + 8 + g] = d[m][2 + j];
          }
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TB * R; i += 256) {
      const int t = i / R, r = i % R;
      float z = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) z += sums[w][t][r];
      joined[t][r] = z;
    }
    if (parts > 1)
      cluster_sync();
    else
      __syncthreads();
    // eight ranks a thread, dealt out to the cluster's blocks
    for (int i = part * 256 + threadIdx.x; i < TB * R / 8; i += parts * 256) {
      const int t = i / (R / 8), r = i % (R / 8) * 8;
      const int id = t0 + t < tokens ? p.ids[t0 + t] : -1;
      if (id < 0 || id >= p.adapters || r0 + r >= (p.rank + 15) / 16 * 16) continue;
      float z[8];
      add_peers(&joined[t][r], parts, z);
      if (p.scaling) {  // (past the rank z stays 0, whatever the factor)
        const float scale = r0 + r < p.rank ? p.scaling[id] : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] *= scale;
      }
      if (!rows) {
        store_terms(l, t0 + t, p.rank, r0 + r, z);
      } else if (r0 + r < p.rank) {
        float4* to = reinterpret_cast<float4*>(l.z + (int64_t)(t0 + t) * p.rank + r0 + r);
        to[0] = make_float4(z[0], z[1], z[2], z[3]);
        to[1] = make_float4(z[4], z[5], z[6], z[7]);
      }
    }
    if (parts > 1)
      cluster_sync();  // (nobody's sums are written over, and no block leaves, while they are read)
    else
      __syncthreads();
  }
  if (!rows && part == 0 && t0 % 128 == 0) {
    const int place = list_adapters(p, t0 / 128, tile);
    write_list(p, l, t0 / 128, tile, place);
  }
}

// ---- z of more tokens -----------------------------------------------------------------------------------------
// Tiles of 128 tokens on tcgen05: a block takes one part of the reduction of a tile (the parts are a cluster,
// which adds its sums), lists the tile's adapters (for the GEMM too), and multiplies the tile by each one's rows (RN of them, from its first on; those past
// its rank are another's, and not used); a token's thread keeps its own adapter's.  (Warp matrix
// instructions, 32 tokens a block: 8192 tokens, 2048 columns, rank 64: 38 us.)
template <int RN>
struct DownSmem {
  static constexpr int kStage = kABM * kABK * 2 + RN * kABK * 2;
  static constexpr int kStages = RN == 128 ? 4 : 6;
  alignas(1024) uint8_t tiles[kStages][kStage];
  alignas(16) float z[128][RN];
  alignas(8) uint64_t full[kStages];
  alignas(8) uint64_t empty[kStages];
  alignas(8) uint64_t acc_full[2];
  alignas(8) uint64_t acc_empty[2];
  alignas(8) uint64_t drain;
  TileAdapters tile;
  uint32_t tmem_base;
  int failed;
};
template <int RN, bool BF16>
__global__ void __launch_bounds__(192, 1)
    adapter_down_tile_kernel(const __grid_constant__ CUtensorMap map_x,
                             const __grid_constant__ CUtensorMap map_a, const AdapterArgs p,
                             const AdapterLists l, int parts) {
  using S = DownSmem<RN>;
  constexpr int kStages = S::kStages;
  constexpr int kColumns = 2 * RN < 32 ? 32 : 2 * RN;
  constexpr uint32_t kIdesc = idesc_f16(kABM, RN, BF16);
  extern __shared__ uint8_t smem_raw[];
  S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                ~static_cast<uintptr_t>(1023));
  const int warp = uniform(threadIdx.x >> 5);
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
    mbar_init(&sm.drain, 1);
    sm.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, kColumns);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // (only now: the GEMM reads x before it waits for this kernel)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int mt = blockIdx.x / parts, part = parts > 1 ? cluster_rank() : 0;
  const int place = list_adapters(p, mt, sm.tile);
  if (part == 0) write_list(p, l, mt, sm.tile, place);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();

  const int slots = uniform(sm.tile.count);
  const int kblocks = (p.inner + kABK - 1) / kABK;
  const int kb0 = (int)((int64_t)kblocks * part / parts);
  const int n = (int)((int64_t)kblocks * (part + 1) / parts) - kb0;
  const uint32_t tmem = uniform(sm.tmem_base);
  volatile int* failed = &sm.failed;
  if (warp == 0) {
    uint32_t g = 0;
    bool ok = true;
    for (int i = 0; i < slots && ok; ++i) {
      const int row = uniform(sm.tile.list[i]) * p.rank;
      for (int k = 0; k < n; ++k, ++g) {
        const int s = g % kStages;
        ok = warp_wait(&sm.empty[s], ((g / kStages) & 1) ^ 1, failed);
        if (!ok) break;
        if (elect_one()) {
          mbar_expect_tx(&sm.full[s], S::kStage);
          tma_load_2d(sm.tiles[s], &map_x, &sm.full[s], (kb0 + k) * kABK, mt * kABM);
          tma_load_2d(sm.tiles[s] + kABM * kABK * 2, &map_a, &sm.full[s], (kb0 + k) * kABK, row);
        }
      }
    }
    for (uint32_t j = g > kStages ? g - kStages : 0; j < g; ++j)
      mbar_wait_drain(&sm.full[j % kStages], (j / kStages) & 1);
  } else if (warp == 1) {
    uint32_t g = 0;
    bool ok = true;
    for (int i = 0; i < slots && ok; ++i) {
      const int b = i & 1;
      ok = warp_wait(&sm.acc_empty[b], ((i >> 1) & 1) ^ 1, failed);
      if (!ok) break;
      fence_after_sync();
      const uint32_t acc = tmem + static_cast<uint32_t>(b * RN);
      for (int k = 0; k < n; ++k, ++g) {
        const int s = g % kStages;
        ok = warp_wait(&sm.full[s], (g / kStages) & 1, failed);
        if (!ok) break;
        fence_after_sync();
        const uint32_t base = smem_addr(sm.tiles[s]);
        const uint64_t da = smem_desc(base), db = smem_desc(base + kABM * kABK * 2);
        if (elect_one()) {
#pragma unroll
          for (int e = 0; e < kABK / 16; ++e)
            mma_kind_f16(acc, da + 2 * e, db + 2 * e, kIdesc, k > 0 || e > 0 ? 1u : 0u);
          mma_commit(&sm.empty[s]);
        }
      }
      if (!ok) break;
      if (elect_one()) mma_commit(&sm.acc_full[b]);
    }
    if (slots > 0) {
      if (elect_one()) mma_commit(&sm.drain);
      mbar_wait_drain(&sm.drain, 0);
    }
  } else {
    const int q = warp & 3;
    const int token = mt * kABM + q * 32 + lane;
    const int id = token < p.tokens ? sm.tile.id[q * 32 + lane] : -1;
    float* to = sm.z[q * 32 + lane];
    for (int i = 0; i < slots; ++i) {
      const int b = i & 1;
      if (!warp_wait(&sm.acc_full[b], (i >> 1) & 1, failed)) break;
      fence_after_sync();
      const bool mine = id >= 0 && id == sm.tile.list[i];
      if (__any_sync(0xffffffffu, mine)) {
        const uint32_t taddr = tmem + static_cast<uint32_t>(b * RN) + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
        for (int c = 0; c < RN; c += 16) {
          uint32_t v[16];
          __syncwarp();
          tmem_load16(taddr + c, v);
          tmem_wait();
          if (mine) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(to + c + j) =
                  make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]),
                              __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
          }
        }
      }
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
    tmem_free(tmem, kColumns);
  }
  if (threadIdx.x == 0 && sm.failed && p.status) atomicExch(p.status, 1);
  if (parts > 1) cluster_sync();
  // eight ranks a thread, the tokens dealt out to the cluster's blocks
  const int groups = (p.rank + 15) / 16 * 2;
  const int m0 = 128 * part / parts, m1 = 128 * (part + 1) / parts;
  for (int i = threadIdx.x; i < (m1 - m0) * groups; i += 192) {
    const int m = m0 + i / groups, r = i % groups * 8, id = sm.tile.id[m];
    if (id < 0) continue;
    float z[8];
    add_peers(&sm.z[m][r], parts, z);
    const float scale = p.scaling ? p.scaling[id] : 1.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = r < p.rank ? z[j] * scale : 0.0f;
    store_terms(l, mt * kABM + m, p.rank, r, z);
  }
  if (parts > 1) cluster_sync();  // (no block leaves while its sums are read)
}

// ---- a few tokens -----------------------------------------------------------------------------------------
// z B of eight ranks
template <bool BF16>
__device__ __forceinline__ float dot8(const float4& z0, const float4& z1, const uint4& v, float y) {
  const float2 e0 = unpack2<BF16>(v.x), e1 = unpack2<BF16>(v.y), e2 = unpack2<BF16>(v.z),
               e3 = unpack2<BF16>(v.w);
  y = fmaf(z0.x, e0.x, y);
  y = fmaf(z0.y, e0.y, y);
  y = fmaf(z0.z, e1.x, y);
  y = fmaf(z0.w, e1.y, y);
  y = fmaf(z1.x, e2.x, y);
  y = fmaf(z1.y, e2.y, y);
  y = fmaf(z1.z, e3.x, y);
  return fmaf(z1.w, e3.y, y);
}

// A block computes 16 features of up to 8 NB tokens, its 8 warps an eighth of the reduction each; then a
// thread adds a feature's z B.  W is read ahead of the wait for z.
template <bool BF16, int NB>
__global__ void __launch_bounds__(256)
    adapted_few_kernel(const AdapterArgs p, const AdapterLists l) {
  constexpr int TB = 8 * NB;
  __shared__ float sums[8][TB][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * 16, tokens = (int)p.tokens;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint16_t* x = static_cast<const uint16_t*>(p.x);
  const uint16_t* w = static_cast<const uint16_t*>(p.w);
  const int units = (p.inner + 31) / 32;
  const int u0 = units * warp / 8, u1 = units * (warp + 1) / 8;
  float d[NB][4] = {};
#pragma unroll 4
  for (int u = u0; u < u1; ++u) {
    const int k = u * 32 + 8 * c;
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
      const float4* z = reinterpret_cast<const float4*>(l.z + (int64_t)t * p.rank);
#pragma unroll 4
      for (int r = 0; r < p.rank; r += 8)
        y = dot8<BF16>(z[r / 4], z[r / 4 + 1], load8(b + r, true), y);
    }
    static_cast<uint16_t*>(p.y)[(int64_t)t * p.outer + n] = (uint16_t)pack2<BF16>(y, 0.0f);
  }
}

// ---- tiles ----------------------------------------------------------------------------------------------
// Stages of 64 columns of x and W come by TMA (128-byte swizzle).  The adapters come in stages of their own,
// 16 ranks of one adapter: z's three terms (zeros for other adapters' tokens) and B, each 16 columns (32-byte
// swizzle), three products with one B.  fp16 B goes in as two bf16 terms (8 of its 11 bits and the rest, exact),
// the second against z's first two: its product with the third is below 2^-26 of z B.  Four warps write the
// stages, the next stage's loads under way while one waits for its place, and they are taken in between the main
// stages, spread over the tile: a sum's order is free.  (The first tile takes them last: z may still be on its
// way.)
// A tile's tokens meet all of its adapters, all but their own times 0, and 0 times an infinity is a NaN.  So
// eight columns of B with one that is not finite go in as zeros, and the epilogue adds them to their own
// adapter's tokens: one request's broken adapter does not reach another's.
template <int NT, bool BF16>
struct AdaptedCfg {
  static constexpr int kATile = kABM * kABK * 2;
  static constexpr int kBTile = NT * kABK * 2;
  static constexpr int kStage = kATile + kBTile;
  static constexpr int kZTile = kABM * 32;  // a term
  static constexpr int kExtra = kTerms * kZTile + (BF16 ? 1 : 2) * NT * 32;
  // (three in fp16 at 128 columns would leave adapter_down_kernel's blocks no room beside this kernel's: 65 tokens
  // 17.4 -> 21.5 us)
  static constexpr int kExtras = NT == 64 ? 4 : BF16 ? 3 : 2;
  static constexpr int kStages = (224 * 1024 - kExtras * kExtra) / kStage;
  static constexpr int kTmem = 2 * NT;  // two accumulators, a power of two
};
// Marks of tiles that left columns of B out, in a ring over the block's tiles that have stages of adapters at
// all.  A stage is filled once the one kExtras before it has been multiplied, in a tile that began behind the
// epilogue of its last but one; so at most the tiles of kExtras + 1 stages, and one before them, have marks that
// are still to be read.
constexpr int kMarks = 8;
template <int NT, bool BF16>
struct AdaptedSmem {
  static_assert(AdaptedCfg<NT, BF16>::kExtras + 2 <= kMarks, "marks are read before they are written over");
  alignas(1024) uint8_t tiles[AdaptedCfg<NT, BF16>::kStages][AdaptedCfg<NT, BF16>::kStage];
  alignas(1024) uint8_t extra[AdaptedCfg<NT, BF16>::kExtras][AdaptedCfg<NT, BF16>::kExtra];
  alignas(8) uint64_t full[AdaptedCfg<NT, BF16>::kStages];
  alignas(8) uint64_t empty[AdaptedCfg<NT, BF16>::kStages];
  alignas(8) uint64_t extra_full[AdaptedCfg<NT, BF16>::kExtras];
  alignas(8) uint64_t extra_empty[AdaptedCfg<NT, BF16>::kExtras];
  alignas(8) uint64_t acc_full[2];
  alignas(8) uint64_t acc_empty[2];
  alignas(8) uint64_t drain;
  uint32_t tmem_base;
  int failed;
  int broken[kMarks];  // 1 + the last tile that left columns of B out
};
template <int NT, bool BF16>
constexpr size_t adapted_smem_bytes() { return sizeof(AdaptedSmem<NT, BF16>) + 1024; }

// eight fp16 values in place as bf16, and what that leaves, also bf16
__device__ __forceinline__ void bf16_terms(uint4* at, uint4* rest) {
  const uint4 v = *at;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 e = unpack2<false>(w[j]);
    hi[j] = pack2<true>(e.x, e.y);
    const float2 near = unpack2<true>(hi[j]);
    lo[j] = pack2<true>(e.x - near.x, e.y - near.y);
  }
  *at = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  *rest = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// Shared-memory matrix descriptor: K-major tile with 32-byte rows, 32-byte swizzle (16-byte piece j of row m
// at piece j ^ (m / 4 % 2)); 8-row groups 256 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_32(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(256 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)6 << 61);
}

struct AdaptedGemm {
  AdapterArgs a;
  AdapterLists l;
  int m_tiles, n_tiles, kblocks, splits;
  bool rows;  // the adapters are added row by row
  bool wide;  // y's rows are 32-byte aligned
};

// The columns of B that stages [q0, q1) of M tile mt left out, for 32 of a token's features.
template <bool BF16>
__device__ __noinline__ void add_broken(const AdaptedGemm& p, int token, int mt, int col, int q0, int q1,
                                        float (&v)[32]) {
  const int slot = p.l.place[token], rank = p.a.rank, width = (rank + 15) / 16;
  if (slot == 255) return;
  const int id = p.l.list[mt * 128 + slot];
  for (int r0 = 0; r0 < rank; r0 += 8) {
    const int q = slot * width + r0 / 16;
    if (q < q0 || q >= q1) continue;
    const uint16_t* terms = p.l.z16 + ((int64_t)token * width + r0 / 16) * (16 * kTerms) + r0 % 16;
    float z[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      z[r] = unpack2<true>(terms[32 + r]).x + unpack2<true>(terms[16 + r]).x + unpack2<true>(terms[r]).x;
#pragma unroll 1
    for (int j = 0; j < 32 && col + j < p.a.outer; ++j) {
      const uint16_t* b =
          static_cast<const uint16_t*>(p.a.b) + ((int64_t)id * p.a.outer + col + j) * rank + r0;
      if (!not_finite<BF16>(load8(b, true))) continue;
#pragma unroll
      for (int r = 0; r < 8; ++r) v[j] = fmaf(z[r], unpack2<BF16>(b[r]).x, v[j]);
    }
  }
}

// A token's NT features by a warp: the sums at `at` and z B.  The ranks of a feature lie on LANES neighbouring
// lanes, eight each, so that a load of the warp is one stretch of B and z stays in registers; 32 features at a
// time, whose parts are exchanged so that each lane ends with a feature of its own.  (Eight features a thread,
// each with all of its ranks: 30 of 52 us at 128 tokens of rank 64.)
template <int NT, bool BF16, int LANES>
__device__ __forceinline__ void add_row(const AdaptedGemm& p, int id, int token, int col,
                                        const float* at, int lane) {
  const int rank = p.a.rank, outer = p.a.outer;
  const int piece = lane % LANES, f0 = lane / LANES;
  constexpr int kStep = 32 / LANES;
  const bool any = id >= 0 && id < p.a.adapters, mine = any && 8 * piece < rank;
  float4 z0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), z1 = z0;
  if (mine) {
    const float4* z = reinterpret_cast<const float4*>(p.l.z + (int64_t)token * rank + 8 * piece);
    z0 = z[0];
    z1 = z[1];
  }
  const uint16_t* b = static_cast<const uint16_t*>(p.a.b) +
                      ((int64_t)(any ? id : 0) * outer + col) * rank + 8 * piece;
  uint16_t* y = static_cast<uint16_t*>(p.a.y) + (int64_t)token * outer + col;
#pragma unroll(LANES <= 4 ? 4 : 2)
  for (int g = 0; g < NT; g += 32) {
    float e[LANES] = {};
    if (any) {
      uint4 v[LANES];
#pragma unroll
      for (int i = 0; i < LANES; ++i) {
        const int f = g + i * kStep + f0;
        v[i] = load8(b + (int64_t)f * rank, mine && col + f < outer);
      }
#pragma unroll
      for (int i = 0; i < LANES; ++i) e[i] = dot8<BF16>(z0, z1, v[i], 0.0f);
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < d; ++i) {
          const bool upper = piece & d;
          const float keep = upper ? e[i + d] : e[i], send = upper ? e[i] : e[i + d];
          e[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
        }
    }
    const int f = g + piece * kStep + f0;
    if (col + f < outer) y[f] = (uint16_t)pack2<BF16>(at[f] + e[0], 0.0f);
  }
}

template <int NT, bool BF16>
__global__ void __launch_bounds__(kAdaptedThreads, 1)
    adapted_gemm_kernel(const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_w, const AdaptedGemm p) {
  using C = AdaptedCfg<NT, BF16>;
  using S = AdaptedSmem<NT, BF16>;
  constexpr uint32_t kIdesc = idesc_f16(kABM, NT, BF16), kExtraIdesc = idesc_f16(kABM, NT, true);
  extern __shared__ uint8_t smem_raw[];
  S& sm = *reinterpret_cast<S*>(
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
    for (int m = 0; m < kMarks; ++m) sm.broken[m] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, C::kTmem);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // (with a split reduction, a tile's blocks are a cluster, and have one tile each; with rows too)
  const int ntiles = p.m_tiles * p.n_tiles * p.splits;
  const int width = (p.a.rank + 15) / 16;  // stages that an adapter adds
  // tile t: reduction part, M tile, N tile, k blocks [kb0, kb1)
  struct Tile {
    int part, mt, nt, kb0, kb1;
  };
  auto tile_of = [&](int t) {
    Tile r;
    r.part = t % p.splits;
    t /= p.splits;
    r.mt = t / p.n_tiles;
    r.nt = t - r.mt * p.n_tiles;
    r.kb0 = (int)((int64_t)p.kblocks * r.part / p.splits);
    r.kb1 = (int)((int64_t)p.kblocks * (r.part + 1) / p.splits);
    return r;
  };
  // its adapters' stages [q0, q1), read behind the wait for adapter_down_kernel
  auto extra_of = [&](const Tile& tl, int& q0, int& q1) {
    const int all = p.rows ? 0 : uniform(p.l.count[tl.mt]) * width;
    q0 = all * tl.part / p.splits;
    q1 = all * (tl.part + 1) / p.splits;
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
          const uint64_t db = smem_desc_32(base + kTerms * C::kZTile);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kTerms; ++k)
              mma_kind_f16(acc, smem_desc_32(base + k * C::kZTile), db, kExtraIdesc, 1u);
            if constexpr (!BF16) {
              const uint64_t low = smem_desc_32(base + kTerms * C::kZTile + NT * 32);
#pragma unroll
              for (int k = 0; k < 2; ++k)
                mma_kind_f16(acc, smem_desc_32(base + k * C::kZTile), low, kExtraIdesc, 1u);
            }
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
      if (ok && i == 0 && !p.rows) {
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
    // ---- epilogue: one token per thread (with rows nothing before the cluster's sums waits for z)
    if (!p.rows) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int q = warp & 3;
    const int outer = p.a.outer;
    int i = 0;
    uint32_t met = 0;  // tiles with stages of adapters
    for (int t = blockIdx.x; t < ntiles; t += gridDim.x, ++i) {
      const Tile tl = tile_of(t);
      const int b = i & 1;
      if (!warp_wait(&sm.acc_full[b], (i >> 1) & 1, failed)) break;
      fence_after_sync();
      const int row = tl.mt * kABM + q * 32 + lane;
      const uint32_t taddr = tmem + static_cast<uint32_t>(b * NT) + ((uint32_t)(q * 32) << 16);
      int q0 = 0, q1 = 0;
      extra_of(tl, q0, q1);  // (by whole warps)
      const bool broken =
          q1 > q0 && *const_cast<volatile int*>(&sm.broken[met++ % kMarks]) == t + 1;
#pragma unroll 1
      for (int c = 0; c < NT; c += 32) {
        float v[32];
        __syncwarp();
        tmem_load32(taddr + c, v);
        const int col = tl.nt * NT + c;
        if (row < p.a.tokens) {
          if (broken) add_broken<BF16>(p, row, tl.mt, col, q0, q1, v);
          if (p.splits > 1 || p.rows) {
            // (every copy into the tiles has been multiplied: they hold the sums)
            float* at = reinterpret_cast<float*>(sm.tiles) + (q * 32 + lane) * (NT + 4) + c;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<float4*>(at + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
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
  } else if (!p.rows) {
    // ---- the adapters' stages: a thread copies one of the tile's tokens' z and every 128th feature's B
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x - 192;
    const int tokens = (int)p.a.tokens, rank = p.a.rank, outer = p.a.outer;
    constexpr int kRows = (NT + 127) / 128, kBehind = C::kExtras - 1;
    const int piece = (tid >> 2 & 1) << 4;  // of the first half of the ranks
    uint32_t h = 0;    // stages issued
    uint32_t met = 0;  // tiles with stages, this one among them
    bool ok = true;
    // stage j has arrived: looked over, to the other proxy (it is read by the MMA), one arrival a warp
    auto hand_over = [&](uint32_t j, int t) {
      uint8_t* at = sm.extra[j % C::kExtras] + kTerms * C::kZTile;
#pragma unroll
      for (int e = 0; e < kRows; ++e)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (tid + 128 * e >= NT) continue;
          uint4* v = reinterpret_cast<uint4*>(at + (tid + 128 * e) * 32 + (piece ^ (k << 4)));
          const bool broken = not_finite<BF16>(*v);
          if (broken) *v = make_uint4(0, 0, 0, 0);
          if constexpr (!BF16) bf16_terms(v, v + NT * 2);
          if (broken) {
            *const_cast<volatile int*>(&sm.broken[(met - 1) % kMarks]) = t + 1;
          }
        }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.extra_full[j % C::kExtras]);
    };
    for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
      const Tile tl = tile_of(t);
      int q0, q1;
      extra_of(tl, q0, q1);
      met += q1 > q0;
      const int token = tl.mt * kABM + tid;
      const int place = token < tokens ? p.l.place[token] : 255;
      const uint16_t* z = p.l.z16 + (int64_t)(token < tokens ? token : 0) * width * (16 * kTerms);
      for (int q = q0; q < q1; ++q, ++h) {
        const int s = h % C::kExtras;
        ok = warp_wait(&sm.extra_empty[s], ((h / C::kExtras) & 1) ^ 1, failed);
        if (!ok) break;
        const int slot = q / width, group = q - slot * width;
        const int id = p.l.list[tl.mt * 128 + slot];
        uint8_t* at = sm.extra[s];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int to = piece ^ (k << 4);
          const bool mine = place == slot;
#pragma unroll
          for (int h = 0; h < kTerms; ++h)
            copy_async16(at + h * C::kZTile + tid * 32 + to, z + (group * kTerms + h) * 16 + 8 * k, mine);
#pragma unroll
          for (int e = 0; e < kRows; ++e) {
            const int row = tid + 128 * e, col = tl.nt * NT + row, r0 = group * 16 + 8 * k;
            const bool there = col < outer && r0 < rank;
            if (row < NT)
              copy_async16(at + kTerms * C::kZTile + row * 32 + to,
                           static_cast<const uint16_t*>(p.a.b) +
                               (there ? ((int64_t)id * outer + col) * rank + r0 : 0),
                           there);
          }
        }
        copy_async_commit();
        if (q - q0 >= kBehind) {
          copy_async_wait<kBehind>();
          hand_over(h - kBehind, t);
        }
      }
      copy_async_wait<0>();
      if (!ok) break;
      for (uint32_t j = h - (q1 - q0 < kBehind ? q1 - q0 : kBehind); j != h; ++j) hand_over(j, t);
    }
  }
  fence_before_sync();
  __syncthreads();
  if (p.splits > 1 || p.rows) {
    // the cluster's sums of this tile
    if (p.splits > 1) cluster_sync();
    const Tile tl = tile_of(blockIdx.x);
    float* sums = reinterpret_cast<float*>(sm.tiles);
    const int left = (int)p.a.tokens - tl.mt * kABM, rows = left < kABM ? left : kABM;
    // eight features a thread, the tokens dealt out to the cluster's blocks; for rows into this block's memory
    float* own = p.splits > 1 ? sums + kABM * (NT + 4) : sums;
    if (p.splits > 1)
      for (int e = threadIdx.x; e < (kABM + p.splits - 1) / p.splits * (NT / 8);
           e += kAdaptedThreads) {
        const int m = e / (NT / 8) * p.splits + tl.part, c = e % (NT / 8) * 8, col = tl.nt * NT + c;
        if (m >= rows || col >= p.a.outer) continue;
        float v[8];
        add_peers(sums + m * (NT + 4) + c, p.splits, v);
        if (p.rows) {
          float4* to = reinterpret_cast<float4*>(own + m / p.splits * (NT + 4) + c);
          to[0] = make_float4(v[0], v[1], v[2], v[3]);
          to[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          store_16b<BF16>(p.a.y, (int64_t)(tl.mt * kABM + m) * p.a.outer + col, v);
        }
      }
    if (p.rows) {
      if (p.splits > 1) __syncthreads();
      // (z's kernel ran after whatever wrote the ids)
      const int mine = tl.mt * kABM + (warp + kAdaptedThreads / 32 * lane) * p.splits + tl.part;
      const int ids = mine < p.a.tokens ? p.a.ids[mine] : -1;  // lane j: of the warp's j-th token
      asm volatile("griddepcontrol.wait;" ::: "memory");
      int turn = 0;
      for (int i = warp; i * p.splits + tl.part < rows; i += kAdaptedThreads / 32, ++turn) {
        const int token = tl.mt * kABM + i * p.splits + tl.part, col = tl.nt * NT;
        const int id = __shfl_sync(0xffffffffu, ids, turn);
        const float* at = own + i * (NT + 4);
        if (p.a.rank <= 8)
          add_row<NT, BF16, 1>(p, id, token, col, at, lane);
        else if (p.a.rank <= 16)
          add_row<NT, BF16, 2>(p, id, token, col, at, lane);
        else if (p.a.rank <= 32)
          add_row<NT, BF16, 4>(p, id, token, col, at, lane);
        else if (p.a.rank <= 64)
          add_row<NT, BF16, 8>(p, id, token, col, at, lane);
        else
          add_row<NT, BF16, 16>(p, id, token, col, at, lane);
      }
    }
    if (p.splits > 1) cluster_sync();  // (no block leaves while its sums are read)
  }
  if (warp == 1) {
    __syncwarp();
    fence_after_sync();
    tmem_free(tmem, C::kTmem);
  }
  if (threadIdx.x == 0 && sm.failed && p.a.status) atomicExch(p.a.status, 1);
}

// ---- host side ----------------------------------------------------------------------------------
static int64_t ceil_of(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t up_256(int64_t b) { return (b + 255) / 256 * 256; }

// z: blocks of 8 tokens up to kDownTokens, tiles of 128 above; the reduction in parts until the card is full,
// at least 256 columns each.  The GEMM: as the gated block's, tiles of 256 columns while they
// fill more than half of the SMs, else narrower ones, and long reductions split, at least 8 stages a part.
static AdapterPlan plan_of(int64_t tokens, int inner, int outer) {
  const int64_t sms = sm_count() > 0 ? sm_count() : 1;
  AdapterPlan pl;
  const bool few = tokens <= kDownTokens;
  // (4 tokens a block while two blocks of those fit an SM)
  pl.take = tokens <= sms ? 4 : 8;
  const int64_t blocks = ceil_of(tokens, few ? pl.take : kABM);
  int64_t parts = (few ? 2 : 1) * sms / blocks;
  if (parts > ceil_of(inner, 256)) parts = ceil_of(inner, 256);
  pl.parts = (int)(parts < 1 ? 1 : parts > kMostParts ? kMostParts : parts);
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
      pl.splits = (int)(s < 1 ? 1 : s > kMostParts ? kMostParts : s);
    }
  }
  return pl;
}

struct AdapterBytes {
  int64_t z, count, list, place, all;
};
static AdapterBytes bytes_of(int64_t tokens, int rank) {
  AdapterBytes b;
  const int64_t tiles = ceil_of(tokens, kABM);
  const bool few = tokens <= kRowTokens;
  b.z = up_256(few ? tokens * rank * 4 : tokens * ceil_of(rank, 16) * 32 * kTerms);
  b.count = few ? 0 : up_256(tiles * 4);
  b.list = few ? 0 : up_256(tiles * 128 * 4);
  b.place = few ? 0 : up_256(tokens);
  b.all = b.z + b.count + b.list + b.place;
  return b;
}

int64_t adapters_workspace(int64_t tokens, int rank) {
  return tokens == 0 ? 0 : bytes_of(tokens, rank).all;
}

template <bool BF16, int MB>
static cudaError_t down(const AdapterArgs& a, const AdapterLists& l, const AdapterPlan& pl, bool rows,
                        cudaStream_t s) {
  auto* kern = adapter_down_kernel<BF16, MB>;
  return launch_clusters(kern, dim3((unsigned)(ceil_of(a.tokens, pl.take) * pl.parts)), dim3(256), 0,
                         s, pl.parts, a, l, rows, pl.parts, pl.take);
}
template <int RN, bool BF16>
static cudaError_t down_tiles(const AdapterArgs& a, const AdapterLists& l, const AdapterPlan& pl,
                              cudaStream_t s) {
  constexpr auto dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto* kern = adapter_down_tile_kernel<RN, BF16>;
  constexpr size_t smem = sizeof(DownSmem<RN>) + 1024;
  static std::mutex mu;
  static bool done[64] = {};
  const cudaError_t e = allow_smem(kern, smem, mu, done);
  if (e != cudaSuccess) return e;
  // (without adapters nothing of A is read, and the map only has to be one)
  const bool any = a.adapters > 0;
  CUtensorMap mx, ma;
  if (!make_map(&mx, a.x, a.tokens, a.inner, kABM, dt) ||
      !make_map(&ma, any ? a.a : a.x, any ? (uint64_t)a.adapters * a.rank : a.tokens, a.inner, RN, dt))
    return cudaErrorInvalidValue;
  return launch_clusters(kern, dim3((unsigned)(ceil_of(a.tokens, kABM) * pl.parts)), dim3(192), smem, s,
                         pl.parts, mx, ma, a, l, pl.parts);
}

template <int NT, bool BF16>
static cudaError_t tiles(const AdapterArgs& a, const AdapterLists& l, const AdapterPlan& pl,
                         cudaStream_t s) {
  constexpr auto dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto* kern = adapted_gemm_kernel<NT, BF16>;
  static std::mutex mu;
  static bool done[64] = {};
  cudaError_t e = allow_smem(kern, adapted_smem_bytes<NT, BF16>(), mu, done);
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
  p.rows = a.tokens <= kRowTokens;
  p.wide = a.outer % 16 == 0 && reinterpret_cast<uintptr_t>(a.y) % 32 == 0;
  const int64_t all = (int64_t)p.m_tiles * p.n_tiles * p.splits;
  const int64_t sms = sm_count() > 0 ? sm_count() : all;
  return launch_clusters(kern, dim3((unsigned)(all < sms || p.splits > 1 || p.rows ? all : sms)),
                         dim3(kAdaptedThreads), adapted_smem_bytes<NT, BF16>(), s, p.splits, mx, mw, p);
}

template <bool BF16>
static cudaError_t adapted(const AdapterArgs& a, uint8_t* ws, cudaStream_t s) {
  const AdapterPlan pl = plan_of(a.tokens, a.inner, a.outer);
  const AdapterBytes by = bytes_of(a.tokens, a.rank);
  AdapterLists l;
  l.z = reinterpret_cast<float*>(ws);
  l.z16 = reinterpret_cast<uint16_t*>(ws);
  l.count = reinterpret_cast<int32_t*>(ws + by.z);
  l.list = reinterpret_cast<int32_t*>(ws + by.z + by.count);
  l.place = ws + by.z + by.count + by.list;
  const bool few = a.tokens <= kFewAdapted, rows = a.tokens <= kRowTokens;
  cudaError_t e;
  if (a.tokens <= kDownTokens) {
    e = a.rank <= 16   ? down<BF16, 1>(a, l, pl, rows, s)
        : a.rank <= 32 ? down<BF16, 2>(a, l, pl, rows, s)
                       : down<BF16, 4>(a, l, pl, rows, s);
  } else {
    e = a.rank <= 16   ? down_tiles<16, BF16>(a, l, pl, s)
        : a.rank <= 32 ? down_tiles<32, BF16>(a, l, pl, s)
        : a.rank <= 64 ? down_tiles<64, BF16>(a, l, pl, s)
                       : down_tiles<128, BF16>(a, l, pl, s);
  }
  if (e != cudaSuccess) return e;
  if (few) {
    auto go = [&](auto* kern) {
      return launch_pdl(kern, dim3((unsigned)ceil_of(a.outer, 16)), dim3(256), 0, s, a, l);
    };
    return a.tokens <= 8    ? go(adapted_few_kernel<BF16, 1>)
           : a.tokens <= 16 ? go(adapted_few_kernel<BF16, 2>)
                            : go(adapted_few_kernel<BF16, 4>);
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
