// The balance loss of a router over groups of tokens, the experts' counts, and the logits' gradient
// (sm_100a).
//
//   p_te  softmax over e, or sigmoid_te / sum_e sigmoid_te, of the tokens that the mask keeps (N of them)
//   c_e   routes to expert e,   P_e = sum_t p_te
//   loss = E / (k N^2) sum_e c_e P_e
//   dlogit_te = dloss E / (k N^2) p_te (c_e - sum_i p_ti c_i)  [sigmoid: times 1 - sigmoid_te]
//
// The counts carry no gradient.  They enter the gradient less their mean (sum_e p = 1, so nothing changes),
// which keeps the difference's bits when the experts are nearly even.  A row whose logits are all -inf has
// p = 0.  A token's sums are fp32; so is P_e within a block, where a lane adds at most 256 tokens, and in 64 bits
// over the blocks, in a fixed order.
//
// The logits are read once forward; backward reads them again and writes the gradient.  131072 x 128 fp32,
// top-8: forward 26.0 us (71 MB; 29 instructions executed a logit, at 0.59 of the issue slots: a warp's few steps
// wait for one another, and for a block's start and end), backward 23.9 (134 MB, 0.86 of a copy's rate).
// A token lies on a few lanes of a warp (about 16 columns a lane), so that a warp takes several at a time
// and a row's two reductions are a few shuffles; a lane keeps its columns, and adds them in registers.
#include "exf_balance.h"
#include "exf_common.cuh"
#include "exf_launch.h"
#include "exf_norm.cuh"

namespace exf {

constexpr int kBalanceThreads = 256;

// e^x within 2^-21: 2^t of the rounded product t = x log2(e), corrected by what the rounding left, x - t ln 2.
// Below 2^-126 it is 0 (a subnormal one would cost every call four instructions more: 27.9 us for 26.0).
__device__ __forceinline__ float exp_near(float x) {
  // (0 below -150; -inf would make a NaN of the rest; NaN stays)
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(x), "f"(-150.0f));
  const float t = x * 1.44269502f;
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return fmaf(e, fmaf(t, 1.90465432e-9f, fmaf(t, -0.693147182f, x)), e);
}

// A row's scores on `lanes` neighbouring lanes, in place of its logits, times the returned factor, the inverse
// of their sum; SLOPE: 1 - sigmoid in `slope`.  Columns past the last hold -inf.
template <int C, bool SIGMOID, bool SLOPE>
__device__ __forceinline__ float scores(float (&x)[C], float (&slope)[SLOPE ? C : 1], int lanes) {
  float m = x[0];
#pragma unroll
  for (int j = 1; j < C; ++j) m = fmaxf(m, x[j]);
  for (int d = lanes / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float sum = 0.0f;
  // sigmoid(x) is e^x to the last bit where the row's largest is below -18 (e^-18 < 2^-25): that row is a
  // softmax too
  if (!SIGMOID || m < -18.0f) {
    const float shift = m > -__int_as_float(0x7f800000) ? m : 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      x[j] = exp_near(x[j] - shift);
      if (SLOPE) slope[j] = 1.0f;
      sum += x[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const bool high = x[j] >= 0.0f;
      const float e = exp_near(-fabsf(x[j]));
      float r;  // (of 1 to 2)
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
      const float low = e * r;
      if (SLOPE) slope[j] = high ? low : r;
      x[j] = high ? r : low;
      sum += x[j];
    }
  }
  __syncwarp();
  for (int d = lanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return sum == 0.0f ? 0.0f : 1.0f / sum;
}

// A lane's columns: unit u = lane + lanes * i of V columns each.
template <typename T, int V, int NV>
__device__ __forceinline__ void fetch_logits(const T* row, int l, int lanes, int units, bool there,
                                             Pack<T, V> (&k)[NV]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (there && l + lanes * i < units) k[i].read(row + (l + lanes * i) * V);
}
template <typename T, int V, int NV>
__device__ __forceinline__ void take_logits(const Pack<T, V> (&k)[NV], int l, int lanes, int units,
                                            float (&x)[NV * V]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) x[i * V + j] = k[i].get(j);
  if (lanes * NV == units) return;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (l + lanes * i >= units) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[i * V + j] = -__int_as_float(0x7f800000);
    }
}

// Block b of a group takes tokens [T b / blocks, T (b + 1) / blocks): its sums of p, counts and number of
// tokens.
template <typename T, int V, int NV, bool SIGMOID>
__global__ void __launch_bounds__(kBalanceThreads, (NV * V <= 16 ? 4 : 2) / (V > 1 ? 1 : 2))
    balance_sums_kernel(const BalanceArgs a, const void* ids, bool ids64, int lanes, float* psum,
                        int32_t* pcount, int32_t* pvalid, int32_t* ticket) {
  extern __shared__ float shared[];  // [warps][experts] sums, [experts] counts
  constexpr int kWarps = kBalanceThreads / 32;
  const int e = a.experts, units = e / V;
  int32_t* count = reinterpret_cast<int32_t*>(shared + kWarps * e);
  __shared__ int valid;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int i = threadIdx.x; i < e; i += kBalanceThreads) count[i] = 0;
  if (threadIdx.x == 0) valid = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int group = blockIdx.y;
  const int64_t t0 = a.tokens * blockIdx.x / gridDim.x, t1 = a.tokens * (blockIdx.x + 1) / gridDim.x;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)group * a.tokens : nullptr;

  const int per_warp = 32 / lanes, lane = threadIdx.x & 31, l = lane % lanes;
  const T* logits = static_cast<const T*>(a.logits) + (int64_t)group * a.tokens * e;
  float acc[NV * V] = {};
  int mine = 0;
  Pack<T, V> next[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) next[i].clear();
  const int64_t first = t0 + (threadIdx.x >> 5) * per_warp + lane / lanes, step = kWarps * per_warp;
  auto kept = [&](int64_t t) { return t < t1 && !(mask && !mask[t]); };
  // (the mask is read a token further ahead than the logits, which wait for it)
  bool there = kept(first), ahead = kept(first + step);
  fetch_logits<T, V, NV>(logits + first * e, l, lanes, units, there, next);
  // the routes are counted while the first logits are on their way (a block has fewer than 2^32 of them)
  const uint32_t routes = (uint32_t)(t1 - t0) * (uint32_t)a.top_k;
  const int64_t at = ((int64_t)group * a.tokens + t0) * a.top_k;
  constexpr int kRoutes = 8;
  for (uint32_t i0 = threadIdx.x; i0 < routes; i0 += kRoutes * kBalanceThreads) {
    int32_t id[kRoutes];
#pragma unroll
    for (int j = 0; j < kRoutes; ++j) {
      const uint32_t i = i0 + j * kBalanceThreads;
      id[j] = -1;
      if (i < routes && !(mask && !mask[t0 + i / (uint32_t)a.top_k])) {
        if (ids64) {
          const int64_t wide = static_cast<const int64_t*>(ids)[at + i];
          if (wide >= 0 && wide < e) id[j] = (int32_t)wide;
        } else {
          id[j] = static_cast<const int32_t*>(ids)[at + i];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kRoutes; ++j)
      if (id[j] >= 0 && id[j] < e) atomicAdd(count + id[j], 1);
  }
  for (int64_t t = first; t - lane / lanes < t1; t += step) {
    float x[NV * V], none[1];
    take_logits<T, V, NV>(next, l, lanes, units, x);
    const bool now = there;
    mine += now && l == 0;
    // the next token's logits are on their way during this one's sums
    there = ahead;
    fetch_logits<T, V, NV>(logits + (t + step) * e, l, lanes, units, there, next);
    ahead = kept(t + 2 * step);
    const float inv = scores<NV * V, SIGMOID, false>(x, none, lanes);
    if (now) {  // (a token left out went along with whatever was there)
#pragma unroll
      for (int j = 0; j < NV * V; ++j) acc[j] = fmaf(x[j], inv, acc[j]);
    }
  }
  // the lanes of a warp that share columns, then the warps
#pragma unroll
  for (int j = 0; j < NV * V; ++j)
    for (int d = lanes; d < 32; d <<= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], d);
  if (lane < lanes) {
#pragma unroll
    for (int j = 0; j < NV * V; ++j) {
      const int u = l + lanes * (j / V);
      if (u < units) shared[(threadIdx.x >> 5) * e + u * V + j % V] = acc[j];
    }
  }
  if (mine) atomicAdd(&valid, mine);
  __syncthreads();
  const int64_t slot = (int64_t)group * gridDim.x + blockIdx.x;
  for (int c = threadIdx.x; c < e; c += kBalanceThreads) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += shared[w * e + c];
    psum[slot * e + c] = s;
    pcount[slot * e + c] = count[c];
  }
  if (threadIdx.x == 0) {
    pvalid[slot] = valid;
    if (blockIdx.x == 0) ticket[group] = 0;
  }
}

// The joined sums: a block takes 8 experts of a group (a sector of each block's sums), 64 threads an expert;
// the last block of a group to finish adds the experts' products c_e P_e, in order.
constexpr int kJoinThreads = 512;
__global__ void __launch_bounds__(kJoinThreads)
    balance_join_kernel(const float* psum, const int32_t* pcount, const int32_t* pvalid, int blocks,
                        int experts, int top_k, double* product, int32_t* ticket, float* loss,
                        int32_t* counts, int32_t* valid) {
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ double sums[kWarps][8];
  __shared__ int32_t routes[kWarps][8];
  __shared__ int tokens;
  __shared__ bool last;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int group = blockIdx.y;
  const int64_t base = (int64_t)group * blocks;
  const int x = threadIdx.x & 7, c = blockIdx.x * 8 + x;
  double s = 0.0;
  int32_t r = 0;
  if (c < experts) {
#pragma unroll 5
    for (int b = threadIdx.x >> 3; b < blocks; b += kJoinThreads / 8) {
      s += (double)__ldcg(psum + (base + b) * experts + c);
      r += __ldcg(pcount + (base + b) * experts + c);
    }
  }
#pragma unroll
  for (int d = 8; d < 32; d <<= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, d);
    r += __shfl_xor_sync(0xffffffffu, r, d);
  }
  if ((threadIdx.x & 31) < 8) {
    sums[threadIdx.x >> 5][x] = s;
    routes[threadIdx.x >> 5][x] = r;
  }
  __syncthreads();
  if (threadIdx.x < 8) {
#pragma unroll
    for (int i = 1; i < kWarps; ++i) {
      s += sums[i][x];
      r += routes[i][x];
    }
    if (c < experts) counts[(int64_t)group * experts + c] = r;
    double total = c < experts ? s * (double)r : 0.0;
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) total += __shfl_xor_sync(0xffu, total, d);
    if (x == 0) {
      product[(int64_t)group * gridDim.x + blockIdx.x] = total;
      __threadfence();
      last = atomicAdd(ticket + group, 1) == (int)gridDim.x - 1;
      tokens = 0;
    }
  }
  __syncthreads();
  if (!last) return;
  int n = 0;
  for (int b = threadIdx.x; b < blocks; b += kJoinThreads) n += __ldcg(pvalid + base + b);
  if (n) atomicAdd(&tokens, n);
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    double total = 0.0;
    for (int i = 0; i < gridDim.x; ++i)
      total += __ldcg(product + (int64_t)group * gridDim.x + i);
    const double t = (double)tokens;
    loss[group] = tokens ? (float)(total * experts / ((double)top_k * t * t)) : 0.0f;
    valid[group] = tokens;
  }
}

template <typename T, int V, int NV, bool SIGMOID>
__global__ void __launch_bounds__(kBalanceThreads)
    balance_backward_kernel(const BalanceArgs a, int lanes, const float* dloss, const int32_t* counts,
                            const int32_t* valid, T* dlogits) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kWarps = kBalanceThreads / 32;
  const int e = a.experts, units = e / V, group = blockIdx.y;
  const uint8_t* mask = a.mask ? a.mask + (int64_t)group * a.tokens : nullptr;
  const int per_warp = 32 / lanes, lane = threadIdx.x & 31, l = lane % lanes;
  const T* logits = static_cast<const T*>(a.logits) + (int64_t)group * a.tokens * e;
  T* out = dlogits + (int64_t)group * a.tokens * e;
  const double n = (double)valid[group];
  const float size = n > 0.0 ? (float)((double)dloss[group] * e / (a.top_k * n * n)) : 0.0f;
  const int middle = (int)(n * a.top_k / e);
  float c[NV * V];
#pragma unroll
  for (int j = 0; j < NV * V; ++j) {
    const int u = l + lanes * (j / V);
    c[j] = u < units ? (float)(counts[(int64_t)group * e + u * V + j % V] - middle) : 0.0f;
  }
  const int64_t first = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * per_warp;
  for (int64_t base = first; base < a.tokens; base += (int64_t)gridDim.x * kWarps * per_warp) {
    const int64_t t = base + lane / lanes;
    const bool in = t < a.tokens;
    const bool there = in && !(mask && !mask[t]);
    Pack<T, V> k[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) k[i].clear();
    float x[NV * V], slope[SIGMOID ? NV * V : 1];
    fetch_logits<T, V, NV>(logits + t * e, l, lanes, units, there, k);
    take_logits<T, V, NV>(k, l, lanes, units, x);
    const float inv = scores<NV * V, SIGMOID, SIGMOID>(x, slope, lanes);
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < NV * V; ++j) dot = fmaf(x[j], c[j], dot);
    for (int d = lanes / 2; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    dot *= inv;
    if (!in) continue;  // (the loop's condition is the warp's: no lane waits for another after it)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = l + lanes * i;
      if (u < units) {
        float d[V] = {};
        if (there) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            d[j] = size * (x[i * V + j] * inv * (c[i * V + j] - dot));
            if (SIGMOID) d[j] *= slope[SIGMOID ? i * V + j : 0];
          }
        }
        store_pack<T, V>(out + t * e + u * V, d);
      }
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------
// Blocks a group of the forward pass: all groups together four on an SM, at least 8 tokens a warp, and at most 256
// (without that bound a group that is a block's alone is added in as many steps as a warp has tokens of it: 131072
// tokens of 100 experts with even scores, 2e-5 off).
static int64_t balance_blocks(int groups, int64_t tokens) {
  const int64_t sms = sm_count() > 0 ? sm_count() : 1;
  const int64_t most = (4 * sms + groups - 1) / groups;
  const int64_t need = (tokens + 63) / 64, least = (tokens + 2047) / 2048;
  return need < most ? need : least > most ? least : most;
}
static int join_blocks(int experts) { return (experts + 7) / 8; }

// products, then the blocks' sums, counts and numbers of tokens, then the tickets
int64_t balance_workspace(int groups, int64_t tokens, int experts) {
  return groups * (8 * (int64_t)join_blocks(experts) + 4 +
                   balance_blocks(groups, tokens) * (8 * (int64_t)experts + 4));
}

// f(logits' type, V, NV, sigmoid) of the call's layout: vectors where rows allow them, 16 columns a lane,
// 32 for more than 512 experts
template <typename T, int V, typename F>
static cudaError_t balance_v(const BalanceArgs& a, F f) {
  const int units = a.experts / V;
  int lanes = 1;
  while (lanes < 32 && lanes * (16 / V) < units) lanes *= 2;
  using std::integral_constant;
  auto pick = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    return a.sigmoid ? f(T(), integral_constant<int, V>(), nv, std::true_type(), lanes)
                     : f(T(), integral_constant<int, V>(), nv, std::false_type(), lanes);
    (void)NV;
  };
  return lanes * (16 / V) >= units ? pick(integral_constant<int, 16 / V>())
                                   : pick(integral_constant<int, 32 / V>());
}
template <typename T, typename F>
static cudaError_t balance_t(const BalanceArgs& a, const void* out, F f) {
  constexpr int V = 16 / sizeof(T);
  return a.experts % V == 0 && norm_aligned(a.logits) && norm_aligned(out)
             ? balance_v<T, V>(a, f)
             : balance_v<T, 1>(a, f);
}
template <typename F>
static cudaError_t balance_dispatch(const BalanceArgs& a, const void* out, F f) {
  if (a.dtype == EXF_F32) return balance_t<float>(a, out, f);
  if (a.dtype == EXF_BF16) return balance_t<__nv_bfloat16>(a, out, f);
  return balance_t<__half>(a, out, f);
}

cudaError_t launch_balance_loss(const BalanceArgs& a, const void* ids, bool ids64, void* workspace,
                                float* loss, int32_t* counts, int32_t* valid, cudaStream_t s) {
  const int64_t blocks = balance_blocks(a.groups, a.tokens);
  if (blocks == 0) {  // no tokens
    cudaError_t e = cudaMemsetAsync(loss, 0, a.groups * sizeof(float), s);
    if (e == cudaSuccess) e = cudaMemsetAsync(valid, 0, a.groups * sizeof(int32_t), s);
    if (e == cudaSuccess)
      e = cudaMemsetAsync(counts, 0, (size_t)a.groups * a.experts * sizeof(int32_t), s);
    return e;
  }
  double* product = static_cast<double*>(workspace);
  float* psum = reinterpret_cast<float*>(product + (int64_t)a.groups * join_blocks(a.experts));
  int32_t* pcount = reinterpret_cast<int32_t*>(psum + a.groups * blocks * a.experts);
  int32_t* pvalid = pcount + a.groups * blocks * a.experts;
  int32_t* ticket = pvalid + a.groups * blocks;
  const cudaError_t err =
      balance_dispatch(a, nullptr, [&](auto t, auto v, auto nv, auto sigmoid, int lanes) {
        return launch_pdl(
            balance_sums_kernel<decltype(t), decltype(v)::value, decltype(nv)::value,
                                decltype(sigmoid)::value>,
            dim3((unsigned)blocks, a.groups), dim3(kBalanceThreads),
            (kBalanceThreads / 32 + 1) * (size_t)a.experts * 4, s, a, ids, ids64, lanes, psum, pcount,
            pvalid, ticket);
      });
  if (err != cudaSuccess) return err;
  return launch_pdl(balance_join_kernel, dim3(join_blocks(a.experts), a.groups), dim3(kJoinThreads), 0, s,
                    static_cast<const float*>(psum), static_cast<const int32_t*>(pcount),
                    static_cast<const int32_t*>(pvalid), (int)blocks, a.experts, a.top_k, product,
                    ticket, loss, counts, valid);
}

cudaError_t launch_balance_loss_backward(const BalanceArgs& a, const float* dloss,
                                         const int32_t* counts, const int32_t* valid, void* dlogits,
                                         cudaStream_t s) {
  return balance_dispatch(a, dlogits, [&](auto t, auto v, auto nv, auto sigmoid, int lanes) {
    const int64_t sms = sm_count() > 0 ? sm_count() : 1;
    const int64_t most = (8 * sms + a.groups - 1) / a.groups;
    const int64_t per_block = kBalanceThreads / lanes;
    const int64_t need = (a.tokens + per_block - 1) / per_block;
    return launch_pdl(balance_backward_kernel<decltype(t), decltype(v)::value, decltype(nv)::value,
                                              decltype(sigmoid)::value>,
                      dim3((unsigned)(need < most ? need : most), a.groups), dim3(kBalanceThreads),
                      0, s, a, lanes, dloss, counts, valid, static_cast<decltype(t)*>(dlogits));
  });
}

}  // namespace exf
