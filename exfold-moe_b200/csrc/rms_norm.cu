// Root-mean-square norm with the residual's addition, and its gradients (sm_100a).
//
//   s = round(x + residual)  (or x),  v = 1 / sqrt(mean_j s_j^2 + eps),  y_j = s_j v w_j
//   ds_j = v (w_j dy_j - s_j v mean_i(w_i dy_i s_i v)) + (the upstream gradient of s)_j
//   dw_j = sum over rows of dy_j s_j v
//
// The norm is taken of the sum as it is stored, so that y belongs to the residual stream that the next
// layer sees and the gradients need nothing but that stream: v is computed again from it, in the reduction
// that the gradient needs anyway, and no statistics are kept.  Sums are fp32; a sum of squares that leaves
// fp32's range is taken again in 64 bits.
//
// Bound by memory: a value is read and written once.  A row lies in the registers of its threads between
// its reduction and its results.
#include <mutex>

#include "exf_launch.h"
#include "exf_norm.cuh"

namespace exf {

// ---- forward ------------------------------------------------------------------------------------
// G threads a row, NV units of V elements a thread (unit u = thread + G * i); NV = 0: rows of any length,
// read again after the reduction.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(1024)
    rms_norm_kernel(const NormArgs a, int g, T* y) {
  __shared__ float part[32];
  __shared__ double part64[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_block = blockDim.x / g;
  const int64_t row = (int64_t)blockIdx.x * per_block + threadIdx.x / g;
  const int t = threadIdx.x % g;
  const bool live = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride;
  const T* r = a.residual ? static_cast<const T*>(a.residual) + (live ? row : 0) * a.r_stride : nullptr;
  T* sum_out = a.residual && live ? static_cast<T*>(a.sum) + row * a.cols : nullptr;
  const int units = a.cols / V;

  constexpr int N = NV > 0 ? NV : 1;
  float s[N][V];
  float q = 0.0f;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = t + g * i;
      if (u < units) {
        load_sum<T, V>(x + u * V, r ? r + u * V : nullptr, s[i]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) s[i][j] = 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) q = fmaf(s[i][j], s[i][j], q);
  } else {
    for (int u = t; u < units; u += g) {
      load_sum<T, V>(x + u * V, r ? r + u * V : nullptr, s[0]);
#pragma unroll
      for (int j = 0; j < V; ++j) q = fmaf(s[0][j], s[0][j], q);
    }
  }
  // up to two units' weights are on their way during the reduction
  constexpr bool kEarly = NV == 1 || NV == 2 || V == 1 && NV == 4;
  float w[N][V];
  if constexpr (kEarly) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + g * i < units) load_weight<T, V>(a.weight, a.weight_f32, (t + g * i) * V, w[i]);
  }
  const float v = inverse_norm(q, a, g, part, part64, [&] {
    double d = 0.0;
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d = fma((double)s[i][j], (double)s[i][j], d);
    } else {
      for (int u = t; u < units; u += g) {
        load_sum<T, V>(x + u * V, r ? r + u * V : nullptr, s[0]);
#pragma unroll
        for (int j = 0; j < V; ++j) d = fma((double)s[0][j], (double)s[0][j], d);
      }
    }
    return d;
  });
  if (!live) return;
  T* out = y + row * a.cols;
  auto finish = [&](int u, float (&e)[V], float (&we)[V]) {
    if (!kEarly) load_weight<T, V>(a.weight, a.weight_f32, u * V, we);
    if (sum_out) store_pack<T, V>(sum_out + u * V, e);
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = e[j] * v * we[j];
    store_pack<T, V>(out + u * V, e);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + g * i < units) finish(t + g * i, s[i], w[kEarly ? i : 0]);
  } else {
    for (int u = t; u < units; u += g) {
      load_sum<T, V>(x + u * V, r ? r + u * V : nullptr, s[0]);
      finish(u, s[0], w[0]);
    }
  }
}

// ---- backward -----------------------------------------------------------------------------------
// Blocks that stay: a thread keeps its columns from row to row and adds dw in registers; each block's sums
// go to part [blocks][cols] and rms_norm_join_kernel adds them in order.  (NV = 0: the sums stay in part.)
template <typename T, int V, int NV>
__global__ void __launch_bounds__(1024)
    rms_norm_backward_kernel(const NormArgs a, int g, const T* dy, const T* ds,
                             T* dx, float* part_dw) {
  __shared__ float part[2][32];
  __shared__ double part64[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_block = blockDim.x / g;
  const int sub = threadIdx.x / g, t = threadIdx.x % g;
  const int units = a.cols / V;
  const float mean = 1.0f / (float)a.cols;
  constexpr int N = NV > 0 ? NV : 1;
  float acc[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) acc[i][j] = 0.0f;
  bool first = true;
  for (int64_t base = (int64_t)blockIdx.x * per_block; base < a.rows;
       base += (int64_t)gridDim.x * per_block) {
    const int64_t row = base + sub;
    const bool live = row < a.rows;
    const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride;
    const T* up = dy + (live ? row : 0) * (int64_t)a.cols;
    const T* side = ds ? ds + (live ? row : 0) * (int64_t)a.cols : nullptr;
    float s[N][V], d[N][V];
    float q = 0.0f, c = 0.0f;
    auto take = [&](int u, float (&sv)[V], float (&dv)[V]) {
      float w[V];
      load_pack<T, V>(x + u * V, sv);
      load_pack<T, V>(up + u * V, dv);
      load_weight<T, V>(a.weight, a.weight_f32, u * V, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        q = fmaf(sv[j], sv[j], q);
        c = fmaf(dv[j] * w[j], sv[j], c);
      }
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (t + g * i < units) {
          take(t + g * i, s[i], d[i]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) s[i][j] = d[i][j] = 0.0f;
        }
      }
    } else {
      for (int u = t; u < units; u += g) take(u, s[0], d[0]);
    }
    q = row_sum(q, g, part[0]);
    c = row_sum(c, g, part[1]);
    float v = rsqrtf(q * mean + a.eps);
    float k = c * mean * v;
    const bool again = out_of_range(q, a.eps) || !(fabsf(c) < 3.0e38f);
    if (g > 32 ? again : __any_sync(0xffffffffu, again)) {
      double q64 = 0.0, c64 = 0.0;
      for (int u = t; u < units; u += g) {
        float e[V], o[V], w[V];
        load_pack<T, V>(x + u * V, e);
        load_pack<T, V>(up + u * V, o);
        load_weight<T, V>(a.weight, a.weight_f32, u * V, w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          q64 = fma((double)e[j], (double)e[j], q64);
          c64 = fma((double)o[j] * (double)w[j], (double)e[j], c64);
        }
      }
      q64 = row_sum(q64, g, part64);
      c64 = row_sum(c64, g, part64);
      if (again) {
        const double v64 = 1.0 / sqrt(q64 / a.cols + (double)a.eps);
        v = (float)v64;
        k = (float)(c64 / a.cols * v64);
      }
    }
    auto give = [&](int u, const float (&sv)[V], const float (&dv)[V], float (&sum)[V], bool add) {
      if (part_dw) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float e = dv[j] * (sv[j] * v);
          sum[j] = add ? sum[j] + e : e;
        }
      }
      if (dx) {
        float w[V], o[V], e[V];
        load_weight<T, V>(a.weight, a.weight_f32, u * V, w);
        if (side) load_pack<T, V>(side + u * V, o);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          e[j] = v * fmaf(-(sv[j] * v), k, dv[j] * w[j]);
          if (side) e[j] += o[j];
        }
        store_pack<T, V>(dx + row * a.cols + u * V, e);
      }
    };
    if (live) {
      if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (t + g * i < units) give(t + g * i, s[i], d[i], acc[i], true);
      } else {
        for (int u = t; u < units; u += g) {
          load_pack<T, V>(x + u * V, s[0]);
          load_pack<T, V>(up + u * V, d[0]);
          float* at = part_dw ? part_dw + (int64_t)blockIdx.x * a.cols + u * V : nullptr;
          if (at && !first) {
#pragma unroll
            for (int j = 0; j < V; ++j) acc[0][j] = at[j];
          }
          give(u, s[0], d[0], acc[0], !first);
          if (at) {
#pragma unroll
            for (int j = 0; j < V; ++j) at[j] = acc[0][j];
          }
        }
      }
    }
    first = false;
  }
  if (NV == 0 || !part_dw) return;
  // the block's rows beside one another are added in order
  extern __shared__ float sums[];  // [per_block][cols] where a block has several rows
  float* to = part_dw + (int64_t)blockIdx.x * a.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = t + g * i;
    if (u < units) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        (per_block > 1 ? sums + sub * a.cols : to)[u * V + j] = acc[i][j];
    }
  }
  if (per_block > 1) {
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      float e = 0.0f;
      for (int b = 0; b < per_block; ++b) e += sums[b * a.cols + c];
      to[c] = e;
    }
  }
}

// dw [cols] from the blocks' sums: 32 columns a block, 16 threads a column.
template <typename W>
__global__ void __launch_bounds__(512) rms_norm_join_kernel(const float* part, int blocks, int cols,
                                                            W* dw) {
  __shared__ float sums[16][33];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), j = threadIdx.x >> 5;
  float e = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int b = j; b < blocks; b += 16) e += __ldcg(part + (int64_t)b * cols + c);
  }
  sums[j][threadIdx.x & 31] = e;
  __syncthreads();
  if (j == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 16; ++i) e += sums[i][threadIdx.x];
    dw[c] = from_f32<W>(e);
  }
}

// ---- host side ----------------------------------------------------------------------------------
template <typename T, int V>
static cudaError_t forward_v(const NormArgs& a, void* y, cudaStream_t s) {
  const int64_t units = a.cols / V;
  // few rows: a unit a thread, the shortest chain; else two (single elements: four), so that more loads
  // are in flight a thread
  const int per = a.rows < 296 ? 1 : V > 1 ? 2 : 4;
  const int g = norm_threads(units, per, 8);
  const int block = g <= 32 ? 128 : g;
  const int per_block = block / g;
  const int64_t grid = (a.rows + per_block - 1) / per_block;
  const int need = (int)((units + g - 1) / g);
  auto* out = static_cast<T*>(y);
  auto go = [&](auto* kern) {
    return launch_pdl(kern, dim3((unsigned)grid), dim3(block), 0, s, a, g, out);
  };
  if (need <= 1) return go(rms_norm_kernel<T, V, 1>);
  if (V > 1) {
    if (need <= 2) return go(rms_norm_kernel<T, V, 2>);
    if (need <= 4) return go(rms_norm_kernel<T, V, (V > 1 ? 4 : 1)>);
  } else {
    if (need <= 4) return go(rms_norm_kernel<T, V, 4>);
    if (need <= 16) return go(rms_norm_kernel<T, V, (V > 1 ? 1 : 16)>);
  }
  return go(rms_norm_kernel<T, V, 0>);
}

template <typename T>
static cudaError_t forward_t(const NormArgs& a, void* y, cudaStream_t s) {
  return norm_vectors<T>(a) && norm_aligned(y) ? forward_v<T, 16 / sizeof(T)>(a, y, s)
                                               : forward_v<T, 1>(a, y, s);
}

cudaError_t launch_rms_norm(const NormArgs& a, void* y, cudaStream_t s) {
  if (a.dtype == EXF_F32) return forward_t<float>(a, y, s);
  if (a.dtype == EXF_BF16) return forward_t<__nv_bfloat16>(a, y, s);
  return forward_t<__half>(a, y, s);
}

// Blocks of the backward pass: four on an SM at 256 threads; at most a row each.
static int64_t backward_blocks(int64_t rows, int block, int per_block) {
  const int64_t sms = sm_count() > 0 ? sm_count() : 1;
  const int64_t most = sms * (block <= 256 ? 4 : block <= 512 ? 2 : 1);
  const int64_t need = (rows + per_block - 1) / per_block;
  return need < most ? need : most;
}

int64_t norm_backward_workspace(int64_t rows, int cols) {
  const int64_t sms = sm_count() > 0 ? sm_count() : 1;
  const int64_t blocks = rows < 4 * sms ? rows : 4 * sms;  // the most that any layout takes
  return blocks * cols * (int64_t)sizeof(float);
}

template <typename T, int V>
static cudaError_t backward_v(const NormArgs& a, const void* dy, const void* ds, void* dx, void* dw,
                              float* part, cudaStream_t s) {
  const int64_t units = a.cols / V;
  const int g = norm_threads(units, V > 1 ? 2 : 4, 8);
  const int block = g <= 32 ? 128 : g;
  const int per_block = block / g;
  const int64_t blocks = backward_blocks(a.rows, block, per_block);
  const int need = (int)((units + g - 1) / g);
  const size_t smem = per_block > 1 ? (size_t)per_block * a.cols * sizeof(float) : 0;
  auto go = [&](auto* kern) {
    return launch_pdl(kern, dim3((unsigned)blocks), dim3(block), smem, s, a, g,
                      static_cast<const T*>(dy), static_cast<const T*>(ds), static_cast<T*>(dx),
                      dw ? part : nullptr);
  };
  cudaError_t e;
  if (need <= 1)
    e = go(rms_norm_backward_kernel<T, V, 1>);
  else if (V > 1 && need <= 2)
    e = go(rms_norm_backward_kernel<T, V, 2>);
  else if (V == 1 && need <= 4)
    e = go(rms_norm_backward_kernel<T, V, (V > 1 ? 1 : 4)>);
  else if (V == 1 && need <= 8)
    e = go(rms_norm_backward_kernel<T, V, (V > 1 ? 1 : 8)>);
  else
    e = go(rms_norm_backward_kernel<T, V, 0>);
  if (e != cudaSuccess || !dw) return e;
  const dim3 grid((unsigned)((a.cols + 31) / 32));
  if (a.weight_f32)
    return launch_pdl(rms_norm_join_kernel<float>, grid, dim3(512), 0, s,
                      static_cast<const float*>(part), (int)blocks, a.cols, static_cast<float*>(dw));
  return launch_pdl(rms_norm_join_kernel<T>, grid, dim3(512), 0, s, static_cast<const float*>(part),
                    (int)blocks, a.cols, static_cast<T*>(dw));
}

template <typename T>
static cudaError_t backward_t(const NormArgs& a, const void* dy, const void* ds, void* dx, void* dw,
                              float* part, cudaStream_t s) {
  return norm_vectors<T>(a) && norm_aligned(dy) && norm_aligned(ds) && norm_aligned(dx)
             ? backward_v<T, 16 / sizeof(T)>(a, dy, ds, dx, dw, part, s)
             : backward_v<T, 1>(a, dy, ds, dx, dw, part, s);
}

cudaError_t launch_rms_norm_backward(const NormArgs& a, const void* dy, const void* ds, void* dx,
                                     void* dw, void* workspace, cudaStream_t s) {
  float* part = static_cast<float*>(workspace);
  if (a.dtype == EXF_F32) return backward_t<float>(a, dy, ds, dx, dw, part, s);
  if (a.dtype == EXF_BF16) return backward_t<__nv_bfloat16>(a, dy, ds, dx, dw, part, s);
  return backward_t<__half>(a, dy, ds, dx, dw, part, s);
}

}  // namespace exf
