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

#include "exf_launch.h"
#include "exf_norm.cuh"

namespace exf {

// ---- forward ------------------------------------------------------------------------------------
// Blocks that stay: G threads a row, NU units of V elements a thread.  The next
// row's loads are issued before this row is reduced, so that memory stays busy through the reduction and
// its barrier, and the weights stay in registers: 32768 x 4096 bf16 with a residual 175 us, 6.1 TB/s, 0.94 of
// a copy's rate.  (A block a row, without either: 255 us.)  G <= 32: a block holds 128 / G rows, and nothing waits but lanes for lanes.
template <typename T, typename W, int V, int NU, int THREADS>
__global__ void __launch_bounds__(THREADS)
    rms_norm_kernel(const NormArgs a, int g, T* y) {
  __shared__ float part[2][32];
  __shared__ double part64[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_block = blockDim.x / g;
  const int t = threadIdx.x % g;
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.residual);
  T* sum = static_cast<T*>(a.sum);
  const int64_t step = (int64_t)gridDim.x * per_block;
  const int64_t first = (int64_t)blockIdx.x * per_block;
  int64_t row = first + threadIdx.x / g;
  const Units<V> n(row, a.cols, t, g);
  const bool extra = V == 2 && n.odd >= 0 && t == 0;

  Pack<T, V> nx[NU], nr[NU], s[NU];
  float nx1 = 0.0f, nr1 = 0.0f;
  Weights<W, V, NU> w;
  auto fetch = [&](int64_t at) {
    const T* xr = x + at * a.x_stride + n.column(0);
    const T* rr = r + at * a.r_stride + n.column(0);
    const bool live = at < a.rows;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (n.has(i) && live) {
        nx[i].read(xr + n.step(i) * V);
        if (r) nr[i].read(rr + n.step(i) * V);
      } else {
        nx[i].clear();
        nr[i].clear();
      }
    }
    if (extra && live) {
      nx1 = to_f32<T>(x[at * a.x_stride + n.odd]);
      if (r) nr1 = to_f32<T>(r[at * a.r_stride + n.odd]);
    }
  };
  fetch(row);
  w.init(a.weight, t, n);
  const float mean = 1.0f / (float)a.cols;
  // every thread of a block (G <= 32: of a warp) takes as many turns
  int b = 0;
  for (int64_t base = first; base < a.rows; base += step, row += step, b ^= 1) {
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      s[i] = r ? rounded_sum<T, V>(nx[i], nr[i]) : nx[i];
#pragma unroll
      for (int j = 0; j < V; ++j) q = fmaf(s[i].get(j), s[i].get(j), q);
    }
    const float s1 = r ? to_f32<T>(from_f32<T>(nx1 + nr1)) : nx1;
    if (V == 2) q = fmaf(s1, s1, q);
    const bool live = row < a.rows;
    const int64_t at = row * a.cols;
    fetch(row + step);
    if (r && live) {
      T* to = sum + at + n.column(0);
#pragma unroll
      for (int i = 0; i < NU; ++i)
        if (n.has(i)) s[i].write(to + n.step(i) * V);
      if (extra) sum[at + n.odd] = from_f32<T>(s1);
    }
    const int64_t mine = live ? row : 0;
    const float v = inverse_norm<T>(q, mean, a, g, t, x + mine * a.x_stride,
                                    r ? r + mine * a.r_stride : nullptr, part[b], part64);
    if (live) {
      T* to = y + at + n.column(0);
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        s[i].anew();
        w.w[i].anew();
        if (n.has(i)) {
          float e[V];
#pragma unroll
          for (int j = 0; j < V; ++j) e[j] = s[i].get(j) * v * w.w[i].get(j);
          store_pack<T, V>(to + n.step(i) * V, e);
        }
      }
      if (extra) y[at + n.odd] = from_f32<T>(s1 * v * w.single);
    }
  }
}

// Rows of any length, read again after the reduction; a block a row.
template <typename T, int V>
__global__ void __launch_bounds__(1024) rms_norm_long_kernel(const NormArgs a, T* y) {
  __shared__ float part[32];
  __shared__ double part64[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.r_stride : nullptr;
  const int units = a.cols / V;
  float s[V];
  float q = 0.0f;
#pragma unroll 4
  for (int u = threadIdx.x; u < units; u += 1024) {
    load_sum<T, V>(x + u * V, r ? r + u * V : nullptr, s);
#pragma unroll
    for (int j = 0; j < V; ++j) q = fmaf(s[j], s[j], q);
  }
  const float mean = 1.0f / (float)a.cols;
  const float v = inverse_norm<T>(q, mean, a, 1024, threadIdx.x, x, r, part, part64);
#pragma unroll 4
  for (int u = threadIdx.x; u < units; u += 1024) {
    float w[V];
    load_sum<T, V>(x + u * V, r ? r + u * V : nullptr, s);
    load_weight<T, V>(a.weight, a.weight_f32, u * V, w);
    if (r) store_pack<T, V>(static_cast<T*>(a.sum) + row * a.cols + u * V, s);
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = s[j] * v * w[j];
    store_pack<T, V>(y + row * a.cols + u * V, s);
  }
}

// ---- backward -----------------------------------------------------------------------------------
// The same blocks and layout; a thread keeps its columns from row to row and adds dw in registers.  Each
// block's sums go to part_dw [blocks][cols], and rms_norm_join_kernel adds them in order.  16384 x 4096 bf16
// with the gradient of the sum: 92 us, 5.8 TB/s, 0.89 of a copy's rate; 16384 columns, a block of 1024 threads
// whose registers hold no row ahead, 0.53.
template <typename T, typename W, int V, int NU, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1)
    rms_norm_backward_kernel(const NormArgs a, int g, const T* dy, const T* ds, T* dx,
                             float* part_dw) {
  __shared__ float2 part[2][32];
  __shared__ double part64[32];
  extern __shared__ float sums[];  // [per_block][cols] where a block has several rows
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per_block = blockDim.x / g;
  const int sub = threadIdx.x / g, t = threadIdx.x % g;
  const float mean = 1.0f / (float)a.cols;
  const T* x = static_cast<const T*>(a.x);
  const int64_t step = (int64_t)gridDim.x * per_block;
  const int64_t first = (int64_t)blockIdx.x * per_block;
  int64_t row = first + sub;
  const Units<V> n(row, a.cols, t, g);
  const bool extra = V == 2 && n.odd >= 0 && t == 0;

  Pack<T, V> nx[NU], ny[NU], nd[NU];
  float nx1 = 0.0f, ny1 = 0.0f, nd1 = 0.0f;
  Weights<W, V, NU> w;
  float acc[NU][V], acc1 = 0.0f;
  auto fetch = [&](int64_t at) {
    const T* xr = x + at * a.x_stride + n.column(0);
    const T* yr = dy + at * a.cols + n.column(0);
    const T* dr = ds + at * a.cols + n.column(0);
    const bool live = at < a.rows;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      if (n.has(i) && live) {
        nx[i].read(xr + n.step(i) * V);
        ny[i].read(yr + n.step(i) * V);
        if (ds) nd[i].read(dr + n.step(i) * V);
      } else {
        nx[i].clear();
        ny[i].clear();
        nd[i].clear();
      }
    }
    if (extra && live) {
      nx1 = to_f32<T>(x[at * a.x_stride + n.odd]);
      ny1 = to_f32<T>(dy[at * a.cols + n.odd]);
      if (ds) nd1 = to_f32<T>(ds[at * a.cols + n.odd]);
    }
  };
  // (1024 threads have no registers for the row after this one)
  constexpr bool kAhead = THREADS < 1024;
  if (kAhead) fetch(row);
  w.init(a.weight, t, n);
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) acc[i][j] = 0.0f;
  int b = 0;
  for (int64_t base = first; base < a.rows; base += step, row += step, b ^= 1) {
    Pack<T, V> s[NU], d[NU], o[NU];
    float q = 0.0f, c = 0.0f;
    if (!kAhead) fetch(row);
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      s[i] = nx[i];
      d[i] = ny[i];
      o[i] = nd[i];
      w.w[i].anew();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float e = s[i].get(j);
        q = fmaf(e, e, q);
        c = fmaf(d[i].get(j) * w.w[i].get(j), e, c);
      }
    }
    const float s1 = nx1, d1 = ny1, o1 = nd1;
    if (extra) {
      q = fmaf(s1, s1, q);
      c = fmaf(d1 * w.single, s1, c);
    }
    if (kAhead) fetch(row + step);
    const float2 both = row_sum(make_float2(q, c), g, part[b]);
    q = both.x;
    c = both.y;
    float v = rsqrtf(q * mean + a.eps);
    float k = c * mean * v;
    const bool again = out_of_range(q, a.eps) || !(fabsf(c) < 3.0e38f);
    if (g > 32 ? again : __any_sync(0xffffffffu, again)) {
      const int64_t mine = row < a.rows ? row : 0;
      const double2 d64 = sums_64<T>(x + mine * a.x_stride, nullptr, dy + mine * a.cols, a.weight,
                                     std::is_same<W, float>::value, a.cols, t, g);
      const double q64 = row_sum(d64.x, g, part64);
      if (g > 32) __syncthreads();
      const double c64 = row_sum(d64.y, g, part64);
      if (g > 32) __syncthreads();
      if (again) {
        const double v64 = 1.0 / sqrt(q64 / a.cols + (double)a.eps);
        v = (float)v64;
        k = (float)(c64 / a.cols * v64);
      }
    }
    if (row < a.rows) {
      T* to = dx + row * a.cols + n.column(0);
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        s[i].anew();
        d[i].anew();
        w.w[i].anew();
        float e[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float hat = s[i].get(j) * v, up = d[i].get(j);
          acc[i][j] = fmaf(up, hat, acc[i][j]);
          e[j] = v * fmaf(-hat, k, up * w.w[i].get(j));
          if (ds) e[j] += o[i].get(j);
        }
        if (dx && n.has(i)) store_pack<T, V>(to + n.step(i) * V, e);
      }
      if (extra) {
        const float hat = s1 * v;
        acc1 = fmaf(d1, hat, acc1);
        float e = v * fmaf(-hat, k, d1 * w.single);
        if (ds) e += o1;
        if (dx) dx[row * a.cols + n.odd] = from_f32<T>(e);
      }
    }
  }
  if (!part_dw) return;
  float* to = part_dw + (int64_t)blockIdx.x * a.cols;
  float* mine = per_block > 1 ? sums + sub * a.cols : to;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if (n.has(i)) {
#pragma unroll
      for (int j = 0; j < V; ++j) mine[n.column(i) + j] = acc[i][j];
    }
  }
  if (extra) mine[n.odd] = acc1;
  // the block's rows beside one another are added in order
  if (per_block > 1) {
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
      float e = 0.0f;
      for (int p = 0; p < per_block; ++p) e += sums[p * a.cols + c];
      to[c] = e;
    }
  }
}

// Rows of any length, read again after the reduction; dw is added in part_dw itself, by the thread of its
// column.
template <typename T, int V>
__global__ void __launch_bounds__(1024)
    rms_norm_backward_long_kernel(const NormArgs a, const T* dy, const T* ds, T* dx,
                                  float* part_dw) {
  __shared__ float2 part[32];
  __shared__ double part64[2][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int units = a.cols / V;
  const float mean = 1.0f / (float)a.cols;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* up = dy + row * a.cols;
    float s[V], d[V], w[V];
    float q = 0.0f, c = 0.0f;
#pragma unroll 2
    for (int u = threadIdx.x; u < units; u += 1024) {
      load_pack<T, V>(x + u * V, s);
      load_pack<T, V>(up + u * V, d);
      load_weight<T, V>(a.weight, a.weight_f32, u * V, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        q = fmaf(s[j], s[j], q);
        c = fmaf(d[j] * w[j], s[j], c);
      }
    }
    const float2 both = row_sum(make_float2(q, c), 1024, part);
    q = both.x;
    c = both.y;
    float v = rsqrtf(q * mean + a.eps);
    float k = c * mean * v;
    if (out_of_range(q, a.eps) || !(fabsf(c) < 3.0e38f)) {
      const double2 d64 = sums_64<T>(x, nullptr, up, a.weight, a.weight_f32, a.cols, threadIdx.x, 1024);
      const double q64 = row_sum(d64.x, 1024, part64[0]);
      const double c64 = row_sum(d64.y, 1024, part64[1]);
      const double v64 = 1.0 / sqrt(q64 / a.cols + (double)a.eps);
      v = (float)v64;
      k = (float)(c64 / a.cols * v64);
    }
    float* to = part_dw ? part_dw + (int64_t)blockIdx.x * a.cols : nullptr;
#pragma unroll 2
    for (int u = threadIdx.x; u < units; u += 1024) {
      float e[V], o[V];
      load_pack<T, V>(x + u * V, s);
      load_pack<T, V>(up + u * V, d);
      load_weight<T, V>(a.weight, a.weight_f32, u * V, w);
      if (ds) load_pack<T, V>(ds + row * a.cols + u * V, o);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float hat = s[j] * v;
        e[j] = v * fmaf(-hat, k, d[j] * w[j]);
        if (ds) e[j] += o[j];
        if (to) to[u * V + j] = row == blockIdx.x ? d[j] * hat : fmaf(d[j], hat, to[u * V + j]);
      }
      if (dx) store_pack<T, V>(dx + row * a.cols + u * V, e);
    }
    __syncthreads();  // (the sums' shared memory is free for the next row)
  }
}

// dw [cols] from the blocks' sums: 8 columns (a sector of each row) a block, 64 threads a column, so that
// short rows fill the card too.
template <typename W>
__global__ void __launch_bounds__(512) rms_norm_join_kernel(const float* part, int blocks, int cols,
                                                            W* dw) {
  __shared__ float sums[16][8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int x = threadIdx.x & 7, c = blockIdx.x * 8 + x;
  float e = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int b = threadIdx.x >> 3; b < blocks; b += 64) e += __ldcg(part + (int64_t)b * cols + c);
  }
  e += __shfl_xor_sync(0xffffffffu, e, 8);
  e += __shfl_xor_sync(0xffffffffu, e, 16);
  if ((threadIdx.x & 31) < 8) sums[threadIdx.x >> 5][x] = e;
  __syncthreads();
  if (threadIdx.x < 8 && c < cols) {
#pragma unroll
    for (int i = 1; i < 16; ++i) e += sums[i][x];
    dw[c] = from_f32<W>(e);
  }
}

// ---- host side ----------------------------------------------------------------------------------
template <typename T, typename W, int V>
static cudaError_t forward_v(const NormArgs& a, void* y, cudaStream_t s) {
  constexpr int NU = V > 2 ? 2 : 8;
  const int64_t units = a.cols / V > 0 ? a.cols / V : 1;
  auto* out = static_cast<T*>(y);
  if (units > 1024 * NU)
    return launch_pdl(rms_norm_long_kernel<T, V == 2 ? 1 : V>, dim3((unsigned)a.rows), dim3(1024), 0, s, a, out);
  auto go = [&](auto* kern, int g, int block) {
    const int64_t need = (a.rows + block / g - 1) / (block / g);
    const unsigned grid =
        even_grid(stay_grid(reinterpret_cast<const void*>(kern), block, 0, need), need);
    return launch_pdl(kern, dim3(grid), dim3(block), 0, s, a, g, out);
  };
  // few rows: half as many units a thread, the shorter chain
  const int g = norm_threads<V>(units, a.rows <= 148 ? NU / 2 : NU, 8);
  const int block = g <= 32 ? 128 : g;
  if (block <= 256) return go(rms_norm_kernel<T, W, V, NU, 256>, g, block);
  return go(rms_norm_kernel<T, W, V, NU, 1024>, g, block);
}

template <typename T>
static cudaError_t forward_t(const NormArgs& a, void* y, cudaStream_t s) {
  return norm_dispatch<T>(a, norm_unit<T>(a, y), [&](auto w, auto v) {
    return forward_v<T, decltype(w), decltype(v)::value>(a, y, s);
  });
}

cudaError_t launch_rms_norm(const NormArgs& a, void* y, cudaStream_t s) {
  if (a.dtype == EXF_F32) return forward_t<float>(a, y, s);
  if (a.dtype == EXF_BF16) return forward_t<__nv_bfloat16>(a, y, s);
  return forward_t<__half>(a, y, s);
}

// The backward pass's blocks: few on an SM, so that their sums stay few; more where the blocks are small.
static int64_t backward_blocks(int cols) {
  return (cols <= 1024 ? 8 : 4) * (int64_t)(sm_count() > 0 ? sm_count() : 1);
}

int64_t norm_backward_workspace(int64_t rows, int cols) {
  const int64_t most = backward_blocks(cols);
  return (rows < most ? rows : most) * cols * (int64_t)sizeof(float);
}

template <typename T, typename W, int V>
static cudaError_t backward_v(const NormArgs& a, const void* dy, const void* ds, void* dx, void* dw,
                              float* part, cudaStream_t s) {
  constexpr int NU = V > 2 ? 2 : 8;
  const int64_t units = a.cols / V > 0 ? a.cols / V : 1;
  const int64_t sms = sm_count() > 0 ? sm_count() : 1;
  auto* up = static_cast<const T*>(dy);
  auto* side = static_cast<const T*>(ds);
  auto* out = static_cast<T*>(dx);
  float* sums = dw ? part : nullptr;
  unsigned blocks;
  cudaError_t e;
  if (units > 1024 * NU) {
    blocks = (unsigned)(a.rows < sms ? a.rows : sms);
    e = launch_pdl(rms_norm_backward_long_kernel<T, V == 2 ? 1 : V>, dim3(blocks), dim3(1024), 0, s, a, up, side,
                   out, sums);
  } else {
    const int g = norm_threads<V>(units, NU, 8);
    const int block = g <= 32 ? 128 : g;
    const int per_block = block / g;
    const size_t smem = per_block > 1 ? (size_t)per_block * a.cols * sizeof(float) : 0;
    const int64_t need = (a.rows + per_block - 1) / per_block;
    auto go = [&](auto* kern) {
      const int64_t most = backward_blocks(a.cols);
      blocks = stay_grid(reinterpret_cast<const void*>(kern), block, smem,
                         need < most ? need : most);
      blocks = even_grid(blocks, need);
      return launch_pdl(kern, dim3(blocks), dim3(block), smem, s, a, g, up, side, out, sums);
    };
    e = block <= 256   ? go(rms_norm_backward_kernel<T, W, V, NU, 256>)
        : block <= 512 ? go(rms_norm_backward_kernel<T, W, V, NU, 512>)
                       : go(rms_norm_backward_kernel<T, W, V, NU, 1024>);
  }
  if (e != cudaSuccess || !dw) return e;
  const dim3 grid((unsigned)((a.cols + 7) / 8));
  return launch_pdl(rms_norm_join_kernel<W>, grid, dim3(512), 0, s, static_cast<const float*>(part),
                    (int)blocks, a.cols, static_cast<W*>(dw));
}

template <typename T>
static cudaError_t backward_t(const NormArgs& a, const void* dy, const void* ds, void* dx, void* dw,
                              float* part, cudaStream_t s) {
  return norm_dispatch<T>(a, norm_unit<T>(a, dy, ds, dx), [&](auto w, auto v) {
    return backward_v<T, decltype(w), decltype(v)::value>(a, dy, ds, dx, dw, part, s);
  });
}

cudaError_t launch_rms_norm_backward(const NormArgs& a, const void* dy, const void* ds, void* dx,
                                     void* dw, void* workspace, cudaStream_t s) {
  float* part = static_cast<float*>(workspace);
  if (a.dtype == EXF_F32) return backward_t<float>(a, dy, ds, dx, dw, part, s);
  if (a.dtype == EXF_BF16) return backward_t<__nv_bfloat16>(a, dy, ds, dx, dw, part, s);
  return backward_t<__half>(a, dy, ds, dx, dw, part, s);
}

}  // namespace exf
