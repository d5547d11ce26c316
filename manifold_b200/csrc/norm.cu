// Layer norm over the last dimension and its backward pass (the readout's
// and the scan layers' nn.LayerNorm, gfn/model.py:113, gfn/layers/parallel.py:27):
//
//   mu = mean(x), rstd = (mean((x - mu)^2) + eps)^-1/2, xh = (x - mu) rstd
//   y  = xh w + b
//   g  = dy w,  dx = rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Statistics and sums are float32; the variance is taken about the mean in a
// second pass over the row, so a large common offset costs no accuracy.  The
// weight gradients are summed in a fixed order (per-block partial rows, then
// one pass over the blocks): no atomics, the same bits on every run.
#include "abi.h"
#include "lm_ops.cuh"

using namespace gfn;
using namespace gfn_abi;

namespace {

constexpr int NORM_THREADS = 256;

struct NormArgs {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  void* y;    // forward: y; backward: dx
  float2* stats;  // (mean, rstd) per row
  float* part;    // backward: [blocks][2][D] partial sums of dw, db
  void* dw;
  void* db;
  long long rows, xs, ds;  // row strides of x and dy, in elements
  int D, blocks;
  float eps;
};

// Sum over the block; `buf` is reused, so the leading barrier separates calls.
GFN_DEV float block_sum(float v, float* buf) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NORM_THREADS / 32; ++k) s += buf[k];
  return s;
}

template <typename T, typename W>
__global__ void __launch_bounds__(NORM_THREADS) norm_forward_kernel(const NormArgs p) {
  __shared__ float buf[NORM_THREADS / 32];
  const W* w = static_cast<const W*>(p.w);
  const W* b = static_cast<const W*>(p.b);
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.xs;
    T* y = static_cast<T*>(p.y) + r * p.D;
    float s = 0.f;
    for (int i = threadIdx.x; i < p.D; i += NORM_THREADS) s += to_f(x[i]);
    const float mu = block_sum(s, buf) / p.D;
    s = 0.f;
    for (int i = threadIdx.x; i < p.D; i += NORM_THREADS) {
      const float c = to_f(x[i]) - mu;
      s += c * c;
    }
    const float rstd = rsqrtf(block_sum(s, buf) / p.D + p.eps);
    for (int i = threadIdx.x; i < p.D; i += NORM_THREADS) {
      float v = (to_f(x[i]) - mu) * rstd;
      if (w) v *= to_f(w[i]);
      if (b) v += to_f(b[i]);
      y[i] = from_f<T>(v);
    }
    if (p.stats && threadIdx.x == 0) p.stats[r] = make_float2(mu, rstd);
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(NORM_THREADS) norm_dx_kernel(const NormArgs p) {
  __shared__ float buf[NORM_THREADS / 32];
  const W* w = static_cast<const W*>(p.w);
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.xs;
    const T* dy = static_cast<const T*>(p.dy) + r * p.ds;
    T* dx = static_cast<T*>(p.y) + r * p.D;
    const float2 st = p.stats[r];
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < p.D; i += NORM_THREADS) {
      const float g = to_f(dy[i]) * (w ? to_f(w[i]) : 1.f);
      s1 += g;
      s2 += g * ((to_f(x[i]) - st.x) * st.y);
    }
    const float m1 = block_sum(s1, buf) / p.D, m2 = block_sum(s2, buf) / p.D;
    for (int i = threadIdx.x; i < p.D; i += NORM_THREADS) {
      const float g = to_f(dy[i]) * (w ? to_f(w[i]) : 1.f);
      dx[i] = from_f<T>(st.y * (g - m1 - ((to_f(x[i]) - st.x) * st.y) * m2));
    }
  }
}

// Partial dw, db of one block's rows: thread per column.  grid (columns, blocks)
template <typename T>
__global__ void __launch_bounds__(NORM_THREADS) norm_dw_kernel(const NormArgs p) {
  const int i = blockIdx.x * NORM_THREADS + threadIdx.x;
  if (i >= p.D) return;
  float sw = 0.f, sb = 0.f;
  for (long long r = blockIdx.y; r < p.rows; r += p.blocks) {
    const float2 st = p.stats[r];
    const float d = to_f(static_cast<const T*>(p.dy)[r * p.ds + i]);
    sw += d * ((to_f(static_cast<const T*>(p.x)[r * p.xs + i]) - st.x) * st.y);
    sb += d;
  }
  p.part[(2LL * blockIdx.y) * p.D + i] = sw;
  p.part[(2LL * blockIdx.y + 1) * p.D + i] = sb;
}

template <typename W>
__global__ void __launch_bounds__(NORM_THREADS) norm_dw_sum_kernel(const NormArgs p) {
  const int i = blockIdx.x * NORM_THREADS + threadIdx.x;
  if (i >= p.D) return;
  float sw = 0.f, sb = 0.f;
  for (int k = 0; k < p.blocks; ++k) {
    sw += p.part[(2LL * k) * p.D + i];
    sb += p.part[(2LL * k + 1) * p.D + i];
  }
  if (p.dw) static_cast<W*>(p.dw)[i] = from_f<W>(sw);
  if (p.db) static_cast<W*>(p.db)[i] = from_f<W>(sb);
}

constexpr int NORM_MAX_BLOCKS = 296;

int norm_blocks(long long rows) { return (int)(rows < NORM_MAX_BLOCKS ? rows : NORM_MAX_BLOCKS); }

template <typename T, typename W>
int norm_run(const NormArgs& p, bool backward, cudaStream_t s) {
  const unsigned grid = (unsigned)(p.rows < (1 << 20) ? p.rows : (1 << 20));
  if (!backward) {
    norm_forward_kernel<T, W><<<grid, NORM_THREADS, 0, s>>>(p);
    return launch_status("norm_forward_kernel");
  }
  if (p.y) {
    norm_dx_kernel<T, W><<<grid, NORM_THREADS, 0, s>>>(p);
    const int st = launch_status("norm_dx_kernel");
    if (st) return st;
  }
  if (!p.dw && !p.db) return GFN_OK;
  const unsigned gc = (unsigned)((p.D + NORM_THREADS - 1) / NORM_THREADS);
  norm_dw_kernel<T><<<dim3(gc, p.blocks), NORM_THREADS, 0, s>>>(p);
  norm_dw_sum_kernel<W><<<gc, NORM_THREADS, 0, s>>>(p);
  return launch_status("norm_dw kernels");
}

// (element type, weight type): the weights are float32 or of the elements' type
int norm_dispatch(const NormArgs& p, int dtype, int wdtype, bool backward, cudaStream_t s) {
  if (dtype == GFN_F32 && wdtype == GFN_F32) return norm_run<float, float>(p, backward, s);
  if (dtype == GFN_BF16 && wdtype == GFN_F32) return norm_run<__nv_bfloat16, float>(p, backward, s);
  if (dtype == GFN_BF16 && wdtype == GFN_BF16) return norm_run<__nv_bfloat16, __nv_bfloat16>(p, backward, s);
  if (dtype == GFN_F16 && wdtype == GFN_F32) return norm_run<__half, float>(p, backward, s);
  if (dtype == GFN_F16 && wdtype == GFN_F16) return norm_run<__half, __half>(p, backward, s);
  return fail(GFN_ERR_UNSUPPORTED, "layer_norm: element type %d with weight type %d", dtype, wdtype);
}

size_t type_size(int dtype) { return dtype == GFN_F32 ? 4 : 2; }

}  // namespace

extern "C" {

int gfn_layer_norm_forward(const void* x, long long x_row_stride, const void* weight, const void* bias,
                           int dtype, int weight_dtype, long long rows, int dim, float eps, void* y,
                           float* stats, gfn_stream_t stream) {
  if (rows < 0 || dim <= 0 || (rows > 0 && (!x || !y)))
    return fail(GFN_ERR_INVALID, "layer_norm_forward: rows=%lld dim=%d or a NULL operand", rows, dim);
  if (x_row_stride < dim && rows > 1)
    return fail(GFN_ERR_INVALID, "layer_norm_forward: row stride %lld below dim %d", x_row_stride, dim);
  if (reinterpret_cast<uintptr_t>(stats) & 7u)
    return fail(GFN_ERR_ALIGN, "layer_norm_forward: stats must be 8-byte aligned");
  if (rows == 0) return GFN_OK;
  NormArgs p = {};
  p.x = x; p.w = weight; p.b = bias; p.y = y; p.stats = reinterpret_cast<float2*>(stats);
  p.rows = rows; p.xs = x_row_stride; p.D = dim; p.eps = eps;
  return norm_dispatch(p, dtype, weight_dtype, false, reinterpret_cast<cudaStream_t>(stream));
}

long long gfn_layer_norm_backward_workspace_floats(long long rows, int dim) {
  if (rows < 0 || dim <= 0) return -1;
  return 2LL * norm_blocks(rows) * dim;
}

int gfn_layer_norm_backward(const void* x, long long x_row_stride, const void* dy, long long dy_row_stride,
                            const void* weight, const float* stats, int dtype, int weight_dtype,
                            long long rows, int dim, void* dx, void* dweight, void* dbias, float* workspace,
                            long long workspace_floats, gfn_stream_t stream) {
  if (rows < 0 || dim <= 0 || (rows > 0 && (!x || !dy || !stats)))
    return fail(GFN_ERR_INVALID, "layer_norm_backward: rows=%lld dim=%d or a NULL operand", rows, dim);
  if ((x_row_stride < dim || dy_row_stride < dim) && rows > 1)
    return fail(GFN_ERR_INVALID, "layer_norm_backward: a row stride below dim %d", dim);
  if (reinterpret_cast<uintptr_t>(stats) & 7u)
    return fail(GFN_ERR_ALIGN, "layer_norm_backward: stats must be 8-byte aligned");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {  // sums over no rows
    const size_t n = (size_t)dim * type_size(weight_dtype);
    if (dweight) {
      cudaError_t e = cudaMemsetAsync(dweight, 0, n, s);
      if (e != cudaSuccess) return cuda_status(e, "layer_norm_backward: dweight");
    }
    if (dbias) {
      cudaError_t e = cudaMemsetAsync(dbias, 0, n, s);
      if (e != cudaSuccess) return cuda_status(e, "layer_norm_backward: dbias");
    }
    return GFN_OK;
  }
  if ((dweight || dbias) && (!workspace || workspace_floats < gfn_layer_norm_backward_workspace_floats(rows, dim)))
    return fail(GFN_ERR_INVALID, "layer_norm_backward: workspace of %lld floats, %lld needed", workspace_floats,
                gfn_layer_norm_backward_workspace_floats(rows, dim));
  NormArgs p = {};
  p.x = x; p.dy = dy; p.w = weight; p.y = dx; p.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  p.part = workspace; p.dw = dweight; p.db = dbias; p.rows = rows; p.xs = x_row_stride; p.ds = dy_row_stride;
  p.D = dim; p.blocks = norm_blocks(rows);
  return norm_dispatch(p, dtype, weight_dtype, true, s);
}

}  // extern "C"
