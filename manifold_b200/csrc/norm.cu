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
//
// Both passes are bound by HBM.  A row is held in registers by the threads
// that share it, 16 elements each, and read once.
#include "abi.h"
#include "lm_ops.cuh"
#include "umma.cuh"

using namespace gfn;
using namespace gfn_abi;

namespace {

constexpr int NORM_THREADS = 256;
constexpr int NORM_EPT = 16;  // elements per thread

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
  int wpr;          // warps that share a row
  int chunk_rows;   // backward: rows per stage
  int stages;
  long long bulk;   // chunks that arrive by bulk copies; the rest is read in place
};

// VEC neighbouring elements: one access of up to 16 bytes.
template <typename T, int VEC>
GFN_DEV void load_vec(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = to_f(*p);
  } else {
    static_assert(sizeof(T) * VEC == 16 || sizeof(T) * VEC == 32, "");
#pragma unroll
    for (int h = 0; h < (int)(sizeof(T) * VEC / 16); ++h) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[h];
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < (int)(16 / sizeof(T)); ++i) f[h * (16 / sizeof(T)) + i] = to_f(e[i]);
    }
  }
}

template <typename T, int VEC>
GFN_DEV void store_vec(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f<T>(f[0]);
  } else {
    static_assert(sizeof(T) * VEC == 16, "");
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f<T>(f[i]);
    __stcs(reinterpret_cast<uint4*>(p), u);
  }
}

GFN_DEV void group_barrier(int group, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
}

// Sums over the warps that share a row.  `buf` [2][warps of the block], used in
// turn: a warp is at most one sum ahead of its group.
template <int N>
GFN_DEV void row_sum(float (&v)[N], float* buf, int warps, int wpr, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (wpr == 1) return;
  const int w = threadIdx.x >> 5, g = w / wpr;
  float* b = buf + turn * warps * N;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) b[w * N + i] = v[i];
  }
  group_barrier(g, wpr * 32);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int k = 0; k < wpr; ++k) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += b[(g * wpr + k) * N + i];
  }
}

// wpr warps per row, one row per group; blocks of max(256, 32 wpr) threads.
template <typename T, typename W, int VEC>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const NormArgs p) {
  constexpr int NV = NORM_EPT / VEC;
  __shared__ float buf[2 * 32];
  const int tpr = p.wpr * 32, warps = blockDim.x >> 5;
  const long long row = (long long)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  if (row >= p.rows) return;  // a whole group: its barriers are its own
  const int l = threadIdx.x % tpr, D = p.D;
  const T* x = static_cast<const T*>(p.x) + row * p.xs;
  float v[NV][VEC];
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * tpr + l) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
    if (e < D) load_vec<T, VEC>(x + e, v[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[0] += v[i][j];
  }
  int turn = 0;
  row_sum<1>(s, buf, warps, p.wpr, turn);
  const float mu = s[0] / D;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * tpr + l) * VEC < D) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] -= mu;
        s[0] = fmaf(v[i][j], v[i][j], s[0]);
      }
    }
  }
  row_sum<1>(s, buf, warps, p.wpr, turn);
  const float rstd = rsqrtf(s[0] / D + p.eps);
  T* y = static_cast<T*>(p.y) + row * D;
  const W* w = static_cast<const W*>(p.w);
  const W* b = static_cast<const W*>(p.b);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * tpr + l) * VEC;
    if (e < D) {
      float wv[VEC], bv[VEC];
      if (w) load_vec<W, VEC>(w + e, wv);
      if (b) load_vec<W, VEC>(b + e, bv);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] *= rstd;
        if (w) v[i][j] *= wv[j];
        if (b) v[i][j] += bv[j];
      }
      store_vec<T, VEC>(y + e, v[i]);
    }
  }
  if (p.stats && l == 0) p.stats[row] = make_float2(mu, rstd);
}

// NW warps compute, one more fetches: chunks of rows travel through a ring of
// stages by bulk copies (a whole number of 16 bytes per chunk, whatever the
// row length), so loads are in flight while rows are computed, at no cost in
// registers.  dx is written from registers; dw and db of all the block's rows
// stay there and leave once, as one partial row per block.
template <typename T, typename W, int VEC, int NW>
__global__ void __launch_bounds__((NW + 1) * 32, NW == 8 ? 2 : 1) norm_backward_kernel(const NormArgs p) {
  constexpr int NV = NORM_EPT / VEC;
  extern __shared__ __align__(128) char ring[];
  __shared__ uint64_t full[4], empty[4];
  __shared__ float buf[2 * NW * 2];
  const int warp = threadIdx.x >> 5, D = p.D;
  const long long chunks = (p.rows + p.chunk_rows - 1) / p.chunk_rows;
  const int bytes = p.chunk_rows * D * (int)sizeof(T);  // of one operand's chunk
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NW);
    }
    fence_mbar_init();
  }
  __syncthreads();
  if (warp == NW) {
    if ((threadIdx.x & 31) == 0) {
      int it = 0;
      for (long long c = blockIdx.x; c < p.bulk; c += gridDim.x, ++it) {
        const int st = it % p.stages;
        if (it >= p.stages) mbar_wait(&empty[st], (it / p.stages - 1) & 1);
        char* dst = ring + (size_t)st * 2 * bytes;
        const long long first = c * p.chunk_rows * (long long)D;
        mbar_arrive_expect_tx(&full[st], 2 * bytes);
        bulk_g2s(dst, static_cast<const T*>(p.x) + first, bytes, &full[st]);
        bulk_g2s(dst + bytes, static_cast<const T*>(p.dy) + first, bytes, &full[st]);
      }
    }
    __syncwarp();
    __syncthreads();  // the one before the partial sums
    __syncthreads();
    return;
  }
  const int tpr = p.wpr * 32, group = warp / p.wpr, groups = NW / p.wpr, l = threadIdx.x % tpr;
  const W* w = static_cast<const W*>(p.w);
  float wv[NV][VEC], aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * tpr + l) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      wv[i][j] = 1.f;
      aw[i][j] = ab[i][j] = 0.f;
    }
    if (w && e < D) load_vec<W, VEC>(w + e, wv[i]);
  }
  int it = 0, turn = 0;
  float2 next = make_float2(0.f, 0.f);  // statistics of this group's next row, fetched ahead
  {
    const long long row = (long long)blockIdx.x * p.chunk_rows + group;
    if (row < p.rows) next = p.stats[row];
  }
  for (long long c = blockIdx.x; c < chunks; c += gridDim.x, ++it) {
    const int st = it % p.stages;
    const bool bulk = c < p.bulk;
    const long long first = c * p.chunk_rows;
    const int rows = (int)min((long long)p.chunk_rows, p.rows - first);
    const T* cx = reinterpret_cast<const T*>(ring + (size_t)st * 2 * bytes);
    const T* cd = reinterpret_cast<const T*>(ring + (size_t)st * 2 * bytes + bytes);
    if (bulk) mbar_wait(&full[st], (it / p.stages) & 1);
    for (int r = group; r < rows; r += groups) {
      const long long row = first + r;
      const T* x = bulk ? cx + r * D : static_cast<const T*>(p.x) + row * p.xs;
      const T* dy = bulk ? cd + r * D : static_cast<const T*>(p.dy) + row * p.ds;
      const float2 stat = next;
      {
        const long long ahead = r + groups < rows ? row + groups : first + (long long)gridDim.x * p.chunk_rows + group;
        if (ahead < p.rows) next = p.stats[ahead];
      }
      float xh[NV][VEC], g[NV][VEC];
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (i * tpr + l) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xh[i][j] = stat.x;
          g[i][j] = 0.f;
        }
        if (e < D) {
          load_vec<T, VEC>(x + e, xh[i]);
          load_vec<T, VEC>(dy + e, g[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xh[i][j] = (xh[i][j] - stat.x) * stat.y;
          aw[i][j] = fmaf(g[i][j], xh[i][j], aw[i][j]);
          ab[i][j] += g[i][j];
          g[i][j] *= wv[i][j];
          s[0] += g[i][j];
          s[1] = fmaf(g[i][j], xh[i][j], s[1]);
        }
      }
      row_sum<2>(s, buf, NW, p.wpr, turn);
      const float m1 = s[0] / D, m2 = s[1] / D;
      if (p.y) {
        T* dx = static_cast<T*>(p.y) + row * D;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e = (i * tpr + l) * VEC;
#pragma unroll
          for (int j = 0; j < VEC; ++j) g[i][j] = stat.y * (g[i][j] - m1 - xh[i][j] * m2);
          if (e < D) store_vec<T, VEC>(dx + e, g[i]);
        }
      }
    }
    if (bulk) {
      __syncwarp();
      if ((threadIdx.x & 31) == 0) umma::mbar_arrive(&empty[st]);
    }
  }
  // dw, db: the groups' sums meet in shared memory (the ring is free: every
  // copy has landed and been read), in the order of the groups
  __syncthreads();
  if (!p.part) {
    __syncthreads();
    return;
  }
  float* sums = reinterpret_cast<float*>(ring);  // [groups][2][tpr * NORM_EPT]
  const int width = tpr * NORM_EPT;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int e = (i * tpr + l) * VEC + j;
      sums[(group * 2) * width + e] = aw[i][j];
      sums[(group * 2 + 1) * width + e] = ab[i][j];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * D; e += NW * 32) {
    const int k = e >= D, col = e - k * D;
    float t = 0.f;
    for (int g = 0; g < groups; ++g) t += sums[(g * 2 + k) * width + col];
    p.part[((long long)blockIdx.x * 2 + k) * D + col] = t;
  }
}

// Rows beyond the registers' reach: the row is read from memory (mostly L2)
// once per pass over it.
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
__global__ void __launch_bounds__(NORM_THREADS) norm_forward_long_kernel(const NormArgs p) {
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
__global__ void __launch_bounds__(NORM_THREADS) norm_dx_long_kernel(const NormArgs p) {
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
__global__ void __launch_bounds__(NORM_THREADS) norm_dw_long_kernel(const NormArgs p) {
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

// The blocks' partial rows, in order: 32 columns x 8 slices of the blocks.
// grid (columns / 32, dw or db)
template <typename W>
__global__ void __launch_bounds__(NORM_THREADS) norm_dw_sum_kernel(const NormArgs p) {
  __shared__ float buf[8][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, k = blockIdx.y;
  const int per = (p.blocks + 7) / 8, b1 = min(p.blocks, (slice + 1) * per);
  float s = 0.f;
  if (col < p.D) {
#pragma unroll 8
    for (int b = slice * per; b < b1; ++b) s += p.part[((long long)b * 2 + k) * p.D + col];
  }
  buf[slice][lane] = s;
  __syncthreads();
  W* out = static_cast<W*>(k ? p.db : p.dw);
  if (slice == 0 && col < p.D && out) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += buf[i][lane];
    out[col] = from_f<W>(s);
  }
}

constexpr int NORM_MAX_BLOCKS = 296;
constexpr int NORM_SMEM = 100 * 1024;  // ring per block: two blocks per SM

int norm_blocks(long long rows) { return (int)(rows < NORM_MAX_BLOCKS ? rows : NORM_MAX_BLOCKS); }

// Warps per row: the smallest power of two whose registers hold the row.
int warps_per_row(int D) {
  int w = 1;
  while (w * 32 * NORM_EPT < D) w *= 2;
  return w;
}

template <typename T, typename W, int VEC, int NW>
int norm_backward_run(NormArgs p, cudaStream_t s) {
  const int groups = NW / p.wpr, row = p.D * (int)sizeof(T);
  int unit = 1;  // rows that make whole 16-byte pieces
  while ((long long)unit * row % 16) unit *= 2;
  int rows = groups > unit ? groups : unit;
  while (rows * row <= 4096 && p.rows / (2 * rows) >= NORM_MAX_BLOCKS) rows *= 2;  // short rows: longer copies
  const size_t sums = (size_t)NW * 32 * NORM_EPT * 2 * 4;
  const bool bulk = (reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.dy)) % 16 == 0 &&
                    (p.rows == 1 || (p.xs == p.D && p.ds == p.D)) && (size_t)rows * row * 4 <= NORM_SMEM;
  if (!bulk) rows = groups;
  p.chunk_rows = rows;
  p.stages = bulk ? (int)(NORM_SMEM / ((size_t)rows * row * 2)) : 1;
  if (p.stages > 4) p.stages = 4;
  p.bulk = bulk ? p.rows / rows : 0;
  const long long chunks = (p.rows + rows - 1) / rows;
  const int most = NW == 8 ? NORM_MAX_BLOCKS : NORM_MAX_BLOCKS / 2;
  p.blocks = (int)(chunks < most ? chunks : most);
  if (!p.dw && !p.db) p.part = nullptr;
  size_t smem = bulk ? (size_t)p.stages * rows * row * 2 : 0;
  if (smem < sums) smem = sums;
  cudaError_t e = cudaFuncSetAttribute(norm_backward_kernel<T, W, VEC, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem);
  if (e != cudaSuccess) return cuda_status(e, "norm_backward_kernel: shared memory");
  norm_backward_kernel<T, W, VEC, NW><<<p.blocks, (NW + 1) * 32, smem, s>>>(p);
  if (p.part) norm_dw_sum_kernel<W><<<dim3((p.D + 31) / 32, 2), NORM_THREADS, 0, s>>>(p);
  return launch_status("norm_backward_kernel");
}

template <typename T, typename W, int VEC>
int norm_short_run(const NormArgs& p, bool backward, cudaStream_t s) {
  if (backward) return p.wpr <= 8 ? norm_backward_run<T, W, VEC, 8>(p, s) : norm_backward_run<T, W, VEC, 16>(p, s);
  const int threads = p.wpr * 32 > 256 ? p.wpr * 32 : 256, per = threads / (p.wpr * 32);
  const long long blocks = (p.rows + per - 1) / per;
  if (blocks > 0x7fffffffLL) return fail(GFN_ERR_UNSUPPORTED, "layer_norm_forward: %lld blocks", blocks);
  norm_forward_kernel<T, W, VEC><<<(unsigned)blocks, threads, 0, s>>>(p);
  return launch_status("norm_forward_kernel");
}

template <typename T, typename W>
int norm_run(NormArgs p, bool backward, cudaStream_t s) {
  p.wpr = warps_per_row(p.D);
  if (p.wpr <= (backward ? 16 : 32)) {
    constexpr int VEC = 16 / sizeof(T);
    const uintptr_t ends = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.dy) |
                           reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.w) |
                           reinterpret_cast<uintptr_t>(p.b);
    const bool vec = p.D % VEC == 0 && ends % 16 == 0 && (p.rows == 1 || (p.xs % VEC == 0 && p.ds % VEC == 0));
    return vec ? norm_short_run<T, W, VEC>(p, backward, s) : norm_short_run<T, W, 1>(p, backward, s);
  }
  const unsigned grid = (unsigned)(p.rows < (1 << 20) ? p.rows : (1 << 20));
  if (!backward) {
    norm_forward_long_kernel<T, W><<<grid, NORM_THREADS, 0, s>>>(p);
    return launch_status("norm_forward_long_kernel");
  }
  if (p.y) {
    norm_dx_long_kernel<T, W><<<grid, NORM_THREADS, 0, s>>>(p);
    const int st = launch_status("norm_dx_long_kernel");
    if (st) return st;
  }
  if (!p.dw && !p.db) return GFN_OK;
  p.blocks = norm_blocks(p.rows);
  norm_dw_long_kernel<T><<<dim3((p.D + NORM_THREADS - 1) / NORM_THREADS, p.blocks), NORM_THREADS, 0, s>>>(p);
  norm_dw_sum_kernel<W><<<dim3((p.D + 31) / 32, 2), NORM_THREADS, 0, s>>>(p);
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
  p.D = dim;
  return norm_dispatch(p, dtype, weight_dtype, true, s);
}

}  // extern "C"
