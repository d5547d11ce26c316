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
// Both passes are bound by HBM.  A row is held in registers by the WPR warps
// that share it (64 bytes a thread forward, 16 elements backward) and read
// once.
#include "lm_host.h"
#include "lm_ops.cuh"
#include "umma.cuh"

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
  int w32;          // weights are float32 (else of the elements' type)
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

// w[e .. e + VEC) as float32, whichever type it has
template <typename T, int VEC>
GFN_DEV void load_weight(const void* w, int w32, int e, float (&f)[VEC]) {
  if (sizeof(T) == 4 || w32) load_vec<float, VEC>(static_cast<const float*>(w) + e, f);
  else load_vec<T, VEC>(static_cast<const T*>(w) + e, f);
}

// Sums over the WPR warps that share a row (named barrier per group).  `buf`
// holds two sets of sums, used in turn: a warp is at most one sum ahead.
template <int N, int WPR>
GFN_DEV void row_sum(float (&v)[N], float* buf, int warps, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if constexpr (WPR > 1) {
    const int w = threadIdx.x >> 5, g = w / WPR;
    float* b = buf + turn * warps * N;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) b[w * N + i] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(g + 1), "n"(WPR * 32) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int k = 0; k < WPR; ++k) v[i] += b[(g * WPR + k) * N + i];
    }
  }
}

constexpr int norm_forward_threads(int wpr) { return wpr * 32 > NORM_THREADS ? wpr * 32 : NORM_THREADS; }

// WPR warps per row, one row per group of warps.  One pass over x: 49 us at
// 65536 x 512 float32 (5.5 TB/s with the launch), 22 us at 20480 x 1024
// bfloat16, where converting and reducing 16-bit values takes about as long as
// the memory.
template <typename T, int VEC, int WPR, int EPT>
__global__ void __launch_bounds__(norm_forward_threads(WPR), VEC == 1 ? 1 : 1024 / norm_forward_threads(WPR)) norm_forward_kernel(const NormArgs p) {
  constexpr int TPR = WPR * 32, NV = EPT / VEC, THREADS = norm_forward_threads(WPR);
  __shared__ float buf[2 * THREADS / 32];
  const long long row = (long long)blockIdx.x * (THREADS / TPR) + threadIdx.x / TPR;
  if (row >= p.rows) return;  // a whole group: its barriers are its own
  const int l = threadIdx.x % TPR, D = p.D;
  const T* x = static_cast<const T*>(p.x) + row * p.xs;
  float v[NV][VEC];
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * TPR + l) * VEC;
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
  row_sum<1, WPR>(s, buf, THREADS / 32, turn);
  const float mu = s[0] / D;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * TPR + l) * VEC < D) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] -= mu;
        s[0] = fmaf(v[i][j], v[i][j], s[0]);
      }
    }
  }
  row_sum<1, WPR>(s, buf, THREADS / 32, turn);
  const float rstd = rsqrtf(s[0] / D + p.eps);
  T* y = static_cast<T*>(p.y) + row * D;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * TPR + l) * VEC;
    if (e < D) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] *= rstd;
      float c[VEC];
      if (p.w) {
        load_weight<T, VEC>(p.w, p.w32, e, c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] *= c[j];
      }
      if (p.b) {
        load_weight<T, VEC>(p.b, p.w32, e, c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] += c[j];
      }
      store_vec<T, VEC>(y + e, v[i]);
    }
  }
  if (p.stats && l == 0) p.stats[row] = make_float2(mu, rstd);
}

// Chunks of rows travel through a ring of stages by bulk copies (a whole number
// of 16 bytes per chunk, whatever the row length), so loads are in flight while
// rows are computed, at no cost in registers; one thread refills the stage that
// was read a chunk ago.  N operands with contiguous rows; blocks take chunks
// in turn; work(rows of operand 0, chunk) is called by every warp.
template <typename T, int N, int NW>
struct RowRing {
  uint64_t full[4], empty[4];

  template <class Work>
  GFN_DEV void run(const NormArgs& p, char* ring, const T* const (&src)[N], Work work) {
    const int bytes = p.chunk_rows * p.D * (int)sizeof(T);  // of one operand's chunk
    if (threadIdx.x == 0) {
      for (int i = 0; i < p.stages; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], NW);
      }
      fence_mbar_init();
    }
    __syncthreads();
    auto refill = [&](long long c, int st) {
      mbar_arrive_expect_tx(&full[st], N * bytes);
#pragma unroll
      for (int k = 0; k < N; ++k)
        bulk_g2s(ring + (size_t)(st * N + k) * bytes, src[k] + c * p.chunk_rows * (long long)p.D, bytes, &full[st]);
    };
    if (threadIdx.x == 0) {
      for (int i = 0; i < p.stages; ++i) {
        const long long c = blockIdx.x + (long long)i * gridDim.x;
        if (c < p.bulk) refill(c, i);
      }
    }
    int st = 0, phase = 0;
    for (long long c = blockIdx.x; c < p.bulk; c += gridDim.x) {
      if (threadIdx.x == 0 && c != blockIdx.x) {  // the stage of a chunk ago, once all warps have read it
        const long long ahead = c + (long long)(p.stages - 1) * gridDim.x;
        const int was = st ? st - 1 : p.stages - 1;
        if (ahead < p.bulk) {
          mbar_wait(&empty[was], st ? phase : phase ^ 1);
          refill(ahead, was);
        }
      }
      __syncwarp();
      mbar_wait(&full[st], phase);
      work(reinterpret_cast<const T*>(ring + (size_t)st * N * bytes), c);
      __syncwarp();
      if ((threadIdx.x & 31) == 0) umma::mbar_arrive(&empty[st]);
      if (++st == p.stages) {
        st = 0;
        phase ^= 1;
      }
    }
  }
};

// The forward over many contiguous rows that do not start on 16 bytes: single
// elements come from shared memory, and the weights stay in registers.  (From
// 128-bit rows the direct kernel is as fast: 49 against 51 us at 65536 x 512
// float32; here 39 against 70 us at 20011 x 1001 bfloat16.)
template <typename T, int WPR, int EPT>
__global__ void __launch_bounds__(256, 3) norm_forward_ring_kernel(const NormArgs p) {
  constexpr int VEC = 1, NW = 8, TPR = WPR * 32, GROUPS = NW / WPR, NV = EPT / VEC;
  extern __shared__ __align__(128) char ring[];
  __shared__ RowRing<T, 1, NW> rows;
  __shared__ float buf[2 * NW];
  const int D = p.D, group = (threadIdx.x >> 5) / WPR, l = threadIdx.x % TPR;
  float wv[NV][VEC], bv[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * TPR + l) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      wv[i][j] = 1.f;
      bv[i][j] = 0.f;
    }
    if (p.w && e < D) load_weight<T, VEC>(p.w, p.w32, e, wv[i]);
    if (p.b && e < D) load_weight<T, VEC>(p.b, p.w32, e, bv[i]);
  }
  int turn = 0;
  auto one = [&](const T* x, long long row) {
    float v[NV][VEC], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * TPR + l) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
      if (e < D) load_vec<T, VEC>(x + e, v[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += v[i][j];
    }
    row_sum<1, WPR>(s, buf, NW, turn);
    const float mu = s[0] / D;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * TPR + l) * VEC < D) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[i][j] -= mu;
          s[0] = fmaf(v[i][j], v[i][j], s[0]);
        }
      }
    }
    row_sum<1, WPR>(s, buf, NW, turn);
    const float rstd = rsqrtf(s[0] / D + p.eps);
    T* y = static_cast<T*>(p.y) + row * D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * TPR + l) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] *= rstd;  // rounded before the weight, as in norm_forward_kernel
        v[i][j] = p.b ? __fadd_rn(__fmul_rn(v[i][j], wv[i][j]), bv[i][j]) : v[i][j] * wv[i][j];
      }
      if (e < D) store_vec<T, VEC>(y + e, v[i]);
    }
    if (p.stats && l == 0) p.stats[row] = make_float2(mu, rstd);
  };
  const T* const src[1] = {static_cast<const T*>(p.x)};
  rows.run(p, ring, src, [&](const T* x, long long c) {
    for (int r = group; r < p.chunk_rows; r += GROUPS) one(x + r * D, c * p.chunk_rows + r);
  });
  for (long long row = p.bulk * p.chunk_rows + (long long)blockIdx.x * GROUPS + group; row < p.rows;
       row += (long long)gridDim.x * GROUPS)  // what is left of a chunk
    one(static_cast<const T*>(p.x) + row * D, row);
}

// dx is written from registers; dw and db of all the block's rows stay there
// and leave once, as one partial row per block.  One pass over x and dy: 76 us
// at 65536 x 512 float32, the sums of the partial rows included (5.3 TB/s);
// 39 us at 20011 x 1001 bfloat16, bound there by single-element accesses.  A
// pass of its own for dw and db took 2.6 times as long.
template <typename T, int VEC, int WPR, int EPT_>
struct NormBackward {
  static constexpr int NW = WPR > 8 ? WPR : 8, TPR = WPR * 32, GROUPS = NW / WPR, EPT = EPT_, NV = EPT / VEC;
  float wv[NV][VEC], aw[NV][VEC], ab[NV][VEC];
  int l, turn = 0;

  GFN_DEV void row(const NormArgs& p, const T* x, const T* dy, T* dx, float2 stat, float* buf) {
    const int D = p.D;
    float xh[NV][VEC], g[NV][VEC];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * TPR + l) * VEC;
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
    row_sum<2, WPR>(s, buf, NW, turn);
    if (dx) {
      const float m1 = s[0] / D, m2 = s[1] / D;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (i * TPR + l) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[i][j] = stat.y * (g[i][j] - m1 - xh[i][j] * m2);
        if (e < D) store_vec<T, VEC>(dx + e, g[i]);
      }
    }
  }
};

template <typename T, int VEC, int WPR, int EPT_>
__global__ void __launch_bounds__(NormBackward<T, VEC, WPR, EPT_>::NW * 32, WPR > 8 ? 1 : 2)
    norm_backward_kernel(const NormArgs p) {
  using Work = NormBackward<T, VEC, WPR, EPT_>;
  constexpr int NW = Work::NW, TPR = Work::TPR, GROUPS = Work::GROUPS, NV = Work::NV, EPT = Work::EPT;
  extern __shared__ __align__(128) char ring[];
  __shared__ RowRing<T, 2, NW> ops;
  __shared__ float buf[2 * NW * 2];
  const int warp = threadIdx.x >> 5, D = p.D, group = warp / WPR;
  Work k;
  k.l = threadIdx.x % TPR;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * TPR + k.l) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      k.wv[i][j] = 1.f;
      k.aw[i][j] = k.ab[i][j] = 0.f;
    }
    if (p.w && e < D) load_weight<T, VEC>(p.w, p.w32, e, k.wv[i]);
  }
  T* dx = static_cast<T*>(p.y);
  float2 next = make_float2(0.f, 0.f);  // statistics of this group's next row, fetched ahead
  const long long stride = (long long)gridDim.x * p.chunk_rows;
  {
    const long long row = (long long)blockIdx.x * p.chunk_rows + group;
    if (row < p.rows) next = p.stats[row];
  }
  const T* const src[2] = {static_cast<const T*>(p.x), static_cast<const T*>(p.dy)};
  ops.run(p, ring, src, [&](const T* cx, long long c) {
    const T* cd = cx + p.chunk_rows * D;
    const long long first = c * p.chunk_rows;
    for (int r = group; r < p.chunk_rows; r += GROUPS) {
      const float2 stat = next;
      const long long ahead = r + GROUPS < p.chunk_rows ? first + r + GROUPS : first + stride + group;
      if (ahead < p.rows) next = p.stats[ahead];
      k.row(p, cx + r * D, cd + r * D, dx ? dx + (first + r) * D : nullptr, stat, buf);
    }
  });
  long long c = blockIdx.x;
  if (c < p.bulk) c += (p.bulk - c + gridDim.x - 1) / gridDim.x * gridDim.x;
  for (; c * p.chunk_rows < p.rows; c += gridDim.x) {  // rows read in place
    const long long first = c * p.chunk_rows;
    const int rows = (int)min((long long)p.chunk_rows, p.rows - first);
    for (int r = group; r < rows; r += GROUPS) {
      const long long row = first + r;
      k.row(p, static_cast<const T*>(p.x) + row * p.xs, static_cast<const T*>(p.dy) + row * p.ds,
            dx ? dx + row * D : nullptr, p.stats[row], buf);
    }
  }
  if (!p.part) return;
  // dw, db: the groups' sums meet in shared memory (the ring is free: every
  // copy has landed and been read), in the order of the groups
  __syncthreads();
  float* sums = reinterpret_cast<float*>(ring);  // [GROUPS][2][TPR * EPT]
  constexpr int WIDTH = TPR * EPT;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int e = (i * TPR + k.l) * VEC + j;
      sums[(group * 2) * WIDTH + e] = k.aw[i][j];
      sums[(group * 2 + 1) * WIDTH + e] = k.ab[i][j];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * D; e += NW * 32) {
    const int which = e >= D, col = e - which * D;
    float t = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) t += sums[(g * 2 + which) * WIDTH + col];
    p.part[((long long)blockIdx.x * 2 + which) * D + col] = t;
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

// The blocks' partial rows, in order: 32 columns x 32 slices of the blocks.
// grid (columns / 32, dw or db)
template <typename W>
__global__ void __launch_bounds__(1024) norm_dw_sum_kernel(const NormArgs p) {
  constexpr int PER = 10;  // partial rows per slice, all in flight; 32 PER >= NORM_MAX_BLOCKS
  __shared__ float buf[32][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, k = blockIdx.y;
  float v[PER], s = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = slice * PER + i;
    v[i] = b < p.blocks && col < p.D ? p.part[((long long)b * 2 + k) * p.D + col] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) s += v[i];
  buf[lane][slice] = s;
  __syncthreads();
  s = warp_sum(buf[slice][lane]);  // warp `slice` sums column `slice` of the tile
  W* out = static_cast<W*>(k ? p.db : p.dw);
  const int c = blockIdx.x * 32 + slice;
  if (lane == 0 && c < p.D && out) out[c] = from_f<W>(s);
}

constexpr int NORM_MAX_BLOCKS = 296;
constexpr int NORM_SMEM = 100 * 1024;  // ring per block: two blocks per SM
constexpr int RING_SMEM = 64 * 1024;   // forward: three blocks per SM
constexpr int RING_ROWS = 4096;        // rows from which the forward streams through the ring

int norm_blocks(long long rows) { return (int)(rows < NORM_MAX_BLOCKS ? rows : NORM_MAX_BLOCKS); }

template <typename W>
void norm_dw_sum(const NormArgs& p, cudaStream_t s) {
  norm_dw_sum_kernel<W><<<dim3((p.D + 31) / 32, 2), 1024, 0, s>>>(p);
}

// How the rows of `operands` contiguous operands travel through the ring; false
// where they do not (rows apart, odd addresses, rows too long for two stages).
bool plan_ring(NormArgs* p, int groups, int operands, int row, int smem, bool whole) {
  int unit = 1;  // rows that make whole 16-byte pieces
  while ((long long)unit * row % 16) unit *= 2;
  int rows = groups > unit ? groups : unit;
  while (rows * row <= 4096 && p->rows / (2 * rows) >= NORM_MAX_BLOCKS) rows *= 2;  // short rows: longer copies
  if (!whole || (size_t)rows * row * 2 * operands > (size_t)smem) return false;
  p->chunk_rows = rows;
  p->stages = (int)(smem / ((size_t)rows * row * operands));
  if (p->stages > 4) p->stages = 4;
  p->bulk = p->rows / rows;
  return true;
}

template <typename T, int VEC, int WPR, int EPT>
int norm_backward_run(NormArgs p, cudaStream_t s) {
  using Work = NormBackward<T, VEC, WPR, EPT>;
  const int row = p.D * (int)sizeof(T);
  const size_t sums = (size_t)Work::NW * 32 * Work::EPT * 2 * 4;
  const bool whole = (reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.dy)) % 16 == 0 &&
                     (p.rows == 1 || (p.xs == p.D && p.ds == p.D));
  const bool bulk = plan_ring(&p, Work::GROUPS, 2, row, NORM_SMEM, whole);
  if (!bulk) {
    p.chunk_rows = Work::GROUPS;
    p.bulk = 0;
  }
  const int rows = p.chunk_rows;
  const long long chunks = (p.rows + rows - 1) / rows;
  const int most = WPR > 8 ? NORM_MAX_BLOCKS / 2 : NORM_MAX_BLOCKS;
  p.blocks = (int)(chunks < most ? chunks : most);
  if (!p.dw && !p.db) p.part = nullptr;
  size_t smem = bulk ? (size_t)p.stages * rows * row * 2 : 0;
  if (smem < sums) smem = sums;
  static std::atomic<unsigned long long> done{0};
  const int st = shared_limit(norm_backward_kernel<T, VEC, WPR, EPT>, NORM_SMEM, &done, "norm_backward_kernel: shared memory");
  if (st) return st;
  norm_backward_kernel<T, VEC, WPR, EPT><<<p.blocks, Work::NW * 32, smem, s>>>(p);
  if (p.part) {
    if (p.w32) norm_dw_sum<float>(p, s);
    else norm_dw_sum<T>(p, s);
  }
  return launch_status("norm_backward_kernel");
}

template <typename T, int VEC, int WPR, int EPT>
int norm_forward_run(const NormArgs& p, cudaStream_t s) {
  constexpr int threads = norm_forward_threads(WPR), per = threads / (WPR * 32);
  const long long blocks = (p.rows + per - 1) / per;
  if (blocks > 0x7fffffffLL) return fail(GFN_ERR_UNSUPPORTED, "layer_norm_forward: %lld blocks", blocks);
  norm_forward_kernel<T, VEC, WPR, EPT><<<(unsigned)blocks, threads, 0, s>>>(p);
  return launch_status("norm_forward_kernel");
}

template <typename T, int WPR, int EPT>
int norm_forward_ring_run(const NormArgs& p, cudaStream_t s) {
  const int smem = (int)((size_t)p.stages * p.chunk_rows * p.D * sizeof(T));
  static std::atomic<unsigned long long> done{0};
  const int st = shared_limit(norm_forward_ring_kernel<T, WPR, EPT>, RING_SMEM, &done,
                              "norm_forward_ring_kernel: shared memory");
  if (st) return st;
  const long long most = NORM_MAX_BLOCKS * 3 / 2;
  norm_forward_ring_kernel<T, WPR, EPT><<<(unsigned)(p.bulk < most ? p.bulk : most), 256, smem, s>>>(p);
  return launch_status("norm_forward_ring_kernel");
}

// Elements per thread in the forward: 64 bytes of vectors, or 16 single
// elements; half of that where it holds the row in one warp (bfloat16 65536 x
// 512: 35 against 41 us).
template <typename T, int VEC>
constexpr int norm_forward_ept() {
  return VEC == 1 ? 16 : 64 / (int)sizeof(T);
}

// The fewest warps whose registers hold a row.
template <typename T, int VEC>
int norm_short_run(const NormArgs& p, bool backward, cudaStream_t s) {
  if (backward) {
    if constexpr (VEC <= 4) {
      if (p.D <= 128) return norm_backward_run<T, VEC, 1, 4>(p, s);
    }
    if (p.D <= 256) return norm_backward_run<T, VEC, 1, 8>(p, s);
    if (p.D <= 512) return norm_backward_run<T, VEC, 1, 16>(p, s);
    if (p.D <= 1024) return norm_backward_run<T, VEC, 2, 16>(p, s);
    if (p.D <= 2048) return norm_backward_run<T, VEC, 4, 16>(p, s);
    if (p.D <= 4096) return norm_backward_run<T, VEC, 8, 16>(p, s);
    return norm_backward_run<T, VEC, 16, 16>(p, s);
  }
  if constexpr (VEC == 1) {
    NormArgs q = p;
    const bool whole = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.xs == p.D;
    const int groups = p.D <= 512 ? 8 : p.D <= 1024 ? 4 : p.D <= 2048 ? 2 : 1;
    if (p.D <= 4096 && p.rows >= RING_ROWS && plan_ring(&q, groups, 1, p.D * (int)sizeof(T), RING_SMEM, whole)) {
      if (p.D <= 128) return norm_forward_ring_run<T, 1, 4>(q, s);
      if (groups == 8) return norm_forward_ring_run<T, 1, 16>(q, s);
      if (groups == 4) return norm_forward_ring_run<T, 2, 16>(q, s);
      if (groups == 2) return norm_forward_ring_run<T, 4, 16>(q, s);
      return norm_forward_ring_run<T, 8, 16>(q, s);
    }
  }
  constexpr int EPT = norm_forward_ept<T, VEC>(), warp = 32 * EPT;  // elements that one warp holds
  if (p.D <= warp / 2) return norm_forward_run<T, VEC, 1, EPT / 2>(p, s);
  if (p.D <= warp) return norm_forward_run<T, VEC, 1, EPT>(p, s);
  if (p.D <= 2 * warp) return norm_forward_run<T, VEC, 2, EPT>(p, s);
  if (p.D <= 4 * warp) return norm_forward_run<T, VEC, 4, EPT>(p, s);
  if (p.D <= 8 * warp) return norm_forward_run<T, VEC, 8, EPT>(p, s);
  return norm_forward_run<T, VEC, 16, EPT>(p, s);
}

template <typename T, typename W>
int norm_run(NormArgs p, bool backward, cudaStream_t s) {
  p.w32 = sizeof(W) == 4;
  constexpr int VEC = 16 / sizeof(T);
  {
    const uintptr_t ends = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.dy) |
                           reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.w) |
                           reinterpret_cast<uintptr_t>(p.b);
    const bool vec = p.D % VEC == 0 && ends % 16 == 0 && (p.rows == 1 || (p.xs % VEC == 0 && p.ds % VEC == 0));
    const int most = backward || !vec ? 8192 : 16 * 32 * norm_forward_ept<T, VEC>();  // 16 warps' registers
    if (p.D <= most) return vec ? norm_short_run<T, VEC>(p, backward, s) : norm_short_run<T, 1>(p, backward, s);
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
  norm_dw_sum<W>(p, s);
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

namespace gfn_abi {
cudaError_t error_word_norm(int* v, int reset, cudaStream_t s) { return gfn_unit_error_word(v, reset, s); }
}  // namespace gfn_abi

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
