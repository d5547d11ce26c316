// Log probabilities of given tokens, the entropy and the top alternatives of
// every row of logits, and their gradient:
//
//   m = max x, d_j = x_j - m, Z = sum e^d_j
//   lp_t = d_t - log Z            (a given token, or one of the top ones)
//   H    = log Z - (sum e^d_j d_j) / Z
//   dx_j = sum_i g_i (1[j = t_i] - p_j) - g_H p_j (lp_j + H)
//
// The reference's sampling and training loops leave these to torch
// (gfn/model.py:404-469).  A row is read once: each thread keeps a running
// maximum, the sums that belong to it, and where its own maximum stood.  The
// k-th best of those bounds the k-th best logit from below, so that only the
// threads above it read their part again (from L2) to name the alternatives.
// Sums and statistics are float32.
//
// Forward and backward are two reads and a write.  8192 x 32000 float32 with the
// entropy: 162 us (6.5 TB/s) and 300 us (7.0 TB/s), at the memory's rate.  4099 x
// 50257 bfloat16 with 8 alternatives: 98 us (4.2 TB/s), bound by instructions (70%
// issue, 10 an element), and 169 (4.9 TB/s).  Few rows are latency: one of 32000
// over eight blocks takes 7.7 us.
#include "lm_host.h"
#include "lm_ops.cuh"

using namespace gfn;
using namespace gfn_abi;

namespace {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_TOP = 32;       // alternatives at most
constexpr int LP_QUADS = LP_THREADS / 4;
constexpr int LP_CAP = 1024;     // candidates for the alternatives at most (else by rounds)
constexpr int LP_CLUSTER = 8;    // blocks that share a row at most
constexpr float LP_LOG2E = 1.4426950408889634f;
constexpr float LP_LOW = -1000.f;  // e^d is 0 from here on; keeps 0 * -inf out of the entropy

struct LpArgs {
  const void* x;
  long long xs;
  const long long* tokens;
  float* lp;
  float* ent;
  float* top_lp;
  long long* top_id;
  float2* stats;  // (m, log Z) per row
  long long rows, ignore;
  int V, top;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T> struct Two { using type = float2; };
template <> struct Two<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Two<__half> { using type = __half2; };

GFN_DEV float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
GFN_DEV float max_nan(float a, float b) {  // NaN where one is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Orders logits as whole numbers: by value (NaN above all, -0 as 0), then the
// lower token first.  Never 0.
GFN_DEV unsigned long long rank_key(float v, unsigned j) {
  const unsigned b = __float_as_uint(v + 0.f);
  const unsigned o = v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
  return (unsigned long long)o << 32 | (0xffffffffu - j);
}
GFN_DEV float key_value(unsigned long long k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float(o == 0xffffffffu ? 0x7fffffffu : o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// A row in groups of VEC places that start on 16 bytes; token j stands at
// place j + phase.
template <typename T>
struct LpRow {
  static constexpr int VEC = 16 / sizeof(T);
  const T* base;
  int phase, end;  // first place, and behind the last
  GFN_DEV LpRow(const T* x, int V) {
    phase = (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % VEC);
    base = x - phase;
    end = V + phase;
  }
  GFN_DEV int groups() const { return (end + VEC - 1) / VEC; }
  GFN_DEV bool whole(int g) const { return g * VEC >= phase && g * VEC + VEC <= end; }
  // A group's raw elements; those outside the row are -inf.
  GFN_DEV Pack<T, VEC> load(int g) const {
    if (whole(g)) return *reinterpret_cast<const Pack<T, VEC>*>(base + (long long)g * VEC);
    Pack<T, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int i = g * VEC + e;
      r.v[e] = i >= phase && i < end ? base[i] : from_f<T>(-INFINITY);
    }
    return r;
  }
};

GFN_DEV void lp_merge(float& m, float& s, float& u, float m2, float s2, float u2) {
  const float mn = fmaxf(m, m2), base = mn == -INFINITY ? 0.f : mn;
  const float c1 = exp2_fast((m - base) * LP_LOG2E), c2 = exp2_fast((m2 - base) * LP_LOG2E);
  // far maxima count as LP_LOW away: their factor is 0, and their distance times a sum could be infinite
  u = c1 * (u + fmaxf(m - base, LP_LOW) * s) + c2 * (u2 + fmaxf(m2 - base, LP_LOW) * s2);
  s = c1 * s + c2 * s2;
  m = mn;
}

// The largest of a group; NaN does not count.
template <typename T, int VEC>
GFN_DEV float group_max(const Pack<T, VEC>& p) {
  if constexpr (sizeof(T) == 4) {
    float m = p.v[0];
#pragma unroll
    for (int e = 1; e < VEC; ++e) m = fmaxf(m, p.v[e]);
    return m;
  } else {
    using T2 = typename Two<T>::type;
    const T2* h = reinterpret_cast<const T2*>(&p);
    T2 m = h[0];
#pragma unroll
    for (int e = 1; e < VEC / 2; ++e) m = __hmax2(m, h[e]);
    return fmaxf(to_f(m.x), to_f(m.y));
  }
}

// Adds N groups (g, g + THREADS, ...) to a thread's running maximum m, its
// group gi, s = sum e^(x-m) and u = sum e^(x-m) (x - m).  The difference is taken
// before the factor log2 e: in one fused step it would be off by up to half a
// unit of |m| log2 e, and a row's only token would not have probability 1.
template <typename T, int VEC, int N, bool ENT, bool TOP>
GFN_DEV void lp_add(const Pack<T, VEC> (&raw)[N], int g, float& m, float& s, float& u, int& gi) {
  float mn = m;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float gm = group_max<T, VEC>(raw[k]);
    if (TOP && gm > mn) gi = g + k * LP_THREADS;
    mn = fmaxf(mn, gm);
  }
  const float base = mn == -INFINITY ? 0.f : mn, c = exp2_fast((m - base) * LP_LOG2E);
  if (ENT) u = c * (u + fmaxf(m - base, LP_LOW) * s);
  m = mn;
  F2 s2 = f2(s * c, 0.f), u2 = f2(u, 0.f);
  const F2 nb = f2(-base), l2 = f2(LP_LOG2E);
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      F2 d = f2(to_f(raw[k].v[e]), to_f(raw[k].v[e + 1])) + nb;
      float lo, hi;
      if (ENT) {
        split(d, lo, hi);
        d = f2(max_nan(lo, LP_LOW), max_nan(hi, LP_LOW));
      }
      split(d * l2, lo, hi);
      const F2 ex = f2(exp2_fast(lo), exp2_fast(hi));
      s2 = s2 + ex;
      if (ENT) u2 = fma2(ex, d, u2);
    }
  }
  float a, b;
  split(s2, a, b);
  s = a + b;
  if (ENT) {
    split(u2, a, b);
    u = a + b;
  }
}

struct LpShared {
  float3 warp[LP_WARPS];
  float3 part[LP_CLUSTER];                       // of every block of the row, in the first one
  unsigned long long quads[LP_QUADS];
  unsigned long long tau;
  int count, holding;
  unsigned short holders[LP_THREADS];
  unsigned long long best[LP_WARPS];
  unsigned long long cand[LP_CAP];
  unsigned long long list[LP_CLUSTER * LP_TOP];  // every block's alternatives, in the first one
};

// This block's `top` best keys of the groups [g0, g1), to list[0 .. top) of
// the row's first block.  (m, gi): the thread's largest logit and its group.
template <typename T, class Put>
GFN_DEV void lp_top(LpShared& sh, const LpRow<T>& row, int g0, int g1, int top, float m, int gi, bool odd, Put put) {
  constexpr int VEC = LpRow<T>::VEC;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool mine = g0 + tid < g1;
  // what the thread's best key is at least, and at most
  const int hi = min(gi * VEC + VEC, row.end) - 1 - row.phase, lo = max(gi * VEC - row.phase, 0);
  const unsigned long long low = mine ? rank_key(m, (unsigned)hi) : 0ull, high = mine ? rank_key(m, (unsigned)lo) : 0ull;
  unsigned long long q = low;
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const unsigned long long t = __shfl_xor_sync(0xffffffffu, q, o);
    q = t > q ? t : q;
  }
  if ((lane & 3) == 0) sh.quads[tid >> 2] = q;
  if (tid == 0) {
    sh.count = 0;
    sh.holding = 0;
    sh.tau = 0;
  }
  __syncthreads();
  if (tid < LP_QUADS) {
    const unsigned long long k = sh.quads[tid];
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < LP_QUADS; ++i) above += sh.quads[i] > k;
    if (above == top - 1 && k) sh.tau = k;  // keys above 0 differ
  }
  __syncthreads();
  const unsigned long long tau = sh.tau;
  // The threads that may hold one of them, and their groups shared out to all:
  // a thread reading its own again (the first form) kept every warp busy with
  // a few lanes (4099 x 50257 bfloat16, 8 alternatives: 290 us against 99).
  // Of logits of -inf, the first 64 tokens hold enough: fewer than `top` are above.
  if (!odd && mine && high >= tau && (m > -INFINITY || lo < 2 * LP_TOP))
    sh.holders[atomicAdd(&sh.holding, 1)] = (unsigned short)tid;
  __syncthreads();
  const int per = (g1 - g0 + LP_THREADS - 1) / LP_THREADS, visits = sh.holding * per;
  const float floor = key_value(tau);  // -inf, or 0 as a key, lets every logit through
  for (int v = tid; v < visits; v += LP_THREADS) {
    const int g = g0 + sh.holders[v / per] + (v % per) * LP_THREADS;
    if (g >= g1) continue;
    const Pack<T, VEC> p = row.load(g);
    float f[VEC], gm = -INFINITY;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      f[e] = to_f(p.v[e]);
      gm = fmaxf(gm, f[e]);
    }
    if (tau && gm < floor) continue;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int j = g * VEC + e - row.phase;
      if (j < 0 || j >= row.end - row.phase) continue;
      if (f[e] == -INFINITY && j >= 2 * LP_TOP) continue;
      const unsigned long long k = rank_key(f[e], (unsigned)j);
      if (k < tau) continue;
      const int at = atomicAdd(&sh.count, 1);
      if (at < LP_CAP) sh.cand[at] = k;
    }
  }
  __syncthreads();
  const int n = sh.count;
  if (!odd && n <= LP_CAP) {
    for (int i = tid; i < n; i += LP_THREADS) {
      const unsigned long long k = sh.cand[i];
      int above = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) above += sh.cand[j] > k;
      if (above < top) put(above, k);
    }
    for (int i = n + tid; i < top; i += LP_THREADS) put(i, 0ull);
    return;
  }
  // One alternative a round, the largest key below the last: rows with NaN or
  // +inf, and rows whose large logits stand so that a thread holds them all.
  unsigned long long last = ~0ull;
  for (int r = 0; r < top; ++r) {
    unsigned long long b = 0;
    for (int g = g0 + tid; g < g1; g += LP_THREADS) {
      const Pack<T, VEC> p = row.load(g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int i = g * VEC + e;
        if (i < row.phase || i >= row.end) continue;
        const unsigned long long k = rank_key(to_f(p.v[e]), (unsigned)(i - row.phase));
        if (k < last && k > b) b = k;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const unsigned long long t = __shfl_xor_sync(0xffffffffu, b, o);
      b = t > b ? t : b;
    }
    if (lane == 0) sh.best[warp] = b;
    __syncthreads();
    b = sh.best[0];
#pragma unroll
    for (int w = 1; w < LP_WARPS; ++w) b = sh.best[w] > b ? sh.best[w] : b;
    __syncthreads();
    if (tid == 0) put(r, b);
    last = b;  // 0 from the last element on: every later round gives 0
  }
}

template <typename T, bool ENT, bool TOP, bool SHARED_ROW>
__global__ void __launch_bounds__(LP_THREADS) logprob_kernel(const LpArgs p) {
  constexpr int VEC = LpRow<T>::VEC, UNROLL = 32 / VEC;
  __shared__ LpShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int parts = SHARED_ROW ? gridDim.y : 1, part = SHARED_ROW ? blockIdx.y : 0;  // a cluster along y
  if (SHARED_ROW) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const long long r = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + r * p.xs;
  const LpRow<T> row(x, p.V);
  const int G = row.groups();
  const int g0 = (int)((long long)G * part / parts), g1 = (int)((long long)G * (part + 1) / parts);
  // the given token's logit, fetched beside the row
  long long token = -1;
  float xt = 0.f;
  bool valid = false;
  if (part == 0 && tid == 0 && p.tokens) {
    token = p.tokens[r];
    valid = (unsigned long long)token < (unsigned)p.V;
    if (valid) xt = to_f(x[token]);
  }
  float m = -INFINITY, s = 0.f, u = 0.f;
  int gi = g0 + tid;
  for (int g = gi; g < g1;) {
    const int last = g + (UNROLL - 1) * LP_THREADS;
    if (last < g1 && row.whole(g) && row.whole(last)) {
      Pack<T, VEC> raw[UNROLL];
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) raw[k] = *reinterpret_cast<const Pack<T, VEC>*>(row.base + (long long)(g + k * LP_THREADS) * VEC);
      lp_add<T, VEC, UNROLL, ENT, TOP>(raw, g, m, s, u, gi);
      g += UNROLL * LP_THREADS;
    } else if (sizeof(T) == 4 && g + LP_THREADS < g1 && row.whole(g)) {
      // fewer groups, or the row's end among them: still all at once (up to seven
      // one by one took 178 us instead of 162 at 8192 x 32000; with 16 bits it is
      // up to three, and this costs more, 103 against 98 at 4099 x 50257)
      Pack<T, VEC> raw[UNROLL];
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        if (g + k * LP_THREADS < g1) raw[k] = row.load(g + k * LP_THREADS);
        else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) raw[k].v[e] = from_f<T>(-INFINITY);
        }
      }
      lp_add<T, VEC, UNROLL, ENT, TOP>(raw, g, m, s, u, gi);
      g += UNROLL * LP_THREADS;
    } else {
      const Pack<T, VEC> raw[1] = {row.load(g)};
      lp_add<T, VEC, 1, ENT, TOP>(raw, g, m, s, u, gi);
      g += LP_THREADS;
    }
  }
  float bm = m, bs = s, bu = u;
#pragma unroll
  for (int o = 16; o; o >>= 1)
    lp_merge(bm, bs, bu, __shfl_xor_sync(0xffffffffu, bm, o), __shfl_xor_sync(0xffffffffu, bs, o),
             __shfl_xor_sync(0xffffffffu, bu, o));
  if (lane == 0) sh.warp[warp] = make_float3(bm, bs, bu);
  __syncthreads();
  bm = sh.warp[lane % LP_WARPS].x;
  bs = sh.warp[lane % LP_WARPS].y;
  bu = sh.warp[lane % LP_WARPS].z;
#pragma unroll
  for (int o = LP_WARPS / 2; o; o >>= 1)
    lp_merge(bm, bs, bu, __shfl_xor_sync(0xffffffffu, bm, o), __shfl_xor_sync(0xffffffffu, bs, o),
             __shfl_xor_sync(0xffffffffu, bu, o));
  // the same bits for every thread: lanes merge in different orders
  bm = __shfl_sync(0xffffffffu, bm, 0);
  bs = __shfl_sync(0xffffffffu, bs, 0);
  bu = __shfl_sync(0xffffffffu, bu, 0);
  // the first block runs by now, so that its shared memory can be written
  if (SHARED_ROW) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (TOP) {
    auto put = [&](int i, unsigned long long k) {
      if (SHARED_ROW) {
        const uint32_t at = dsmem_addr(&sh.list[part * LP_TOP + i], 0);
        asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(k) : "memory");
      } else {
        sh.list[i] = k;
      }
    };
    lp_top<T>(sh, row, g0, g1, p.top, m, gi, !(bs < INFINITY) || bm == INFINITY, put);
  }
  if (SHARED_ROW) {
    if (tid == 0) {
      const uint32_t at = dsmem_addr(&sh.part[part], 0);
      dsmem_st(at, bm);
      dsmem_st(at + 4, bs);
      dsmem_st(at + 8, bu);
    }
    cluster_sync();
    if (part != 0) return;
    bm = sh.part[0].x;
    bs = sh.part[0].y;
    bu = sh.part[0].z;
    for (int q = 1; q < parts; ++q) lp_merge(bm, bs, bu, sh.part[q].x, sh.part[q].y, sh.part[q].z);
  } else if (TOP) {
    __syncthreads();
  }
  const bool empty = bm == -INFINITY && bs == 0.f;  // no logit above -inf
  const float base = empty ? 0.f : bm, lz = empty ? INFINITY : logf(bs);
  if (tid == 0) {
    if (p.stats) p.stats[r] = make_float2(base, lz);
    if (ENT) p.ent[r] = empty ? 0.f : lz - bu / bs;
    if (p.tokens) {
      float v = 0.f;
      if (token != p.ignore) {
        v = valid ? (empty ? -INFINITY : (xt - base) - lz) : __int_as_float(0x7fffffff);
        if (!valid) gfn_flag_error(kDevErrBadToken);
      }
      p.lp[r] = v;
    }
  }
  if (TOP) {
    auto write = [&](int i, unsigned long long k) {
      const float v = key_value(k);
      p.top_id[r * p.top + i] = (long long)(0xffffffffu - (unsigned)k);
      p.top_lp[r * p.top + i] = empty ? -INFINITY : (v - base) - lz;
    };
    if (!SHARED_ROW) {
      if (tid < p.top) write(tid, sh.list[tid]);
    } else if (tid < parts * LP_TOP && (tid & (LP_TOP - 1)) < p.top) {
      const unsigned long long k = sh.list[tid];
      int above = 0;
      for (int q = 0; q < parts; ++q)
        for (int i = 0; i < p.top; ++i) above += sh.list[q * LP_TOP + i] > k;
      if (k && above < p.top) write(above, k);
    }
  }
}

template <typename T, bool ENT, bool TOP>
int lp_launch(const LpArgs& p, cudaStream_t s) {
  int sms = 0;
  const int st = sm_count(&sms);
  if (st != GFN_OK) return st;
  // Few rows: up to eight blocks share one, as long as each has 8 KB to read
  // and there are not two blocks per SM yet
  // (256 x 50257 bfloat16: four blocks a row 29 us, two 20).
  int parts = 1;
  const long long bytes = (long long)p.V * sizeof(T);
  while (parts < LP_CLUSTER && p.rows * parts < 2LL * sms && bytes / (2 * parts) >= 8192) parts *= 2;
  if (parts == 1) {
    logprob_kernel<T, ENT, TOP, false><<<(unsigned)p.rows, LP_THREADS, 0, s>>>(p);
    return launch_status("logprob_kernel");
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.rows, (unsigned)parts);
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = s;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 1;
  at.val.clusterDim.y = (unsigned)parts;
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logprob_kernel<T, ENT, TOP, true>, p);
  return e == cudaSuccess ? GFN_OK : cuda_status(e, "logprob_kernel");
}

template <typename T>
int lp_dispatch(const LpArgs& p, cudaStream_t s) {
  if (p.ent) return p.top ? lp_launch<T, true, true>(p, s) : lp_launch<T, true, false>(p, s);
  return p.top ? lp_launch<T, false, true>(p, s) : lp_launch<T, false, false>(p, s);
}

// ----------------------------------------------------------------- gradient
struct LpGradArgs {
  const void* x;
  void* dx;
  const long long* tokens;
  const long long* top_id;
  const float2* stats;
  const float* ent;
  const float* g_lp;
  const float* g_ent;
  const float* g_top;
  long long xs, rows, ignore;
  int V, top, blocks;  // blocks per row
};

GFN_DEV void store_two(float* p, float a, float b) {
  p[0] = a;
  p[1] = b;
}
GFN_DEV void store_two(__nv_bfloat16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }
GFN_DEV void store_two(__half* p, float a, float b) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b); }

// A block owns THREADS * UNROLL groups of one row.  The part that every
// element has, p_j (A + B d_j), is written in one go; then the block puts
// right the given token's element and those of the alternatives.
template <typename T, int VEC, bool ENT>
__global__ void __launch_bounds__(LP_THREADS) logprob_grad_kernel(const LpGradArgs p) {
  constexpr int UNROLL = VEC == 1 ? 8 : 4, RUN = LP_THREADS * UNROLL * VEC;
  __shared__ long long id[LP_TOP + 1];
  __shared__ float g[LP_TOP + 1];
  const int tid = threadIdx.x;
  const long long r = blockIdx.x / p.blocks;
  const int block = blockIdx.x % p.blocks;
  const T* x = static_cast<const T*>(p.x) + r * p.xs;
  T* dx = static_cast<T*>(p.dx) + r * p.V;
  const int phase = VEC > 1 ? (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % VEC) : 0, end = p.V + phase;
  const int start = block * RUN;
  // places are counted from `start`: the last block's would pass 2^31 behind the longest rows
  const int front = phase - start, left = end - start;
  const T* from = x - phase + start;
  T* to = dx - phase + start;
  Pack<T, VEC> raw[UNROLL];
#pragma unroll
  for (int k = 0; k < UNROLL; ++k) {
    const int i = (k * LP_THREADS + tid) * VEC;
    if (i >= front && i + VEC <= left) raw[k] = *reinterpret_cast<const Pack<T, VEC>*>(from + i);
  }
  const float2 st = p.stats[r];
  const bool empty = st.y == INFINITY;
  if (tid <= LP_TOP) {
    long long t = -1;
    float v = 0.f;
    if (tid == 0) {
      if (p.tokens && p.g_lp) {
        t = p.tokens[r];
        if (t == p.ignore) t = -1;
        else v = (unsigned long long)t < (unsigned)p.V ? p.g_lp[r] : __int_as_float(0x7fffffff);
      }
    } else if (tid <= p.top && p.g_top) {
      t = p.top_id[r * p.top + tid - 1];
      v = p.g_top[r * p.top + tid - 1];
    }
    id[tid] = t;
    g[tid] = empty ? 0.f : v;
  }
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int i = 0; i <= LP_TOP; ++i) total += i <= p.top ? g[i] : 0.f;
  const float ge = ENT && !empty ? p.g_ent[r] : 0.f;
  const float A = ENT ? -total - ge * ((empty ? 0.f : p.ent[r]) - (empty ? 0.f : st.y)) : -total, B = -ge;
  const float nz = -st.y * LP_LOG2E;
  auto grad = [&](float lo, float hi, float& a, float& b) {
    F2 d = f2(lo, hi) + f2(-st.x);
    if (ENT) {
      split(d, lo, hi);
      d = f2(max_nan(lo, LP_LOW), max_nan(hi, LP_LOW));
    }
    split(fma2(d, f2(LP_LOG2E), f2(nz)), lo, hi);
    split(f2(exp2_fast(lo), exp2_fast(hi)) * (ENT ? fma2(f2(B), d, f2(A)) : f2(A)), a, b);
  };
  auto grad1 = [&](float v) {
    float a, b;
    grad(v, v, a, b);
    return a;
  };
#pragma unroll
  for (int k = 0; k < UNROLL; ++k) {
    const int i = (k * LP_THREADS + tid) * VEC;
    if (i >= front && i + VEC <= left) {
      Pack<T, VEC> o;
      if constexpr (VEC == 1) o.v[0] = from_f<T>(grad1(to_f(raw[k].v[0])));
      else {
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          float a, b;
          grad(to_f(raw[k].v[e]), to_f(raw[k].v[e + 1]), a, b);
          store_two(&o.v[e], a, b);
        }
      }
      *reinterpret_cast<Pack<T, VEC>*>(to + i) = o;
    } else {
      for (int j = max(i, front); j < min(i + VEC, left); ++j) to[j] = from_f<T>(grad1(to_f(from[j])));
    }
  }
  __syncthreads();
  if (tid <= p.top && id[tid] >= 0 && id[tid] < p.V) {
    const long long j = id[tid];
    const long long at = j + phase - start;
    if (at < 0 || at >= RUN) return;
    float sum = 0.f;
    for (int i = 0; i <= p.top; ++i) {
      if (id[i] != j) continue;
      if (i < tid) return;  // the first of the same token writes
      sum += g[i];
    }
    dx[j] = from_f<T>(grad1(to_f(x[j])) + sum);
  }
}

template <typename T, int VEC>
int lp_grad_launch(LpGradArgs p, cudaStream_t s) {
  constexpr int RUN = LP_THREADS * (VEC == 1 ? 8 : 4) * VEC;
  p.blocks = (int)(((long long)p.V + VEC - 1 + RUN - 1) / RUN);
  if (p.rows * p.blocks > 0x7fffffffLL) return fail(GFN_ERR_UNSUPPORTED, "token_logprobs: %lld rows of %d", p.rows, p.V);
  if (p.g_ent) logprob_grad_kernel<T, VEC, true><<<(unsigned)(p.rows * p.blocks), LP_THREADS, 0, s>>>(p);
  else logprob_grad_kernel<T, VEC, false><<<(unsigned)(p.rows * p.blocks), LP_THREADS, 0, s>>>(p);
  return launch_status("logprob_grad_kernel");
}

template <typename T>
int lp_grad_dispatch(const LpGradArgs& p, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  // logits and gradient in one phase, row by row
  const bool vec = (reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.dx)) % 16 == 0 &&
                   (p.rows == 1 || (p.xs - p.V) % VEC == 0);
  return vec ? lp_grad_launch<T, VEC>(p, s) : lp_grad_launch<T, 1>(p, s);
}

int lp_check(const char* what, long long rows, int vocab, int top, bool null) {
  if (rows < 0 || vocab <= 0 || top < 0 || (rows > 0 && null))
    return fail(GFN_ERR_INVALID, "%s: rows=%lld vocab=%d top=%d or a NULL operand", what, rows, vocab, top);
  if (top > LP_TOP || top > vocab)
    return fail(GFN_ERR_UNSUPPORTED, "%s: %d alternatives of %d tokens, %d at most", what, top, vocab, LP_TOP);
  if (rows > 0x7fffffffLL || vocab > 0x7fffff00)
    return fail(GFN_ERR_UNSUPPORTED, "%s: %lld rows of %d", what, rows, vocab);
  return GFN_OK;
}

}  // namespace

namespace gfn_abi {
cudaError_t error_word_logprobs(int* v, int reset, cudaStream_t s) { return gfn_unit_error_word(v, reset, s); }
}  // namespace gfn_abi

extern "C" {

int gfn_token_logprobs_forward(const void* logits, long long logits_row_stride, int dtype, long long rows, int vocab,
                               const long long* tokens, long long ignore_index, int top, float* logprobs,
                               float* entropy, float* top_logprobs, long long* top_tokens, float* stats,
                               gfn_stream_t stream) {
  const int st = lp_check("token_logprobs", rows, vocab, top,
                          !logits || (tokens && !logprobs) || (top > 0 && (!top_logprobs || !top_tokens)));
  if (st != GFN_OK || rows == 0) return st;
  LpArgs p = {};
  p.x = logits; p.xs = logits_row_stride; p.tokens = tokens; p.lp = logprobs; p.ent = entropy;
  p.top_lp = top_logprobs; p.top_id = top_tokens; p.stats = reinterpret_cast<float2*>(stats);
  p.rows = rows; p.ignore = ignore_index; p.V = vocab; p.top = top;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == GFN_F32) return lp_dispatch<float>(p, s);
  if (dtype == GFN_BF16) return lp_dispatch<__nv_bfloat16>(p, s);
  if (dtype == GFN_F16) return lp_dispatch<__half>(p, s);
  return fail(GFN_ERR_UNSUPPORTED, "token_logprobs: element type %d", dtype);
}

int gfn_token_logprobs_backward(const void* logits, long long logits_row_stride, int dtype, long long rows, int vocab,
                                const long long* tokens, long long ignore_index, int top, const long long* top_tokens,
                                const float* stats, const float* entropy, const float* d_logprobs,
                                const float* d_entropy, const float* d_top, void* dlogits, gfn_stream_t stream) {
  const int st = lp_check("token_logprobs backward", rows, vocab, top,
                          !logits || !stats || !dlogits || (d_logprobs && !tokens) || (d_entropy && !entropy) ||
                              (d_top && !top_tokens));
  if (st != GFN_OK || rows == 0) return st;
  LpGradArgs p = {};
  p.x = logits; p.dx = dlogits; p.tokens = tokens; p.top_id = top_tokens;
  p.stats = reinterpret_cast<const float2*>(stats);
  p.ent = entropy; p.g_lp = d_logprobs; p.g_ent = d_entropy; p.g_top = d_top;
  p.xs = logits_row_stride; p.rows = rows; p.ignore = ignore_index; p.V = vocab; p.top = d_top ? top : 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == GFN_F32) return lp_grad_dispatch<float>(p, s);
  if (dtype == GFN_BF16) return lp_grad_dispatch<__nv_bfloat16>(p, s);
  if (dtype == GFN_F16) return lp_grad_dispatch<__half>(p, s);
  return fail(GFN_ERR_UNSUPPORTED, "token_logprobs backward: element type %d", dtype);
}

}  // extern "C"
