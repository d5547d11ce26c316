// Linear attention with a decay for each head: a state S [K, V] per sequence
// and head,
//
//   S_t = g S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
//
// the gated scan (gfn/scan.py:11-104) with a matrix for a state.  In blocks of
// C tokens, i, j = 0 .. n - 1 within one and S the state before it:
//
//   O  = scale ((Q K^T) o M) V + scale diag(g^(i+1)) Q S,   M_ij = g^(i-j), j <= i
//   S' = g^n S + (diag(g^(n-1-j)) K)^T V
//
// The gradients are the same pass with other operands: with do for q, v for k,
// k for v and the transposed state it gives dq; from the last token to the
// first, with the state's gradient R for S,
//
//   dv = pass(k, q, do; R),   dk = pass(v, do, q; R^T),
//   R' = g (g^(n-1) R + scale sum of g^(n-1-j) q_j do_j^T)
//
// State, sums and powers of g are float32.  The products run on the tensor
// cores with float32 accumulators; what is rounded for them:
//   bfloat16: P = (Q K^T) o M and S as operands, to bfloat16, once each (the
//     outputs are rounded to it too); the state's own update takes g^.. k in
//     three bfloat16 pieces (24 bits), so that the state stays float32-exact.
//   float16: operands as tf32, which holds float16 exactly and P and S to 11
//     bits at float32's range (a float16 P or S could overflow); g^.. k in two
//     tf32 pieces.
//   float32: every operand in two tf32 pieces, three products (2^-22).
// The scores' powers of g come from ex2.approx (2^-22 relative, 0 below 2^-126),
// which is below what the operands lose.
//
// Why mma.sync: scores are masked, g^.. applied and the result multiplied again
// without leaving the registers, and so is k where it is split.  Through tensor
// memory those steps would keep about 70% of today's issue slots.  1 x 65536 x 8
// heads of 64 in bfloat16: outputs 86 us (tensor pipe 50%, issue 39%, 12 warps an
// SM), segments' states 46 (56%, 36%), their join 7; the bytes would take 41.  What
// is left is latency between the steps of a block of tokens.  Larger tiles a warp
// do better than more warps: 8 warps of half the columns took 108 us for the outputs.
#pragma once
#include <type_traits>

#include "decay_attn.h"
#include "lm_host.h"
#include "lm_ops.cuh"

namespace gfn_attn {

using namespace gfn;
using namespace gfn_abi;

GFN_DEV int length_of(const PassArgs& p, int b) {
  if (!p.lengths) return p.L;
  const long long n = p.lengths64 ? static_cast<const long long*>(p.lengths)[b] : static_cast<const int*>(p.lengths)[b];
  return (int)(n < 0 ? 0 : n > p.L ? p.L : n);
}

GFN_DEV float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// log2 of a decay in [0, 1] (taken as the nearer end outside); 0 becomes a
// finite number whose every multiple from one on is a power of 0.
GFN_DEV float log2_decay(float g) {
  g = g > 1.f ? 1.f : g < 0.f ? 0.f : g;
  return g == 0.f ? -1e30f : log2f(g);
}
GFN_DEV float power(float lg, int n) { return exp2f(lg * (float)n); }

// ---------------------------------------------------------------- fragments
// Operands of one tensor-core step.  Lane l stands at g = l / 4, t = l % 4.
// 16-bit types: m16n8k16, pairs of neighbours of the contraction in a register.
// tf32: m16n8k8, where place t of the contraction is its element 2 t and place
// t + 4 its element 2 t + 1 on both sides, so that two neighbours are read at
// once, accumulators serve as operands as they are, and a 16-bit step's
// registers hold two tf32 steps.
template <typename T>
struct Math {  // float32
  static constexpr int KS = 8, PIECES = 2;
  using State = float;
  static constexpr int PAD = 4, STATE_PAD = 4;
  struct A {
    unsigned v[PIECES][4];
  };
  struct B {
    unsigned v[PIECES][2];
  };
};
struct Math16 {
  static constexpr int KS = 16, PAD = 8;
  struct A {
    unsigned v[4];
  };
  struct B {
    unsigned v[2];
  };
};
template <>
struct Math<__nv_bfloat16> : Math16 {
  using State = __nv_bfloat16;
  static constexpr int STATE_PAD = 8;
};
template <>
struct Math<__half> : Math16 {
  using State = float;  // tf32 values
  static constexpr int STATE_PAD = 4;
};

GFN_DEV void mma_bf16(float (&c)[4], const unsigned (&a)[4], const unsigned (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
GFN_DEV void mma_f16(float (&c)[4], const unsigned (&a)[4], const unsigned (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
GFN_DEV void mma_tf32(float (&c)[4], const unsigned (&a)[4], const unsigned (&b)[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
GFN_DEV unsigned tf32(float v) {
  unsigned r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}
// WIDE: the first piece stops at tf32's largest number.  Values between that and
// float32's largest, as finfo.max is, round to infinity otherwise and leave
// inf - inf; but everywhere this conversion costs 10 to 16% of a float32 pass.
template <bool WIDE, int N>
GFN_DEV void pieces(float v, unsigned (&r)[N]) {
  if constexpr (WIDE) asm("cvt.rna.satfinite.tf32.f32 %0, %1;" : "=r"(r[0]) : "f"(v));
  else r[0] = tf32(v);
  if constexpr (N > 1) r[1] = tf32(v - __uint_as_float(r[0]));
}

template <int PA, int PB>
GFN_DEV void mma_pieces(float (&c)[4], const unsigned (&a)[PA][4], const unsigned (&b)[PB][2]) {
  if constexpr (PA > 1) mma_tf32(c, a[1], b[0]);
  if constexpr (PB > 1) mma_tf32(c, a[0], b[1]);
  mma_tf32(c, a[0], b[0]);
}
// c += a b with the products of a step summed by themselves first: the tensor
// cores cut where float32 addition rounds, three times a step, and over an output's
// steps that adds up (40 x 72 heads: error 1.3e-6, so 7.8e-7; 443 -> 453 us trained).
GFN_DEV void mma_apart(float (&c)[4], const unsigned (&a)[2][4], const unsigned (&b)[2][2]) {
  float d[4] = {};
  mma_pieces(d, a, b);
  split(f2(c[0], c[1]) + f2(d[0], d[1]), c[0], c[1]);
  split(f2(c[2], c[3]) + f2(d[2], d[3]), c[2], c[3]);
}
template <typename T>
GFN_DEV void mma(float (&c)[4], const typename Math<T>::A& a, const typename Math<T>::B& b) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) mma_bf16(c, a.v, b.v);
  else if constexpr (std::is_same_v<T, __half>) mma_f16(c, a.v, b.v);
  else mma_pieces(c, a.v, b.v);
}

GFN_DEV void ldsm(unsigned& a, unsigned& b, unsigned& c, unsigned& d, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(smem_u32(p)));
}
GFN_DEV void ldsm_t(unsigned& a, unsigned& b, unsigned& c, unsigned& d, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(smem_u32(p)));
}
GFN_DEV float2 pair(const float* p) { return *reinterpret_cast<const float2*>(p); }

// A, 16 rows from p [row][k].
template <typename T, bool CARE>
GFN_DEV void load_a(typename Math<T>::A& f, const T* p, int ld, int lane) {
  if constexpr (Math<T>::KS == 16) {
    ldsm(f.v[0], f.v[1], f.v[2], f.v[3], p + ((lane & 7) + (lane & 8)) * ld + ((lane >> 4) << 3));
  } else {
    const T* q = p + (lane >> 2) * ld + 2 * (lane & 3);
    const float2 x = pair(q), y = pair(q + 8 * ld);
    const float w[4] = {x.x, y.x, x.y, y.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned r[Math<T>::PIECES];
      pieces<CARE>(w[i], r);
#pragma unroll
      for (int k = 0; k < Math<T>::PIECES; ++k) f.v[k][i] = r[k];
    }
  }
}
// Two neighbouring B of 8 columns each, from p [n][k].
template <typename T, bool CARE, typename E>
GFN_DEV void load_bn(typename Math<T>::B (&f)[2], const E* p, int ld, int lane) {
  if constexpr (Math<T>::KS == 16) {
    ldsm(f[0].v[0], f[0].v[1], f[1].v[0], f[1].v[1], p + ((lane & 7) + ((lane >> 4) << 3)) * ld + (lane & 8));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 x = pair(p + ((lane >> 2) + 8 * h) * ld + 2 * (lane & 3));
      unsigned r[2][Math<T>::PIECES];
      pieces<CARE>(x.x, r[0]);
      pieces<CARE>(x.y, r[1]);
#pragma unroll
      for (int k = 0; k < Math<T>::PIECES; ++k) {
        f[h].v[k][0] = r[0][k];
        f[h].v[k][1] = r[1][k];
      }
    }
  }
}
// The same from p [k][n].
template <typename T, bool CARE, typename E>
GFN_DEV void load_bk(typename Math<T>::B (&f)[2], const E* p, int ld, int lane) {
  if constexpr (Math<T>::KS == 16) {
    ldsm_t(f[0].v[0], f[0].v[1], f[1].v[0], f[1].v[1], p + ((lane & 7) + (lane & 8)) * ld + ((lane >> 4) << 3));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const E* q = p + 2 * (lane & 3) * ld + (lane >> 2) + 8 * h;
      unsigned r[2][Math<T>::PIECES];
      pieces<CARE>(to_f(q[0]), r[0]);
      pieces<CARE>(to_f(q[ld]), r[1]);
#pragma unroll
      for (int k = 0; k < Math<T>::PIECES; ++k) {
        f[h].v[k][0] = r[0][k];
        f[h].v[k][1] = r[1][k];
      }
    }
  }
}

// Two float16 neighbours as tf32 (exact).
GFN_DEV void unpack_f16(unsigned v, unsigned& lo, unsigned& hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  lo = __float_as_uint(f.x);
  hi = __float_as_uint(f.y);
}
// Step q (0, 1) of eight of a 16-bit operand, as tf32.
GFN_DEV void half_step(const Math16::A& f, int q, unsigned (&a)[4]) {
  unpack_f16(f.v[2 * q], a[0], a[2]);
  unpack_f16(f.v[2 * q + 1], a[1], a[3]);
}
GFN_DEV void half_step(const Math16::B& f, int q, unsigned (&b)[2]) { unpack_f16(f.v[q], b[0], b[1]); }

GFN_DEV unsigned pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}
GFN_DEV float2 unpack_bf16(unsigned v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }

// ------------------------------------------------------------------- blocks
// Tokens per block, warps, and who holds what.  A warp has 16 rows of a
// block's output and, of the state, 16 rows (a slab) of SN tiles of 8 columns.
template <typename T, int DK, int DV>
struct Shape {
  static constexpr bool WIDE = DK > 64 || DV > 64;
  static constexpr int W = WIDE ? 8 : 4, THREADS = 32 * W;
  static constexpr int C = sizeof(T) == 4 && (DK > 32 || DV > 32) ? 32 : 64;
  static constexpr int LDK = DK + Math<T>::PAD, LDV = DV + Math<T>::PAD, LS = DV + Math<T>::STATE_PAD;
  static constexpr int ROWS = C / 16, SPLIT = W / ROWS;
  static constexpr int SLABS = DK / 16, SN = DV / 8 / (W / SLABS);
  static constexpr int TK = C * LDK, TV = C * LDV;  // elements of an operand
  static constexpr int STATE_BYTES = DK * LS * (int)sizeof(typename Math<T>::State);
  static constexpr int stage(int kind) { return kind == STATE ? TK + TV : kind == OUTPUT ? 2 * TK + TV : 2 * TK + 2 * TV; }
  // thread blocks of an SM that registers allow (heads up to 32: four instead of
  // three, 4 x 6000 x 4 heads of 32 trained in bfloat16 66 us of kernels to 62; 65 since
  // segments end with a look for bad values)
  static constexpr int most(int kind) {
    return WIDE ? (DK + DV < 256 ? 2 : 1) : kind == STATE || DK == 32 ? 4 : kind == PAIR && sizeof(T) < 4 ? 2 : 3;
  }
  static constexpr int need(int kind, int stages, int buffers) {
    return stages * stage(kind) * (int)sizeof(T) + buffers * STATE_BYTES + 8 * C;
  }
  static constexpr int fit(int kind, int stages, int buffers) {
    const int n = 228 * 1024 / (need(kind, stages, buffers) + 1024);
    return n < most(kind) ? n : most(kind);
  }
  // Operands of two blocks of tokens (one on its way) unless one alone lets an
  // SM hold more thread blocks; the state's operand form twice where that costs
  // none: then a block of tokens takes one barrier instead of two.
  static constexpr int stages(int kind) { return kind == STATE || fit(kind, 2, 1) >= fit(kind, 1, 1) ? 2 : 1; }
  static constexpr int buffers(int kind) {
    return kind == STATE ? 0 : stages(kind) == 2 && fit(kind, 2, 2) >= fit(kind, 2, 1) ? 2 : 1;
  }
  static constexpr int bytes(int kind) { return need(kind, stages(kind), buffers(kind)); }
  static constexpr int resident(int kind) { return fit(kind, stages(kind), buffers(kind)); }
};

template <int BYTES>
GFN_DEV void copy_async(uint32_t to, const void* from, int read) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(read) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(read) : "memory");
}
template <typename T, int D, int LD, int C, int THREADS, bool BACK, int BYTES>
GFN_DEV void fetch_pieces(T* dst, const T* src, const void* any, long long sl, int dim, int n) {
  constexpr int PER = BYTES / sizeof(T), ROW = D / PER, LANES = ROW < THREADS ? ROW : THREADS, STEP = THREADS / LANES;
  const int col = (threadIdx.x % LANES) * PER, r0 = threadIdx.x / LANES;
  if (col >= dim) return;
  const T* from = src + col + (BACK ? -r0 : r0) * sl;
  const long long step = (BACK ? -STEP : STEP) * sl;
  const uint32_t to = smem_u32(dst + r0 * LD + col);
#pragma unroll
  for (int i = 0; i < C / STEP; ++i) {
    const bool live = r0 + i * STEP < n;  // others are filled with zeros: 0 bytes are read
    copy_async<BYTES>(to + i * STEP * LD * (int)sizeof(T), live ? from : any, live ? BYTES : 0);
    from += step;
  }
}
// Brings rows 0 .. n - 1 of a block into shared memory, zeros behind them; row
// r is the r-th token from `at` on (BACK: from there to the front).  Columns
// from `dim` on were zeroed once and stay so.
template <typename T, int D, int LD, int C, int THREADS, bool BACK, bool FULL>
GFN_DEV void fetch(T* dst, const View& v, int b, int h, int dim, int at, int n, int piece) {
  const T* src = static_cast<const T*>(v.p) + b * v.sb + h * v.sh + at * v.sl;
  if (FULL || piece == 16) fetch_pieces<T, D, LD, C, THREADS, BACK, 16>(dst, src, v.p, v.sl, dim, n);
  else if (piece == 8) fetch_pieces<T, D, LD, C, THREADS, BACK, 8>(dst, src, v.p, v.sl, dim, n);
  else if (sizeof(T) == 4 || piece == 4) fetch_pieces<T, D, LD, C, THREADS, BACK, 4>(dst, src, v.p, v.sl, dim, n);
  else if constexpr (sizeof(T) == 2) {  // elements at odd places
    constexpr int AHEAD = 8, COUNT = C * D / THREADS;
    static_assert(COUNT % AHEAD == 0, "");
#pragma unroll 1
    for (int i0 = 0; i0 < COUNT; i0 += AHEAD) {
      T e[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = (i0 + u) * THREADS + threadIdx.x, r = i / D, col = i % D;
        e[u] = col < dim && r < n ? src[(BACK ? -r : r) * v.sl + col] : from_f<T>(0.f);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = (i0 + u) * THREADS + threadIdx.x, r = i / D, col = i % D;
        if (col < dim) dst[r * LD + col] = e[u];
      }
    }
  }
}

// Powers of g that a thread applies to its scores, g^(i-j) s_in: on the two
// tiles that the diagonal crosses, on the one before them, and from tile to
// tile further back.
struct Decay {
  float diag[2][4], first[4], g8;
  int gap;  // the first score's row less its key
  GFN_DEV Decay(float lg, float s_in) {
    const int lane = threadIdx.x & 31;
    gap = (lane >> 2) - 2 * (lane & 3);
    g8 = exp2_fast(8.f * lg);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = gap + 8 * (e >> 1) - (e & 1);
      diag[0][e] = d < 0 ? 0.f : s_in * exp2_fast((float)d * lg);
      diag[1][e] = d < 8 ? 0.f : s_in * exp2_fast((float)(d - 8) * lg);
      first[e] = s_in * exp2_fast((float)(d + 8) * lg);
    }
  }
  // Score e of the diagonal's tile z (keys 8 z .. 8 z + 7): 0 where the key
  // stands behind the row, whatever it holds.
  GFN_DEV float masked(float s, int z, int e) const {
    return gap + 8 * (e >> 1) - (e & 1) - 8 * z < 0 ? 0.f : s * diag[z][e];
  }
};

// Whether N tiles of 16 rows and 8 columns hold NaN or an infinity.
template <typename T, int N>
GFN_DEV bool tiles_are_bad(const T* p, int ld, int lane) {
  float t = 0.f;
#pragma unroll 1
  for (int i = lane; i < 16 * 8 * N; i += 32) t = fmaf(to_f(p[i / (8 * N) * ld + i % (8 * N)]), 0.f, t);
  return __any_sync(0xffffffffu, t != 0.f);
}
// o += s times the values of the diagonal's tile, each row with the keys up to
// its own.  The tensor cores multiply the keys behind a row too, by scores of 0,
// which makes NaN of a NaN or an infinity there.
template <typename T, int N>
GFN_DEV void add_up_to_diagonal(float (&o)[N][4], const float (&s)[2][4], const T* values, int ld, int lane) {
#pragma unroll 1
  for (int j = 0; j < 16; ++j) {
    float w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float even = j & 8 ? s[1][2 * h] : s[0][2 * h], odd = j & 8 ? s[1][2 * h + 1] : s[0][2 * h + 1];
      w[h] = __shfl_sync(0xffffffffu, j & 1 ? odd : even, (lane & 28) | ((j & 7) >> 1));
    }
    const T* v = values + j * ld + 2 * (lane & 3);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float lo = to_f(v[n * 8]), hi = to_f(v[n * 8 + 1]);
      if (j <= lane >> 2) {
        o[n][0] = fmaf(w[0], lo, o[n][0]);
        o[n][1] = fmaf(w[0], hi, o[n][1]);
      }
      if (j <= (lane >> 2) + 8) {
        o[n][2] = fmaf(w[1], lo, o[n][2]);
        o[n][3] = fmaf(w[1], hi, o[n][3]);
      }
    }
  }
}

// attend (see attend_f32) for the 16-bit types: the keys' tiles of 16 one after
// the other, from the diagonal back, so that eight scores are in registers
// instead of a row of them and no branch stands within a tile.  float16 rows and
// values meet state and scores as tf32.
template <typename T, int DA, int LDA, int LDB, int LS, int ON, bool NMAJOR, bool FULL, bool CARE>
GFN_DEV void attend_16(float (&o)[ON][4], const T* rows, const T* keys, const T* values, const typename Math<T>::State* st,
                       int rt, int col0, int kd, int nd, const Decay& g, float w0, float w1) {
  using M = Math<T>;
  constexpr bool HALF = std::is_same_v<T, __half>;
  constexpr int KN = DA / 16;
  const int lane = threadIdx.x & 31;
  typename M::A a[KN];
#pragma unroll
  for (int k = 0; k < KN; ++k) load_a<T, CARE>(a[k], rows + rt * 16 * LDA + k * 16, LDA, lane);
#pragma unroll
  for (int i = 0; i < ON; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
#pragma unroll
  for (int k = 0; k < KN; ++k) {
    if (!FULL && k * 16 >= kd) continue;
    if constexpr (HALF) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        unsigned aq[4];
        half_step(a[k], q, aq);
#pragma unroll
        for (int i = 0; i < ON; ++i) {
          const int col = col0 + i * 8 + (lane >> 2), kk = k * 16 + q * 8 + 2 * (lane & 3);
          unsigned b[2];
          if (NMAJOR) {
            const float2 x = pair(st + col * LS + kk);
            b[0] = __float_as_uint(x.x);
            b[1] = __float_as_uint(x.y);
          } else {
            b[0] = __float_as_uint(st[kk * LS + col]);
            b[1] = __float_as_uint(st[(kk + 1) * LS + col]);
          }
          mma_tf32(o[i], aq, b);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < ON; i += 2) {
        const int col = col0 + i * 8;
        if (!FULL && col >= nd) continue;
        typename M::B b[2];
        if (NMAJOR) load_bn<T, CARE>(b, st + col * LS + k * 16, LS, lane);
        else load_bk<T, CARE>(b, st + k * 16 * LS + col, LS, lane);
        mma<T>(o[i], a[k], b[0]);
        mma<T>(o[i + 1], a[k], b[1]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ON; ++i) {
    o[i][0] *= w0;
    o[i][1] *= w0;
    o[i][2] *= w1;
    o[i][3] *= w1;
  }
  auto scores = [&](int i, float (&s)[2][4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[0][e] = s[1][e] = 0.f;
#pragma unroll
    for (int k = 0; k < KN; ++k) {
      if (!FULL && k * 16 >= kd) continue;
      typename M::B b[2];
      load_bn<T, CARE>(b, keys + i * 16 * LDA + k * 16, LDA, lane);
      mma<T>(s[0], a[k], b[0]);
      mma<T>(s[1], a[k], b[1]);
    }
  };
  auto add = [&](int i, const float (&s)[2][4]) {
    typename M::A p;
    unsigned pq[2][4];
    if constexpr (HALF) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float w[4] = {s[q][0], s[q][2], s[q][1], s[q][3]};
#pragma unroll
        for (int e = 0; e < 4; ++e) pq[q][e] = tf32(w[e]);
      }
    } else {
      p.v[0] = pack_bf16(s[0][0], s[0][1]);
      p.v[1] = pack_bf16(s[0][2], s[0][3]);
      p.v[2] = pack_bf16(s[1][0], s[1][1]);
      p.v[3] = pack_bf16(s[1][2], s[1][3]);
    }
#pragma unroll
    for (int n = 0; n < ON; n += 2) {
      if (!FULL && col0 + n * 8 >= nd) continue;
      typename M::B b[2];
      load_bk<T, CARE>(b, values + i * 16 * LDB + col0 + n * 8, LDB, lane);
      if constexpr (HALF) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            unsigned bq[2];
            half_step(b[z], q, bq);
            mma_tf32(o[n + z], pq[q], bq);
          }
        }
      } else {
        mma<T>(o[n], p, b[0]);
        mma<T>(o[n + 1], p, b[1]);
      }
    }
  };
  float s[2][4];
  scores(rt, s);
#pragma unroll
  for (int z = 0; z < 2; ++z)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[z][e] = g.masked(s[z][e], z, e);
  const T* own = values + rt * 16 * LDB + col0;
  if (CARE && tiles_are_bad<T, ON>(own, LDB, lane)) add_up_to_diagonal<T, ON>(o, s, own, LDB, lane);
  else add(rt, s);
  F2 f0 = f2(g.first[0], g.first[1]), f1 = f2(g.first[2], g.first[3]);
  const F2 g8 = f2(g.g8);
#pragma unroll 2
  for (int i = rt - 1; i >= 0; --i) {
    scores(i, s);
#pragma unroll
    for (int z = 1; z >= 0; --z) {
      split(f2(s[z][0], s[z][1]) * f0, s[z][0], s[z][1]);
      split(f2(s[z][2], s[z][3]) * f1, s[z][2], s[z][3]);
      f0 = f0 * g8;
      f1 = f1 * g8;
    }
    add(i, s);
  }
}

// One warp's 16 rows of a block's output: ON tiles of 8 columns from col0.
// rows, keys [C][LDA] with kd of their columns in use, values [C][LDB]; st: the
// state, seen from this product as [k][n] or (NMAJOR) [n][k].
template <typename T, int C, int DA, int LDA, int LDB, int LS, int ON, bool NMAJOR, bool FULL, bool CARE>
GFN_DEV void attend_f32(float (&o)[ON][4], const T* rows, const T* keys, const T* values, const typename Math<T>::State* st,
                         int rt, int col0, int kd, int nd, const Decay& g, float w0, float w1) {
  using M = Math<T>;
  const int lane = threadIdx.x & 31;
  float s[C / 8][4];
#pragma unroll
  for (int i = 0; i < C / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
  for (int i = 0; i < ON; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
#pragma unroll
  for (int k = 0; k < DA; k += M::KS) {
    if (!FULL && k >= kd) continue;
    typename M::A a;
    load_a<T, CARE>(a, rows + rt * 16 * LDA + k, LDA, lane);
#pragma unroll
    for (int i = 0; i < ON; i += 2) {
      const int col = col0 + i * 8;
      if (!FULL && col >= nd) continue;
      typename M::B b[2];
      if (NMAJOR) load_bn<T, CARE>(b, st + col * LS + k, LS, lane);
      else load_bk<T, CARE>(b, st + k * LS + col, LS, lane);
      mma_apart(o[i], a.v, b[0].v);
      mma_apart(o[i + 1], a.v, b[1].v);
    }
#pragma unroll
    for (int i = 0; i < C / 16; ++i) {
      if (i > rt) continue;  // keys behind the rows
      typename M::B b[2];
      load_bn<T, CARE>(b, keys + i * 16 * LDA + k, LDA, lane);
      mma<T>(s[2 * i], a, b[0]);
      mma<T>(s[2 * i + 1], a, b[1]);
    }
  }
#pragma unroll
  for (int i = 0; i < ON; ++i) {
    o[i][0] *= w0;
    o[i][1] *= w0;
    o[i][2] *= w1;
    o[i][3] *= w1;
  }
  F2 f0 = f2(g.first[0], g.first[1]), f1 = f2(g.first[2], g.first[3]);
  const F2 g8 = f2(g.g8);
#pragma unroll
  for (int i = C / 8 - 1; i >= 0; --i) {
    const int off = 2 * rt - i;  // -1, 0: the diagonal's tiles
    if (off < -1) continue;
    if (off > 0) {
      split(f2(s[i][0], s[i][1]) * f0, s[i][0], s[i][1]);
      split(f2(s[i][2], s[i][3]) * f1, s[i][2], s[i][3]);
      f0 = f0 * g8;
      f1 = f1 * g8;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = off == 0 ? g.masked(s[i][e], 0, e) : g.masked(s[i][e], 1, e);
    }
  }
  const T* own = values + rt * 16 * LDB + col0;
  const bool bad = CARE && tiles_are_bad<T, ON>(own, LDB, lane);
#pragma unroll
  for (int i = 0; i < C / 16; ++i) {
    if (i > rt) continue;
    if (bad && i == rt) {
      const float d[2][4] = {{s[2 * i][0], s[2 * i][1], s[2 * i][2], s[2 * i][3]},
                             {s[2 * i + 1][0], s[2 * i + 1][1], s[2 * i + 1][2], s[2 * i + 1][3]}};
      add_up_to_diagonal<T, ON>(o, d, own, LDB, lane);
      continue;
    }
#pragma unroll
    for (int q = 0; q < 16 / M::KS; ++q) {
      typename M::A a;
      const float w[4] = {s[2 * i + q][0], s[2 * i + q][2], s[2 * i + q][1], s[2 * i + q][3]};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        unsigned r[M::PIECES];
        pieces<CARE>(w[e], r);
#pragma unroll
        for (int z = 0; z < M::PIECES; ++z) a.v[z][e] = r[z];
      }
      const T* v = values + (16 * i + M::KS * q) * LDB + col0;
#pragma unroll
      for (int n = 0; n < ON; n += 2) {
        if (!FULL && col0 + n * 8 >= nd) continue;
        typename M::B b[2];
        load_bk<T, CARE>(b, v + n * 8, LDB, lane);
        mma_apart(o[n], a.v, b[0].v);
        mma_apart(o[n + 1], a.v, b[1].v);
      }
    }
  }
}

template <typename T, int C, int DA, int LDA, int LDB, int LS, int ON, bool NMAJOR, bool FULL, bool CARE>
GFN_DEV void attend(float (&o)[ON][4], const T* rows, const T* keys, const T* values, const typename Math<T>::State* st,
                    int rt, int col0, int kd, int nd, const Decay& g, float w0, float w1) {
  if constexpr (Math<T>::KS == 16)
    attend_16<T, DA, LDA, LDB, LS, ON, NMAJOR, FULL, CARE>(o, rows, keys, values, st, rt, col0, kd, nd, g, w0, w1);
  else
    attend_f32<T, C, DA, LDA, LDB, LS, ON, NMAJOR, FULL, CARE>(o, rows, keys, values, st, rt, col0, kd, nd, g, w0, w1);
}

// Two values in three bfloat16 pieces each (cut, not rounded), which add up to
// them exactly.
GFN_DEV void split3(F2 v, unsigned& hi, unsigned& mid, unsigned& lo) {
  auto cut = [](float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); };
  auto both = [](float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); };
  float x, y;
  split(v, x, y);
  hi = both(x, y);
  v = v + f2(-cut(x), -cut(y));
  split(v, x, y);
  mid = both(x, y);
  split(v + f2(-cut(x), -cut(y)), x, y);
  lo = both(x, y);
}

// Those of a block's sums that came out as NaN once more, term by term: the
// pieces of a product make NaN of an infinity (inf - inf, 0 x inf) that the
// product alone leaves one.  faded: the factor of an infinity whose own has become 0.
template <typename T, int C, int LDK, int LDV, int N>
GFN_DEV void add_again(float (&add)[N][4], const T* keys, const T* values, const float* wt, float faded, int m0, int n0) {
  const int lane = threadIdx.x & 31;
  float s[4 * N];
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) s[i] = add[i / 4][i % 4];
#pragma unroll 1
  for (int i = 0; i < 4 * N; ++i) {
    if (!isnan(s[i])) continue;
    const T* k = keys + m0 + (lane >> 2) + (i & 2) * 4;
    const T* v = values + n0 + (i >> 2) * 8 + 2 * (lane & 3) + (i & 1);
    float sum = 0.f;
#pragma unroll 1
    for (int j = 0; j < C && !isnan(sum); ++j) {
      const float x = to_f(k[j * LDK]), y = to_f(v[j * LDV]), w = wt[j];
      sum += isfinite(x) && isfinite(y) ? x * w * y : x * y * (w == 0.f ? faded : w);
    }
    s[i] = sum;
  }
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) add[i / 4][i % 4] = s[i];
}

// w s + add for a power w of the decay; an infinity stays one while the decay is
// above 0 (lasts), even if w is below float32's range.
GFN_DEV float carried(float s, float w, float add, bool lasts) {
  return w == 0.f && lasts && isinf(s) ? s + add : fmaf(w, s, add);
}

// st = gn st + (diag(wt) keys)^T values for one warp's 16 rows (from m0) and N
// tiles of columns (from n0) of the state.  The products of a block are summed
// by themselves and then added, since the tensor cores cut where float32
// addition rounds: over a long sequence that would drift.
template <typename T, int C, int LDK, int LDV, int N, bool FULL, bool CARE>
GFN_DEV void update(float (&st)[N][4], const T* keys, const T* values, const float* wt, float gn, int m0, int n0, int nd,
                    float faded, bool lasts) {
  using M = Math<T>;
  const int lane = threadIdx.x & 31, t = lane & 3;
  constexpr int AT = N < 8 ? N : 8;  // tiles at a time
#pragma unroll
  for (int at = 0; at < N; at += AT) {
    if (!FULL && n0 + at * 8 >= nd) continue;
    float add[AT][4];
#pragma unroll
    for (int n = 0; n < AT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) add[n][e] = 0.f;
#pragma unroll
    for (int k = 0; k < C; k += M::KS) {
      const T* vals = values + k * LDV + n0 + at * 8;
      if constexpr (std::is_same_v<T, __half>) {
        unsigned raw[4], a[2][2][4];  // step, piece
        ldsm_t(raw[0], raw[1], raw[2], raw[3], keys + (k + (lane & 7) + ((lane >> 4) << 3)) * LDK + m0 + (lane & 8));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float w0 = wt[k + 8 * q + 2 * t], w1 = wt[k + 8 * q + 2 * t + 1];
          unsigned x[4];
          unpack_f16(raw[2 * q], x[0], x[2]);
          unpack_f16(raw[2 * q + 1], x[1], x[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            unsigned r[2];
            pieces<CARE>(__uint_as_float(x[e]) * (e < 2 ? w0 : w1), r);
            a[q][0][e] = r[0];
            a[q][1][e] = r[1];
          }
        }
#pragma unroll
        for (int n = 0; n < AT; n += 2) {
          if (!FULL && n0 + (at + n) * 8 >= nd) continue;
          typename M::B b[2];
          load_bk<T, CARE>(b, vals + n * 8, LDV, lane);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              unsigned bq[2];
              half_step(b[z], q, bq);
              mma_tf32(add[n + z], a[q][1], bq);
              mma_tf32(add[n + z], a[q][0], bq);
            }
          }
        }
      } else if constexpr (M::KS == 16) {
        unsigned raw[4], a[3][4];
        ldsm_t(raw[0], raw[1], raw[2], raw[3], keys + (k + (lane & 7) + ((lane >> 4) << 3)) * LDK + m0 + (lane & 8));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float* w = wt + k + 2 * t + 8 * (e >> 1);
          const float2 x = unpack_bf16(raw[e]);
          split3(f2(x.x, x.y) * f2(w[0], w[1]), a[0][e], a[1][e], a[2][e]);
        }
#pragma unroll
        for (int n = 0; n < AT; n += 2) {
          if (!FULL && n0 + (at + n) * 8 >= nd) continue;
          typename M::B b[2];
          load_bk<T, CARE>(b, vals + n * 8, LDV, lane);
#pragma unroll
          for (int z = 2; z >= 0; --z) {
            mma_bf16(add[n], a[z], b[0].v);
            mma_bf16(add[n + 1], a[z], b[1].v);
          }
        }
      } else {
        unsigned a[2][4];
        const T* q = keys + (k + 2 * t) * LDK + m0 + (lane >> 2);
        const float w0 = wt[k + 2 * t], w1 = wt[k + 2 * t + 1];
        const float x[4] = {to_f(q[0]) * w0, to_f(q[8]) * w0, to_f(q[LDK]) * w1, to_f(q[LDK + 8]) * w1};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          unsigned r[2];
          pieces<CARE>(x[e], r);
          a[0][e] = r[0];
          a[1][e] = r[1];
        }
#pragma unroll
        for (int n = 0; n < AT; n += 2) {
          if (!FULL && n0 + (at + n) * 8 >= nd) continue;
          typename M::B b[2];
          load_bk<T, CARE>(b, vals + n * 8, LDV, lane);
          mma_pieces(add[n], a, b[0].v);
          mma_pieces(add[n + 1], a, b[1].v);
        }
      }
    }
    if (CARE) add_again<T, C, LDK, LDV, AT>(add, keys, values, wt, faded, m0, n0 + at * 8);
#pragma unroll
    for (int n = 0; n < AT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        st[at + n][e] = CARE ? carried(st[at + n][e], gn, add[n][e], lasts) : fmaf(st[at + n][e], gn, add[n][e]);
  }
}

// Writes a warp's rows.  16-bit: lanes 2 i and 2 i + 1 trade a half of two
// neighbouring tiles, so that four lanes write 32 bytes in a row.
template <typename T, int ON, bool BACK>
GFN_DEV void emit(void* out, const float (&o)[ON][4], const PassArgs& p, int b, int h, int dim, int at, int n, int rt, int col0) {
  const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = rt * 16 + (lane >> 2) + 8 * half;
    T* row = static_cast<T*>(out) + (((long long)b * p.L + (BACK ? at - r : at + r)) * p.H + h) * dim;
    if (sizeof(T) == 2 && dim % 4 == 0) {
#pragma unroll
      for (int i = 0; i < ON; i += 2) {
        unsigned w[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const T two[2] = {from_f<T>(o[i + z][2 * half]), from_f<T>(o[i + z][2 * half + 1])};
          w[z] = *reinterpret_cast<const unsigned*>(two);
        }
        const unsigned other = __shfl_xor_sync(0xffffffffu, t & 1 ? w[0] : w[1], 1);
        const int col = col0 + (i + (t & 1)) * 8 + 2 * (t & 2);
        if (r < n && col < dim) *reinterpret_cast<uint2*>(row + col) = t & 1 ? make_uint2(other, w[1]) : make_uint2(w[0], other);
      }
      continue;
    }
    if (r >= n) continue;
#pragma unroll
    for (int i = 0; i < ON; ++i) {
      const int col = col0 + i * 8 + 2 * t;
      const float lo = o[i][2 * half], hi = o[i][2 * half + 1];
      if (sizeof(T) == 4 && dim % 2 == 0) {
        if (col < dim) *reinterpret_cast<float2*>(row + col) = make_float2(lo, hi);
      } else {
        if (col < dim) row[col] = from_f<T>(lo);
        if (col + 1 < dim) row[col + 1] = from_f<T>(hi);
      }
    }
  }
}

// One thread block walks the blocks of C tokens of one segment of a sequence
// and head, the state in registers (float32), the next block's operands on
// their way.  OUTPUT: rows a, keys b, values c.  STATE: keys b, values c.
// PAIR: with a = q, b = k, c = v, d = do, the outputs dv (rows b, keys a,
// values d) and dk (rows c, keys d, values a) of the state's gradient.  dv and dk in
// one launch share the operands and the state: 32 x 2048 x 8 heads of 64 in bfloat16
// 145 us, where the outputs alone take 106 (256 thread blocks: two an SM, or one).
// Returns whether the segment is to be walked again with CARE.
template <typename T, int DK, int DV, bool BACK, int KIND, bool FULL, bool CARE>
GFN_DEV bool attn_walk(const PassArgs& p) {
  using S = Shape<T, DK, DV>;
  using M = Math<T>;
  using Op = typename M::State;
  constexpr int STAGE = S::stage(KIND), BUFS = S::buffers(KIND), STAGES = S::stages(KIND);
  extern __shared__ __align__(128) char attn_shared[];
  T* stage = reinterpret_cast<T*>(attn_shared);
  Op* st_op = reinterpret_cast<Op*>(stage + STAGES * STAGE);
  float* wt = reinterpret_cast<float*>(attn_shared + STAGES * STAGE * sizeof(T) + BUFS * S::STATE_BYTES);  // [2 C]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int len = length_of(p, b);
  const int from = seg * p.seg_len, to = min(from + p.seg_len, len);
  const float lg = log2_decay(p.decay[h]);
  const bool lasts = p.decay[h] > 0.f;
  // the state's place of this warp
  const int m0 = (warp % S::SLABS) * 16, n0 = (warp / S::SLABS) * S::SN * 8;
  const bool holds = FULL || (m0 < p.KD && n0 < p.VD);
  float st[S::SN][4];
  const long long mat = (long long)p.KD * p.VD, bh = (long long)b * p.H + h;
  const float* init = KIND == STATE ? nullptr : p.segs ? p.segs + (bh * p.segments + seg) * mat : p.state ? p.state + bh * mat : nullptr;
  const long long sr = p.segs ? p.segs_sr : p.sr, sc = p.segs ? p.segs_sc : p.sc;
  auto before = [&](int i, int e) {
    const int row = m0 + (lane >> 2) + 8 * (e >> 1), col = n0 + i * 8 + 2 * (lane & 3) + (e & 1);
    return init && row < p.KD && col < p.VD ? init[row * sr + col * sc] : 0.f;
  };
#pragma unroll
  for (int i = 0; i < S::SN; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) st[i][e] = before(i, e);
  {
    uint4* z = reinterpret_cast<uint4*>(attn_shared);
    for (int i = threadIdx.x; i < (int)((STAGES * STAGE * sizeof(T) + BUFS * S::STATE_BYTES) / 16); i += S::THREADS)
      z[i] = make_uint4(0, 0, 0, 0);
    // place C - 1 - e holds g^e (back: g^(e+1)); rows behind a short block take zeros
    for (int i = threadIdx.x; i < 2 * S::C; i += S::THREADS)
      wt[i] = i < S::C ? p.s_update * power(lg, S::C - 1 - i + (BACK ? 1 : 0)) : 0.f;
  }
  __syncthreads();
  auto bring = [&](int c, T* dst) {
    const int done = c * S::C, n = min(S::C, to - from - done), at = BACK ? to - 1 - done : from + done;
    auto keys = [&](T* d, const View& v) { fetch<T, DK, S::LDK, S::C, S::THREADS, BACK, FULL>(d, v, b, h, p.KD, at, n, p.piece); };
    auto vals = [&](T* d, const View& v) { fetch<T, DV, S::LDV, S::C, S::THREADS, BACK, FULL>(d, v, b, h, p.VD, at, n, p.piece); };
    if (KIND == OUTPUT) {
      keys(dst, p.a);
      keys(dst + S::TK, p.b);
      vals(dst + 2 * S::TK, p.c);
    } else if (KIND == STATE) {
      keys(dst, p.b);
      vals(dst + S::TK, p.c);
    } else {
      keys(dst, p.a);
      keys(dst + S::TK, p.b);
      vals(dst + 2 * S::TK, p.c);
      vals(dst + 2 * S::TK + S::TV, p.d);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto lay_out = [&](Op* q) {  // the state as the products take it
    if (KIND == STATE || !holds) return;
    q += (m0 + (lane >> 2)) * S::LS + n0 + 2 * (lane & 3);
#pragma unroll
    for (int i = 0; i < S::SN; ++i) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float x = st[i][2 * half], y = st[i][2 * half + 1];
        Op* at = q + 8 * half * S::LS + i * 8;
        if constexpr (std::is_same_v<T, __nv_bfloat16>) *reinterpret_cast<unsigned*>(at) = pack_bf16(x, y);
        else if constexpr (std::is_same_v<T, __half>) *reinterpret_cast<uint2*>(at) = make_uint2(tf32(x), tf32(y));
        else *reinterpret_cast<float2*>(at) = make_float2(x, y);
      }
    }
  };
  const int blocks = to > from ? (to - from + S::C - 1) / S::C : 0;
  const int rt = warp % S::ROWS, part = warp / S::ROWS;
  const Decay decay(lg, p.s_in);
  const float whole = power(lg, S::C);
  // forward: row i takes g^(i+1) of the state; back: g^i, as the state's
  // gradient arrives with that factor in it
  const int r0 = rt * 16 + (lane >> 2) + (BACK ? 0 : 1);
  const float w0 = p.s_state * power(lg, r0), w1 = p.s_state * power(lg, r0 + 8);
  constexpr bool WATCH = !CARE && sizeof(T) == 4;
  float watch = 0.f;  // turns NaN
  auto note = [&](const auto& o) {
#pragma unroll
    for (const auto& tile : o)
#pragma unroll
      for (const float x : tile) watch = fmaf(x, 0.f, watch);
  };
  // Whether the state holds NaN or an infinity: one that a token brings stays
  // there.  float32 outputs are watched too, for operands beyond tf32's range.
  auto turned_bad = [&] {
    float t = watch;
#pragma unroll
    for (int i = 0; i < S::SN; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) t = fmaf(st[i][e], 0.f, t);
    return t != 0.f;
  };
  if (blocks) bring(0, stage);
  lay_out(st_op);
  for (int c = 0; c < blocks; ++c) {
    const T* cur = stage + (STAGES == 2 ? (c & 1) * STAGE : 0);
    const Op* op = st_op + (BUFS == 2 ? (c & 1) * DK * S::LS : 0);
    const int done = c * S::C, n = min(S::C, to - from - done), at = BACK ? to - 1 - done : from + done;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // and with it everyone has left the other stage
    if (STAGES == 2 && c + 1 < blocks) bring(c + 1, stage + ((c + 1) & 1) * STAGE);
    auto move_on = [&] {
      const T* uk = KIND == OUTPUT ? cur + S::TK : cur;
      const T* uv = KIND == OUTPUT ? cur + 2 * S::TK : KIND == STATE ? cur + S::TK : cur + 2 * S::TK + S::TV;
      const float gn = n == S::C ? whole : power(lg, n);
      if (holds) update<T, S::C, S::LDK, S::LDV, S::SN, FULL, CARE>(st, uk, uv, wt + S::C - n, gn, m0, n0, p.VD, lasts ? p.s_update : 0.f, lasts);
    };
    if (BUFS == 2) {  // the next block's state, beside the outputs of this one
      move_on();
      lay_out(st_op + ((c + 1) & 1) * DK * S::LS);
    }
    if constexpr (KIND != STATE) {
      constexpr int OV = DV / 8 / S::SPLIT;
      float o[OV][4];
      const int col0 = part * OV * 8;
      if (FULL || col0 < p.VD) {
        if constexpr (KIND == OUTPUT)
          attend<T, S::C, DK, S::LDK, S::LDV, S::LS, OV, false, FULL, CARE>(o, cur, cur + S::TK, cur + 2 * S::TK, op, rt, col0, p.KD, p.VD,
                                                               decay, w0, w1);
        else
          attend<T, S::C, DK, S::LDK, S::LDV, S::LS, OV, false, FULL, CARE>(o, cur + S::TK, cur, cur + 2 * S::TK + S::TV, op, rt, col0, p.KD,
                                                               p.VD, decay, w0, w1);
        if (WATCH) note(o);
        emit<T, OV, BACK>(p.o, o, p, b, h, p.VD, at, n, rt, col0);
      }
    }
    if constexpr (KIND == PAIR) {
      constexpr int OK = DK / 8 / S::SPLIT;
      float o[OK][4];
      const int col0 = part * OK * 8;
      if (FULL || col0 < p.KD) {
        attend<T, S::C, DV, S::LDV, S::LDK, S::LS, OK, true, FULL, CARE>(o, cur + 2 * S::TK, cur + 2 * S::TK + S::TV, cur, op, rt, col0, p.VD,
                                                            p.KD, decay, w0, w1);
        if (WATCH) note(o);
        emit<T, OK, BACK>(p.o2, o, p, b, h, p.KD, at, n, rt, col0);
      }
    }
    if (BUFS < 2) move_on();
    if (BUFS == 1) {
      __syncthreads();
      if (STAGES == 1 && c + 1 < blocks) bring(c + 1, stage);
      lay_out(st_op);
    }
  }
  if (!CARE && __syncthreads_or(turned_bad())) return true;
  // tokens behind the sequence: zeros
  if (KIND != STATE && len < p.L) {
    const int z0 = max(from, len), z1 = min(from + p.seg_len, p.L);
    for (int pass = 0; pass < (KIND == PAIR ? 2 : 1); ++pass) {
      const int dim = pass ? p.KD : p.VD;
      T* y = static_cast<T*>(pass ? p.o2 : p.o);
      for (long long i = threadIdx.x; i < (long long)(z1 - z0) * dim; i += S::THREADS)
        y[(((long long)b * p.L + z0 + i / dim) * p.H + h) * dim + i % dim] = from_f<T>(0.f);
    }
  }
  float* out = KIND == STATE ? p.segs + (bh * p.segments + seg) * mat : p.segs ? nullptr : p.state_out ? p.state_out + bh * mat : nullptr;
  if (out) {
#pragma unroll
    for (int i = 0; i < S::SN; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = m0 + (lane >> 2) + 8 * (e >> 1), col = n0 + i * 8 + 2 * (lane & 3) + (e & 1);
        if (row < p.KD && col < p.VD) out[row * p.VD + col] = st[i][e];
      }
  }
  return false;
}

// Segments of finite tokens are walked once.  Others are walked again, by code of
// its own, so that care (see add_up_to_diagonal, add_again) costs next to nothing on the way:
// 32 x 2048 x 8 heads of 64 in bfloat16, trained, 353 us, and 351 without it; asking
// in the walk which infinities the state came with took 397.
template <typename T, int DK, int DV, bool BACK, int KIND, bool FULL>
__device__ __noinline__ void attn_walk_again(const PassArgs& p) {
  attn_walk<T, DK, DV, BACK, KIND, FULL, true>(p);
}
template <typename T, int DK, int DV, bool BACK, int KIND, bool FULL>
__global__ void __launch_bounds__(Shape<T, DK, DV>::THREADS, Shape<T, DK, DV>::resident(KIND))
    attn_kernel(const __grid_constant__ PassArgs p) {
  if (attn_walk<T, DK, DV, BACK, KIND, FULL, false>(p)) attn_walk_again<T, DK, DV, BACK, KIND, FULL>(p);
}

// The states before each segment, from what each segment adds; in place.  JOIN
// segments' parts are on their way at once.
template <bool BACK, int JOIN>
__global__ void __launch_bounds__(256) attn_join_kernel(const PassArgs p) {
  const int mat = p.KD * p.VD, i = blockIdx.x * 256 + threadIdx.x;
  const long long bh = blockIdx.y + (long long)gridDim.y * blockIdx.z;
  if (i >= mat || bh >= (long long)p.B * p.H) return;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H), len = length_of(p, b);
  const float lg = log2_decay(p.decay[h]);
  const bool lasts = p.decay[h] > 0.f;
  const int row = i / p.VD, col = i % p.VD;
  float s = p.state ? p.state[bh * mat + row * p.sr + col * p.sc] : 0.f;
  float* q = p.segs + bh * p.segments * mat + i;
  const float whole = power(lg, p.seg_len);
  for (int k0 = 0; k0 < p.segments; k0 += JOIN) {
    float add[JOIN];
#pragma unroll
    for (int u = 0; u < JOIN; ++u) {
      const int k = BACK ? p.segments - 1 - k0 - u : k0 + u;
      add[u] = k0 + u < p.segments ? q[(long long)k * mat] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < JOIN; ++u) {
      if (k0 + u >= p.segments) continue;
      const int k = BACK ? p.segments - 1 - k0 - u : k0 + u;
      const int n = min(max(len - k * p.seg_len, 0), p.seg_len);
      q[(long long)k * mat] = s;
      s = carried(s, n == p.seg_len ? whole : power(lg, n), add[u], lasts);
    }
  }
  if (p.state_out) p.state_out[bh * mat + i] = s;
}

// The same for many segments of few heads: a warp has 32 cells of the state over
// an eighth of the segments, whose maps s -> g^n s + add are composed, handed on
// and then applied one by one.
template <bool BACK>
__global__ void __launch_bounds__(256) attn_join_long_kernel(const PassArgs p) {
  constexpr int PARTS = 8, AHEAD = 8;
  __shared__ float sums[PARTS][32], gains[PARTS];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int mat = p.KD * p.VD, i = blockIdx.x * 32 + lane;
  const long long bh = blockIdx.y + (long long)gridDim.y * blockIdx.z;
  if (bh >= (long long)p.B * p.H) return;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H), len = length_of(p, b);
  const float lg = log2_decay(p.decay[h]), whole = power(lg, p.seg_len);
  const bool lasts = p.decay[h] > 0.f;
  const bool live = i < mat;
  float* q = p.segs + bh * p.segments * mat + i;
  auto place = [&](int k) { return BACK ? p.segments - 1 - k : k; };
  auto tokens = [&](int k) { return min(max(len - place(k) * p.seg_len, 0), p.seg_len); };
  auto gain = [&](int k) {
    const int n = tokens(k);
    return n == p.seg_len ? whole : power(lg, n);
  };
  const int per = (p.segments + PARTS - 1) / PARTS, from = min(part * per, p.segments), to = min(from + per, p.segments);
  float add[AHEAD], s = 0.f, g = 1.f;
  auto read = [&](int k0) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) add[u] = live && k0 + u < to ? q[(long long)place(k0 + u) * mat] : 0.f;
  };
  for (int k0 = from; k0 < to; k0 += AHEAD) {
    read(k0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (k0 + u >= to) continue;
      const float w = gain(k0 + u);
      s = carried(s, w, add[u], lasts);
      g *= w;
    }
  }
  sums[part][lane] = s;
  if (lane == 0) gains[part] = g;
  __syncthreads();
  if (!live) return;
  const int row = i / p.VD, col = i % p.VD;
  s = p.state ? p.state[bh * mat + row * p.sr + col * p.sc] : 0.f;
  for (int r = 0; r < part; ++r) s = carried(s, gains[r], sums[r][lane], lasts);
  for (int k0 = from; k0 < to; k0 += AHEAD) {
    read(k0);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (k0 + u >= to) continue;
      q[(long long)place(k0 + u) * mat] = s;
      s = carried(s, gain(k0 + u), add[u], lasts);
    }
  }
  if (part == PARTS - 1 && p.state_out) p.state_out[bh * mat + i] = s;
}

// One token: the state is read, moved on and written once.  A thread owns VEC
// columns of every `groups`-th row, and AT rows are on their way at once, the
// first ones beside the token's q, k and v.  64 x 8 heads of 64: 5.5 us, of which the
// 17 MB would take 2.6 (7.4 with the state read after them).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) attn_step_kernel(const PassArgs p) {
  constexpr int AT = 4;
  __shared__ float q[128], k[128], sum[256 * VEC];
  struct alignas(4 * VEC) Cells {
    float c[VEC];
  };
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H;
  const long long mat = (long long)p.KD * p.VD, bh = (long long)b * p.H + h;
  const int cols = p.VD / VEC, groups = 256 / cols, mine = threadIdx.x % cols, group = threadIdx.x / cols;
  const int rows = group < groups ? p.KD : 0;  // the last threads may be left over
  const float* in = p.state ? p.state + bh * mat + mine * VEC : nullptr;
  float* out = p.state_out ? p.state_out + bh * mat + mine * VEC : nullptr;
  Cells s[AT];
  auto read = [&](int r0) {
#pragma unroll
    for (int u = 0; u < AT; ++u) {
      const int r = r0 + u * groups;
      s[u] = {};
      if (in && r < rows) s[u] = *reinterpret_cast<const Cells*>(in + r * p.VD);
    }
  };
  read(group);
  const bool live = length_of(p, b) > 0;
  float g = p.decay[h];
  g = g > 1.f ? 1.f : g < 0.f ? 0.f : g;
  auto at = [&](const View& v) { return static_cast<const T*>(v.p) + b * v.sb + h * v.sh; };
  if ((int)threadIdx.x < p.KD) {
    q[threadIdx.x] = live ? to_f(at(p.a)[threadIdx.x]) * p.s_state : 0.f;
    k[threadIdx.x] = live ? to_f(at(p.b)[threadIdx.x]) : 0.f;
  }
  float v[VEC], acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    v[e] = live ? to_f(at(p.c)[mine * VEC + e]) : 0.f;
    acc[e] = 0.f;
  }
  __syncthreads();
  for (int r0 = group; r0 < rows; r0 += AT * groups) {
    if (r0 != group) read(r0);
#pragma unroll
    for (int u = 0; u < AT; ++u) {
      const int r = r0 + u * groups;
      if (r >= rows) continue;
      if (live) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s[u].c[e] = fmaf(g, s[u].c[e], k[r] * v[e]);
          acc[e] = fmaf(q[r], s[u].c[e], acc[e]);
        }
      }
      if (out) *reinterpret_cast<Cells*>(out + r * p.VD) = s[u];
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[threadIdx.x * VEC + e] = acc[e];
  __syncthreads();
  for (int c = threadIdx.x; c < p.VD; c += 256) {
    float t = 0.f;
#pragma unroll 8
    for (int r = 0; r < groups; ++r) t += sum[r * p.VD + c];
    static_cast<T*>(p.o)[bh * p.VD + c] = from_f<T>(t);
  }
}

// ------------------------------------------------------------------ launches
// FULL: heads as wide as the kernel, and all operands in 16-byte pieces.
template <typename T, int DK, int DV, bool BACK, int KIND, bool FULL>
int attn_launch(const PassArgs& p, cudaStream_t s) {
  using S = Shape<T, DK, DV>;
  static std::atomic<unsigned long long> done;
  const int bytes = S::bytes(KIND);
  const int st = shared_limit(attn_kernel<T, DK, DV, BACK, KIND, FULL>, bytes, &done, "attn_kernel");
  if (st != GFN_OK) return st;
  attn_kernel<T, DK, DV, BACK, KIND, FULL><<<dim3(p.segments, p.H, p.B), S::THREADS, bytes, s>>>(p);
  return launch_status("attn_kernel");
}
template <typename T, int DK, int DV, bool BACK, int KIND>
int attn_run(const PassArgs& p, cudaStream_t s) {
  return p.piece == 16 && p.KD == DK && p.VD == DV ? attn_launch<T, DK, DV, BACK, KIND, true>(p, s)
                                           : attn_launch<T, DK, DV, BACK, KIND, false>(p, s);
}

template <typename T, int DK, int DV, bool BACK, int KIND>
int attn_pass(PassArgs p, bool known, cudaStream_t s) {
  if (p.segments == 1) p.segs = nullptr;
  else if (!known) {
    PassArgs w = p;
    if (KIND == PAIR) {  // the state's rows are q's, its columns do's
      w.b = p.a;
      w.c = p.d;
    }
    int st = attn_run<T, DK, DV, BACK, STATE>(w, s);
    if (st != GFN_OK) return st;
    const int bh = p.B * p.H, y = bh < 32768 ? bh : 32768;
    // one head, 342 segments of 64 x 64: 22 us by one thread a cell, 12 by eight;
    // 40 heads, 3 segments of 128 x 128: 97 by eight, by one 20 with 4 parts
    // under way and 43 with 32; 8 heads, 54 segments: 7.5 with 16, 6.3 with 32
    const bool many = p.segments > 96;
    const dim3 grid((unsigned)((p.KD * p.VD + (many ? 31 : 255)) / (many ? 32 : 256)), y, (bh + y - 1) / y);
    if (many) attn_join_long_kernel<BACK><<<grid, 256, 0, s>>>(w);
    else if (p.segments <= 4) attn_join_kernel<BACK, 4><<<grid, 256, 0, s>>>(w);
    else if (p.segments <= 16) attn_join_kernel<BACK, 16><<<grid, 256, 0, s>>>(w);
    else attn_join_kernel<BACK, 32><<<grid, 256, 0, s>>>(w);
    if ((st = launch_status("attn_join_kernel")) != GFN_OK) return st;
  }
  return attn_run<T, DK, DV, BACK, KIND>(p, s);
}

template <typename T, bool BACK, int KIND>
int attn_dims(const PassArgs& p, bool known, cudaStream_t s) {
  const Dims d = padded(p.KD, p.VD);
  if (d.k == 32) return attn_pass<T, 32, 32, BACK, KIND>(p, known, s);
  if (d.k == 64 && d.v == 64) return attn_pass<T, 64, 64, BACK, KIND>(p, known, s);
  if (d.k == 64) return attn_pass<T, 64, 128, BACK, KIND>(p, known, s);
  if (d.v == 64) return attn_pass<T, 128, 64, BACK, KIND>(p, known, s);
  return attn_pass<T, 128, 128, BACK, KIND>(p, known, s);
}

template <typename T>
int attn_step(const PassArgs& p, cudaStream_t s) {
  const unsigned blocks = (unsigned)(p.B * p.H);
  const bool vec = p.VD % 4 == 0 && (!p.state || aligned16(p.state)) && (!p.state_out || aligned16(p.state_out));
  if (vec) attn_step_kernel<T, 4><<<blocks, 256, 0, s>>>(p);
  else attn_step_kernel<T, 1><<<blocks, 256, 0, s>>>(p);
  return launch_status("attn_step_kernel");
}

template <typename T>
int attn_resident(Kind kind, int kd, int vd) {
  const Dims d = padded(kd, vd);
  if (d.k == 32) return Shape<T, 32, 32>::resident(kind);
  if (d.k == 64) return d.v == 64 ? Shape<T, 64, 64>::resident(kind) : Shape<T, 64, 128>::resident(kind);
  return d.v == 64 ? Shape<T, 128, 64>::resident(kind) : Shape<T, 128, 128>::resident(kind);
}

}  // namespace gfn_attn
