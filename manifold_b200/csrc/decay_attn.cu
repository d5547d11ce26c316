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
#include "lm_host.h"
#include "lm_ops.cuh"

using namespace gfn;
using namespace gfn_abi;

namespace {

struct View {  // [batch][length][heads][dim], inner stride 1
  const void* p;
  long long sb, sl, sh;
};

struct PassArgs {
  View a, b, c, d;      // rows; keys; values; in the two-output pass also d (see attn_kernel)
  void* o;              // [B][L][H][c.dim]
  void* o2;
  const float* decay;
  const float* state;   // before the first token, or nullptr
  float* state_out;     // after the last, or nullptr
  float* segs;          // [B * H][segments][KD][VD]: states by segment, or nullptr (one segment)
  const void* lengths;
  int lengths64;
  int B, L, H, KD, VD;  // dims of the state's rows (keys) and columns (values)
  long long sr, sc;     // strides of the state's rows and columns
  int seg_len, segments;
  float s_in, s_state, s_update;  // factors of the products within a block, with the state, and of the state's update
  int vec;              // operands arrive in 16-byte pieces
};

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
// bfloat16: m16n8k16.  tf32: m16n8k8, where place t of the contraction is its
// element 2 t and place t + 4 its element 2 t + 1 on both sides, so that two
// neighbours are read at once and accumulators serve as operands as they are.
template <typename T>
struct Math {
  static constexpr int KS = 8, PIECES = sizeof(T) == 4 ? 2 : 1;
  using State = float;
  static constexpr int PAD = sizeof(T) == 4 ? 4 : 8, STATE_PAD = 4;
  struct A {
    unsigned v[PIECES][4];
  };
  struct B {
    unsigned v[PIECES][2];
  };
};
template <>
struct Math<__nv_bfloat16> {
  static constexpr int KS = 16;
  using State = __nv_bfloat16;
  static constexpr int PAD = 8, STATE_PAD = 8;
  struct A {
    unsigned v[4];
  };
  struct B {
    unsigned v[2];
  };
};

GFN_DEV void mma_bf16(float (&c)[4], const unsigned (&a)[4], const unsigned (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
template <int N>
GFN_DEV void pieces(float v, unsigned (&r)[N]) {
  r[0] = tf32(v);
  if constexpr (N > 1) r[1] = tf32(v - __uint_as_float(r[0]));
}

template <int PA, int PB>
GFN_DEV void mma_pieces(float (&c)[4], const unsigned (&a)[PA][4], const unsigned (&b)[PB][2]) {
  if constexpr (PA > 1) mma_tf32(c, a[1], b[0]);
  if constexpr (PB > 1) mma_tf32(c, a[0], b[1]);
  mma_tf32(c, a[0], b[0]);
}
template <typename T>
GFN_DEV void mma(float (&c)[4], const typename Math<T>::A& a, const typename Math<T>::B& b) {
  if constexpr (Math<T>::KS == 16) mma_bf16(c, a.v, b.v);
  else mma_pieces(c, a.v, b.v);
}

GFN_DEV void ldsm(unsigned& a, unsigned& b, unsigned& c, unsigned& d, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(smem_u32(p)) : "memory");
}
GFN_DEV void ldsm_t(unsigned& a, unsigned& b, unsigned& c, unsigned& d, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(smem_u32(p)) : "memory");
}
GFN_DEV float2 pair(const float* p) { return *reinterpret_cast<const float2*>(p); }
GFN_DEV float2 pair(const __half* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }

// A, 16 rows from p [row][k].
template <typename T>
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
      pieces(w[i], r);
#pragma unroll
      for (int k = 0; k < Math<T>::PIECES; ++k) f.v[k][i] = r[k];
    }
  }
}
// Two neighbouring B of 8 columns each, from p [n][k].
template <typename T, typename E>
GFN_DEV void load_bn(typename Math<T>::B (&f)[2], const E* p, int ld, int lane) {
  if constexpr (Math<T>::KS == 16) {
    ldsm(f[0].v[0], f[0].v[1], f[1].v[0], f[1].v[1], p + ((lane & 7) + ((lane >> 4) << 3)) * ld + (lane & 8));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 x = pair(p + ((lane >> 2) + 8 * h) * ld + 2 * (lane & 3));
      unsigned r[2][Math<T>::PIECES];
      pieces(x.x, r[0]);
      pieces(x.y, r[1]);
#pragma unroll
      for (int k = 0; k < Math<T>::PIECES; ++k) {
        f[h].v[k][0] = r[0][k];
        f[h].v[k][1] = r[1][k];
      }
    }
  }
}
// The same from p [k][n].
template <typename T, typename E>
GFN_DEV void load_bk(typename Math<T>::B (&f)[2], const E* p, int ld, int lane) {
  if constexpr (Math<T>::KS == 16) {
    ldsm_t(f[0].v[0], f[0].v[1], f[1].v[0], f[1].v[1], p + ((lane & 7) + (lane & 8)) * ld + ((lane >> 4) << 3));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const E* q = p + 2 * (lane & 3) * ld + (lane >> 2) + 8 * h;
      unsigned r[2][Math<T>::PIECES];
      pieces(to_f(q[0]), r[0]);
      pieces(to_f(q[ld]), r[1]);
#pragma unroll
      for (int k = 0; k < Math<T>::PIECES; ++k) {
        f[h].v[k][0] = r[0][k];
        f[h].v[k][1] = r[1][k];
      }
    }
  }
}

GFN_DEV unsigned pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}
GFN_DEV float2 unpack_bf16(unsigned v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }

// ------------------------------------------------------------------- blocks
// Tokens per block and warps: the two stages of operands and the state's
// operand form share an SM's memory with two or three other thread blocks.
template <typename T, int D>
struct Shape {
  static constexpr int W = D == 128 ? 8 : 4, THREADS = 32 * W;
  static constexpr int C = sizeof(T) == 4 && D >= 64 ? 32 : 64;
  static constexpr int LD = D + Math<T>::PAD, LS = D + Math<T>::STATE_PAD;
  static constexpr int ROWS = C / 16, SPLIT = W / ROWS, ON = D / 8 / SPLIT;      // row tiles; output tiles of a warp
  static constexpr int SLABS = D / 16, SN = D / 8 / (W / SLABS > 0 ? W / SLABS : 1);  // the state's rows; its tiles of a warp
  static constexpr int TILE = C * LD;  // elements of one operand
  static int bytes(int operands, bool state) {
    return 2 * operands * TILE * (int)sizeof(T) + (state ? D * LS * (int)sizeof(typename Math<T>::State) : 0) + 4 * C;
  }
};

// Token of row r of a block whose first row (in the pass's order) is token `at`.
template <bool BACK>
GFN_DEV int token_of(int at, int r) { return BACK ? at - r : at + r; }

// Brings rows 0 .. n - 1 of a block into shared memory, zeros behind them.
// Columns from `dim` on were zeroed once and stay so.
template <typename T, int D, bool BACK>
GFN_DEV void fetch(T* dst, const View& v, int b, int h, int dim, int at, int n, int vec) {
  using S = Shape<T, D>;
  const T* src = static_cast<const T*>(v.p) + b * v.sb + h * v.sh;
  if (vec) {
    constexpr int PER = 16 / sizeof(T), LANES = D / PER, STEP = S::THREADS / LANES;
    const int col = (threadIdx.x % LANES) * PER;
    if (col >= dim) return;
#pragma unroll
    for (int r = threadIdx.x / LANES; r < S::C; r += STEP) {
      const T* from = src + (r < n ? (long long)token_of<BACK>(at, r) * v.sl + col : 0);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * S::LD + col)), "l"(from),
                   "r"(r < n ? 16 : 0)
                   : "memory");
    }
  } else {
    for (int i = threadIdx.x; i < S::C * D; i += S::THREADS) {
      const int r = i / D, col = i % D;
      if (col < dim) dst[r * S::LD + col] = r < n ? src[(long long)token_of<BACK>(at, r) * v.sl + col] : from_f<T>(0.f);
    }
  }
}

// One warp's 16 rows of a block's output, ON tiles of 8 columns from col0.
// rows, keys, values: [C][LD]; st: the state, [K][V] or (NMAJOR) [V][K] seen
// from this product.
template <typename T, int D, bool NMAJOR>
GFN_DEV void attend(float (&o)[Shape<T, D>::ON][4], const T* rows, const T* keys, const T* values,
                    const typename Math<T>::State* st, int rt, int col0, float lg, float s_in, float w0, float w1) {
  using S = Shape<T, D>;
  using M = Math<T>;
  const int lane = threadIdx.x & 31;
  float s[S::C / 8][4];
#pragma unroll
  for (int i = 0; i < S::C / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
  for (int i = 0; i < S::ON; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
#pragma unroll
  for (int k = 0; k < D; k += M::KS) {
    typename M::A a;
    load_a<T>(a, rows + rt * 16 * S::LD + k, S::LD, lane);
#pragma unroll
    for (int i = 0; i < S::ON; i += 2) {
      typename M::B b[2];
      const int col = col0 + i * 8;
      if (NMAJOR) load_bn<T>(b, st + col * S::LS + k, S::LS, lane);
      else load_bk<T>(b, st + k * S::LS + col, S::LS, lane);
      mma<T>(o[i], a, b[0]);
      mma<T>(o[i + 1], a, b[1]);
    }
#pragma unroll
    for (int i = 0; i < S::C / 16; ++i) {
      if (i > rt) continue;  // keys behind the rows
      typename M::B b[2];
      load_bn<T>(b, keys + i * 16 * S::LD + k, S::LD, lane);
      mma<T>(s[2 * i], a, b[0]);
      mma<T>(s[2 * i + 1], a, b[1]);
    }
  }
#pragma unroll
  for (int i = 0; i < S::ON; ++i) {
    o[i][0] *= w0;
    o[i][1] *= w0;
    o[i][2] *= w1;
    o[i][3] *= w1;
  }
  // g^(i-j): by powers on the two tiles that the diagonal crosses and on the
  // one before them, by a factor of g^8 from tile to tile further back
  const int gap = (lane >> 2) - 2 * (lane & 3);
  const float g8 = exp2_fast(8.f * lg);
  float f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = s_in * exp2_fast((float)(gap + 8 + 8 * (e >> 1) - (e & 1)) * lg);
#pragma unroll
  for (int i = S::C / 8 - 1; i >= 0; --i) {
    const int off = 2 * rt - i;  // -1, 0: the diagonal's tiles
    if (off < -1) continue;
    if (off > 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] *= f[e];
        f[e] *= g8;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = gap + 8 * off + 8 * (e >> 1) - (e & 1);
        s[i][e] = d < 0 ? 0.f : s[i][e] * (s_in * exp2_fast((float)d * lg));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < S::C / 16; ++i) {
    if (i > rt) continue;
#pragma unroll
    for (int q = 0; q < 16 / M::KS; ++q) {
      typename M::A a;
      if constexpr (M::KS == 16) {
        a.v[0] = pack_bf16(s[2 * i][0], s[2 * i][1]);
        a.v[1] = pack_bf16(s[2 * i][2], s[2 * i][3]);
        a.v[2] = pack_bf16(s[2 * i + 1][0], s[2 * i + 1][1]);
        a.v[3] = pack_bf16(s[2 * i + 1][2], s[2 * i + 1][3]);
      } else {
        const float w[4] = {s[2 * i + q][0], s[2 * i + q][2], s[2 * i + q][1], s[2 * i + q][3]};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          unsigned r[M::PIECES];
          pieces(w[e], r);
#pragma unroll
          for (int z = 0; z < M::PIECES; ++z) a.v[z][e] = r[z];
        }
      }
      const T* v = values + (16 * i + M::KS * q) * S::LD + col0;
#pragma unroll
      for (int n = 0; n < S::ON; n += 2) {
        typename M::B b[2];
        load_bk<T>(b, v + n * 8, S::LD, lane);
        mma<T>(o[n], a, b[0]);
        mma<T>(o[n + 1], a, b[1]);
      }
    }
  }
}

// st += (diag(wt) keys)^T values for one warp's 16 rows (from m0) and SN tiles
// of columns (from n0) of the state.
template <typename T, int D>
GFN_DEV void update(float (&st)[Shape<T, D>::SN][4], const T* keys, const T* values, const float* wt, int m0, int n0) {
  using S = Shape<T, D>;
  using M = Math<T>;
  const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
  for (int k = 0; k < S::C; k += M::KS) {
    if constexpr (M::KS == 16) {
      unsigned raw[4], a[3][4];
      ldsm_t(raw[0], raw[1], raw[2], raw[3], keys + (k + (lane & 7) + ((lane >> 4) << 3)) * S::LD + m0 + (lane & 8));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 w = *reinterpret_cast<const float2*>(wt + k + 2 * t + 8 * (e >> 1));
        float2 x = unpack_bf16(raw[e]);
        x.x *= w.x;
        x.y *= w.y;
#pragma unroll
        for (int z = 0; z < 3; ++z) {
          a[z][e] = pack_bf16(x.x, x.y);
          const float2 h = unpack_bf16(a[z][e]);
          x.x -= h.x;
          x.y -= h.y;
        }
      }
#pragma unroll
      for (int n = 0; n < S::SN; n += 2) {
        typename M::B b[2];
        load_bk<T>(b, values + k * S::LD + n0 + n * 8, S::LD, lane);
#pragma unroll
        for (int z = 2; z >= 0; --z) {
          mma_bf16(st[n], a[z], b[0].v);
          mma_bf16(st[n + 1], a[z], b[1].v);
        }
      }
    } else {
      unsigned a[2][4];
      const T* q = keys + (k + 2 * t) * S::LD + m0 + (lane >> 2);
      const float2 w = *reinterpret_cast<const float2*>(wt + k + 2 * t);
      const float x[4] = {to_f(q[0]) * w.x, to_f(q[8]) * w.x, to_f(q[S::LD]) * w.y, to_f(q[S::LD + 8]) * w.y};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        unsigned r[2];
        pieces(x[e], r);
        a[0][e] = r[0];
        a[1][e] = r[1];
      }
#pragma unroll
      for (int n = 0; n < S::SN; n += 2) {
        typename M::B b[2];
        load_bk<T>(b, values + k * S::LD + n0 + n * 8, S::LD, lane);
        mma_pieces(st[n], a, b[0].v);
        mma_pieces(st[n + 1], a, b[1].v);
      }
    }
  }
}

template <typename T, int D, bool BACK>
GFN_DEV void emit(void* out, const float (&o)[Shape<T, D>::ON][4], const PassArgs& p, int b, int h, int dim, int at, int n, int rt,
                  int col0) {
  using S = Shape<T, D>;
  const int lane = threadIdx.x & 31;
  T* y = static_cast<T*>(out);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = rt * 16 + (lane >> 2) + 8 * half;
    if (r >= n) continue;
    T* row = y + (((long long)b * p.L + token_of<BACK>(at, r)) * p.H + h) * dim;
#pragma unroll
    for (int i = 0; i < S::ON; ++i) {
      const int col = col0 + i * 8 + 2 * (lane & 3);
      const float lo = o[i][2 * half], hi = o[i][2 * half + 1];
      if (dim % 2 == 0) {
        if (col < dim) {
          if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(row + col) = make_float2(lo, hi);
          else {
            T two[2] = {from_f<T>(lo), from_f<T>(hi)};
            *reinterpret_cast<unsigned*>(row + col) = *reinterpret_cast<const unsigned*>(two);
          }
        }
      } else {
        if (col < dim) row[col] = from_f<T>(lo);
        if (col + 1 < dim) row[col + 1] = from_f<T>(hi);
      }
    }
  }
}

// What a launch does: a segment's output, its part of the state alone, or the
// two outputs dv (rows b = k, keys a = q, values d = do) and dk (rows c = v,
// keys d, values a) of the backward pass.
enum Kind { OUTPUT, STATE, PAIR };

// One thread block walks the blocks of C tokens of one segment of a sequence
// and head, the state in registers (float32), the next block's operands on
// their way.
template <typename T, int D, bool BACK, int KIND>
__global__ void __launch_bounds__(Shape<T, D>::THREADS) attn_kernel(const PassArgs p) {
  using S = Shape<T, D>;
  using M = Math<T>;
  constexpr int OPS = KIND == STATE ? 2 : KIND == OUTPUT ? 3 : 4;
  extern __shared__ __align__(128) char attn_shared[];
  T* stage = reinterpret_cast<T*>(attn_shared);  // [2][OPS][TILE]
  typename M::State* st_op = reinterpret_cast<typename M::State*>(stage + 2 * OPS * S::TILE);
  float* wt = reinterpret_cast<float*>(attn_shared + 2 * OPS * S::TILE * sizeof(T) +
                                       (KIND == STATE ? 0 : D * S::LS * sizeof(typename M::State)));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seg = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int len = length_of(p, b);
  const int from = seg * p.seg_len, to = min(from + p.seg_len, len);
  const float lg = log2_decay(p.decay[h]);
  // the state's place of this warp
  const int m0 = (warp % S::SLABS) * 16, n0 = (warp / S::SLABS) * S::SN * 8;
  float st[S::SN][4];
  const long long mat = (long long)p.KD * p.VD, bh = (long long)b * p.H + h;
  const float* init = KIND == STATE ? nullptr : p.segs ? p.segs + (bh * p.segments + seg) * mat : p.state ? p.state + bh * mat : nullptr;
  const long long sr = p.segs ? p.VD : p.sr, sc = p.segs ? 1 : p.sc;
#pragma unroll
  for (int i = 0; i < S::SN; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = m0 + (lane >> 2) + 8 * (e >> 1), col = n0 + i * 8 + 2 * (lane & 3) + (e & 1);
      st[i][e] = init && row < p.KD && col < p.VD ? init[row * sr + col * sc] : 0.f;
    }
  }
  {
    uint4* z = reinterpret_cast<uint4*>(attn_shared);
    for (int i = threadIdx.x; i < (int)(2 * OPS * S::TILE * sizeof(T) / 16); i += S::THREADS) z[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  auto bring = [&](int c, T* dst) {
    const int done = c * S::C, n = min(S::C, to - from - done), at = BACK ? to - 1 - done : from + done;
    if (KIND == OUTPUT) {
      fetch<T, D, BACK>(dst, p.a, b, h, p.KD, at, n, p.vec);
      fetch<T, D, BACK>(dst + S::TILE, p.b, b, h, p.KD, at, n, p.vec);
      fetch<T, D, BACK>(dst + 2 * S::TILE, p.c, b, h, p.VD, at, n, p.vec);
    } else if (KIND == STATE) {
      fetch<T, D, BACK>(dst, p.b, b, h, p.KD, at, n, p.vec);
      fetch<T, D, BACK>(dst + S::TILE, p.c, b, h, p.VD, at, n, p.vec);
    } else {
      fetch<T, D, BACK>(dst, p.a, b, h, p.KD, at, n, p.vec);
      fetch<T, D, BACK>(dst + S::TILE, p.b, b, h, p.KD, at, n, p.vec);
      fetch<T, D, BACK>(dst + 2 * S::TILE, p.c, b, h, p.VD, at, n, p.vec);
      fetch<T, D, BACK>(dst + 3 * S::TILE, p.d, b, h, p.VD, at, n, p.vec);
    }
  };
  const int blocks = to > from ? (to - from + S::C - 1) / S::C : 0;
  if (blocks) bring(0, stage);
  asm volatile("cp.async.commit_group;" ::: "memory");
  const int rt = warp % S::ROWS, col0 = (warp / S::ROWS) * S::ON * 8;
  // forward: row i takes g^(i+1) of the state; back: g^i, as the state's
  // gradient arrives with that factor in it
  const int r0 = rt * 16 + (lane >> 2) + (BACK ? 0 : 1);
  const float w0 = p.s_state * power(lg, r0), w1 = p.s_state * power(lg, r0 + 8);
  for (int c = 0; c < blocks; ++c) {
    T* cur = stage + (c & 1) * OPS * S::TILE;
    const int done = c * S::C, n = min(S::C, to - from - done), at = BACK ? to - 1 - done : from + done;
    if (KIND != STATE) {
#pragma unroll
      for (int i = 0; i < S::SN; ++i) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          typename M::State* q = st_op + (m0 + (lane >> 2) + 8 * half) * S::LS + n0 + i * 8 + 2 * (lane & 3);
          if constexpr (M::KS == 16) *reinterpret_cast<unsigned*>(q) = pack_bf16(st[i][2 * half], st[i][2 * half + 1]);
          else *reinterpret_cast<float2*>(q) = make_float2(st[i][2 * half], st[i][2 * half + 1]);
        }
      }
    }
    if (threadIdx.x < S::C) {
      const int e = n - 1 - (int)threadIdx.x;
      wt[threadIdx.x] = e < 0 ? 0.f : p.s_update * power(lg, BACK ? e + 1 : e);
    }
    if (c + 1 < blocks) bring(c + 1, stage + ((c + 1) & 1) * OPS * S::TILE);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    if constexpr (KIND == OUTPUT) {
      float o[S::ON][4];
      attend<T, D, false>(o, cur, cur + S::TILE, cur + 2 * S::TILE, st_op, rt, col0, lg, p.s_in, w0, w1);
      emit<T, D, BACK>(p.o, o, p, b, h, p.VD, at, n, rt, col0);
    } else if constexpr (KIND == PAIR) {
      float o[S::ON][4];
      attend<T, D, false>(o, cur + S::TILE, cur, cur + 3 * S::TILE, st_op, rt, col0, lg, p.s_in, w0, w1);
      emit<T, D, BACK>(p.o, o, p, b, h, p.VD, at, n, rt, col0);
      attend<T, D, true>(o, cur + 2 * S::TILE, cur + 3 * S::TILE, cur, st_op, rt, col0, lg, p.s_in, w0, w1);
      emit<T, D, BACK>(p.o2, o, p, b, h, p.KD, at, n, rt, col0);
    }
    const float gn = power(lg, n);
#pragma unroll
    for (int i = 0; i < S::SN; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) st[i][e] *= gn;
    const T* uk = KIND == OUTPUT ? cur + S::TILE : cur;
    const T* uv = KIND == OUTPUT ? cur + 2 * S::TILE : KIND == STATE ? cur + S::TILE : cur + 3 * S::TILE;
    update<T, D>(st, uk, uv, wt, m0, n0);
    __syncthreads();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
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
        if (row < p.KD && col < p.VD) out[(long long)row * p.VD + col] = st[i][e];
      }
  }
}

// The states before each segment, from what each segment adds; in place.
template <bool BACK>
__global__ void __launch_bounds__(256) attn_join_kernel(const PassArgs p) {
  const long long mat = (long long)p.KD * p.VD, i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int bh = blockIdx.y + gridDim.y * blockIdx.z;
  if (i >= mat || bh >= p.B * p.H) return;
  const int b = bh / p.H, h = bh % p.H, len = length_of(p, b);
  const float lg = log2_decay(p.decay[h]);
  const int row = (int)(i / p.VD), col = (int)(i % p.VD);
  float s = p.state ? p.state[bh * mat + row * p.sr + col * p.sc] : 0.f;
  float* q = p.segs + (long long)bh * p.segments * mat + i;
  const float whole = power(lg, p.seg_len);
  for (int k0 = 0; k0 < p.segments; k0 += 8) {
    float add[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int k = BACK ? p.segments - 1 - k0 - u : k0 + u;
      add[u] = k0 + u < p.segments ? q[k * mat] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (k0 + u >= p.segments) continue;
      const int k = BACK ? p.segments - 1 - k0 - u : k0 + u;
      const int n = min(max(len - k * p.seg_len, 0), p.seg_len);
      q[k * mat] = s;
      s = fmaf(n == p.seg_len ? whole : power(lg, n), s, add[u]);
    }
  }
  if (p.state_out) p.state_out[bh * mat + i] = s;
}

// One token: the state is read, moved on and written once.  A thread owns VEC
// columns of every RG-th row.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) attn_step_kernel(const PassArgs p) {
  __shared__ float q[128], k[128], sum[256 * VEC];
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H;
  const long long mat = (long long)p.KD * p.VD, bh = (long long)b * p.H + h;
  const bool live = length_of(p, b) > 0;
  const float gam = fminf(fmaxf(p.decay[h], 0.f), 1.f), g = p.decay[h] != p.decay[h] ? p.decay[h] : gam;
  auto at = [&](const View& v) { return static_cast<const T*>(v.p) + b * v.sb + h * v.sh; };
  const int cols = p.VD / VEC, groups = 256 / cols, mine = threadIdx.x % cols, group = threadIdx.x / cols;
  if (threadIdx.x < p.KD) {
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
  struct alignas(4 * VEC) Cells {
    float c[VEC];
  };
  if (group < groups) {
#pragma unroll 4
    for (int r = group; r < p.KD; r += groups) {
      Cells s = {};
      if (p.state) s = *reinterpret_cast<const Cells*>(p.state + bh * mat + (long long)r * p.VD + mine * VEC);
      if (live) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s.c[e] = fmaf(g, s.c[e], k[r] * v[e]);
          acc[e] = fmaf(q[r], s.c[e], acc[e]);
        }
      }
      if (p.state_out) *reinterpret_cast<Cells*>(p.state_out + bh * mat + (long long)r * p.VD + mine * VEC) = s;
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[threadIdx.x * VEC + e] = acc[e];
  __syncthreads();
  for (int c = threadIdx.x; c < p.VD; c += 256) {
    float t = 0.f;
    for (int r = 0; r < groups; ++r) t += sum[(r * cols + c / VEC) * VEC + c % VEC];
    static_cast<T*>(p.o)[bh * p.VD + c] = from_f<T>(t);
  }
}

// --------------------------------------------------------------------- host
constexpr int SEG_UNIT = 64;

// Tokens of a segment: sequences are cut where they are too few to fill the
// device, into as many parts as give it three thread blocks per SM, of four
// blocks of tokens at least.
void attn_segments(int B, int L, int H, int sms, int* seg_len, int* segments) {
  const long long want = (3LL * sms + (long long)B * H - 1) / ((long long)B * H);
  const long long units = (L + SEG_UNIT - 1) / SEG_UNIT;
  long long n = units / 4;
  if (n > want) n = want;
  if (n < 1) n = 1;
  const long long per = (units + n - 1) / n;
  *seg_len = (int)(per * SEG_UNIT);
  *segments = (int)((units + per - 1) / per);
}

template <typename T, int D, bool BACK, int KIND>
int attn_run(const PassArgs& p, cudaStream_t s) {
  using S = Shape<T, D>;
  static std::atomic<unsigned long long> done;
  const int bytes = S::bytes(KIND == STATE ? 2 : KIND == OUTPUT ? 3 : 4, KIND != STATE);
  const int st = shared_limit(attn_kernel<T, D, BACK, KIND>, bytes, &done, "attn_kernel");
  if (st != GFN_OK) return st;
  attn_kernel<T, D, BACK, KIND><<<dim3(p.segments, p.H, p.B), S::THREADS, bytes, s>>>(p);
  return launch_status("attn_kernel");
}

// States by segment where there are several, then the outputs.
template <typename T, int D, bool BACK, int KIND>
int attn_pass(PassArgs p, float* segs, cudaStream_t s) {
  if (p.segments > 1) {
    PassArgs w = p;
    w.segs = segs;
    if (KIND == PAIR) {  // the state's rows are q's, its columns do's
      w.b = p.a;
      w.c = p.d;
    }
    int st = attn_run<T, D, BACK, STATE>(w, s);
    if (st != GFN_OK) return st;
    const int bh = p.B * p.H, y = bh < 32768 ? bh : 32768;
    attn_join_kernel<BACK><<<dim3((unsigned)((p.KD * p.VD + 255) / 256), y, (bh + y - 1) / y), 256, 0, s>>>(w);
    if ((st = launch_status("attn_join_kernel")) != GFN_OK) return st;
    p.segs = segs;
    p.state_out = nullptr;
  }
  return attn_run<T, D, BACK, KIND>(p, s);
}

template <typename T, bool BACK, int KIND>
int attn_dims(const PassArgs& p, float* segs, cudaStream_t s) {
  const int d = p.KD > p.VD ? p.KD : p.VD;
  if (d <= 32) return attn_pass<T, 32, BACK, KIND>(p, segs, s);
  if (d <= 64) return attn_pass<T, 64, BACK, KIND>(p, segs, s);
  return attn_pass<T, 128, BACK, KIND>(p, segs, s);
}

template <typename T>
int attn_forward(PassArgs p, float* segs, cudaStream_t s) {
  if (p.L == 1) {
    const unsigned blocks = (unsigned)(p.B * p.H);
    const bool vec = p.VD % 4 == 0 && (!p.state || aligned16(p.state)) && (!p.state_out || aligned16(p.state_out));
    if (vec) attn_step_kernel<T, 4><<<blocks, 256, 0, s>>>(p);
    else attn_step_kernel<T, 1><<<blocks, 256, 0, s>>>(p);
    return launch_status("attn_step_kernel");
  }
  return attn_dims<T, false, OUTPUT>(p, segs, s);
}

bool pieces16(const View& v, int dim, int size) {
  const long long per = 16 / size;
  return aligned16(v.p) && dim % per == 0 && v.sb % per == 0 && v.sl % per == 0 && v.sh % per == 0;
}

int attn_check(const char* what, int dtype, int batch, int length, int heads, int kdim, int vdim, bool null) {
  if (batch < 0 || length < 0 || heads < 0 || kdim <= 0 || vdim <= 0 || (batch > 0 && heads > 0 && null))
    return fail(GFN_ERR_INVALID, "%s: batch=%d length=%d heads=%d dims %d, %d, or a NULL operand", what, batch, length,
                heads, kdim, vdim);
  if (kdim > 128 || vdim > 128) return fail(GFN_ERR_UNSUPPORTED, "%s: head dims %d, %d above 128", what, kdim, vdim);
  if (batch > 65535 || heads > 65535 || (long long)batch * heads > 0x3fffffffLL || length > 1 << 30)
    return fail(GFN_ERR_UNSUPPORTED, "%s: batch %d, %d heads, length %d", what, batch, heads, length);
  if (dtype != GFN_F32 && dtype != GFN_BF16 && dtype != GFN_F16)
    return fail(GFN_ERR_UNSUPPORTED, "%s: element type %d", what, dtype);
  return GFN_OK;
}

// An empty sequence leaves the state as it was.
int attn_copy_state(const float* from, float* to, long long n, cudaStream_t s) {
  if (!to || n == 0) return GFN_OK;
  const cudaError_t e = from ? cudaMemcpyAsync(to, from, 4 * n, cudaMemcpyDeviceToDevice, s) : cudaMemsetAsync(to, 0, 4 * n, s);
  return e == cudaSuccess ? GFN_OK : cuda_status(e, "decay_attention: state");
}

}  // namespace

extern "C" {

long long gfn_decay_attention_workspace_bytes(int batch, int length, int heads, int kdim, int vdim) {
  if (batch <= 0 || heads <= 0 || length <= 0 || kdim <= 0 || vdim <= 0) return 0;
  int sms = 0, seg_len = 0, segments = 0;
  if (sm_count(&sms) != GFN_OK) return -1;
  attn_segments(batch, length, heads, sms, &seg_len, &segments);
  return segments > 1 ? 4LL * batch * heads * segments * kdim * vdim : 0;
}

int gfn_decay_attention_forward(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
                                const void* v, const long long* v_strides, const float* decay, const float* state,
                                const void* lengths, int lengths_are_64, int dtype, int batch, int length, int heads,
                                int kdim, int vdim, float scale, void* o, float* state_out, void* workspace,
                                long long workspace_bytes, gfn_stream_t stream) {
  int st = attn_check("decay_attention", dtype, batch, length, heads, kdim, vdim,
                      !decay || (length > 0 && (!q || !k || !v || !o)));
  if (st != GFN_OK) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (batch == 0 || heads == 0) return GFN_OK;
  if (length == 0) return attn_copy_state(state, state_out, (long long)batch * heads * kdim * vdim, s);
  int sms = 0;
  if ((st = sm_count(&sms)) != GFN_OK) return st;
  PassArgs p = {};
  auto view = [](const void* x, const long long* t) { return View{x, t[0], t[1], t[2]}; };
  p.a = view(q, q_strides); p.b = view(k, k_strides); p.c = view(v, v_strides);
  p.o = o; p.decay = decay; p.state = state; p.state_out = state_out;
  p.lengths = lengths; p.lengths64 = lengths_are_64; p.B = batch; p.L = length; p.H = heads; p.KD = kdim; p.VD = vdim;
  p.sr = vdim; p.sc = 1; p.s_in = p.s_state = scale; p.s_update = 1.f;
  attn_segments(batch, length, heads, sms, &p.seg_len, &p.segments);
  const int size = dtype == GFN_F32 ? 4 : 2;
  p.vec = pieces16(p.a, kdim, size) && pieces16(p.b, kdim, size) && pieces16(p.c, vdim, size);
  if (length > 1 && p.segments > 1 &&
      (!aligned16(workspace) || !workspace || workspace_bytes < 4LL * batch * heads * p.segments * kdim * vdim))
    return fail(GFN_ERR_INVALID, "decay_attention: a workspace of gfn_decay_attention_workspace_bytes is needed");
  float* segs = static_cast<float*>(workspace);
  if (dtype == GFN_F32) return attn_forward<float>(p, segs, s);
  if (dtype == GFN_BF16) return attn_forward<__nv_bfloat16>(p, segs, s);
  return attn_forward<__half>(p, segs, s);
}

int gfn_decay_attention_backward(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
                                 const void* v, const long long* v_strides, const void* d_o, const long long* do_strides,
                                 const float* decay, const float* state, const float* d_state_out, const void* lengths,
                                 int lengths_are_64, int dtype, int batch, int length, int heads, int kdim, int vdim,
                                 float scale, void* dq, void* dk, void* dv, float* d_state, void* workspace,
                                 long long workspace_bytes, gfn_stream_t stream) {
  int st = attn_check("decay_attention backward", dtype, batch, length, heads, kdim, vdim,
                      !decay || (length > 0 && (!q || !k || !v || !d_o || !dq || !dk || !dv)));
  if (st != GFN_OK) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (batch == 0 || heads == 0) return GFN_OK;
  if (length == 0) return attn_copy_state(d_state_out, d_state, (long long)batch * heads * kdim * vdim, s);
  int sms = 0;
  if ((st = sm_count(&sms)) != GFN_OK) return st;
  auto view = [](const void* x, const long long* t) { return View{x, t[0], t[1], t[2]}; };
  const View vq = view(q, q_strides), vk = view(k, k_strides), vv = view(v, v_strides), vo = view(d_o, do_strides);
  PassArgs p = {};
  p.decay = decay; p.lengths = lengths; p.lengths64 = lengths_are_64; p.B = batch; p.L = length; p.H = heads;
  attn_segments(batch, length, heads, sms, &p.seg_len, &p.segments);
  const int size = dtype == GFN_F32 ? 4 : 2;
  p.vec = pieces16(vq, kdim, size) && pieces16(vk, kdim, size) && pieces16(vv, vdim, size) && pieces16(vo, vdim, size);
  if (p.segments > 1 &&
      (!workspace || !aligned16(workspace) || workspace_bytes < 4LL * batch * heads * p.segments * kdim * vdim))
    return fail(GFN_ERR_INVALID, "decay_attention backward: a workspace of gfn_decay_attention_workspace_bytes is needed");
  float* segs = static_cast<float*>(workspace);
  PassArgs f = p;  // dq
  f.a = vo; f.b = vv; f.c = vk; f.o = dq; f.state = state; f.KD = vdim; f.VD = kdim; f.sr = 1; f.sc = vdim;
  f.s_in = f.s_state = scale; f.s_update = 1.f;
  PassArgs r = p;  // dv and dk
  r.a = vq; r.b = vk; r.c = vv; r.d = vo; r.o = dv; r.o2 = dk; r.state = d_state_out; r.state_out = d_state;
  r.KD = kdim; r.VD = vdim; r.sr = vdim; r.sc = 1; r.s_in = r.s_update = scale; r.s_state = 1.f;
  auto both = [&](auto t) {
    using T = decltype(t);
    const int e = attn_dims<T, false, OUTPUT>(f, segs, s);
    return e != GFN_OK ? e : attn_dims<T, true, PAIR>(r, segs, s);
  };
  if (dtype == GFN_F32) return both(float());
  if (dtype == GFN_BF16) return both(__nv_bfloat16());
  return both(__half());
}

}  // extern "C"
