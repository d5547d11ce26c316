// Gated linear recurrence over long sequences, forward and backward.
//
//   h_t = a_t h_{t-1} + x_t,  h_{-1} = h0       (per batch row and column)
//
// and, for upstream gradients dh_t and dlast (of the last state),
//
//   g_t = dh_t + m_{t+1},  m_t = a_t g_t,  m_L = dlast
//   dx_t = g_t,  da_t = g_t h_{t-1},  dh0 = m_0.
//
// States and messages are float32 whatever the operands' type.  The forward
// for training keeps the state every SCAN_CK steps; the backward recomputes
// h from there, in float32, instead of reading the rounded h of a 16-bit
// output (the bytes are the same: x is read in h's place).
//
// Both directions are bound by HBM, so the operands are read once.  A block
// holds a run of NW * S steps of 32 * VEC columns in registers: warp w keeps
// S steps, lane l VEC columns.  A run maps its incoming state as
// h -> P h + p; the warps' maps meet in shared memory, the blocks' maps in
// global memory, and then the block walks its registers once more to write the
// results.  Many blocks per column tile keep the memory busy when batch * dim
// is far too small to fill the GPU.  Runs form groups of SCAN_GROUP: a run
// composes the maps of its group before it and applies them to the state at
// the group's start, which the group before publishes.  What is composed with
// what does not depend on which block is faster, so results repeat bit for bit.
#pragma once
#include "lm_ops.cuh"

namespace gfn {

constexpr int SCAN_CK = 64;  // steps between kept states

struct GScanArgs {
  const void* a;  // [B, L, D] by strides; null: a == 1
  const void* x;
  const float* h0;     // [B, D] or null (zero)
  void* h;             // forward out [B, L, D]
  float* h_last;       // [B, D] or null
  float* states;       // [B][ceil(L / SCAN_CK)][D]: the state before step k SCAN_CK
  const void* dh;      // backward: [B, L, D] by strides, or null (zero)
  const float* dlast;  // [B, D] or null
  void* da;            // [B, L, D] or null
  void* dx;            // [B, L, D] or null
  float* dh0;          // [B, D] or null
  long long a_sb, a_st, x_sb, x_st, g_sb, g_st;  // batch and step strides, in elements
  unsigned long long* words;  // published words, one run of steps and column each; null: a single run
  unsigned* ticket;
  int B, L, D, nck;
  int nchunks, ctiles;  // runs of steps per column; column tiles per batch row
};

// ------------------------------------------------------------ published words
// A word is two floats in 64 bits, stored and read whole: all ones until it
// is published.  No value carries that pattern (a NaN that would is replaced),
// so no flag and no fence is needed beside the word itself.
constexpr unsigned SCAN_EMPTY = 0xffffffffu;

GFN_DEV unsigned scan_bits(float v) {
  const unsigned u = __float_as_uint(v);
  return u == SCAN_EMPTY ? 0x7fffffffu : u;
}
GFN_DEV unsigned long long scan_word(float lo, float hi) {
  return ((unsigned long long)scan_bits(hi) << 32) | scan_bits(lo);
}
GFN_DEV float word_lo(unsigned long long w) { return __uint_as_float((unsigned)w); }
GFN_DEV float word_hi(unsigned long long w) { return __uint_as_float((unsigned)(w >> 32)); }
GFN_DEV unsigned long long word_load(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
GFN_DEV void word_store(unsigned long long* p, unsigned long long v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

// Product of two runs' gates.  A product of non-zero gates that underflows is
// held at the smallest float, so that an infinite state stays infinite as it
// does step by step (0 * inf would be NaN); its weight is 1e-45.
GFN_DEV float gate_product(float a, float b) {
  const float r = a * b;
  return (r == 0.f && a != 0.f && b != 0.f) ? copysignf(1.4e-45f, r) : r;
}
// P h + p; a zero state passes as p alone (an overflowed P must not make NaN of it).
GFN_DEV float pass(float P, float h, float p) { return h == 0.f ? p : fmaf(P, h, p); }

// Maps of a run of steps and how they compose: `compose(l, e)` applies e first.
struct GatedMap {  // h -> P h + p
  static constexpr int WORDS = 1;
  float P, p;
  GFN_DEV static GatedMap identity() { return {1.f, 0.f}; }
  GFN_DEV static GatedMap compose(GatedMap l, GatedMap e) { return {gate_product(l.P, e.P), pass(l.P, e.p, l.p)}; }
  GFN_DEV void pack(unsigned long long (&w)[WORDS]) const { w[0] = scan_word(P, p); }
  GFN_DEV static GatedMap unpack(const unsigned long long (&w)[WORDS]) { return {word_lo(w[0]), word_hi(w[0])}; }
};
struct GatedState {
  static constexpr int WORDS = 1;
  float h;
  GFN_DEV void pack(unsigned long long (&w)[1]) const { w[0] = scan_word(h, 0.f); }
  GFN_DEV static GatedState unpack(const unsigned long long (&w)[1]) { return {word_lo(w[0])}; }
  GFN_DEV GatedState through(GatedMap m) const { return {pass(m.P, h, m.p)}; }
};

constexpr int SCAN_GROUP = 32;  // runs whose maps are composed; the states pass from group to group

// N maps (or states) that other blocks publish for one column, from `src` on,
// `stride` words apart.
template <class M, int N>
GFN_DEV void await(const unsigned long long* src, long long stride, int ct, int n, M (&out)[N]) {
  unsigned long long got[N][M::WORDS];
  for (int spin = 0;; ++spin) {
    bool ready = true;
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
      for (int i = 0; i < M::WORDS; ++i) {
        got[k][i] = 0;
        if (k < n) got[k][i] = word_load(src + k * stride + i * ct);
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
      for (int i = 0; i < M::WORDS; ++i) ready = ready && (unsigned)got[k][i] != SCAN_EMPTY;
    }
    if (ready) break;
    if (spin == (1 << 22)) {  // seconds: flag it and carry on with what is there
      gfn_flag_error(kDevErrMbarTimeout);
      break;
    }
    __nanosleep(20);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) out[k] = M::unpack(got[k]);
}

template <class M>
GFN_DEV void publish(M m, unsigned long long* dst, int ct) {
  unsigned long long w[M::WORDS];
  m.pack(w);
#pragma unroll
  for (int i = 0; i < M::WORDS; ++i) word_store(dst + i * ct, w[i]);
}

template <class Map, class State, int CT, int NW>
struct ScanShared {
  static constexpr int R = NW * 32 / CT;  // threads per column
  unsigned long long maps[NW][Map::WORDS][CT];  // the warps' maps; then those of all warps before each
  unsigned long long part[R][Map::WORDS][CT];   // maps of parts of the group
  State in[CT];                                 // the state before this run
  unsigned slot;
};

// The state that `chunk` (counted in the direction of the scan) of a column
// tile receives.  Call with the warps' maps in sh.maps; on return (after a
// barrier) sh.maps[w] holds the map of the warps before w, counted in the
// direction of the scan (REV: from the last warp), and sh.in the states.
// R threads serve a column: the last of them chains the warps' maps and
// publishes, all of them fetch their share of the group's earlier maps.
// `words` is the tile's [nchunks][WORDS][CT]; first(c) the state before chunk 0.
template <class Map, class State, int CT, int NW, bool REV, class First>
GFN_DEV void receive(ScanShared<Map, State, CT, NW>& sh, unsigned long long* words, int chunk, int nchunks,
                     int live, First first) {
  constexpr int W = Map::WORDS, R = NW * 32 / CT, GS = SCAN_GROUP / R;
  constexpr int BATCH = GS < 8 ? GS : 8;
  const int c = threadIdx.x % CT, r = threadIdx.x / CT;
  const bool active = c < live, teller = r == R - 1 && active;
  const int pos = chunk % SCAN_GROUP, start = chunk - pos;
  const bool tells = teller && chunk + 1 < nchunks;
  unsigned long long* mine = words + (long long)chunk * W * CT + c;
  Map own = Map::identity();
  __syncthreads();
  if (teller) {
#pragma unroll
    for (int j = 0; j < NW; ++j) {
      const int w = REV ? NW - 1 - j : j;
      unsigned long long x[W], y[W];
      own.pack(y);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        x[i] = sh.maps[w][i][c];
        sh.maps[w][i][c] = y[i];
      }
      own = Map::compose(Map::unpack(x), own);
    }
    if (tells && pos < SCAN_GROUP - 1) publish(own, mine, CT);
  }
  Map acc = Map::identity();  // of the group's runs before this one
  if (pos > 0) {
    if (active && r * GS < pos) {
      for (int k = r * GS; k < min((r + 1) * GS, pos); k += BATCH) {
        const int n = min(BATCH, min((r + 1) * GS, pos) - k);
        Map next[BATCH];
        await<Map, BATCH>(words + (long long)(start + k) * W * CT + c, W * CT, CT, n, next);
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (i < n) acc = Map::compose(next[i], acc);
      }
      unsigned long long x[W];
      acc.pack(x);
#pragma unroll
      for (int i = 0; i < W; ++i) sh.part[r][i][c] = x[i];
    }
    __syncthreads();
    if (teller) {
      acc = Map::identity();
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (j * GS < pos) {
          unsigned long long x[W];
#pragma unroll
          for (int i = 0; i < W; ++i) x[i] = sh.part[j][i][c];
          acc = Map::compose(Map::unpack(x), acc);
        }
      }
    }
  }
  if (teller) {
    State at[1];  // at the group's start
    if (start > 0) await<State, 1>(words + (long long)(start - 1) * W * CT + c, 0, CT, 1, at);
    else at[0] = first(c);
    if (tells && pos == SCAN_GROUP - 1) publish(at[0].through(Map::compose(own, acc)), mine, CT);
    sh.in[c] = at[0].through(acc);
  }
  __syncthreads();
}

// ------------------------------------------------------------ vector accesses
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T, int VEC>
GFN_DEV Pack<T, VEC> load_pack(const T* p) {  // read once: evict first
  Pack<T, VEC> r;
  constexpr int B = sizeof(T) * VEC;
  if constexpr (B == 2) *reinterpret_cast<unsigned short*>(&r) = __ldcs(reinterpret_cast<const unsigned short*>(p));
  else if constexpr (B == 4) *reinterpret_cast<unsigned*>(&r) = __ldcs(reinterpret_cast<const unsigned*>(p));
  else if constexpr (B == 8) *reinterpret_cast<uint2*>(&r) = __ldcs(reinterpret_cast<const uint2*>(p));
  else *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));
  return r;
}
template <typename T, int VEC>
GFN_DEV void store_pack(T* p, const Pack<T, VEC>& r) {
  constexpr int B = sizeof(T) * VEC;
  if constexpr (B == 2) __stcs(reinterpret_cast<unsigned short*>(p), *reinterpret_cast<const unsigned short*>(&r));
  else if constexpr (B == 4) __stcs(reinterpret_cast<unsigned*>(p), *reinterpret_cast<const unsigned*>(&r));
  else if constexpr (B == 8) __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<const uint2*>(&r));
  else __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&r));
}

// Which run of steps and which columns a block computes.  Runs are handed out
// by a ticket in the direction of the scan, all column tiles of one run before
// the next: the blocks that a block waits for have started, so its wait ends.
struct ScanTile {
  int chunk, b, c0, col;  // c0: the tile's first column; col: this lane's first
  bool active;
  long long tile;
};

template <int VEC, class Args>
GFN_DEV ScanTile scan_tile(const Args& p, unsigned* slot) {
  unsigned t = blockIdx.x;
  if (p.words) {
    if (threadIdx.x == 0) *slot = atomicAdd(p.ticket, 1u) + 1u;  // starts at all ones, like the words
    __syncthreads();
    t = *slot;
  }
  ScanTile r;
  const unsigned tiles = (unsigned)p.B * p.ctiles;
  r.chunk = t / tiles;
  r.tile = t - (unsigned)r.chunk * tiles;
  r.b = (int)(r.tile / p.ctiles);
  r.c0 = (int)(r.tile - (long long)r.b * p.ctiles) * (32 * VEC);
  r.col = r.c0 + (threadIdx.x & 31) * VEC;
  r.active = r.col < p.D;
  return r;
}

// ------------------------------------------------------------------ gated scan
template <typename T, int VEC>
GFN_DEV Pack<T, VEC> fill_pack(float v) {
  Pack<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.v[i] = from_f<T>(v);
  return r;
}

// Map of S steps from a zero state; steps beyond the end hold a = 1, x = 0.
template <typename T, int VEC, int S>
GFN_DEV GatedMap run_map(const Pack<T, VEC> (&a)[S], const Pack<T, VEC> (&x)[S], int v) {
  GatedMap m = GatedMap::identity();
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const float g = to_f(a[s].v[v]);
    m.P *= g;
    m.p = fmaf(g, m.p, to_f(x[s].v[v]));
  }
  if (m.P == 0.f) {  // a zero gate, or an underflow?
    bool zero = false;
#pragma unroll
    for (int s = 0; s < S; ++s) zero = zero || to_f(a[s].v[v]) == 0.f;
    if (!zero) m.P = copysignf(1.4e-45f, m.P);
  }
  return m;
}

template <typename T, int VEC, int S, int NW, int OCC>
__global__ void __launch_bounds__(NW * 32, OCC) gscan_forward_kernel(const GScanArgs p) {
  constexpr int CT = 32 * VEC;
  __shared__ ScanShared<GatedMap, GatedState, CT, NW> sh;
  const ScanTile q = scan_tile<VEC>(p, &sh.slot);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = (q.chunk * NW + w) * S;
  const int n = q.active ? max(0, min(S, p.L - t0)) : 0;
  Pack<T, VEC> a[S], x[S];
  const T* xp = static_cast<const T*>(p.x) + q.b * p.x_sb + t0 * p.x_st + q.col;
  const T* ap = static_cast<const T*>(p.a) + q.b * p.a_sb + t0 * p.a_st + q.col;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    x[s] = fill_pack<T, VEC>(0.f);
    a[s] = fill_pack<T, VEC>(1.f);
    if (s < n) {
      x[s] = load_pack<T, VEC>(xp + s * p.x_st);
      if (p.a) a[s] = load_pack<T, VEC>(ap + s * p.a_st);
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    unsigned long long wd[1];
    run_map<T, VEC, S>(a, x, v).pack(wd);
    sh.maps[w][0][lane * VEC + v] = wd[0];
  }
  receive<GatedMap, GatedState, CT, NW, false>(
      sh, p.words + q.tile * p.nchunks * (long long)CT, q.chunk, p.nchunks, p.D - q.c0,
      [&](int c) { return GatedState{p.h0 ? p.h0[(long long)q.b * p.D + q.c0 + c] : 0.f}; });
  if (n <= 0) return;
  float h[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    h[v] = sh.in[lane * VEC + v].through(GatedMap::unpack({sh.maps[w][0][lane * VEC + v]})).h;
  if (p.states && t0 % SCAN_CK == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.states[((long long)q.b * p.nck + t0 / SCAN_CK) * p.D + q.col + v] = h[v];
  }
  T* hp = static_cast<T*>(p.h) + ((long long)q.b * p.L + t0) * p.D + q.col;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    Pack<T, VEC> o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      h[v] = fmaf(to_f(a[s].v[v]), h[v], to_f(x[s].v[v]));
      o.v[v] = from_f<T>(h[v]);
    }
    if (s < n) store_pack<T, VEC>(hp + (long long)s * p.D, o);
  }
  if (p.h_last && t0 + n == p.L) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.h_last[(long long)q.b * p.D + q.col + v] = h[v];
  }
}

// Runs of NW * S = SCAN_CK steps from the last to the first: the state kept
// before the run gives h, the messages pass from run to run as the states do
// in the forward.
template <typename T, int VEC, int S, int NW, int OCC>
__global__ void __launch_bounds__(NW * 32, OCC) gscan_backward_kernel(const GScanArgs p) {
  static_assert(NW * S == SCAN_CK, "one kept state per run");
  constexpr int CT = 32 * VEC;
  __shared__ ScanShared<GatedMap, GatedState, CT, NW> sh;
  __shared__ unsigned long long fmaps[NW][CT];
  const ScanTile q = scan_tile<VEC>(p, &sh.slot);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int run = p.nchunks - 1 - q.chunk;
  const int t0 = run * SCAN_CK + w * S;
  const int n = q.active ? max(0, min(S, p.L - t0)) : 0;
  Pack<T, VEC> a[S], x[S], g[S];
  const T* xp = static_cast<const T*>(p.x) + q.b * p.x_sb + t0 * p.x_st + q.col;
  const T* ap = static_cast<const T*>(p.a) + q.b * p.a_sb + t0 * p.a_st + q.col;
  const T* gp = static_cast<const T*>(p.dh) + q.b * p.g_sb + t0 * p.g_st + q.col;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    x[s] = g[s] = fill_pack<T, VEC>(0.f);
    a[s] = fill_pack<T, VEC>(1.f);
    if (s < n) {
      x[s] = load_pack<T, VEC>(xp + s * p.x_st);
      if (p.a) a[s] = load_pack<T, VEC>(ap + s * p.a_st);
      if (p.dh) g[s] = load_pack<T, VEC>(gp + s * p.g_st);
    }
  }
  float h[VEC];  // before the run
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    h[v] = q.active ? p.states[((long long)q.b * p.nck + run) * p.D + q.col + v] : 0.f;
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    unsigned long long wd[1];
    const GatedMap mf = run_map<T, VEC, S>(a, x, v);
    mf.pack(wd);
    fmaps[w][lane * VEC + v] = wd[0];
    GatedMap mb = {mf.P, 0.f};  // of the message, last step first
#pragma unroll
    for (int s = S - 1; s >= 0; --s) mb.p = to_f(a[s].v[v]) * (to_f(g[s].v[v]) + mb.p);
    mb.pack(wd);
    sh.maps[w][0][lane * VEC + v] = wd[0];
  }
  receive<GatedMap, GatedState, CT, NW, true>(
      sh, p.words + q.tile * p.nchunks * (long long)CT, q.chunk, p.nchunks, p.D - q.c0,
      [&](int c) { return GatedState{p.dlast ? p.dlast[(long long)q.b * p.D + q.c0 + c] : 0.f}; });
  if (!q.active) return;
  float m[VEC], hp[S][VEC];  // hp: h_{t-1}
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    m[v] = sh.in[lane * VEC + v].through(GatedMap::unpack({sh.maps[w][0][lane * VEC + v]})).h;
    for (int j = 0; j < w; ++j) {
      const GatedMap f = GatedMap::unpack({fmaps[j][lane * VEC + v]});
      h[v] = pass(f.P, h[v], f.p);
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      hp[s][v] = h[v];
      h[v] = fmaf(to_f(a[s].v[v]), h[v], to_f(x[s].v[v]));
    }
  }
  const long long o = ((long long)q.b * p.L + t0) * p.D + q.col;
#pragma unroll
  for (int s = S - 1; s >= 0; --s) {
    Pack<T, VEC> oa, ox;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float gt = to_f(g[s].v[v]) + m[v];
      ox.v[v] = from_f<T>(gt);
      oa.v[v] = from_f<T>(gt * hp[s][v]);
      m[v] = to_f(a[s].v[v]) * gt;
    }
    if (s < n) {
      if (p.dx) store_pack<T, VEC>(static_cast<T*>(p.dx) + o + (long long)s * p.D, ox);
      if (p.da) store_pack<T, VEC>(static_cast<T*>(p.da) + o + (long long)s * p.D, oa);
    }
  }
  if (p.dh0 && run == 0 && w == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.dh0[(long long)q.b * p.D + q.col + v] = m[v];
  }
}

// A few steps: one thread per column.  (Length 0 passes the state through.)
template <typename T>
__global__ void __launch_bounds__(128) gscan_forward_seq_kernel(const GScanArgs p) {
  const long long c = blockIdx.x * 128LL + threadIdx.x;
  if (c >= (long long)p.B * p.D) return;
  const long long b = c / p.D, j = c - b * p.D;
  const T* a = p.a ? static_cast<const T*>(p.a) + b * p.a_sb + j : nullptr;
  const T* x = static_cast<const T*>(p.x) + b * p.x_sb + j;
  T* h = static_cast<T*>(p.h) + b * p.L * (long long)p.D + j;
  float s = p.h0 ? p.h0[c] : 0.f;
  if (p.states && p.L) p.states[c] = s;  // one kept state: L <= SCAN_CK
#pragma unroll 4
  for (int t = 0; t < p.L; ++t) {
    s = fmaf(a ? to_f(a[t * p.a_st]) : 1.f, s, to_f(x[t * p.x_st]));
    h[(long long)t * p.D] = from_f<T>(s);
  }
  if (p.h_last) p.h_last[c] = s;
}

// ---------------------------------------------------------------------------
// The scan layer's recurrence (gfn/layers/parallel.py:101-121) from the
// pre-activations z = [zA | zdt | zB]:
//   A = sigma(zA), dt = softplus(zdt) c, c = base_dt 1.5^head
//   v_t = A_t v_{t-1} + zB_t dt_t,  x_t = x_{t-1} + v_t dt_t
// and backward, for upstream gradients gx, gv of the sequences and gxl, gvl
// of the last state:
//   X_t = gx_t + X_{t+1},  l_t = gv_t + dt_t X_t + m_{t+1},  m_t = A_t l_t
//   dzA = l_t v_{t-1} A (1 - A),  dzB = l_t dt_t
//   dzdt = (l_t zB_t + X_t v_t) c sigma(zdt),  dv0 = m_0,  dx0 = X_0.
struct LScanArgs {
  const float* z;   // [B, L, 3D]
  const float* v0;  // [B, D] or null
  const float* x0;
  float* xs;        // [B, L, D]
  float* vs;
  float* v_last;    // [B, D] or null
  float* x_last;
  float* states;    // v before step k SCAN_CK, as in GScanArgs
  const float* gx;  // [B, L, D] or null
  const float* gv;
  const float* gxl; // [B, D] or null
  const float* gvl;
  float* dz;        // [B, L, 3D]
  float* dv0;       // [B, D] or null
  float* dx0;
  unsigned long long* words;  // as in GScanArgs
  unsigned* ticket;
  int B, L, D, H, nck, nchunks, ctiles;
  float base_dt;
};

// 1 / v to one unit in the last place, for v in [1, 6].
GFN_DEV float quick_rcp(float v) { return __fdividef(1.f, v); }

// sigma(z) and its slope sigma(z) sigma(-z) from one exponential that cannot
// overflow: both keep their digits far out, where 1 / (1 + exp(-z)) is
// already 0 or 1.
GFN_DEV float gate(float z, float* slope) {
  const float e = expf(-fabsf(z)), r = quick_rcp(1.f + e), c = e * r;
  *slope = r * c;
  return z >= 0.f ? r : c;
}

// softplus(z) = max(z, 0) + log1p(e), e = exp(-|z|) in [0, 1], and its slope
// sigma(z).  log1p(e) = 2 atanh(y) with y = e / (2 + e) <= 1/3: the odd series
// up to y^15 leaves 1e-9 of the sum, and every term is positive.
GFN_DEV float soft_step(float z, float* slope) {
  const float e = expf(-fabsf(z));
  const float r = quick_rcp((1.f + e) * (2.f + e));  // both quotients from one reciprocal
  const float y = e * ((1.f + e) * r), y2 = y * y, s = (2.f + e) * r;
  float q = 1.f / 15.f;
  q = fmaf(q, y2, 1.f / 13.f);
  q = fmaf(q, y2, 1.f / 11.f);
  q = fmaf(q, y2, 1.f / 9.f);
  q = fmaf(q, y2, 1.f / 7.f);
  q = fmaf(q, y2, 1.f / 5.f);
  q = fmaf(q, y2, 1.f / 3.f);
  q = fmaf(q * y2, y, y);
  *slope = z >= 0.f ? s : e * s;
  return fmaf(2.f, q, fmaxf(z, 0.f));
}

GFN_DEV float head_scale(int col, int hd) {
  float hs = 1.f;
  for (int i = 0; i < col / hd; ++i) hs *= 1.5f;
  return hs;
}

struct LayerMap {  // v -> P v + p, x -> x + Q v + q
  static constexpr int WORDS = 2;
  float P, p, Q, q;
  GFN_DEV static LayerMap identity() { return {1.f, 0.f, 0.f, 0.f}; }
  GFN_DEV static LayerMap compose(LayerMap l, LayerMap e) {
    return {gate_product(l.P, e.P), pass(l.P, e.p, l.p), fmaf(l.Q, e.P, e.Q), e.q + pass(l.Q, e.p, l.q)};
  }
  GFN_DEV void pack(unsigned long long (&w)[2]) const {
    w[0] = scan_word(P, p);
    w[1] = scan_word(Q, q);
  }
  GFN_DEV static LayerMap unpack(const unsigned long long (&w)[2]) {
    return {word_lo(w[0]), word_hi(w[0]), word_lo(w[1]), word_hi(w[1])};
  }
};
struct LayerState {
  static constexpr int WORDS = 1;
  float v, x;
  GFN_DEV void pack(unsigned long long (&w)[1]) const { w[0] = scan_word(v, x); }
  GFN_DEV static LayerState unpack(const unsigned long long (&w)[1]) { return {word_lo(w[0]), word_hi(w[0])}; }
  GFN_DEV LayerState through(LayerMap m) const { return {pass(m.P, v, m.p), x + pass(m.Q, v, m.q)}; }
};

template <int VEC, int S, int NW, int OCC>
__global__ void __launch_bounds__(NW * 32, OCC) lscan_forward_kernel(const LScanArgs p) {
  constexpr int CT = 32 * VEC;
  __shared__ ScanShared<LayerMap, LayerState, CT, NW> sh;
  const ScanTile c = scan_tile<VEC>(p, &sh.slot);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = (c.chunk * NW + w) * S;
  const int n = c.active ? max(0, min(S, p.L - t0)) : 0;
  const float* zp = p.z + ((long long)c.b * p.L + t0) * 3 * p.D + c.col;
  Pack<float, VEC> A[S], dt[S], bv[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {  // beyond the end: A = 1, dt = 0, zB = 0
    A[s] = fill_pack<float, VEC>(INFINITY);
    dt[s] = fill_pack<float, VEC>(-INFINITY);
    bv[s] = fill_pack<float, VEC>(0.f);
    if (s < n) {
      A[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D);
      dt[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D + p.D);
      bv[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D + 2LL * p.D);
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const float scale = p.base_dt * head_scale(c.col + v, p.D / p.H);
    LayerMap m = LayerMap::identity();
    bool zero = false;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float slope;
      A[s].v[v] = gate(A[s].v[v], &slope);
      dt[s].v[v] = soft_step(dt[s].v[v], &slope) * scale;
      bv[s].v[v] *= dt[s].v[v];
      zero = zero || A[s].v[v] == 0.f;
      m.P *= A[s].v[v];
      m.p = fmaf(A[s].v[v], m.p, bv[s].v[v]);
      m.Q = fmaf(dt[s].v[v], m.P, m.Q);
      m.q = fmaf(dt[s].v[v], m.p, m.q);
    }
    if (m.P == 0.f && !zero) m.P = 1.4e-45f;
    unsigned long long wd[2];
    m.pack(wd);
    sh.maps[w][0][lane * VEC + v] = wd[0];
    sh.maps[w][1][lane * VEC + v] = wd[1];
  }
  receive<LayerMap, LayerState, CT, NW, false>(
      sh, p.words + c.tile * p.nchunks * (2LL * CT), c.chunk, p.nchunks, p.D - c.c0, [&](int j) {
        const long long e = (long long)c.b * p.D + c.c0 + j;
        return LayerState{p.v0 ? p.v0[e] : 0.f, p.x0 ? p.x0[e] : 0.f};
      });
  if (n <= 0) return;
  LayerState st[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    st[v] = sh.in[lane * VEC + v].through(
        LayerMap::unpack({sh.maps[w][0][lane * VEC + v], sh.maps[w][1][lane * VEC + v]}));
  if (p.states && t0 % SCAN_CK == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.states[((long long)c.b * p.nck + t0 / SCAN_CK) * p.D + c.col + v] = st[v].v;
  }
  const long long o = ((long long)c.b * p.L + t0) * p.D + c.col;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    Pack<float, VEC> ov, ox;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      st[v].v = fmaf(A[s].v[v], st[v].v, bv[s].v[v]);
      st[v].x = fmaf(st[v].v, dt[s].v[v], st[v].x);
      ov.v[v] = st[v].v;
      ox.v[v] = st[v].x;
    }
    if (s < n) {
      store_pack<float, VEC>(p.vs + o + (long long)s * p.D, ov);
      store_pack<float, VEC>(p.xs + o + (long long)s * p.D, ox);
    }
  }
  if (t0 + n == p.L) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const long long e = (long long)c.b * p.D + c.col + v;
      if (p.v_last) p.v_last[e] = st[v].v;
      if (p.x_last) p.x_last[e] = st[v].x;
    }
  }
}

struct LayerBackMap {  // m -> P m + R X + q, X -> X + G
  static constexpr int WORDS = 2;
  float P, q, R, G;
  GFN_DEV static LayerBackMap identity() { return {1.f, 0.f, 0.f, 0.f}; }
  GFN_DEV static LayerBackMap compose(LayerBackMap l, LayerBackMap e) {
    return {gate_product(l.P, e.P), pass(l.P, e.q, pass(l.R, e.G, l.q)), fmaf(l.P, e.R, l.R), l.G + e.G};
  }
  GFN_DEV void pack(unsigned long long (&w)[2]) const {
    w[0] = scan_word(P, q);
    w[1] = scan_word(R, G);
  }
  GFN_DEV static LayerBackMap unpack(const unsigned long long (&w)[2]) {
    return {word_lo(w[0]), word_hi(w[0]), word_lo(w[1]), word_hi(w[1])};
  }
};
struct LayerBackState {
  static constexpr int WORDS = 1;
  float m, X;
  GFN_DEV void pack(unsigned long long (&w)[1]) const { w[0] = scan_word(m, X); }
  GFN_DEV static LayerBackState unpack(const unsigned long long (&w)[1]) { return {word_lo(w[0]), word_hi(w[0])}; }
  GFN_DEV LayerBackState through(LayerBackMap f) const { return {pass(f.P, m, pass(f.R, X, f.q)), X + f.G}; }
};

template <int VEC, int S, int NW, int OCC>
__global__ void __launch_bounds__(NW * 32, OCC) lscan_backward_kernel(const LScanArgs p) {
  static_assert(NW * S == SCAN_CK, "one kept state per run");
  constexpr int CT = 32 * VEC;
  __shared__ ScanShared<LayerBackMap, LayerBackState, CT, NW> sh;
  __shared__ unsigned long long fmaps[NW][CT];
  const ScanTile c = scan_tile<VEC>(p, &sh.slot);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int run = p.nchunks - 1 - c.chunk;
  const int t0 = run * SCAN_CK + w * S;
  const int n = c.active ? max(0, min(S, p.L - t0)) : 0;
  const long long o = ((long long)c.b * p.L + t0) * p.D + c.col;
  const float* zp = p.z + 3 * (o - c.col) + c.col;
  Pack<float, VEC> A[S], dt[S], zb[S], gx[S], gv[S], sa[S], sd[S];  // sa, sd: slopes of A and dt
#pragma unroll
  for (int s = 0; s < S; ++s) {  // beyond the end: A = 1, dt = 0, zB = 0, no gradients
    A[s] = fill_pack<float, VEC>(INFINITY);
    dt[s] = fill_pack<float, VEC>(-INFINITY);
    zb[s] = gx[s] = gv[s] = fill_pack<float, VEC>(0.f);
    if (s < n) {
      A[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D);
      dt[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D + p.D);
      zb[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D + 2LL * p.D);
      if (p.gx) gx[s] = load_pack<float, VEC>(p.gx + o + (long long)s * p.D);
      if (p.gv) gv[s] = load_pack<float, VEC>(p.gv + o + (long long)s * p.D);
    }
  }
  float h[VEC];  // v before the run
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    h[v] = c.active ? p.states[((long long)c.b * p.nck + run) * p.D + c.col + v] : 0.f;
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const float scale = p.base_dt * head_scale(c.col + v, p.D / p.H);
    GatedMap mf = GatedMap::identity();
    bool zero = false;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      A[s].v[v] = gate(A[s].v[v], &sa[s].v[v]);
      dt[s].v[v] = soft_step(dt[s].v[v], &sd[s].v[v]) * scale;
      sd[s].v[v] *= scale;
      zero = zero || A[s].v[v] == 0.f;
      mf.P *= A[s].v[v];
      mf.p = fmaf(A[s].v[v], mf.p, zb[s].v[v] * dt[s].v[v]);
    }
    if (mf.P == 0.f && !zero) mf.P = 1.4e-45f;
    LayerBackMap mb = LayerBackMap::identity();
    mb.P = mf.P;
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      mb.G += gx[s].v[v];
      mb.q = A[s].v[v] * (fmaf(dt[s].v[v], mb.G, gv[s].v[v]) + mb.q);
      mb.R = A[s].v[v] * (mb.R + dt[s].v[v]);
    }
    unsigned long long wd[2], wf[1];
    mf.pack(wf);
    fmaps[w][lane * VEC + v] = wf[0];
    mb.pack(wd);
    sh.maps[w][0][lane * VEC + v] = wd[0];
    sh.maps[w][1][lane * VEC + v] = wd[1];
  }
  receive<LayerBackMap, LayerBackState, CT, NW, true>(
      sh, p.words + c.tile * p.nchunks * (2LL * CT), c.chunk, p.nchunks, p.D - c.c0, [&](int j) {
        const long long e = (long long)c.b * p.D + c.c0 + j;
        return LayerBackState{p.gvl ? p.gvl[e] : 0.f, p.gxl ? p.gxl[e] : 0.f};
      });
  if (!c.active) return;
  LayerBackState st[VEC];
  float vs[S + 1][VEC];  // v_{t-1} of this warp's steps, and the last step's v
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    st[v] = sh.in[lane * VEC + v].through(
        LayerBackMap::unpack({sh.maps[w][0][lane * VEC + v], sh.maps[w][1][lane * VEC + v]}));
    for (int j = 0; j < w; ++j) {
      const GatedMap f = GatedMap::unpack({fmaps[j][lane * VEC + v]});
      h[v] = pass(f.P, h[v], f.p);
    }
    vs[0][v] = h[v];
#pragma unroll
    for (int s = 0; s < S; ++s) vs[s + 1][v] = fmaf(A[s].v[v], vs[s][v], zb[s].v[v] * dt[s].v[v]);
  }
  float* dz = p.dz + 3 * (o - c.col) + c.col;
#pragma unroll
  for (int s = S - 1; s >= 0; --s) {
    Pack<float, VEC> oa, od, ob;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      st[v].X += gx[s].v[v];
      const float l = fmaf(dt[s].v[v], st[v].X, gv[s].v[v]) + st[v].m;
      oa.v[v] = l * vs[s][v] * sa[s].v[v];
      od.v[v] = (l * zb[s].v[v] + st[v].X * vs[s + 1][v]) * sd[s].v[v];
      ob.v[v] = l * dt[s].v[v];
      st[v].m = A[s].v[v] * l;
    }
    if (s < n) {
      store_pack<float, VEC>(dz + (long long)s * 3 * p.D, oa);
      store_pack<float, VEC>(dz + (long long)s * 3 * p.D + p.D, od);
      store_pack<float, VEC>(dz + (long long)s * 3 * p.D + 2LL * p.D, ob);
    }
  }
  if (run == 0 && w == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const long long e = (long long)c.b * p.D + c.col + v;
      if (p.dv0) p.dv0[e] = st[v].m;
      if (p.dx0) p.dx0[e] = st[v].X;
    }
  }
}

// A few steps, or none: one thread per column (as gscan_forward_seq_kernel).
__global__ void __launch_bounds__(128) lscan_forward_seq_kernel(const LScanArgs p) {
  const long long c = blockIdx.x * 128LL + threadIdx.x;
  if (c >= (long long)p.B * p.D) return;
  const long long b = c / p.D, j = c - b * p.D;
  const float scale = p.base_dt * head_scale((int)j, p.D / p.H);
  float v = p.v0 ? p.v0[c] : 0.f, x = p.x0 ? p.x0[c] : 0.f;
  if (p.states && p.L) p.states[c] = v;
#pragma unroll 4
  for (int t = 0; t < p.L; ++t) {
    const float* z = p.z + (b * p.L + t) * 3 * p.D + j;
    float slope;
    const float dt = soft_step(z[p.D], &slope) * scale;
    v = fmaf(gate(z[0], &slope), v, z[2LL * p.D] * dt);
    x = fmaf(v, dt, x);
    const long long e = (b * p.L + t) * p.D + j;
    p.vs[e] = v;
    p.xs[e] = x;
  }
  if (p.v_last) p.v_last[c] = v;
  if (p.x_last) p.x_last[c] = x;
}

}  // namespace gfn
