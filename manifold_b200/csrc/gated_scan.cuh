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

// M (a map or a state) of `chunk` as its block published it; `words` is the
// column tile's [nchunks][WORDS of a map][32 VEC] words.
template <class M, int W, int VEC>
GFN_DEV void await(const unsigned long long* words, int chunk, M (&out)[VEC]) {
  constexpr int CT = 32 * VEC;
  const unsigned long long* src = words + (long long)chunk * W * CT + (threadIdx.x & 31) * VEC;
  unsigned long long got[VEC][M::WORDS];
  for (int spin = 0;; ++spin) {
    bool ready = true;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
#pragma unroll
      for (int i = 0; i < M::WORDS; ++i) {
        got[v][i] = word_load(src + i * CT + v);
        ready = ready && (unsigned)got[v][i] != SCAN_EMPTY;
      }
    }
    if (ready) break;
    if (spin == (1 << 22)) {  // seconds: flag it and carry on with what is there
      gfn_flag_error(kDevErrMbarTimeout);
      break;
    }
    __nanosleep(20);
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) out[v] = M::unpack(got[v]);
}

template <class M, int W, int VEC>
GFN_DEV void publish(const M (&m)[VEC], unsigned long long* words, int chunk) {
  constexpr int CT = 32 * VEC;
  unsigned long long* dst = words + (long long)chunk * W * CT + (threadIdx.x & 31) * VEC;
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    unsigned long long w[M::WORDS];
    m[v].pack(w);
#pragma unroll
    for (int i = 0; i < M::WORDS; ++i) word_store(dst + i * CT + v, w[i]);
  }
}

// The state that `chunk` (counted in the direction of the scan) of a column
// tile receives, from its own map `own` (of the whole run; used in the last
// run of a group) and `first`, the state before chunk 0.  The whole block
// takes part; `teller` is true in the one warp that publishes.  `found` is
// shared memory for one map per warp and column.
template <class Map, class State, int VEC, int NW>
GFN_DEV void receive(unsigned long long* words, int chunk, int nchunks, bool active, bool teller,
                     const Map (&own)[VEC], const State (&first)[VEC],
                     unsigned long long (*found)[Map::WORDS][32 * VEC], State (&in)[VEC]) {
  constexpr int W = Map::WORDS, K = SCAN_GROUP / NW;
  static_assert(SCAN_GROUP % NW == 0, "each warp fetches the same number of maps");
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pos = chunk % SCAN_GROUP, start = chunk - pos;
  const bool tells = teller && active && chunk + 1 < nchunks;
  if (tells && pos < SCAN_GROUP - 1) publish<Map, W, VEC>(own, words, chunk);
  Map acc[VEC];  // of the group's runs before this one
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = Map::identity();
  if (pos > 0) {
    const int k0 = w * K;
    if (active && k0 < pos) {
      await<Map, W, VEC>(words, start + k0, acc);
      for (int k = k0 + 1; k < min(k0 + K, pos); ++k) {
        Map next[VEC];
        await<Map, W, VEC>(words, start + k, next);
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = Map::compose(next[v], acc[v]);
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        unsigned long long x[W];
        acc[v].pack(x);
#pragma unroll
        for (int i = 0; i < W; ++i) found[w][i][lane * VEC + v] = x[i];
      }
    }
    __syncthreads();
    const int n = (pos + K - 1) / K;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      acc[v] = Map::identity();
      for (int j = 0; j < n && active; ++j) {
        unsigned long long x[W];
#pragma unroll
        for (int i = 0; i < W; ++i) x[i] = found[j][i][lane * VEC + v];
        acc[v] = Map::compose(Map::unpack(x), acc[v]);
      }
    }
  }
  State at[VEC];  // at the group's start
#pragma unroll
  for (int v = 0; v < VEC; ++v) at[v] = first[v];
  if (start > 0 && active) await<State, W, VEC>(words, start - 1, at);
  if (tells && pos == SCAN_GROUP - 1) {
    State end[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) end[v] = at[v].through(Map::compose(own[v], acc[v]));
    publish<State, W, VEC>(end, words, chunk);
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) in[v] = at[v].through(acc[v]);
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
  int chunk, b, col;
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
  r.col = (int)(r.tile - (long long)r.b * p.ctiles) * (32 * VEC) + (threadIdx.x & 31) * VEC;
  r.active = r.col < p.D;
  return r;
}

// ------------------------------------------------------------------ gated scan
template <typename T, int VEC, int S, int NW>
__global__ void __launch_bounds__(NW * 32) gscan_forward_kernel(const GScanArgs p) {
  constexpr int CT = 32 * VEC;
  __shared__ unsigned long long maps[NW][1][CT], found[NW][1][CT];
  __shared__ unsigned slot;
  const ScanTile q = scan_tile<VEC>(p, &slot);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = (q.chunk * NW + w) * S;
  const int n = q.active ? max(0, min(S, p.L - t0)) : 0;
  Pack<T, VEC> a[S], x[S];
  {
    const T* xp = static_cast<const T*>(p.x) + q.b * p.x_sb + t0 * p.x_st + q.col;
    const T* ap = static_cast<const T*>(p.a) + q.b * p.a_sb + t0 * p.a_st + q.col;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        x[s] = load_pack<T, VEC>(xp + s * p.x_st);
        if (p.a) a[s] = load_pack<T, VEC>(ap + s * p.a_st);
      }
    }
    if (!p.a) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) a[s].v[v] = from_f<T>(1.f);
      }
    }
  }
  GatedMap m[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    m[v] = GatedMap::identity();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        const float g = to_f(a[s].v[v]);
        m[v].P *= g;
        m[v].p = fmaf(g, m[v].p, to_f(x[s].v[v]));
      }
    }
    if (m[v].P == 0.f) {  // a zero gate, or an underflow?
      bool zero = false;
#pragma unroll
      for (int s = 0; s < S; ++s) zero = zero || (s < n && to_f(a[s].v[v]) == 0.f);
      if (!zero) m[v].P = copysignf(1.4e-45f, m[v].P);
    }
    unsigned long long wd[1];
    m[v].pack(wd);
    maps[w][0][lane * VEC + v] = wd[0];
  }
  __syncthreads();
  GatedMap before[VEC];  // of the warps before this one
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    before[v] = GatedMap::identity();
    for (int j = 0; j < w; ++j) before[v] = GatedMap::compose(GatedMap::unpack({maps[j][0][lane * VEC + v]}), before[v]);
  }
  unsigned long long* words = p.words + q.tile * p.nchunks * (long long)CT;
  GatedState first[VEC], in[VEC];
  GatedMap own[VEC];  // of the whole run, in the last warp
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    first[v].h = (p.h0 && q.active) ? p.h0[(long long)q.b * p.D + q.col + v] : 0.f;
    own[v] = GatedMap::compose(m[v], before[v]);
  }
  receive<GatedMap, GatedState, VEC, NW>(words, q.chunk, p.nchunks, q.active, w == NW - 1, own, first, found, in);
  float h[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) h[v] = in[v].through(before[v]).h;
  if (n <= 0) return;
  if (p.states && t0 % SCAN_CK == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.states[((long long)q.b * p.nck + t0 / SCAN_CK) * p.D + q.col + v] = h[v];
  }
  T* hp = static_cast<T*>(p.h) + ((long long)q.b * p.L + t0) * p.D + q.col;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (s < n) {
      Pack<T, VEC> o;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        h[v] = fmaf(to_f(a[s].v[v]), h[v], to_f(x[s].v[v]));
        o.v[v] = from_f<T>(h[v]);
      }
      store_pack<T, VEC>(hp + (long long)s * p.D, o);
    }
  }
  if (p.h_last && t0 + n == p.L) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.h_last[(long long)q.b * p.D + q.col + v] = h[v];
  }
}

// Runs of NW * S = SCAN_CK steps from the last to the first: the state kept
// before the run gives h, the messages pass from run to run as the states do
// in the forward.
template <typename T, int VEC, int S, int NW>
__global__ void __launch_bounds__(NW * 32) gscan_backward_kernel(const GScanArgs p) {
  static_assert(NW * S == SCAN_CK, "one kept state per run");
  constexpr int CT = 32 * VEC;
  __shared__ unsigned long long fmaps[NW][CT], maps[NW][CT], found[NW][1][CT];
  __shared__ unsigned slot;
  const ScanTile q = scan_tile<VEC>(p, &slot);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int run = p.nchunks - 1 - q.chunk;
  const int t0 = run * SCAN_CK + w * S;
  const int n = q.active ? max(0, min(S, p.L - t0)) : 0;
  Pack<T, VEC> a[S], x[S], g[S];
  {
    const T* xp = static_cast<const T*>(p.x) + q.b * p.x_sb + t0 * p.x_st + q.col;
    const T* ap = static_cast<const T*>(p.a) + q.b * p.a_sb + t0 * p.a_st + q.col;
    const T* gp = static_cast<const T*>(p.dh) + q.b * p.g_sb + t0 * p.g_st + q.col;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        x[s] = load_pack<T, VEC>(xp + s * p.x_st);
        if (p.a) a[s] = load_pack<T, VEC>(ap + s * p.a_st);
        if (p.dh) g[s] = load_pack<T, VEC>(gp + s * p.g_st);
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (!p.a) a[s].v[v] = from_f<T>(1.f);
        if (!p.dh) g[s].v[v] = from_f<T>(0.f);
      }
    }
  }
  GatedMap mb[VEC];  // of the message, last step first
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    GatedMap mf = GatedMap::identity();
    mb[v] = GatedMap::identity();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        const float c = to_f(a[s].v[v]);
        mf.P *= c;
        mf.p = fmaf(c, mf.p, to_f(x[s].v[v]));
      }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s)
      if (s < n) mb[v].p = to_f(a[s].v[v]) * (to_f(g[s].v[v]) + mb[v].p);
    if (mf.P == 0.f) {
      bool zero = false;
#pragma unroll
      for (int s = 0; s < S; ++s) zero = zero || (s < n && to_f(a[s].v[v]) == 0.f);
      if (!zero) mf.P = copysignf(1.4e-45f, mf.P);
    }
    mb[v].P = mf.P;
    unsigned long long wd[1];
    mf.pack(wd);
    fmaps[w][lane * VEC + v] = wd[0];
    mb[v].pack(wd);
    maps[w][lane * VEC + v] = wd[0];
  }
  __syncthreads();
  GatedMap after[VEC];  // of the warps behind this one, whose messages arrive first
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    after[v] = GatedMap::identity();
    for (int j = NW - 1; j > w; --j)
      after[v] = GatedMap::compose(GatedMap::unpack({maps[j][lane * VEC + v]}), after[v]);
  }
  unsigned long long* words = p.words + q.tile * p.nchunks * (long long)CT;
  // h_{t-1} of this warp's steps, from the kept state
  float hp[S][VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float h = 0.f;
    if (q.active) h = p.states[((long long)q.b * p.nck + run) * p.D + q.col + v];
    for (int j = 0; j < w; ++j) {
      const GatedMap f = GatedMap::unpack({fmaps[j][lane * VEC + v]});
      h = pass(f.P, h, f.p);
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      hp[s][v] = h;
      if (s < n) h = fmaf(to_f(a[s].v[v]), h, to_f(x[s].v[v]));
    }
  }
  GatedState first[VEC], in[VEC];
  GatedMap own[VEC];  // of the whole run, in the first warp
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    first[v].h = (p.dlast && q.active) ? p.dlast[(long long)q.b * p.D + q.col + v] : 0.f;
    own[v] = GatedMap::compose(mb[v], after[v]);
  }
  receive<GatedMap, GatedState, VEC, NW>(words, q.chunk, p.nchunks, q.active, w == 0, own, first, found, in);
  float m[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) m[v] = in[v].through(after[v]).h;
  const long long o = ((long long)q.b * p.L + t0) * p.D + q.col;
#pragma unroll
  for (int s = S - 1; s >= 0; --s) {
    if (s < n) {
      Pack<T, VEC> oa, ox;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float gt = to_f(g[s].v[v]) + m[v];
        ox.v[v] = from_f<T>(gt);
        oa.v[v] = from_f<T>(gt * hp[s][v]);
        m[v] = to_f(a[s].v[v]) * gt;
      }
      if (p.dx) store_pack<T, VEC>(static_cast<T*>(p.dx) + o + (long long)s * p.D, ox);
      if (p.da) store_pack<T, VEC>(static_cast<T*>(p.da) + o + (long long)s * p.D, oa);
    }
  }
  if (p.dh0 && run == 0 && w == 0 && q.active) {
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

// sigma(z) and sigma(-z) from one exponential that cannot overflow: both keep
// their digits far out, where 1 / (1 + exp(-z)) is already 0 or 1.
GFN_DEV float gate(float z, float* complement) {
  const float e = expf(-fabsf(z)), r = 1.f / (1.f + e);
  *complement = z >= 0.f ? e * r : r;
  return z >= 0.f ? r : e * r;
}

GFN_DEV float gate(float z) {
  float c;
  return gate(z, &c);
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

template <int VEC, int S, int NW>
__global__ void __launch_bounds__(NW * 32) lscan_forward_kernel(const LScanArgs p) {
  constexpr int CT = 32 * VEC;
  __shared__ unsigned long long maps[NW][2][CT], found[NW][2][CT];
  __shared__ unsigned slot;
  const ScanTile c = scan_tile<VEC>(p, &slot);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = (c.chunk * NW + w) * S;
  const int n = c.active ? max(0, min(S, p.L - t0)) : 0;
  const float* zp = p.z + ((long long)c.b * p.L + t0) * 3 * p.D + c.col;
  Pack<float, VEC> A[S], dt[S], bv[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (s < n) {
      A[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D);
      dt[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D + p.D);
      bv[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D + 2LL * p.D);
    }
  }
  LayerMap m[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const float hs = head_scale(c.col + v, p.D / p.H);
    m[v] = LayerMap::identity();
    bool zero = false;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        A[s].v[v] = gate(A[s].v[v]);
        dt[s].v[v] = (softplus_f(dt[s].v[v]) * p.base_dt) * hs;
        bv[s].v[v] *= dt[s].v[v];
        zero = zero || A[s].v[v] == 0.f;
        m[v].P *= A[s].v[v];
        m[v].p = fmaf(A[s].v[v], m[v].p, bv[s].v[v]);
        m[v].Q = fmaf(dt[s].v[v], m[v].P, m[v].Q);
        m[v].q = fmaf(dt[s].v[v], m[v].p, m[v].q);
      }
    }
    if (m[v].P == 0.f && !zero) m[v].P = 1.4e-45f;
    unsigned long long wd[2];
    m[v].pack(wd);
    maps[w][0][lane * VEC + v] = wd[0];
    maps[w][1][lane * VEC + v] = wd[1];
  }
  __syncthreads();
  LayerMap before[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    before[v] = LayerMap::identity();
    for (int j = 0; j < w; ++j)
      before[v] = LayerMap::compose(LayerMap::unpack({maps[j][0][lane * VEC + v], maps[j][1][lane * VEC + v]}),
                                    before[v]);
  }
  unsigned long long* words = p.words + c.tile * p.nchunks * (2LL * CT);
  LayerState first[VEC], in[VEC];
  LayerMap own[VEC];  // of the whole run, in the last warp
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const long long e = (long long)c.b * p.D + c.col + v;
    first[v].v = (p.v0 && c.active) ? p.v0[e] : 0.f;
    first[v].x = (p.x0 && c.active) ? p.x0[e] : 0.f;
    own[v] = LayerMap::compose(m[v], before[v]);
  }
  receive<LayerMap, LayerState, VEC, NW>(words, c.chunk, p.nchunks, c.active, w == NW - 1, own, first, found, in);
  LayerState st[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) st[v] = in[v].through(before[v]);
  if (n <= 0) return;
  if (p.states && t0 % SCAN_CK == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.states[((long long)c.b * p.nck + t0 / SCAN_CK) * p.D + c.col + v] = st[v].v;
  }
  const long long o = ((long long)c.b * p.L + t0) * p.D + c.col;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (s < n) {
      Pack<float, VEC> ov, ox;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        st[v].v = fmaf(A[s].v[v], st[v].v, bv[s].v[v]);
        st[v].x = fmaf(st[v].v, dt[s].v[v], st[v].x);
        ov.v[v] = st[v].v;
        ox.v[v] = st[v].x;
      }
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

template <int VEC, int S, int NW>
__global__ void __launch_bounds__(NW * 32) lscan_backward_kernel(const LScanArgs p) {
  static_assert(NW * S == SCAN_CK, "one kept state per run");
  constexpr int CT = 32 * VEC;
  __shared__ unsigned long long fmaps[NW][CT], maps[NW][2][CT], found[NW][2][CT];
  __shared__ unsigned slot;
  const ScanTile c = scan_tile<VEC>(p, &slot);
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int run = p.nchunks - 1 - c.chunk;
  const int t0 = run * SCAN_CK + w * S;
  const int n = c.active ? max(0, min(S, p.L - t0)) : 0;
  const long long o = ((long long)c.b * p.L + t0) * p.D + c.col;
  const float* zp = p.z + 3 * (o - c.col) + c.col;
  Pack<float, VEC> za[S], zd[S], zb[S], gx[S], gv[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (s < n) {
      za[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D);
      zd[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D + p.D);
      zb[s] = load_pack<float, VEC>(zp + (long long)s * 3 * p.D + 2LL * p.D);
      if (p.gx) gx[s] = load_pack<float, VEC>(p.gx + o + (long long)s * p.D);
      if (p.gv) gv[s] = load_pack<float, VEC>(p.gv + o + (long long)s * p.D);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      if (!p.gx) gx[s].v[v] = 0.f;
      if (!p.gv) gv[s].v[v] = 0.f;
    }
  }
  float scale[VEC];
  LayerBackMap mb[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    scale[v] = head_scale(c.col + v, p.D / p.H);
    GatedMap mf = GatedMap::identity();
    bool zero = false;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        const float A = gate(za[s].v[v]), dt = (softplus_f(zd[s].v[v]) * p.base_dt) * scale[v];
        zero = zero || A == 0.f;
        mf.P *= A;
        mf.p = fmaf(A, mf.p, zb[s].v[v] * dt);
      }
    }
    if (mf.P == 0.f && !zero) mf.P = 1.4e-45f;
    mb[v] = LayerBackMap::identity();
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      if (s < n) {
        const float A = gate(za[s].v[v]), dt = (softplus_f(zd[s].v[v]) * p.base_dt) * scale[v];
        mb[v].G += gx[s].v[v];
        mb[v].q = A * (fmaf(dt, mb[v].G, gv[s].v[v]) + mb[v].q);
        mb[v].R = A * (mb[v].R + dt);
      }
    }
    mb[v].P = mf.P;
    unsigned long long wd[2], wf[1];
    mf.pack(wf);
    fmaps[w][lane * VEC + v] = wf[0];
    mb[v].pack(wd);
    maps[w][0][lane * VEC + v] = wd[0];
    maps[w][1][lane * VEC + v] = wd[1];
  }
  __syncthreads();
  LayerBackMap after[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    after[v] = LayerBackMap::identity();
    for (int j = NW - 1; j > w; --j)
      after[v] = LayerBackMap::compose(
          LayerBackMap::unpack({maps[j][0][lane * VEC + v], maps[j][1][lane * VEC + v]}), after[v]);
  }
  unsigned long long* words = p.words + c.tile * p.nchunks * (2LL * CT);
  float vs[S + 1][VEC];  // v_{t-1} of this warp's steps, and the last step's v
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float h = 0.f;
    if (c.active) h = p.states[((long long)c.b * p.nck + run) * p.D + c.col + v];
    for (int j = 0; j < w; ++j) {
      const GatedMap f = GatedMap::unpack({fmaps[j][lane * VEC + v]});
      h = pass(f.P, h, f.p);
    }
    vs[0][v] = h;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n)
        h = fmaf(gate(za[s].v[v]), h, zb[s].v[v] * ((softplus_f(zd[s].v[v]) * p.base_dt) * scale[v]));
      vs[s + 1][v] = h;
    }
  }
  LayerBackState first[VEC], in[VEC];
  LayerBackMap own[VEC];  // of the whole run, in the first warp
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const long long e = (long long)c.b * p.D + c.col + v;
    first[v].m = (p.gvl && c.active) ? p.gvl[e] : 0.f;
    first[v].X = (p.gxl && c.active) ? p.gxl[e] : 0.f;
    own[v] = LayerBackMap::compose(mb[v], after[v]);
  }
  receive<LayerBackMap, LayerBackState, VEC, NW>(words, c.chunk, p.nchunks, c.active, w == 0, own, first, found, in);
  LayerBackState st[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) st[v] = in[v].through(after[v]);
  float* dz = p.dz + 3 * (o - c.col) + c.col;
#pragma unroll
  for (int s = S - 1; s >= 0; --s) {
    if (s < n) {
      Pack<float, VEC> oa, od, ob;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float nA;
        const float A = gate(za[s].v[v], &nA);
        const float dt = (softplus_f(zd[s].v[v]) * p.base_dt) * scale[v];
        st[v].X += gx[s].v[v];
        const float l = fmaf(dt, st[v].X, gv[s].v[v]) + st[v].m;
        oa.v[v] = l * vs[s][v] * (A * nA);
        od.v[v] = (l * zb[s].v[v] + st[v].X * vs[s + 1][v]) * (p.base_dt * scale[v]) * gate(zd[s].v[v]);
        ob.v[v] = l * dt;
        st[v].m = A * l;
      }
      store_pack<float, VEC>(dz + (long long)s * 3 * p.D, oa);
      store_pack<float, VEC>(dz + (long long)s * 3 * p.D + p.D, od);
      store_pack<float, VEC>(dz + (long long)s * 3 * p.D + 2LL * p.D, ob);
    }
  }
  if (run == 0 && w == 0 && c.active) {
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
  const float hs = head_scale((int)j, p.D / p.H);
  float v = p.v0 ? p.v0[c] : 0.f, x = p.x0 ? p.x0[c] : 0.f;
  if (p.states && p.L) p.states[c] = v;
#pragma unroll 4
  for (int t = 0; t < p.L; ++t) {
    const float* z = p.z + (b * p.L + t) * 3 * p.D + j;
    const float dt = (softplus_f(z[p.D]) * p.base_dt) * hs;
    v = fmaf(gate(z[0]), v, z[2LL * p.D] * dt);
    x = fmaf(v, dt, x);
    const long long e = (b * p.L + t) * p.D + j;
    p.vs[e] = v;
    p.xs[e] = x;
  }
  if (p.v_last) p.v_last[c] = v;
  if (p.x_last) p.x_last[c] = x;
}

}  // namespace gfn
