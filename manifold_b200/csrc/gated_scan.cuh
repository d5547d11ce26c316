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
// is far too small to fill the GPU.  Runs form groups: a run composes the maps
// of its group before it and applies them to the state at the group's start,
// which the group before publishes.  What is composed with what does not
// depend on which block is faster, so results repeat bit for bit.
// (Looking back for the nearest state instead did not, and one block per
// column with no split took 33.7 ms where this takes 62 us, at 1 x 65536 x 512.)
//
// Measured on B200 (CUDA events around workspace clearing and kernel; copy
// bandwidth 6.46 TB/s):
//   forward   128 x 512 x 512 float32    75 us, 5.4 TB/s
//             16 x 2048 x 512 float32    46 us, 4.4 TB/s
//             1 x 65536 x 512 bfloat16   62 us, 3.2 TB/s
//             3 x 5003 x 1001 bfloat16   54 us, 1.7 TB/s (rows off 16 bytes)
//   backward  118, 74, 100 and 84 us: 5.7, 4.5, 3.3 and 1.8 TB/s
// (With products of gates in plain float32, wrong where they leave its range, 44,
// 59 and 52 us forward and 71, 96 and 80 backward for the last three.)
// With many columns they run at the memory's rate.  With few, what is left is
// the way of a map through global memory and the wait for the group's state,
// about 6,000 of a block's 14,000 cycles per run; off 16 bytes, the loads'
// latency and 67 (forward) to 114 (backward) instructions per element.
#pragma once
#include <cfloat>
#include <type_traits>

#include "lm_ops.cuh"
#include "umma.cuh"

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
  int group;            // runs whose maps are composed; the states pass from group to group
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

// ------------------------------------------------------------ products of gates
// A product P of the gates of many steps leaves float32's range long before
// P h does, and may come back (256 gates of 0.5, then 256 of 1.9).  It is held in
// 32 bits of wider range: a product from 2^-99 to 2^100, 0 or NaN is that float,
// and codes that are other floats stand for 2^-278 to 2^-99 and 2^100 to 2^278
// with 20 bits after the point, as the high word of a float64 has them (one such
// rounding is eight of float32's, on a product that has decayed or grown by 2^99).
// Above that it is infinite: any state would be.  Below it is GAIN_TINY: every
// finite state has underflowed to zero, an infinite one stays infinite.  Both
// remain, whatever gates follow, as such a state does step by step.
constexpr unsigned GAIN_TINY = 1u, GAIN_INF = 0x7f800000u;
constexpr unsigned GAIN_LOW_CODES = 0x00800000u, GAIN_HIGH_CODES = 0x72000000u;  // of 2^-278 and of 2^100
constexpr unsigned GAIN_PLAIN = 0x0e000000u;  // 2^-99: floats from here to GAIN_HIGH_CODES are themselves
constexpr float GAIN_LEAST = 0x1p-99f;
constexpr int GAIN_STUCK = 1 << 20;  // |e| of a product beyond the codes

GFN_DEV unsigned gain_magnitude(float g) { return __float_as_uint(g) & 0x7fffffffu; }
GFN_DEV bool gain_plain(float g) { return gain_magnitude(g) - GAIN_PLAIN < GAIN_HIGH_CODES - GAIN_PLAIN; }

struct Gain {  // m 2^e
  float m;     // of either sign, from 1 on; 0 or NaN
  int e;

  GFN_DEV static Gain of_plain(float g) {
    return {__uint_as_float((__float_as_uint(g) & 0x807fffffu) | 0x3f800000u), (int)(gain_magnitude(g) >> 23) - 127};
  }
  GFN_DEV static Gain of(float g) {
    const unsigned u = gain_magnitude(g), sign = __float_as_uint(g) & 0x80000000u;
    if (gain_plain(g)) return of_plain(g);
    if (u == 0 || u > GAIN_INF) return {g, 0};
    if (u == GAIN_TINY || u == GAIN_INF)
      return {__uint_as_float(sign | 0x3f800000u), u == GAIN_TINY ? -GAIN_STUCK : GAIN_STUCK};
    const unsigned w = u < GAIN_PLAIN ? u - GAIN_LOW_CODES : u - GAIN_HIGH_CODES;
    return {__uint_as_float(sign | ((w & 0x000fffffu) << 3) | 0x3f800000u),
            (int)(w >> 20) + (u < GAIN_PLAIN ? -278 : 100)};
  }
  // this, then l (fewer than 64 products are multiplied before they are packed)
  GFN_DEV void append(Gain l) {
    m *= l.m;
    if (e > -GAIN_STUCK / 2 && e < GAIN_STUCK / 2) e += l.e;
  }
  GFN_DEV float pack() const {
    const unsigned u = gain_magnitude(m), sign = __float_as_uint(m) & 0x80000000u;
    const int x = (int)(u >> 23) - 127 + e;
    if (u == 0) return e < GAIN_STUCK / 2 ? m : __uint_as_float(0x7fffffffu);  // 0 after an infinity: NaN
    if (u > GAIN_INF) return m;
    if (x >= -99 && x < 100) return __uint_as_float(sign | (u + ((unsigned)e << 23)));
    if (x < -278) return __uint_as_float(sign | GAIN_TINY);
    if (x >= 278) return __uint_as_float(sign | GAIN_INF);
    const unsigned w = ((u & 0x007fffffu) + 4u) >> 3;  // to 20 bits; 2^20 moves into the exponent
    return __uint_as_float(sign | ((x < 0 ? ((unsigned)(x + 278) << 20) + GAIN_LOW_CODES
                                          : ((unsigned)(x - 100) << 20) + GAIN_HIGH_CODES) + w));
  }
  GFN_DEV float carry(float h, float p) const {  // P h + p
    const double P = (double)m * __hiloint2double((max(-1000, min(1000, e)) + 1023) << 20, 0);
    return (float)fma(P, (double)h, (double)p);
  }
};

// A P below 2^-99 drops a state below 2^73 times what is added to it: at most
// 2^-26 of that, half of a rounding.
GFN_DEV bool gain_small(float P) { return fabsf(P) < GAIN_LEAST; }
GFN_DEV bool gain_drops(float h, float p) { return fabsf(h) <= fminf(0x1p73f * fabsf(p), FLT_MAX); }
// P h + p for a packed P.
GFN_DEV float carry(float P, float h, float p) {
  if (gain_plain(P)) return fmaf(P, h, p);
  return h == 0.f || (gain_small(P) && gain_drops(h, p)) ? p : Gain::of(P).carry(h, p);
}
// The same for other factors.  In both a zero state passes as p alone (an infinite P must not make NaN of it).
GFN_DEV float pass(float P, float h, float p) { return h == 0.f ? p : fmaf(P, h, p); }

// The rare ways through a run or a group are calls: in line their registers
// would be taken from the walk over the operands.
//
// The packed product of n gates, mantissas and exponents multiplied apart.
__device__ __noinline__ float gain_of_gates(const float* gates, int n) {
  Gain r = {1.f, 0};
  float special = 1.f;
  for (int s = 0; s < n; ++s) {
    float g = gates[s];
    if (g == 0.f || !(fabsf(g) < INFINITY)) {
      special *= g;
    } else {
      if (fabsf(g) < 0x1p-126f) {  // subnormal
        g *= 0x1p32f;
        r.e -= 32;
      }
      const unsigned u = __float_as_uint(g);
      r.m *= __uint_as_float((u & 0x807fffffu) | 0x3f800000u);
      r.e += (int)((u >> 23) & 255u) - 127;
    }
  }
  return special != 1.f ? special : r.pack();  // 0, an infinity or NaN among the gates decides
}

// The same of S gates, given as float32's products of every 8 of them and the
// largest magnitude among them.  Such a product is right if it is in the plain
// range and no part of it can have left float32's normal range on the way: with
// magnitudes up to 2^(26 / 8) what follows a part grows by 2^26 at most, so the
// part was at least 2^-126.
template <int S, class Gate>
GFN_DEV float gain_run(const float (&eights)[S / 8], float largest, Gate gate) {
  static_assert(S <= 32, "");
  float all = eights[0];
  bool right = largest <= 9.5f && gain_plain(eights[0]);
#pragma unroll
  for (int k = 1; k < S / 8; ++k) {
    all *= eights[k];
    right = right && gain_plain(eights[k]);
  }
  if (right && gain_plain(all) && (S <= 16 || largest <= 1.f)) return all;
  if (right) {
    Gain r = Gain::of_plain(eights[0]);
#pragma unroll
    for (int k = 1; k < S / 8; ++k) {
      const Gain l = Gain::of_plain(eights[k]);
      r = {r.m * l.m, r.e + l.e};
    }
    return r.pack();
  }
  float gates[S];
#pragma unroll
  for (int s = 0; s < S; ++s) gates[s] = gate(s);
  return gain_of_gates(gates, S);
}

// Maps of a run of steps, and chains of them: append(l) puts l behind what is
// there.  Chain is right for every P.  Quick serves the usual case in float32,
// products of at most 1 that drop what they are handed where they are below 2^-99;
// where that does not hold, ok turns false and the maps have to be gone through
// again as a Chain.  append_plain(l) is for a P from 2^-99 to 1.
struct GatedMap {  // h -> P h + p
  static constexpr int WORDS = 1;
  float P, p;
  GFN_DEV void pack(unsigned long long (&w)[WORDS]) const { w[0] = scan_word(P, p); }
  GFN_DEV static GatedMap unpack(const unsigned long long (&w)[WORDS]) { return {word_lo(w[0]), word_hi(w[0])}; }
  struct Chain {
    Gain P = {1.f, 0};
    float p = 0.f;
    GFN_DEV void append(GatedMap l) {
      p = carry(l.P, p, l.p);
      P.append(Gain::of(l.P));
    }
    GFN_DEV GatedMap map() const { return {P.pack(), p}; }
  };
  struct Quick {
    float P = 1.f, p = 0.f;
    bool ok = true;
    GFN_DEV void append_plain(GatedMap l) {
      p = fmaf(l.P, p, l.p);
      P *= l.P;
    }
    GFN_DEV void append(GatedMap l) {
      if (gain_small(l.P)) {
        ok = ok && (gain_drops(p, l.p) || (l.P == 0.f && fabsf(p) < INFINITY));
        l.P = 0.f;
      }
      ok = ok && fabsf(l.P) <= 1.f;
      append_plain(l);
    }
    GFN_DEV bool right() const { return ok; }
    GFN_DEV GatedMap map() const { return {ok ? P : INFINITY, p}; }
  };
};
struct GatedState {
  static constexpr int WORDS = 1;
  float h;
  GFN_DEV void pack(unsigned long long (&w)[1]) const { w[0] = scan_word(h, 0.f); }
  GFN_DEV static GatedState unpack(const unsigned long long (&w)[1]) { return {word_lo(w[0])}; }
  GFN_DEV GatedState through(GatedMap m) const { return {carry(m.P, h, m.p)}; }
  GFN_DEV bool through(const GatedMap::Quick& m, GatedState& out) const {  // whether it can
    const bool small = gain_small(m.P);
    out.h = fmaf(small ? 0.f : m.P, h, m.p);
    return m.right() && (!small || gain_drops(h, m.p));
  }
};

constexpr int SCAN_GROUP = 32;  // the most runs in a group

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
  unsigned slot[2];                             // tickets drawn ahead
  uint64_t bar;                                 // the staged operands' arrival
  // the thread that issues the copies: neither a teller nor, where there are others, a `beside`
  static constexpr int ISSUER = R > 2 ? CT : 0;

  GFN_DEV void init() {
    if (threadIdx.x == 0) {
      mbar_init(&bar, 1);
      fence_mbar_init();
    }
    __syncthreads();
  }
};

// The map of warp j of a run (counted in the direction of the scan) for column c,
// and in its place what is before it.
template <class Map, bool REV, int CT, int NW, class Chain>
GFN_DEV Map before_warp(const Chain& before, unsigned long long (*maps)[Map::WORDS][CT], int j, int c) {
  unsigned long long x[Map::WORDS], y[Map::WORDS];
  unsigned long long(&at)[Map::WORDS][CT] = maps[REV ? NW - 1 - j : j];
  before.map().pack(y);
#pragma unroll
  for (int i = 0; i < Map::WORDS; ++i) {
    x[i] = at[i][c];
    at[i][c] = y[i];
  }
  return Map::unpack(x);
}
template <class Map, bool REV, int CT, int NW>
__device__ __noinline__ Map chain_warps(unsigned long long (*maps)[Map::WORDS][CT], int c) {
  typename Map::Chain all;
  for (int j = 0; j < NW; ++j) all.append(before_warp<Map, REV, CT, NW>(all, maps, j, c));
  return all.map();
}
// `at` through the n maps of the group before a run, which are all published.
template <class Map, class State>
__device__ __noinline__ State chain_group(State at, const unsigned long long* words, long long stride, int ct, int n) {
  typename Map::Chain all;
  for (int k = 0; k < n; ++k) {
    Map next[1];
    await<Map, 1>(words + k * stride, 0, ct, 1, next);
    all.append(next[0]);
    all.P = Gain::of(all.P.pack());
  }
  return at.through(all.map());
}

// The state that `chunk` (counted in the direction of the scan) of a column
// tile receives.  Call with the warps' maps in sh.maps; on return (after a
// barrier) sh.maps[w] holds the map of the warps before w, counted in the
// direction of the scan (REV: from the last warp), and sh.in the states.
// R threads serve a column: the last of them chains the warps' maps and
// publishes, all of them fetch their share of the group's earlier maps.
// `words` is the tile's [nchunks][WORDS][CT]; first(c) the state before chunk 0;
// beside(c) runs on another thread per column, between the barriers, and ahead()
// on all threads once this block's map is out.
template <class Map, class State, int CT, int NW, bool REV, class First, class Beside, class Ahead>
GFN_DEV void receive(ScanShared<Map, State, CT, NW>& sh, unsigned long long* words, int chunk, int nchunks,
                     int group, int live, First first, Beside beside, Ahead ahead) {
  static_assert(ScanShared<Map, State, CT, NW>::R >= 2, "a second thread per column");
  constexpr int W = Map::WORDS, R = NW * 32 / CT, GS = SCAN_GROUP / R;
  constexpr int BATCH = GS < 8 ? GS : 8;
  const int c = threadIdx.x % CT, r = threadIdx.x / CT;
  const bool active = c < live, teller = r == R - 1 && active;
  const int pos = chunk % group, start = chunk - pos;
  const bool tells = teller && chunk + 1 < nchunks;
  unsigned long long* mine = words + (long long)chunk * W * CT + c;
  Map own;  // of this run
  __syncthreads();
  if (teller) {
    float P = 1.f;
    bool plain = true;  // a product of at most 1, and no part of it below the plain range
#pragma unroll
    for (int j = 0; j < NW; ++j) {
      const float f = word_lo(sh.maps[j][0][c]);
      plain = plain && fabsf(f) <= 1.f;
      P *= f;
    }
    if (plain && fabsf(P) >= GAIN_LEAST) {
      typename Map::Quick all;
#pragma unroll
      for (int j = 0; j < NW; ++j) all.append_plain(before_warp<Map, REV, CT, NW>(all, sh.maps, j, c));
      own = all.map();
    } else {
      own = chain_warps<Map, REV, CT, NW>(sh.maps, c);
    }
    if (tells && pos < group - 1) publish(own, mine, CT);
  }
  ahead();
  if (r == 0) beside(c);
  typename Map::Quick acc;  // of the group's runs before this one
  if (pos > 0) {
    if (active && r * GS < pos) {
      for (int k = r * GS; k < min((r + 1) * GS, pos); k += BATCH) {
        const int n = min(BATCH, min((r + 1) * GS, pos) - k);
        Map next[BATCH];
        await<Map, BATCH>(words + (long long)(start + k) * W * CT + c, W * CT, CT, n, next);
        float least = 1.f, most = 0.f;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          if (i < n) {
            least = fminf(least, fabsf(next[i].P));
            most = fmaxf(most, fabsf(next[i].P));
          }
        }
        if (least >= GAIN_LEAST && most <= 1.f) {  // a NaN goes through as one
#pragma unroll
          for (int i = 0; i < BATCH; ++i)
            if (i < n) acc.append_plain(next[i]);
        } else {
#pragma unroll
          for (int i = 0; i < BATCH; ++i)
            if (i < n) acc.append(next[i]);
        }
      }
      unsigned long long x[W];
      acc.map().pack(x);
#pragma unroll
      for (int i = 0; i < W; ++i) sh.part[r][i][c] = x[i];
    }
    __syncthreads();
    if (teller) {
      acc = typename Map::Quick();
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (j * GS < pos) {
          unsigned long long x[W];
#pragma unroll
          for (int i = 0; i < W; ++i) x[i] = sh.part[j][i][c];
          acc.append(Map::unpack(x));
        }
      }
    }
  }
  if (teller) {
    State at[1], in;  // at the group's start; before this run
    if (start > 0) await<State, 1>(words + (long long)(start - 1) * W * CT + c, 0, CT, 1, at);
    else at[0] = first(c);
    if (!at[0].through(acc, in)) in = chain_group<Map, State>(at[0], words + (long long)start * W * CT + c, W * CT, CT, pos);
    if (tells && pos == group - 1) publish(in.through(own), mine, CT);
    sh.in[c] = in;
  }
  __syncthreads();
}

// ------------------------------------------------------------ vector accesses
// VEC neighbouring elements as they lie in memory, in whole registers: 16-bit
// pairs stay packed until a value is used.
template <typename T, int VEC>
struct Pack {
  static constexpr int BYTES = sizeof(T) * VEC, N = (BYTES + 3) / 4;
  unsigned u[N];

  GFN_DEV float get(int v) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[v]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return __uint_as_float((v & 1) ? u[v >> 1] & 0xffff0000u : u[v >> 1] << 16);
    else return __half2float(__ushort_as_half((unsigned short)((v & 1) ? u[v >> 1] >> 16 : u[v >> 1] & 0xffffu)));
  }
  GFN_DEV static Pack of(const float (&f)[VEC]) {
    Pack r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) r.u[v] = __float_as_uint(f[v]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const T lo = from_f<T>(f[2 * i]), hi = from_f<T>(2 * i + 1 < VEC ? f[2 * i + 1] : 0.f);
        r.u[i] = (unsigned)bits16(lo) | ((unsigned)bits16(hi) << 16);
      }
    }
    return r;
  }
  GFN_DEV static Pack fill(float v) {
    float f[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = v;
    return of(f);
  }
  GFN_DEV static Pack load(const T* p) {  // read once: evict first
    Pack r;
    if constexpr (BYTES == 2) r.u[0] = __ldcs(reinterpret_cast<const unsigned short*>(p));
    else if constexpr (N == 1) r.u[0] = __ldcs(reinterpret_cast<const unsigned*>(p));
    else {
      const uint2 x = __ldcs(reinterpret_cast<const uint2*>(p));
      r.u[0] = x.x;
      r.u[1] = x.y;
    }
    return r;
  }
  GFN_DEV void store(T* p) const {
    if constexpr (BYTES == 2) __stcs(reinterpret_cast<unsigned short*>(p), (unsigned short)u[0]);
    else if constexpr (N == 1) __stcs(reinterpret_cast<unsigned*>(p), u[0]);
    else __stcs(reinterpret_cast<uint2*>(p), make_uint2(u[0], u[1]));
  }
  GFN_DEV static unsigned short bits16(__nv_bfloat16 x) { return __bfloat16_as_ushort(x); }
  GFN_DEV static unsigned short bits16(__half x) { return __half_as_ushort(x); }
};

// Which run of steps and which columns a block computes.  Runs are numbered in
// the direction of the scan, all column tiles of one run before the next, and
// handed out by a ticket: whatever a block waits for has a lower number, and
// the lowest unfinished number is always being computed, so every wait ends.
// A block draws its ticket one run ahead.
struct ScanTile {
  int chunk, b, c0, col;  // c0: the tile's first column; col: this lane's first
  int first, t0;          // the run's first step and this warp's
  int n;                  // steps of this lane: 0 beyond the end or the columns
  long long tile;
};

template <int VEC, int S, int NW, bool REV, class Args>
GFN_DEV ScanTile scan_tile(const Args& p, unsigned t) {
  ScanTile r;
  const unsigned tiles = (unsigned)p.B * p.ctiles;
  r.chunk = t / tiles;
  r.tile = t - (unsigned)r.chunk * tiles;
  r.b = (int)(r.tile / p.ctiles);
  r.c0 = (int)(r.tile - (long long)r.b * p.ctiles) * (32 * VEC);
  r.col = r.c0 + (threadIdx.x & 31) * VEC;
  r.first = (REV ? p.nchunks - 1 - r.chunk : r.chunk) * (NW * S);
  r.t0 = r.first + (threadIdx.x >> 5) * S;
  r.n = r.col < p.D ? max(0, min(S, p.L - r.t0)) : 0;
  return r;
}

struct ScanTurn {
  unsigned cur, next, drawn, total;

  template <class Args>
  GFN_DEV ScanTurn(const Args& p, unsigned (&slot)[2]) {
    total = (unsigned)p.B * p.ctiles * (unsigned)p.nchunks;
    cur = blockIdx.x;
    if (p.words) {
      if (threadIdx.x == 0) slot[1] = atomicAdd(p.ticket, 1u) + 1u;  // starts at all ones, like the words
      __syncthreads();
      cur = slot[1];
    }
  }
  // Drawn once this run's operands have arrived, so that every block that
  // runs has drawn its first before any draws its second.
  template <class Args>
  GFN_DEV void draw(const Args& p) {
    if (p.words && threadIdx.x == 0) drawn = atomicAdd(p.ticket, 1u) + 1u;
  }
  template <class Args>
  GFN_DEV void tell(const Args& p, unsigned (&slot)[2], int it) const {
    if (p.words && threadIdx.x == 0) slot[it & 1] = drawn;
  }
  // after a barrier that follows tell()
  template <class Args>
  GFN_DEV void hear(const Args& p, const unsigned (&slot)[2], int it) {
    next = p.words ? slot[it & 1] : cur + gridDim.x;
  }
};

// -------------------------------------------------------------------- operands
// How a run's operands reach the registers:
//   TMA     rows that start on 16 bytes: one thread issues a tensor copy per
//           operand for the NEXT run as soon as this run's values are in
//           registers, so the memory stays busy through the exchange of maps;
//   PLAIN   any other rows: each lane loads one column's elements when the run
//           begins.  (Pairs of 16-bit elements assembled from the aligned words
//           around them measured slower: 63 against 49 us forward and 86
//           against 78 backward at 3 x 5003 x 1001.)
enum { SCAN_TMA, SCAN_PLAIN };

// S rows of this lane, `step` elements apart, of which n exist.
template <typename T, int VEC, int S>
GFN_DEV void load_rows(Pack<T, VEC> (&out)[S], const T* src, long long step, int n) {
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (s < n) out[s] = Pack<T, VEC>::load(src + s * step);
}

// The operands as [batch][step][column] tensors with boxes of one run's steps
// of one column tile.
struct ScanMaps {
  CUtensorMap m[3];
};

// Shared memory for one run's rows, [operand][NW * S][32 VEC], and the barrier
// on which they arrive.
template <typename T, int VEC, int S, int NW>
struct Stage {
  static constexpr int ROW = 32 * VEC * sizeof(T), OPERAND = NW * S * ROW;  // bytes
  char* base;
  uint64_t* bar;

  GFN_DEV void expect(int operands) const { mbar_arrive_expect_tx(bar, (uint32_t)(operands * OPERAND)); }
  GFN_DEV void fetch(int operand, const CUtensorMap* map, int col, const ScanTile& q) const {
    umma::tma_load_3d(base + operand * OPERAND, map, bar, col, q.first, q.b);
  }
  GFN_DEV Pack<T, VEC> take(int operand, int s) const {
    Pack<T, VEC> r;
    const char* from = base + operand * OPERAND + ((threadIdx.x >> 5) * S + s) * ROW + (threadIdx.x & 31) * r.BYTES;
    if constexpr (r.N == 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(from);
      r.u[0] = x.x;
      r.u[1] = x.y;
    } else {
      r.u[0] = *reinterpret_cast<const unsigned*>(from);
    }
    return r;
  }
};

// Keeps packed values packed: without it the compiler carries the unpacked
// floats of the first pass over to the second, in twice the registers.
template <typename T, int VEC, int S>
GFN_DEV void keep_packed(Pack<T, VEC> (&a)[S]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int i = 0; i < Pack<T, VEC>::N; ++i) asm volatile("" : "+r"(a[s].u[i]));
    }
  }
}

// ------------------------------------------------------------------ gated scan
// Map of S steps from a zero state; steps beyond the end hold a = 1, x = 0.
template <typename T, int VEC, int S>
GFN_DEV GatedMap run_map(const Pack<T, VEC> (&a)[S], const Pack<T, VEC> (&x)[S], int v) {
  float eights[S / 8], p = 0.f, largest = 0.f;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const float g = a[s].get(v);
    eights[s / 8] = s % 8 ? eights[s / 8] * g : g;
    largest = fmaxf(largest, fabsf(g));
    p = fmaf(g, p, x[s].get(v));
  }
  return {gain_run<S>(eights, largest, [&](int s) { return a[s].get(v); }), p};
}

template <int MODE, typename T, int VEC, int S, int NW, int OCC>
__global__ void __launch_bounds__(NW * 32, OCC) gscan_forward_kernel(const GScanArgs p, const __grid_constant__ ScanMaps maps) {
  constexpr int CT = 32 * VEC;
  extern __shared__ __align__(128) unsigned staged[];
  __shared__ ScanShared<GatedMap, GatedState, CT, NW> sh;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Stage<T, VEC, S, NW> stage = {reinterpret_cast<char*>(staged), &sh.bar};
  auto row = [](const void* base, const ScanTile& q, long long sb, long long st, int t, int col) {
    return static_cast<const T*>(base) + q.b * sb + t * st + col;
  };
  auto fetch = [&](unsigned turn) {
    if (MODE != SCAN_TMA || threadIdx.x != sh.ISSUER) return;
    const ScanTile q = scan_tile<VEC, S, NW, false>(p, turn);
    stage.expect(1 + (p.a != nullptr));
    stage.fetch(0, &maps.m[0], q.c0, q);
    if (p.a) stage.fetch(1, &maps.m[1], q.c0, q);
  };
  if constexpr (MODE == SCAN_TMA) sh.init();
  ScanTurn turn(p, sh.slot);
  if (turn.cur < turn.total) fetch(turn.cur);
  for (int it = 0; turn.cur < turn.total; turn.cur = turn.next, ++it) {
    const ScanTile q = scan_tile<VEC, S, NW, false>(p, turn.cur);
    Pack<T, VEC> a[S], x[S];
    if constexpr (MODE == SCAN_TMA) {
      mbar_wait(&sh.bar, it & 1);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        x[s] = stage.take(0, s);
        a[s] = stage.take(1, s);
      }
    } else {
      load_rows<T, VEC, S>(x, row(p.x, q, p.x_sb, p.x_st, q.t0, q.col), p.x_st, q.n);
      if (p.a) load_rows<T, VEC, S>(a, row(p.a, q, p.a_sb, p.a_st, q.t0, q.col), p.a_st, q.n);
    }
    turn.draw(p);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s >= q.n) x[s] = Pack<T, VEC>::fill(0.f);
      if (s >= q.n || !p.a) a[s] = Pack<T, VEC>::fill(1.f);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      unsigned long long wd[1];
      run_map<T, VEC, S>(a, x, v).pack(wd);
      sh.maps[w][0][lane * VEC + v] = wd[0];
    }
    turn.tell(p, sh.slot, it);
    receive<GatedMap, GatedState, CT, NW, false>(
        sh, p.words + q.tile * p.nchunks * (long long)CT, q.chunk, p.nchunks, p.group, p.D - q.c0,
        [&](int c) { return GatedState{p.h0 ? p.h0[(long long)q.b * p.D + q.c0 + c] : 0.f}; },
        [](int) {},
        [&] {
          turn.hear(p, sh.slot, it);
          if (turn.next < turn.total) fetch(turn.next);
        });
    if (q.n <= 0) continue;
    keep_packed(a);
    keep_packed(x);
    float h[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      h[v] = sh.in[lane * VEC + v].through(GatedMap::unpack({sh.maps[w][0][lane * VEC + v]})).h;
    if (p.states && q.t0 % SCAN_CK == 0) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) p.states[((long long)q.b * p.nck + q.t0 / SCAN_CK) * p.D + q.col + v] = h[v];
    }
    T* hp = static_cast<T*>(p.h) + ((long long)q.b * p.L + q.t0) * p.D + q.col;
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[v] = fmaf(a[s].get(v), h[v], x[s].get(v));
      if (s < q.n) Pack<T, VEC>::of(h).store(hp + (long long)s * p.D);
    }
    if (p.h_last && q.t0 + q.n == p.L) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) p.h_last[(long long)q.b * p.D + q.col + v] = h[v];
    }
  }
}

// h before each warp's steps, from the state kept before the run and the
// warps' maps: column c, one thread.
template <int CT, int NW>
GFN_DEV void chain_states(const unsigned long long (*maps)[CT], const float* kept, int c, int live,
                          float (*start)[CT]) {
  if (c >= live) return;
  float h = kept[c];
#pragma unroll
  for (int j = 0; j < NW; ++j) {
    start[j][c] = h;
    const GatedMap f = GatedMap::unpack({maps[j][c]});
    h = carry(f.P, h, f.p);
  }
}

// Runs of NW * S steps from the last to the first: the state kept before the
// run gives h, the messages pass from run to run as the states do in the
// forward.
template <int MODE, typename T, int VEC, int S, int NW, int OCC>
__global__ void __launch_bounds__(NW * 32, OCC) gscan_backward_kernel(const GScanArgs p, const __grid_constant__ ScanMaps maps) {
  static_assert(NW * S % SCAN_CK == 0, "a kept state at every run's start");
  constexpr int CT = 32 * VEC;
  extern __shared__ __align__(128) unsigned staged[];
  __shared__ ScanShared<GatedMap, GatedState, CT, NW> sh;
  __shared__ unsigned long long fmaps[NW][CT];
  __shared__ float hstart[NW][CT];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Stage<T, VEC, S, NW> stage = {reinterpret_cast<char*>(staged), &sh.bar};
  auto row = [](const void* base, const ScanTile& q, long long sb, long long st, int t, int col) {
    return static_cast<const T*>(base) + q.b * sb + t * st + col;
  };
  auto fetch = [&](unsigned turn) {
    if (MODE != SCAN_TMA || threadIdx.x != sh.ISSUER) return;
    const ScanTile q = scan_tile<VEC, S, NW, true>(p, turn);
    stage.expect(1 + (p.a != nullptr) + (p.dh != nullptr));
    stage.fetch(0, &maps.m[0], q.c0, q);
    if (p.a) stage.fetch(1, &maps.m[1], q.c0, q);
    if (p.dh) stage.fetch(2, &maps.m[2], q.c0, q);
  };
  if constexpr (MODE == SCAN_TMA) sh.init();
  ScanTurn turn(p, sh.slot);
  if (turn.cur < turn.total) fetch(turn.cur);
  for (int it = 0; turn.cur < turn.total; turn.cur = turn.next, ++it) {
    const ScanTile q = scan_tile<VEC, S, NW, true>(p, turn.cur);
    Pack<T, VEC> a[S], x[S], g[S];
    if constexpr (MODE == SCAN_TMA) {
      mbar_wait(&sh.bar, it & 1);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        x[s] = stage.take(0, s);
        a[s] = stage.take(1, s);
        g[s] = stage.take(2, s);
      }
    } else {
      load_rows<T, VEC, S>(x, row(p.x, q, p.x_sb, p.x_st, q.t0, q.col), p.x_st, q.n);
      if (p.a) load_rows<T, VEC, S>(a, row(p.a, q, p.a_sb, p.a_st, q.t0, q.col), p.a_st, q.n);
      if (p.dh) load_rows<T, VEC, S>(g, row(p.dh, q, p.g_sb, p.g_st, q.t0, q.col), p.g_st, q.n);
    }
    turn.draw(p);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s >= q.n) x[s] = Pack<T, VEC>::fill(0.f);
      if (s >= q.n || !p.a) a[s] = Pack<T, VEC>::fill(1.f);
      if (s >= q.n || !p.dh) g[s] = Pack<T, VEC>::fill(0.f);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      unsigned long long wd[1];
      const GatedMap mf = run_map<T, VEC, S>(a, x, v);
      mf.pack(wd);
      fmaps[w][lane * VEC + v] = wd[0];
      GatedMap mb = {mf.P, 0.f};  // of the message, last step first
#pragma unroll
      for (int s = S - 1; s >= 0; --s) mb.p = a[s].get(v) * (g[s].get(v) + mb.p);
      mb.pack(wd);
      sh.maps[w][0][lane * VEC + v] = wd[0];
    }
    turn.tell(p, sh.slot, it);
    const int run = p.nchunks - 1 - q.chunk;
    receive<GatedMap, GatedState, CT, NW, true>(
        sh, p.words + q.tile * p.nchunks * (long long)CT, q.chunk, p.nchunks, p.group, p.D - q.c0,
        [&](int c) { return GatedState{p.dlast ? p.dlast[(long long)q.b * p.D + q.c0 + c] : 0.f}; },
        [&](int c) {
          chain_states<CT, NW>(fmaps, p.states + ((long long)q.b * p.nck + q.first / SCAN_CK) * p.D + q.c0, c, p.D - q.c0, hstart);
        },
        [&] {
          turn.hear(p, sh.slot, it);
          if (turn.next < turn.total) fetch(turn.next);
        });
    if (q.n <= 0) continue;
    keep_packed(a);
    keep_packed(x);
    keep_packed(g);
    float m[VEC], hp[S][VEC];  // hp: h_{t-1}
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      m[v] = sh.in[lane * VEC + v].through(GatedMap::unpack({sh.maps[w][0][lane * VEC + v]})).h;
      hp[0][v] = hstart[w][lane * VEC + v];
#pragma unroll
      for (int s = 1; s < S; ++s) hp[s][v] = fmaf(a[s - 1].get(v), hp[s - 1][v], x[s - 1].get(v));
    }
    const long long o = ((long long)q.b * p.L + q.t0) * p.D + q.col;
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      float oa[VEC], ox[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        ox[v] = g[s].get(v) + m[v];
        oa[v] = ox[v] * hp[s][v];
        m[v] = a[s].get(v) * ox[v];
      }
      if (s < q.n) {
        const long long e = o + (long long)s * p.D;
        if (p.dx) Pack<T, VEC>::of(ox).store(static_cast<T*>(p.dx) + e);
        if (p.da) Pack<T, VEC>::of(oa).store(static_cast<T*>(p.da) + e);
      }
    }
    if (p.dh0 && run == 0 && w == 0) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) p.dh0[(long long)q.b * p.D + q.col + v] = m[v];
    }
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
  int B, L, D, H, nck, nchunks, ctiles, group;
  float base_dt;
};

// 1 / v to one unit in the last place, for v in [1, 6].
GFN_DEV float quick_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
GFN_DEV F2 quick_rcp(F2 v) {
  float lo, hi;
  split(v, lo, hi);
  return f2(quick_rcp(lo), quick_rcp(hi));
}

// Two gates at a time, sigma(z) and its slope sigma(z) sigma(-z), from one
// exponential each that cannot overflow: both keep their digits far out, where
// 1 / (1 + exp(-z)) is already 0 or 1.
GFN_DEV void gates(float z0, float z1, float& a0, float& a1, F2& slope) {
  const F2 e = f2(expf(-fabsf(z0)), expf(-fabsf(z1)));
  const F2 r = quick_rcp(e + f2(1.f)), c = e * r;
  slope = r * c;
  float r0, r1, c0, c1;
  split(r, r0, r1);
  split(c, c0, c1);
  a0 = z0 >= 0.f ? r0 : c0;
  a1 = z1 >= 0.f ? r1 : c1;
}

// Two steps at a time: softplus(z) = max(z, 0) + log1p(e), e = exp(-|z|) in
// [0, 1], and its slope sigma(z).  log1p(e) = 2 atanh(y) with
// y = e / (2 + e) <= 1/3, and atanh(y) / y as a polynomial in y^2 (interpolated
// at the Chebyshev nodes of [0, 1/9]: within 8e-9 of it, an eighth of a
// float32 rounding), so that a small step keeps its digits, which log(1 + e)
// would lose.
GFN_DEV F2 soft_steps(float z0, float z1, F2& slope) {
  const F2 e = f2(expf(-fabsf(z0)), expf(-fabsf(z1)));
  const F2 e1 = e + f2(1.f), e2 = e + f2(2.f);
  const F2 r = quick_rcp(e1 * e2);  // both quotients from one reciprocal
  const F2 y = e * (e1 * r), y2 = y * y, s = e2 * r, c = e * s;
  F2 q = f2(0.14078889f);
  q = fma2(q, y2, f2(0.13982579f));
  q = fma2(q, y2, f2(0.20012298f));
  q = fma2(q, y2, f2(0.33333161f));
  q = fma2(q * y2, y, y);
  float s0, s1, c0, c1;
  split(s, s0, s1);
  split(c, c0, c1);
  slope = f2(z0 >= 0.f ? s0 : c0, z1 >= 0.f ? s1 : c1);
  return fma2(f2(2.f), q, f2(fmaxf(z0, 0.f), fmaxf(z1, 0.f)));
}

GFN_DEV float head_scale(int col, int hd) {
  float hs = 1.f;
  for (int i = 0; i < col / hd; ++i) hs *= 1.5f;
  return hs;
}

struct LayerMap {  // v -> P v + p, x -> x + Q v + q
  static constexpr int WORDS = 2;
  float P, p, Q, q;
  GFN_DEV void pack(unsigned long long (&w)[2]) const {
    w[0] = scan_word(P, p);
    w[1] = scan_word(Q, q);
  }
  GFN_DEV static LayerMap unpack(const unsigned long long (&w)[2]) {
    return {word_lo(w[0]), word_hi(w[0]), word_lo(w[1]), word_hi(w[1])};
  }
  struct Chain {
    Gain P = {1.f, 0};
    float p = 0.f, Q = 0.f, q = 0.f;
    GFN_DEV void append(LayerMap l) {
      Q = P.carry(l.Q, Q);
      q += pass(l.Q, p, l.q);
      p = carry(l.P, p, l.p);
      P.append(Gain::of(l.P));
    }
    GFN_DEV LayerMap map() const { return {P.pack(), p, Q, q}; }
  };
  struct Quick {
    float P = 1.f, p = 0.f, Q = 0.f, q = 0.f, most = 0.f;  // most: the largest Q appended
    bool ok = true;
    GFN_DEV void append_plain(LayerMap l) {
      most = fmaxf(most, l.Q);
      Q = fmaf(l.Q, P, Q);
      q += pass(l.Q, p, l.q);
      p = fmaf(l.P, p, l.p);
      P *= l.P;
    }
    GFN_DEV void append(LayerMap l) {
      if (gain_small(l.P)) {
        ok = ok && (gain_drops(p, l.p) || (l.P == 0.f && fabsf(p) < INFINITY));
        l.P = 0.f;
      }
      ok = ok && fabsf(l.P) <= 1.f;
      append_plain(l);
    }
    // Q adds up to 32 terms of Q P with a P below 2^-99 that may have been 0
    GFN_DEV bool right() const { return ok && most <= fminf(0x1p68f * Q, FLT_MAX); }
    GFN_DEV LayerMap map() const { return {right() ? P : INFINITY, p, Q, q}; }
  };
};
struct LayerState {
  static constexpr int WORDS = 1;
  float v, x;
  GFN_DEV void pack(unsigned long long (&w)[1]) const { w[0] = scan_word(v, x); }
  GFN_DEV static LayerState unpack(const unsigned long long (&w)[1]) { return {word_lo(w[0]), word_hi(w[0])}; }
  GFN_DEV LayerState through(LayerMap m) const { return {carry(m.P, v, m.p), x + pass(m.Q, v, m.q)}; }
  GFN_DEV bool through(const LayerMap::Quick& m, LayerState& out) const {
    const bool small = gain_small(m.P);
    out = {fmaf(small ? 0.f : m.P, v, m.p), x + pass(m.Q, v, m.q)};
    return m.right() && (!small || gain_drops(v, m.p));
  }
};

// 20 bytes per element, and 72 instructions: two exponentials, two reciprocals
// and a polynomial, two steps at a time where packed arithmetic does both (one
// at a time 86 instructions and 134 us).  Runs of 128 steps of 32 columns, two
// blocks per SM: at 32 x 2048 x 512 132 us, 5.1 TB/s (runs of 64 steps of 64
// columns 155 us); at 1 x 20000 x 256, where 8 column tiles leave 5 rounds of
// blocks, 43 us.
template <int MODE, int VEC, int S, int NW, int OCC>
__global__ void __launch_bounds__(NW * 32, OCC) lscan_forward_kernel(const LScanArgs p, const __grid_constant__ ScanMaps maps) {
  constexpr int CT = 32 * VEC;
  extern __shared__ __align__(128) unsigned staged[];
  __shared__ ScanShared<LayerMap, LayerState, CT, NW> sh;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Stage<float, VEC, S, NW> stage = {reinterpret_cast<char*>(staged), &sh.bar};
  auto fetch = [&](unsigned turn) {
    if (MODE != SCAN_TMA || threadIdx.x != sh.ISSUER) return;
    const ScanTile c = scan_tile<VEC, S, NW, false>(p, turn);
    stage.expect(3);
#pragma unroll
    for (int k = 0; k < 3; ++k) stage.fetch(k, &maps.m[0], k * p.D + c.c0, c);
  };
  if constexpr (MODE == SCAN_TMA) sh.init();
  ScanTurn turn(p, sh.slot);
  if (turn.cur < turn.total) fetch(turn.cur);
  for (int it = 0; turn.cur < turn.total; turn.cur = turn.next, ++it) {
    const ScanTile c = scan_tile<VEC, S, NW, false>(p, turn.cur);
    Pack<float, VEC> pa[S], pd[S], pb[S];
    if constexpr (MODE == SCAN_TMA) {
      mbar_wait(&sh.bar, it & 1);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        pa[s] = stage.take(0, s);
        pd[s] = stage.take(1, s);
        pb[s] = stage.take(2, s);
      }
    } else {
      const float* zp = p.z + ((long long)c.b * p.L + c.t0) * 3 * p.D + c.col;
      load_rows<float, VEC, S>(pa, zp, 3LL * p.D, c.n);
      load_rows<float, VEC, S>(pd, zp + p.D, 3LL * p.D, c.n);
      load_rows<float, VEC, S>(pb, zp + 2LL * p.D, 3LL * p.D, c.n);
    }
    turn.draw(p);
    if (c.n < S) {  // beyond the end: A = 1, dt = 0
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (s >= c.n) {
          pa[s] = Pack<float, VEC>::fill(INFINITY);
          pd[s] = Pack<float, VEC>::fill(-INFINITY);
          pb[s] = Pack<float, VEC>::fill(0.f);
        }
      }
    }
    float A[S][VEC], dt[S][VEC], bv[S][VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float scale = p.base_dt * head_scale(c.col + v, p.D / p.H);
      LayerMap m = {1.f, 0.f, 0.f, 0.f};
      float eights[S / 8];
#pragma unroll
      for (int s = 0; s < S; s += 2) {
        F2 slope;
        gates(pa[s].get(v), pa[s + 1].get(v), A[s][v], A[s + 1][v], slope);
        const F2 d = soft_steps(pd[s].get(v), pd[s + 1].get(v), slope) * f2(scale);
        split(d, dt[s][v], dt[s + 1][v]);
        split(d * f2(pb[s].get(v), pb[s + 1].get(v)), bv[s][v], bv[s + 1][v]);
      }
#pragma unroll
      for (int s = 0; s < S; ++s) {
        m.P *= A[s][v];
        eights[s / 8] = s % 8 ? eights[s / 8] * A[s][v] : A[s][v];
        m.p = fmaf(A[s][v], m.p, bv[s][v]);
        m.Q = fmaf(dt[s][v], m.P, m.Q);
        m.q = fmaf(dt[s][v], m.p, m.q);
      }
      m.P = gain_run<S>(eights, 1.f, [&](int s) { return A[s][v]; });
      unsigned long long wd[2];
      m.pack(wd);
      sh.maps[w][0][lane * VEC + v] = wd[0];
      sh.maps[w][1][lane * VEC + v] = wd[1];
    }
    turn.tell(p, sh.slot, it);
    receive<LayerMap, LayerState, CT, NW, false>(
        sh, p.words + c.tile * p.nchunks * (2LL * CT), c.chunk, p.nchunks, p.group, p.D - c.c0,
        [&](int j) {
          const long long e = (long long)c.b * p.D + c.c0 + j;
          return LayerState{p.v0 ? p.v0[e] : 0.f, p.x0 ? p.x0[e] : 0.f};
        },
        [](int) {},
        [&] {
          turn.hear(p, sh.slot, it);
          if (turn.next < turn.total) fetch(turn.next);
        });
    if (c.n <= 0) continue;
    LayerState st[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      st[v] = sh.in[lane * VEC + v].through(
          LayerMap::unpack({sh.maps[w][0][lane * VEC + v], sh.maps[w][1][lane * VEC + v]}));
    if (p.states && c.t0 % SCAN_CK == 0) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) p.states[((long long)c.b * p.nck + c.t0 / SCAN_CK) * p.D + c.col + v] = st[v].v;
    }
    const long long o = ((long long)c.b * p.L + c.t0) * p.D + c.col;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float ov[VEC], ox[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        st[v].v = fmaf(A[s][v], st[v].v, bv[s][v]);
        st[v].x = fmaf(st[v].v, dt[s][v], st[v].x);
        ov[v] = st[v].v;
        ox[v] = st[v].x;
      }
      if (s < c.n) {
        Pack<float, VEC>::of(ov).store(p.vs + o + (long long)s * p.D);
        Pack<float, VEC>::of(ox).store(p.xs + o + (long long)s * p.D);
      }
    }
    if (c.t0 + c.n == p.L) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const long long e = (long long)c.b * p.D + c.col + v;
        if (p.v_last) p.v_last[e] = st[v].v;
        if (p.x_last) p.x_last[e] = st[v].x;
      }
    }
  }
}

struct LayerBackMap {  // m -> P m + R X + q, X -> X + G
  static constexpr int WORDS = 2;
  float P, q, R, G;
  GFN_DEV void pack(unsigned long long (&w)[2]) const {
    w[0] = scan_word(P, q);
    w[1] = scan_word(R, G);
  }
  GFN_DEV static LayerBackMap unpack(const unsigned long long (&w)[2]) {
    return {word_lo(w[0]), word_hi(w[0]), word_lo(w[1]), word_hi(w[1])};
  }
  struct Chain {
    Gain P = {1.f, 0};
    float q = 0.f, R = 0.f, G = 0.f;
    GFN_DEV void append(LayerBackMap l) {
      q = carry(l.P, q, pass(l.R, G, l.q));
      R = carry(l.P, R, l.R);
      G += l.G;
      P.append(Gain::of(l.P));
    }
    GFN_DEV LayerBackMap map() const { return {P.pack(), q, R, G}; }
  };
  struct Quick {
    float P = 1.f, q = 0.f, R = 0.f, G = 0.f;
    bool ok = true;
    GFN_DEV void append_plain(LayerBackMap l) {
      q = fmaf(l.P, q, pass(l.R, G, l.q));
      R = fmaf(l.P, R, l.R);
      G += l.G;
      P *= l.P;
    }
    GFN_DEV void append(LayerBackMap l) {
      if (gain_small(l.P)) {
        ok = ok && gain_drops(q, pass(l.R, G, l.q)) && gain_drops(R, l.R);
        l.P = 0.f;
      }
      ok = ok && fabsf(l.P) <= 1.f;
      append_plain(l);
    }
    GFN_DEV bool right() const { return ok; }
    GFN_DEV LayerBackMap map() const { return {ok ? P : INFINITY, q, R, G}; }
  };
};
struct LayerBackState {
  static constexpr int WORDS = 1;
  float m, X;
  GFN_DEV void pack(unsigned long long (&w)[1]) const { w[0] = scan_word(m, X); }
  GFN_DEV static LayerBackState unpack(const unsigned long long (&w)[1]) { return {word_lo(w[0]), word_hi(w[0])}; }
  GFN_DEV LayerBackState through(LayerBackMap f) const { return {carry(f.P, m, pass(f.R, X, f.q)), X + f.G}; }
  GFN_DEV bool through(const LayerBackMap::Quick& f, LayerBackState& out) const {
    const bool small = gain_small(f.P);
    const float in = pass(f.R, X, f.q);
    out = {fmaf(small ? 0.f : f.P, m, in), X + f.G};
    return f.right() && (!small || gain_drops(m, in));
  }
};

// 28 bytes per element (32 with a gradient of v) and 128 instructions, issued
// at 55% of the rate: instructions, the exchange's waits and memory share the
// time.  The gates, steps and slopes stay in registers between the two walks
// (recomputing them took 298 us); v is recomputed from its kept state instead
// of read.  At 32 x 2048 x 512 226 us, 4.2 TB/s.
template <int MODE, int VEC, int S, int NW, int OCC>
__global__ void __launch_bounds__(NW * 32, OCC) lscan_backward_kernel(const LScanArgs p, const __grid_constant__ ScanMaps maps) {
  static_assert(NW * S % SCAN_CK == 0, "a kept state at every run's start");
  constexpr int CT = 32 * VEC;
  extern __shared__ __align__(128) unsigned staged[];
  __shared__ ScanShared<LayerBackMap, LayerBackState, CT, NW> sh;
  __shared__ unsigned long long fmaps[NW][CT];
  __shared__ float vstart[NW][CT];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Stage<float, VEC, S, NW> stage = {reinterpret_cast<char*>(staged), &sh.bar};
  auto fetch = [&](unsigned turn) {
    if (MODE != SCAN_TMA || threadIdx.x != sh.ISSUER) return;
    const ScanTile c = scan_tile<VEC, S, NW, true>(p, turn);
    stage.expect(3 + (p.gx != nullptr) + (p.gv != nullptr));
#pragma unroll
    for (int k = 0; k < 3; ++k) stage.fetch(k, &maps.m[0], k * p.D + c.c0, c);
    if (p.gx) stage.fetch(3, &maps.m[1], c.c0, c);
    if (p.gv) stage.fetch(4, &maps.m[2], c.c0, c);
  };
  if constexpr (MODE == SCAN_TMA) sh.init();
  ScanTurn turn(p, sh.slot);
  if (turn.cur < turn.total) fetch(turn.cur);
  for (int it = 0; turn.cur < turn.total; turn.cur = turn.next, ++it) {
    const ScanTile c = scan_tile<VEC, S, NW, true>(p, turn.cur);
    Pack<float, VEC> pa[S], pd[S], pb[S], px[S], pv[S];
    if constexpr (MODE == SCAN_TMA) {
      mbar_wait(&sh.bar, it & 1);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        pa[s] = stage.take(0, s);
        pd[s] = stage.take(1, s);
        pb[s] = stage.take(2, s);
        px[s] = stage.take(3, s);
        pv[s] = stage.take(4, s);
      }
    } else {
      const long long o = ((long long)c.b * p.L + c.t0) * p.D + c.col;
      const float* zp = p.z + 3 * (o - c.col) + c.col;
      load_rows<float, VEC, S>(pa, zp, 3LL * p.D, c.n);
      load_rows<float, VEC, S>(pd, zp + p.D, 3LL * p.D, c.n);
      load_rows<float, VEC, S>(pb, zp + 2LL * p.D, 3LL * p.D, c.n);
      if (p.gx) load_rows<float, VEC, S>(px, p.gx + o, p.D, c.n);
      if (p.gv) load_rows<float, VEC, S>(pv, p.gv + o, p.D, c.n);
    }
    turn.draw(p);
    if (c.n < S || !p.gx || !p.gv) {  // beyond the end: A = 1, dt = 0, no gradients
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (s >= c.n) {
          pa[s] = Pack<float, VEC>::fill(INFINITY);
          pd[s] = Pack<float, VEC>::fill(-INFINITY);
          pb[s] = Pack<float, VEC>::fill(0.f);
        }
        if (s >= c.n || !p.gx) px[s] = Pack<float, VEC>::fill(0.f);
        if (s >= c.n || !p.gv) pv[s] = Pack<float, VEC>::fill(0.f);
      }
    }
    float A[S][VEC], dt[S][VEC], zb[S][VEC], gx[S][VEC], gv[S][VEC];
    float sa[S][VEC], sd[S][VEC];  // slopes of A and dt
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const F2 scale = f2(p.base_dt * head_scale(c.col + v, p.D / p.H));
      float eights[S / 8], mp = 0.f;
#pragma unroll
      for (int s = 0; s < S; s += 2) {
        F2 slope;
        gates(pa[s].get(v), pa[s + 1].get(v), A[s][v], A[s + 1][v], slope);
        split(slope, sa[s][v], sa[s + 1][v]);
        const F2 d = soft_steps(pd[s].get(v), pd[s + 1].get(v), slope) * scale;
        split(d, dt[s][v], dt[s + 1][v]);
        split(slope * scale, sd[s][v], sd[s + 1][v]);
      }
#pragma unroll
      for (int s = 0; s < S; ++s) {
        zb[s][v] = pb[s].get(v);
        gx[s][v] = px[s].get(v);
        gv[s][v] = pv[s].get(v);
        eights[s / 8] = s % 8 ? eights[s / 8] * A[s][v] : A[s][v];
        mp = fmaf(A[s][v], mp, zb[s][v] * dt[s][v]);
      }
      const GatedMap mf = {gain_run<S>(eights, 1.f, [&](int s) { return A[s][v]; }), mp};
      LayerBackMap mb = {mf.P, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        mb.G += gx[s][v];
        mb.q = A[s][v] * (fmaf(dt[s][v], mb.G, gv[s][v]) + mb.q);
        mb.R = A[s][v] * (mb.R + dt[s][v]);
      }
      unsigned long long wd[2], wf[1];
      mf.pack(wf);
      fmaps[w][lane * VEC + v] = wf[0];
      mb.pack(wd);
      sh.maps[w][0][lane * VEC + v] = wd[0];
      sh.maps[w][1][lane * VEC + v] = wd[1];
    }
    turn.tell(p, sh.slot, it);
    const int run = p.nchunks - 1 - c.chunk;
    receive<LayerBackMap, LayerBackState, CT, NW, true>(
        sh, p.words + c.tile * p.nchunks * (2LL * CT), c.chunk, p.nchunks, p.group, p.D - c.c0,
        [&](int j) {
          const long long e = (long long)c.b * p.D + c.c0 + j;
          return LayerBackState{p.gvl ? p.gvl[e] : 0.f, p.gxl ? p.gxl[e] : 0.f};
        },
        [&](int j) {
          chain_states<CT, NW>(fmaps, p.states + ((long long)c.b * p.nck + c.first / SCAN_CK) * p.D + c.c0, j, p.D - c.c0, vstart);
        },
        [&] {
          turn.hear(p, sh.slot, it);
          if (turn.next < turn.total) fetch(turn.next);
        });
    if (c.n <= 0) continue;
    LayerBackState st[VEC];
    float vs[S + 1][VEC];  // v_{t-1} of this warp's steps, and the last step's v
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      st[v] = sh.in[lane * VEC + v].through(
          LayerBackMap::unpack({sh.maps[w][0][lane * VEC + v], sh.maps[w][1][lane * VEC + v]}));
      vs[0][v] = vstart[w][lane * VEC + v];
#pragma unroll
      for (int s = 0; s < S; ++s) vs[s + 1][v] = fmaf(A[s][v], vs[s][v], zb[s][v] * dt[s][v]);
    }
    float* dz = p.dz + 3 * ((long long)c.b * p.L + c.t0) * p.D + c.col;
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      float oa[VEC], od[VEC], ob[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        st[v].X += gx[s][v];
        const float l = fmaf(dt[s][v], st[v].X, gv[s][v]) + st[v].m;
        oa[v] = l * vs[s][v] * sa[s][v];
        od[v] = (l * zb[s][v] + st[v].X * vs[s + 1][v]) * sd[s][v];
        ob[v] = l * dt[s][v];
        st[v].m = A[s][v] * l;
      }
      if (s < c.n) {
        Pack<float, VEC>::of(oa).store(dz + 3LL * s * p.D);
        Pack<float, VEC>::of(od).store(dz + (3LL * s + 1) * p.D);
        Pack<float, VEC>::of(ob).store(dz + (3LL * s + 2) * p.D);
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
}

// A few steps, or none: one thread per column (as gscan_forward_seq_kernel).
__global__ void __launch_bounds__(128) lscan_forward_seq_kernel(const LScanArgs p) {
  const long long c = blockIdx.x * 128LL + threadIdx.x;
  if (c >= (long long)p.B * p.D) return;
  const long long b = c / p.D, j = c - b * p.D;
  const float scale = p.base_dt * head_scale((int)j, p.D / p.H);
  float v = p.v0 ? p.v0[c] : 0.f, x = p.x0 ? p.x0[c] : 0.f;
  if (p.states && p.L) p.states[c] = v;
  for (int t = 0; t < p.L; t += 2) {
    const float* z = p.z + (b * p.L + t) * 3 * p.D + j;
    const long long e = (b * p.L + t) * p.D + j;
    const bool two = t + 1 < p.L;
    const float *z1 = two ? z + 3LL * p.D : z;
    F2 slope;
    float A0, A1, dt0, dt1;
    gates(z[0], z1[0], A0, A1, slope);
    split(soft_steps(z[p.D], z1[p.D], slope) * f2(scale), dt0, dt1);
    v = fmaf(A0, v, z[2LL * p.D] * dt0);
    x = fmaf(v, dt0, x);
    p.vs[e] = v;
    p.xs[e] = x;
    if (two) {
      v = fmaf(A1, v, z1[2LL * p.D] * dt1);
      x = fmaf(v, dt1, x);
      p.vs[e + p.D] = v;
      p.xs[e + p.D] = x;
    }
  }
  if (p.v_last) p.v_last[c] = v;
  if (p.x_last) p.x_last[c] = x;
}

}  // namespace gfn
