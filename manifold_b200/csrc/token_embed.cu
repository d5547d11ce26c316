// Embedding of token ids and the gradient of its table:
//
//   y_n  = scale W[id_n]
//   dW_v = scale (sum of dy_n over the n with id_n = v)
//
// (the reference's nn.Embedding, gfn/model.py:52-66, whose gradient it leaves
// to torch).  Both are bound by HBM.  The gradient sorts the tokens by id, a
// stable radix sort, so that every row of the table has one owner that sums
// its tokens in a fixed order (that of the sequence; rows of more than two runs
// of 32 tokens by parts): no float atomics, the same bits on every run.  Sums are
// float32 and are rounded once.
//
// Kernels, us, on one B200: 65536 tokens of 50257 x 1024 bfloat16 looked up 34
// (185 MB, 5.4 TB/s); 65536 of 32000 x 512 float32, lookup 30 (4.4 TB/s written),
// gradient 66: sort and 65 MB of zeros 26, sums 32 (134 MB read), joins 8.
#include "lm_host.h"
#include "lm_ops.cuh"

using namespace gfn;
using namespace gfn_abi;

namespace {

constexpr int EMBED_THREADS = 256;
constexpr int EMBED_GROUPS = 4;  // groups of 16 bytes a thread has on their way at once

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, 1994).
struct Divisor {
  unsigned d, shift;
  unsigned long long m;
};
Divisor divisor(unsigned d) {
  unsigned l = 0;
  while (l < 31 && (1u << l) < d) ++l;
  return {d, 31 + l, (1ull << (31 + l)) / d + 1};
}
GFN_DEV unsigned quotient(unsigned n, const Divisor& v) { return (unsigned)((n * v.m) >> v.shift); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

GFN_DEV long long id_at(const void* ids, bool wide, long long n) {
  return wide ? static_cast<const long long*>(ids)[n] : (long long)static_cast<const int*>(ids)[n];
}

// ------------------------------------------------------------------ forward
struct EmbedArgs {
  const void* ids;
  const void* w;
  void* y;
  long long N, ws, total;  // tokens, row stride of the table, items of all rows
  int V, D, wide;
  float scale;
  Divisor per_row;  // groups or other items of a row
};

// The 16 bytes at address `at`, which is a multiple of the element's size only,
// out of the two aligned ones that hold them.
GFN_DEV uint4 cut_out(uintptr_t at, const uint4& lo, const uint4& hi) {
  unsigned w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = at & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = at & 4 ? w[i + 1] : w[i];
  const unsigned sh = (unsigned)(at & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], sh), __funnelshift_r(w[1], w[2], sh), __funnelshift_r(w[2], w[3], sh),
                    __funnelshift_r(w[3], w[4], sh));
}

// y in groups of VEC elements, which rows of table and y are made of (16 bytes
// where they are; else elements).
template <typename T, int VEC>
__global__ void __launch_bounds__(EMBED_THREADS) embed_kernel(const EmbedArgs p) {
  constexpr int TILE = EMBED_THREADS * EMBED_GROUPS;
  const long long first = (long long)blockIdx.x * TILE;
  const T* w = static_cast<const T*>(p.w);
  const long long row0 = first / p.per_row.d;
  const unsigned rem = (unsigned)(first - row0 * p.per_row.d);
  const T* src[EMBED_GROUPS];
  Pack<T, VEC> v[EMBED_GROUPS];
#pragma unroll
  for (int u = 0; u < EMBED_GROUPS; ++u) {
    const unsigned at = threadIdx.x + u * EMBED_THREADS, off = rem + at, r = quotient(off, p.per_row);
    src[u] = nullptr;
    if (first + at < p.total) {
      const long long id = id_at(p.ids, p.wide, row0 + r);
      if ((unsigned long long)id < (unsigned)p.V) src[u] = w + id * p.ws + (long long)(off - r * p.per_row.d) * VEC;
      else gfn_flag_error(kDevErrBadToken);
    }
  }
#pragma unroll
  for (int u = 0; u < EMBED_GROUPS; ++u)
    if (src[u]) v[u] = *reinterpret_cast<const Pack<T, VEC>*>(src[u]);
#pragma unroll
  for (int u = 0; u < EMBED_GROUPS; ++u) {
    const long long g = first + threadIdx.x + u * EMBED_THREADS;
    if (g >= p.total) continue;
    Pack<T, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o.v[e] = from_f<T>(src[u] ? to_f(v[u].v[e]) * p.scale : 0.f);
    reinterpret_cast<Pack<T, VEC>*>(p.y)[g] = o;
  }
}

// Rows off 16 bytes, y on them.  A row is 2 VEC single elements (those before
// its first and behind its last whole 16 bytes of y, some of them none) and
// the groups between, each cut out of two loads.  20011 x 1001 bfloat16: 24 us,
// against 27 where groups over the rows' ends were fetched by elements in a loop
// (33 with the rest of them sped up as here).
template <typename T>
__global__ void __launch_bounds__(EMBED_THREADS) embed_across_kernel(const EmbedArgs p) {
  constexpr int TILE = EMBED_THREADS * EMBED_GROUPS, VEC = 16 / sizeof(T);
  const long long first = (long long)blockIdx.x * TILE;
  const T* w = static_cast<const T*>(p.w);
  const uintptr_t begin = reinterpret_cast<uintptr_t>(w), end = reinterpret_cast<uintptr_t>(w + (p.V - 1) * p.ws + p.D);
  const long long row0 = first / p.per_row.d;
  const unsigned rem = (unsigned)(first - row0 * p.per_row.d);
  const T* src[EMBED_GROUPS];
  int col[EMBED_GROUPS], width[EMBED_GROUPS];  // width: 0 nothing, 1 an element, VEC a group
  uint4 lo[EMBED_GROUPS], hi[EMBED_GROUPS];
  T one[EMBED_GROUPS];
#pragma unroll
  for (int u = 0; u < EMBED_GROUPS; ++u) {
    const unsigned at = threadIdx.x + u * EMBED_THREADS, r = quotient(rem + at, p.per_row);
    const int i = (int)(rem + at - r * p.per_row.d);
    const int head = (int)((VEC - (unsigned long long)(row0 + r) * (unsigned)p.D % VEC) % VEC);
    const int groups = (p.D - head) / VEC, behind = head + groups * VEC;
    width[u] = 0;
    src[u] = nullptr;
    if (first + at >= p.total) continue;
    if (i < VEC) {
      col[u] = i;
      width[u] = i < head;
    } else if (i < 2 * VEC) {
      col[u] = behind + i - VEC;
      width[u] = col[u] < p.D;
    } else {
      col[u] = head + (i - 2 * VEC) * VEC;
      width[u] = i - 2 * VEC < groups ? VEC : 0;
    }
    if (!width[u]) continue;
    const long long id = id_at(p.ids, p.wide, row0 + r);
    if ((unsigned long long)id < (unsigned)p.V) src[u] = w + id * p.ws + col[u];
    else gfn_flag_error(kDevErrBadToken);
  }
  auto within = [&](int u) {
    const uintptr_t q = reinterpret_cast<uintptr_t>(src[u]) & ~(uintptr_t)15;
    return q >= begin && q + 32 <= end;
  };
#pragma unroll
  for (int u = 0; u < EMBED_GROUPS; ++u) {
    if (!src[u]) continue;
    if (width[u] == 1) one[u] = *src[u];
    else if (within(u)) {
      const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src[u]) & ~(uintptr_t)15);
      lo[u] = q[0];
      hi[u] = q[1];
    }
  }
#pragma unroll
  for (int u = 0; u < EMBED_GROUPS; ++u) {
    if (!width[u]) continue;
    const unsigned at = threadIdx.x + u * EMBED_THREADS;
    T* y = static_cast<T*>(p.y) + (row0 + quotient(rem + at, p.per_row)) * p.D + col[u];
    if (width[u] == 1) {
      *y = from_f<T>(src[u] ? to_f(one[u]) * p.scale : 0.f);
      continue;
    }
    Pack<T, VEC> o;
    if (!src[u]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.v[e] = from_f<T>(0.f);
    } else if (within(u)) {
      const uint4 bits = cut_out(reinterpret_cast<uintptr_t>(src[u]), lo[u], hi[u]);
      const T* v = reinterpret_cast<const T*>(&bits);
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.v[e] = from_f<T>(to_f(v[e]) * p.scale);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.v[e] = from_f<T>(to_f(src[u][e]) * p.scale);
    }
    *reinterpret_cast<Pack<T, VEC>*>(y) = o;
  }
}

template <typename T>
int embed_forward(EmbedArgs p, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const bool rows = aligned16(p.w) && aligned16(p.y) && p.D % VEC == 0 && p.ws % VEC == 0;
  const bool across = !rows && aligned16(p.y) && p.D >= 8 * VEC;  // shorter rows are mostly ends
  const int items = rows ? p.D / VEC : across ? 2 * VEC + p.D / VEC : p.D;
  p.total = p.N * items;
  p.per_row = divisor((unsigned)items);
  const long long blocks = (p.total + EMBED_THREADS * EMBED_GROUPS - 1) / (EMBED_THREADS * EMBED_GROUPS);
  if (blocks > 0x7fffffffLL) return fail(GFN_ERR_UNSUPPORTED, "embed: %lld x %d elements", p.N, p.D);
  if (rows) embed_kernel<T, VEC><<<(unsigned)blocks, EMBED_THREADS, 0, s>>>(p);
  else if (across) embed_across_kernel<T><<<(unsigned)blocks, EMBED_THREADS, 0, s>>>(p);
  else embed_kernel<T, 1><<<(unsigned)blocks, EMBED_THREADS, 0, s>>>(p);
  return launch_status("embed_kernel");
}

// ----------------------------------------------------------------- gradient
// The sort: digits of up to 9 bits, least significant first.  A tile of
// tokens is ranked by a block; where it writes a digit follows from the counts
// of every digit in every tile, which the kernel before left in global memory.
// A key and its token travel as one 64-bit word.  Three launches of 7 to 10 us
// (65536 tokens, 17% issue) are latency: counts of 64 tiles, eight barriers,
// scattered stores.  One cluster of eight blocks that keeps all in shared memory
// took 33 us for the same, since eight SMs then do all the ranking.
constexpr int SORT_THREADS = 256, SORT_WARPS = 8;
constexpr int SORT_BITS = 9, SORT_BINS = 1 << SORT_BITS, SORT_TILES = 256;
constexpr int SORT_ITEMS = 4, SORT_SUB = SORT_THREADS * SORT_ITEMS;      // tokens of a thread, of a tile's part
constexpr int SORT_ALONE = 8, SORT_ONE = SORT_THREADS * SORT_ALONE;      // where one block sorts them all
// Tokens (in sorted order) that one group of threads sums.
constexpr int SUM_RUN = 32, SUM_THREADS = 128, SUM_AHEAD = 8, SUM_WORDS = 4 * SUM_RUN + 2;
constexpr int SUM_COLS = 4;  // columns of a thread where rows are not whole groups of 16 bytes

struct SortArgs {
  const void* ids;
  uint2* sorted[2];  // (key, token)
  unsigned* counts;  // [passes][tiles][bins]
  void* dw;
  long long dw_bytes;
  long long padding;
  int N, V, wide, tiles, subs, bits, passes;  // subs: parts of SORT_SUB tokens in a tile; bits of a digit
};

// The token's row, or V where it takes no part (padding, or outside the table).
GFN_DEV unsigned sort_key(const SortArgs& p, long long n, bool flag) {
  const long long id = id_at(p.ids, p.wide, n);
  if ((unsigned long long)id >= (unsigned)p.V) {
    if (flag) gfn_flag_error(kDevErrBadToken);
    return p.V;
  }
  return id == p.padding ? (unsigned)p.V : (unsigned)id;
}

// Part `part` of `parts` of the table's gradient becomes zero: the blocks
// beyond the sort's own fill it meanwhile.
GFN_DEV void zero_part(void* dw, long long bytes, long long part, long long parts) {
  char* b = static_cast<char*>(dw);
  const long long head = min((16 - (long long)(reinterpret_cast<uintptr_t>(b) & 15)) & 15, bytes);
  const long long groups = (bytes - head) / 16, tail = head + groups * 16;
  const long long per = (groups + parts - 1) / parts;
  const long long end = min((part + 1) * per, groups);
  uint4* g = reinterpret_cast<uint4*>(b + head);
  for (long long i = part * per + threadIdx.x; i < end; i += blockDim.x) g[i] = make_uint4(0, 0, 0, 0);
  if (part == 0) {
    for (long long i = threadIdx.x; i < head; i += blockDim.x) b[i] = 0;
    for (long long i = tail + threadIdx.x; i < bytes; i += blockDim.x) b[i] = 0;
  }
}

// Stage `stage` of `stages` of that filling, by the blocks from `first` on.
GFN_DEV void zero_stage(const SortArgs& p, int first, int stage, int stages) {
  const long long n = gridDim.x - first;
  zero_part(p.dw, p.dw_bytes, stage * n + (blockIdx.x - first), n * stages);
}

// The counts of the first digit, and zeros for those of the later ones.
__global__ void __launch_bounds__(SORT_THREADS) embed_count_kernel(const SortArgs p) {
  if ((int)blockIdx.x >= p.tiles) return zero_stage(p, p.tiles, 0, p.passes + 1);
  __shared__ unsigned bins[SORT_BINS];
  const int n_bins = 1 << p.bits;
  for (int i = threadIdx.x; i < n_bins; i += SORT_THREADS) bins[i] = 0;
  __syncthreads();
  const long long from = (long long)blockIdx.x * p.subs * SORT_SUB, to = min(from + (long long)p.subs * SORT_SUB, (long long)p.N);
  const unsigned mask = n_bins - 1;
  for (long long n = from + threadIdx.x; n < to; n += SORT_THREADS) atomicAdd(&bins[sort_key(p, n, true) & mask], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < n_bins; i += SORT_THREADS) {
    p.counts[(long long)blockIdx.x * n_bins + i] = bins[i];
    for (int q = 1; q < p.passes; ++q) p.counts[((long long)q * p.tiles + blockIdx.x) * n_bins + i] = 0;
  }
}

struct SortShared {
  unsigned warp[SORT_WARPS][SORT_BINS];  // a warp's count of each digit, then where its first one goes
  unsigned next[SORT_BINS];              // where the block's next one goes
  unsigned sums[SORT_WARPS];
};

// Exclusive sums over the bins of `v[2]` (this thread's bins 2 t and 2 t + 1).
GFN_DEV void scan_bins(SortShared& sh, const unsigned (&v)[2], unsigned (&out)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned s = v[0] + v[1], inc = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) sh.sums[warp] = inc;
  __syncthreads();
  unsigned before = 0;
#pragma unroll
  for (int w = 0; w < SORT_WARPS; ++w) before += w < warp ? sh.sums[w] : 0u;
  out[0] = before + inc - s;
  out[1] = out[0] + v[0];
  __syncthreads();
}

// Ranks THREADS * ITEMS tokens from `from` on (below `to`), given by `item`, by
// the digit of their key at `shift`, and hands each with its place to `put`;
// sh.next moves on.
template <int ITEMS, class Item, class Put>
GFN_DEV void rank_part(SortShared& sh, long long from, long long to, unsigned shift, unsigned mask, Item item, Put put) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint2 k[ITEMS];
  unsigned rank[ITEMS];
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const long long n = from + (warp * ITEMS + r) * 32 + lane;
    k[r] = n < to ? item(n) : make_uint2(0u, 0u);
  }
  for (int w = 0; w < SORT_WARPS; ++w)
    for (int i = threadIdx.x; i <= (int)mask; i += SORT_THREADS) sh.warp[w][i] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const bool live = from + (warp * ITEMS + r) * 32 + lane < to;
    const unsigned d = live ? (k[r].x >> shift) & mask : ~0u;
    const unsigned same = __match_any_sync(0xffffffffu, d), before = __popc(same & ((1u << lane) - 1));
    rank[r] = live ? sh.warp[warp][d] + before : 0u;
    __syncwarp();
    if (live && before == 0) sh.warp[warp][d] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int b = threadIdx.x; b <= (int)mask; b += SORT_THREADS) {
    unsigned at = sh.next[b];
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) {
      const unsigned c = sh.warp[w][b];
      sh.warp[w][b] = at;
      at += c;
    }
    sh.next[b] = at;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ITEMS; ++r)
    if (from + (warp * ITEMS + r) * 32 + lane < to) put(k[r], sh.warp[warp][(k[r].x >> shift) & mask] + rank[r]);
  __syncthreads();
}

// One digit of the sort.  The counts of the next digit are collected on the way.
__global__ void __launch_bounds__(SORT_THREADS) embed_rank_kernel(const SortArgs p, int pass) {
  if ((int)blockIdx.x >= p.tiles) return zero_stage(p, p.tiles, pass + 1, p.passes + 1);
  __shared__ SortShared sh;
  const int n_bins = 1 << p.bits;
  const unsigned mask = n_bins - 1, shift = pass * p.bits;
  const unsigned* counts = p.counts + (long long)pass * p.tiles * n_bins;
  unsigned total[2] = {0, 0}, before[2] = {0, 0}, start[2];
  if ((int)threadIdx.x < n_bins / 2) {
#pragma unroll 16
    for (int t = 0; t < p.tiles; ++t) {
      const uint2 c = reinterpret_cast<const uint2*>(counts + (long long)t * n_bins)[threadIdx.x];
      total[0] += c.x;
      total[1] += c.y;
      if (t < (int)blockIdx.x) {
        before[0] += c.x;
        before[1] += c.y;
      }
    }
  }
  scan_bins(sh, total, start);
  sh.next[2 * threadIdx.x] = start[0] + before[0];
  sh.next[2 * threadIdx.x + 1] = start[1] + before[1];
  const long long from = (long long)blockIdx.x * p.subs * SORT_SUB, to = min(from + (long long)p.subs * SORT_SUB, (long long)p.N);
  const uint2* in = pass & 1 ? p.sorted[0] : p.sorted[1];
  uint2* out = pass & 1 ? p.sorted[1] : p.sorted[0];
  unsigned* following = pass + 1 < p.passes ? p.counts + (long long)(pass + 1) * p.tiles * n_bins : nullptr;
  for (long long at = from; at < to; at += SORT_SUB)
    rank_part<SORT_ITEMS>(
        sh, at, to, shift, mask,
        [&](long long n) { return pass == 0 ? make_uint2(sort_key(p, n, false), (unsigned)n) : in[n]; },
        [&](uint2 k, unsigned place) {
          out[place] = k;
          if (following) atomicAdd(&following[(place / (p.subs * SORT_SUB)) * n_bins + ((k.x >> (shift + p.bits)) & mask)], 1u);
        });
}

// The whole sort of up to SORT_ONE tokens by one block; the others fill zeros.
__global__ void __launch_bounds__(SORT_THREADS) embed_sort_kernel(const SortArgs p) {
  if (blockIdx.x >= 1) return zero_stage(p, 1, 0, 1);
  __shared__ SortShared sh;
  __shared__ uint2 items[SORT_ONE];
  const int n_bins = 1 << p.bits;
  const unsigned mask = n_bins - 1;
  for (int n = threadIdx.x; n < p.N; n += SORT_THREADS) items[n] = make_uint2(sort_key(p, n, true), n);
  uint2* out = (p.passes - 1) & 1 ? p.sorted[1] : p.sorted[0];
  for (int pass = 0; pass < p.passes; ++pass) {
    const unsigned shift = pass * p.bits;
    for (int i = threadIdx.x; i < SORT_BINS; i += SORT_THREADS) sh.next[i] = 0;
    __syncthreads();
    for (int n = threadIdx.x; n < p.N; n += SORT_THREADS) atomicAdd(&sh.next[(items[n].x >> shift) & mask], 1u);
    __syncthreads();
    const unsigned v[2] = {sh.next[2 * threadIdx.x], sh.next[2 * threadIdx.x + 1]};
    unsigned start[2];
    scan_bins(sh, v, start);
    sh.next[2 * threadIdx.x] = start[0];
    sh.next[2 * threadIdx.x + 1] = start[1];
    const bool last = pass == p.passes - 1;
    rank_part<SORT_ALONE>(
        sh, 0, p.N, shift, mask, [&](long long n) { return items[n]; },
        [&](uint2 k, unsigned place) { (last ? out : items)[place] = k; });  // every thread has read its own by now
  }
}

struct SumArgs {
  const uint2* sorted;  // (key, token)
  const void* dy;
  void* dw;
  float* part;  // [runs][2][D]: what a run's first and last row have of a row that goes on in the neighbour
  long long ds;
  int N, V, D;
  float scale;
};

// A group of blockDim.x threads sums SUM_RUN sorted tokens (a run) over the
// columns of its threads, VEC each.  A row of the table whose tokens begin in
// one run and end in the next belongs to the first.  Longer ones leave a part
// for each run in `part`: [0] of a run's first row, [1] of its last.  Eight tokens'
// rows are on their way at once.  65536 x 512 float32: 29 to 32 us, 63% of DRAM's
// rate; 20011 x 1001 bfloat16 24 us, by single elements, four columns a thread (30
// with one: the work on keys and places is shared by the columns).
template <typename T, int VEC, int COLS>
__global__ void __launch_bounds__(SUM_THREADS) embed_sum_kernel(const SumArgs p) {
  extern __shared__ unsigned sum_shared[];
  unsigned* key = sum_shared + threadIdx.y * SUM_WORDS + 1;  // key[-1] .. key[2 SUM_RUN]
  unsigned* pos = key + 2 * SUM_RUN + 1;
  const long long run = (long long)blockIdx.x * blockDim.y + threadIdx.y, from = run * SUM_RUN;
  const unsigned none = (unsigned)p.V;
  for (int i = (int)threadIdx.x - 1; i <= 2 * SUM_RUN; i += blockDim.x) {
    const long long n = from + i;
    const uint2 k = n >= 0 && n < p.N ? p.sorted[n] : make_uint2(n < 0 ? ~0u : none, 0u);
    key[i] = k.x;
    if (i >= 0 && i < 2 * SUM_RUN) pos[i] = k.y;
  }
  const unsigned far = from > SUM_RUN && from < p.N ? p.sorted[from - SUM_RUN - 1].x : ~0u;  // the last key before the run before
  __syncthreads();
  // COLS groups of VEC columns, blockDim.x groups apart
  const int first = (blockIdx.y * blockDim.x * COLS + threadIdx.x) * VEC, gap = blockDim.x * VEC;
  if (first >= p.D || key[0] >= none) return;
  const T* dy = static_cast<const T*>(p.dy) + first;
  float acc[COLS][VEC];
  auto clear = [&] {
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[c][e] = 0.f;
  };
  clear();
  // the first row, where it began before: the run before has it if it ends here and began there
  bool open = key[0] == key[-1];
  const bool skip = open && far != key[0] && key[SUM_RUN] != key[0];
  const unsigned skipped = skip ? key[0] : ~0u;
  // the last row, where it goes on: this run has it if it began here and ends in the next
  const unsigned final = key[SUM_RUN - 1];
  const bool goes_on = final < none && key[SUM_RUN] == final, began = key[0] != final || !open;
  const bool whole = goes_on && began && key[2 * SUM_RUN] != final;
  const int end = whole ? 2 * SUM_RUN : SUM_RUN;
  auto store = [&](float* dst) {
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      if (first + c * gap >= p.D) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e) dst[first + c * gap + e] = acc[c][e];
    }
  };
  for (int i0 = 0; i0 < end; i0 += SUM_AHEAD) {
    if (i0 >= SUM_RUN && key[i0] != final) break;
    Pack<T, VEC> v[SUM_AHEAD][COLS];
#pragma unroll
    for (int i = 0; i < SUM_AHEAD; ++i) {
      const unsigned k = key[i0 + i];
      if (k < none && k != skipped && (i0 < SUM_RUN || k == final)) {
        const T* row = dy + (long long)pos[i0 + i] * p.ds;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
          if (first + c * gap < p.D) v[i][c] = *reinterpret_cast<const Pack<T, VEC>*>(row + c * gap);
      }
    }
#pragma unroll
    for (int i = 0; i < SUM_AHEAD; ++i) {
      const unsigned k = key[i0 + i];
      if (k >= none || (i0 >= SUM_RUN && k != final)) return;
      if (k == skipped) {
        open = false;
        continue;
      }
#pragma unroll
      for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[c][e] += to_f(v[i][c].v[e]);
      if (key[i0 + i + 1] == k) continue;
      if (open) store(p.part + run * 2 * p.D);
      else {
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          if (first + c * gap >= p.D) continue;
          Pack<T, VEC> o;
#pragma unroll
          for (int e = 0; e < VEC; ++e) o.v[e] = from_f<T>(acc[c][e] * p.scale);
          *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(p.dw) + (long long)k * p.D + first + c * gap) = o;
        }
      }
      open = false;
      clear();
    }
  }
  if (goes_on && !whole) store(p.part + (run * 2 + (open ? 0 : 1)) * p.D);
}

// Rows of more than two runs: the run in which such a row begins adds the
// parts over JOIN_COLS columns.  A warp looks at one run and adds a row of up to JOIN_SHORT parts by itself; longer ones are added by
// the whole block, in eight interleaved sums.
constexpr int JOIN_RUNS = 8, JOIN_COLS = 128, JOIN_SHORT = 8, JOIN_AHEAD = 10;

template <typename T>
__global__ void __launch_bounds__(32 * JOIN_RUNS) embed_join_kernel(const SumArgs p) {
  constexpr int PER = JOIN_COLS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long runs = ((long long)p.N + SUM_RUN - 1) / SUM_RUN, base = (long long)blockIdx.x * JOIN_RUNS;
  __shared__ unsigned row[JOIN_RUNS];
  __shared__ long long stop[JOIN_RUNS];  // behind the last run whose first token is the row's
  __shared__ float sums[JOIN_RUNS][JOIN_COLS];
  auto first_part = [&](long long run, int from, float (&acc)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int col = from + lane + 32 * j;
      acc[j] = col < p.D ? p.part[(run * 2 + 1) * p.D + col] : 0.f;
    }
  };
  auto add_parts = [&](long long r, long long end, int step, int from, float (&acc)[PER]) {
    for (; r < end; r += JOIN_AHEAD * step) {
      float v[JOIN_AHEAD][PER];
#pragma unroll
      for (int u = 0; u < JOIN_AHEAD; ++u)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int col = from + lane + 32 * j;
          v[u][j] = r + u * step < end && col < p.D ? p.part[(r + u * step) * 2 * p.D + col] : 0.f;
        }
#pragma unroll
      for (int u = 0; u < JOIN_AHEAD; ++u)
#pragma unroll
        for (int j = 0; j < PER; ++j) acc[j] += v[u][j];
    }
  };
  {
    const long long run = base + warp, from = run * SUM_RUN, end = from + SUM_RUN;
    unsigned k = p.V;
    if (end + SUM_RUN < p.N) {
      k = p.sorted[end + SUM_RUN].x;
      const unsigned own = p.sorted[end - 1].x;
      const unsigned next = p.sorted[end].x, begin = p.sorted[from].x, before = from > 0 ? p.sorted[from - 1].x : ~0u;
      if (own != k || next != k || (begin == k && before == k)) k = p.V;
    }
    bool wide = false;
    if (k < (unsigned)p.V) {
      // the first run that does not begin with k (sorted: those that do come first), by steps of 32 runs, then of one
      long long last = run + 1;
      for (int step = 32; step; step = step == 32 ? 1 : 0) {
        for (;;) {
          const long long r = last + (step == 32 ? 31 + 32 * lane : lane);
          const int n = __popc(__ballot_sync(0xffffffffu, r < runs && p.sorted[r * SUM_RUN].x == k));
          last += n * step;
          if (n < 32) break;
        }
      }
      wide = last - run > JOIN_SHORT;
      if (wide) {
        if (lane == 0) stop[warp] = last;
      } else {
        for (int at = blockIdx.y * JOIN_COLS; at < p.D; at += gridDim.y * JOIN_COLS) {
          float acc[PER];
          first_part(run, at, acc);
          add_parts(run + 1, last, 1, at, acc);
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const int col = at + lane + 32 * j;
            if (col < p.D) static_cast<T*>(p.dw)[(long long)k * p.D + col] = from_f<T>(acc[j] * p.scale);
          }
        }
      }
    }
    if (lane == 0) row[warp] = wide ? k : (unsigned)p.V;
  }
  __syncthreads();
  for (int w = 0; w < JOIN_RUNS; ++w) {
    const unsigned k = row[w];
    if (k >= (unsigned)p.V) continue;
    const long long run = base + w, last = stop[w];
    for (int from = blockIdx.y * JOIN_COLS; from < p.D; from += gridDim.y * JOIN_COLS) {
      float acc[PER] = {};
      if (warp == 0) first_part(run, from, acc);
      add_parts(run + 1 + warp, last, JOIN_RUNS, from, acc);
#pragma unroll
      for (int j = 0; j < PER; ++j) sums[warp][lane + 32 * j] = acc[j];
      __syncthreads();
      if (threadIdx.x < JOIN_COLS && from + (int)threadIdx.x < p.D) {
        float t = sums[0][threadIdx.x];
#pragma unroll
        for (int g = 1; g < JOIN_RUNS; ++g) t += sums[g][threadIdx.x];
        static_cast<T*>(p.dw)[(long long)k * p.D + from + threadIdx.x] = from_f<T>(t * p.scale);
      }
      __syncthreads();
    }
  }
}

// How the tokens are divided and where the workspace holds what.
struct Plan {
  int bits, passes, tiles, subs;
  long long runs, items, counts, part, bytes;
};
Plan embed_plan(long long N, int V, int D) {
  Plan q = {};
  int need = 1;
  while (need < 32 && ((unsigned)V >> need)) ++need;  // V itself is a key
  q.passes = (need + SORT_BITS - 1) / SORT_BITS;
  q.bits = (need + q.passes - 1) / q.passes;
  const long long parts = (N + SORT_SUB - 1) / SORT_SUB;
  q.subs = (int)((parts + SORT_TILES - 1) / SORT_TILES);
  if (q.subs < 1) q.subs = 1;
  q.tiles = (int)((parts + q.subs - 1) / q.subs);
  q.runs = (N + SUM_RUN - 1) / SUM_RUN;
  auto up = [](long long b) { return (b + 255) / 256 * 256; };
  q.items = up(8 * N);
  q.counts = 2 * q.items;
  q.part = q.counts + up(4LL * q.passes * q.tiles << q.bits);
  q.bytes = q.part + up(8 * q.runs * D);
  return q;
}

template <typename T>
int embed_sum(const SumArgs& p, long long runs, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = aligned16(p.dy) && aligned16(p.dw) && p.D % VEC == 0 && (p.N == 1 || p.ds % VEC == 0);
  const int per = vec ? VEC : SUM_COLS, need = (p.D + per - 1) / per;
  int lanes = 8;
  while (lanes < SUM_THREADS && lanes < need) lanes *= 2;
  const dim3 block((unsigned)lanes, (unsigned)(SUM_THREADS / lanes));
  const dim3 grid((unsigned)((runs + block.y - 1) / block.y), (unsigned)((need + lanes - 1) / lanes));
  if (grid.y > 65535) return fail(GFN_ERR_UNSUPPORTED, "token_embed backward: dim %d", p.D);
  const int shared = (int)block.y * SUM_WORDS * 4;
  if (vec) embed_sum_kernel<T, VEC, 1><<<grid, block, shared, s>>>(p);
  else embed_sum_kernel<T, 1, SUM_COLS><<<grid, block, shared, s>>>(p);
  const int st = launch_status("embed_sum_kernel");
  if (st != GFN_OK || runs < 3) return st;
  const int cols = (p.D + JOIN_COLS - 1) / JOIN_COLS;
  const dim3 joins((unsigned)((runs + JOIN_RUNS - 1) / JOIN_RUNS), (unsigned)(cols < 65535 ? cols : 65535));
  embed_join_kernel<T><<<joins, 32 * JOIN_RUNS, 0, s>>>(p);
  return launch_status("embed_join_kernel");
}

}  // namespace

namespace gfn_abi {
cudaError_t error_word_token_embed(int* v, int reset, cudaStream_t s) { return gfn_unit_error_word(v, reset, s); }
}  // namespace gfn_abi

extern "C" {

int gfn_token_embed_forward(const void* ids, int ids_are_64, long long tokens, const void* weight,
                            long long weight_row_stride, int dtype, int vocab, int dim, float scale, void* y,
                            gfn_stream_t stream) {
  if (tokens < 0 || vocab <= 0 || dim <= 0 || (tokens > 0 && (!ids || !weight || !y)))
    return fail(GFN_ERR_INVALID, "token_embed: tokens=%lld vocab=%d dim=%d or a NULL operand", tokens, vocab, dim);
  if (dim > 1 << 30) return fail(GFN_ERR_UNSUPPORTED, "token_embed: dim %d above 2^30", dim);
  if (tokens == 0) return GFN_OK;
  EmbedArgs p = {};
  p.ids = ids; p.w = weight; p.y = y; p.N = tokens; p.ws = weight_row_stride; p.V = vocab; p.D = dim;
  p.wide = ids_are_64 != 0; p.scale = scale;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == GFN_F32) return embed_forward<float>(p, s);
  if (dtype == GFN_BF16) return embed_forward<__nv_bfloat16>(p, s);
  if (dtype == GFN_F16) return embed_forward<__half>(p, s);
  return fail(GFN_ERR_UNSUPPORTED, "token_embed: element type %d", dtype);
}

long long gfn_token_embed_backward_workspace_bytes(long long tokens, int vocab, int dim) {
  if (tokens < 0 || tokens > 0x7fffffffLL || vocab <= 0 || dim <= 0) return -1;
  return embed_plan(tokens, vocab, dim).bytes;
}

int gfn_token_embed_backward(const void* ids, int ids_are_64, long long tokens, const void* dy,
                             long long dy_row_stride, int dtype, int vocab, int dim, float scale,
                             long long padding_id, void* dweight, void* workspace, long long workspace_bytes,
                             gfn_stream_t stream) {
  if (tokens < 0 || vocab <= 0 || dim <= 0 || !dweight || (tokens > 0 && (!ids || !dy || !workspace)))
    return fail(GFN_ERR_INVALID, "token_embed backward: tokens=%lld vocab=%d dim=%d or a NULL operand", tokens, vocab,
                dim);
  if (tokens > 0x7fffffffLL || vocab == 0x7fffffff)
    return fail(GFN_ERR_UNSUPPORTED, "token_embed backward: %lld tokens, vocabulary of %d", tokens, vocab);
  if (dtype != GFN_F32 && dtype != GFN_BF16 && dtype != GFN_F16)
    return fail(GFN_ERR_UNSUPPORTED, "token_embed backward: element type %d", dtype);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const long long dw_bytes = (long long)vocab * dim * (dtype == GFN_F32 ? 4 : 2);
  if (tokens == 0) {
    const cudaError_t e = cudaMemsetAsync(dweight, 0, (size_t)dw_bytes, s);
    return e == cudaSuccess ? GFN_OK : cuda_status(e, "token_embed backward");
  }
  const Plan q = embed_plan(tokens, vocab, dim);
  if (workspace_bytes < q.bytes || !aligned16(workspace))
    return fail(GFN_ERR_INVALID, "token_embed backward: a workspace of %lld bytes, 16-byte aligned, is needed", q.bytes);
  int sms = 0;
  int st = sm_count(&sms);
  if (st != GFN_OK) return st;
  char* ws = static_cast<char*>(workspace);
  SortArgs a = {};
  a.ids = ids;
  a.sorted[0] = reinterpret_cast<uint2*>(ws);
  a.sorted[1] = reinterpret_cast<uint2*>(ws + q.items);
  a.counts = reinterpret_cast<unsigned*>(ws + q.counts);
  a.dw = dweight; a.dw_bytes = dw_bytes; a.padding = padding_id;
  a.N = (int)tokens; a.V = vocab; a.wide = ids_are_64 != 0;
  a.tiles = q.tiles; a.subs = q.subs; a.bits = q.bits; a.passes = q.passes;
  const unsigned fill = (unsigned)(4 * sms);
  if (tokens <= SORT_ONE) {
    embed_sort_kernel<<<1 + fill, SORT_THREADS, 0, s>>>(a);
    if ((st = launch_status("embed_sort_kernel")) != GFN_OK) return st;
  } else {
    embed_count_kernel<<<(unsigned)q.tiles + fill, SORT_THREADS, 0, s>>>(a);
    if ((st = launch_status("embed_count_kernel")) != GFN_OK) return st;
    for (int pass = 0; pass < q.passes; ++pass) {
      embed_rank_kernel<<<(unsigned)q.tiles + fill, SORT_THREADS, 0, s>>>(a, pass);
      if ((st = launch_status("embed_rank_kernel")) != GFN_OK) return st;
    }
  }
  SumArgs b = {};
  b.sorted = a.sorted[(q.passes - 1) & 1];
  b.dy = dy; b.dw = dweight; b.part = reinterpret_cast<float*>(ws + q.part);
  b.ds = dy_row_stride; b.N = a.N; b.V = vocab; b.D = dim; b.scale = scale;
  if (dtype == GFN_F32) return embed_sum<float>(b, q.runs, s);
  if (dtype == GFN_BF16) return embed_sum<__nv_bfloat16>(b, q.runs, s);
  return embed_sum<__half>(b, q.runs, s);
}

}  // extern "C"
