// Shaping of a row of logits before sampling, in one pass: penalties for the
// tokens of the row's history, an additive bias, the temperature and a
// grammar mask.  For token j of a row whose history holds it `seen` times in
// all and c times after the prompt:
//
//   s = x > 0 ? x / rep : x rep                 where seen > 0
//   s = s - (freq c + pres [c > 0])
//   y = (s + bias_j) / temp, or -inf where the mask's bit j is clear
//
// The reference samples from bare logits (gfn/model.py:404-469).  A block
// owns a run of the vocabulary of one row: it counts the history's tokens in
// that run in shared memory (integer atomics, so the order does not matter)
// and then streams its logits once.
//
// 256 x 50257 bfloat16 with biases, masks and up to 2048 tokens of history takes
// 35 us as one call among others with lengths spread over the history (3.1 TB/s),
// and 41 us by CUDA events around a single call behind a cleared L2, as the other
// figures here are taken; 9 us a call, launch and checks included, for one row of
// 32000.  The bytes would take 17 us: the rest is instructions, 59 per element
// there, 25 without history (27 us) and 14 without bias and mask too.
#include "abi.h"
#include "lm_ops.cuh"

using namespace gfn;
using namespace gfn_abi;

namespace {

constexpr int LOGITS_THREADS = 512;
constexpr unsigned LOGITS_SEEN = 0x80000000u;  // the token occurs in the prompt; low bits: generated count

struct LogitsArgs {
  const void* x;
  void* y;
  const long long* tokens;
  const long long* lengths;
  const long long* prompts;
  const float* rep_rows;
  const float* freq_rows;
  const float* pres_rows;
  const float* temp_rows;
  const float* bias;
  const unsigned* allowed;
  long long xs, ts, bs, as;  // row strides of logits, tokens, bias, mask
  int B, V, T;
  int bias_groups;  // rows of the bias have the logits' phase
  float rep, freq, pres, temp;
};

// VEC neighbouring tokens.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Group {
  T v[VEC];
};

// Quotients by a row's penalty and temperature are products with 1 / d, since a
// long history puts a penalised token before almost every warp and a division at
// each then costs a third of the time (256 x 50257 bfloat16 with 2048 tokens: 53 us
// against 41).  Rows whose 1 / d could leave float32's range divide.
struct RowTerms {
  float rep, inv_rep, freq, pres, temp, inv_temp;
  bool divides;
};
GFN_DEV bool reciprocal_serves(float d) { return d >= 0x1p-100f && d <= 0x1p100f; }

// v / d given 1 / d.  For 16-bit results the product's two roundings do; for
// float32 ones (EXACT) it is corrected by its residual, which makes it the rounded
// quotient (Markstein, 1990) unless the residual loses digits: `odd` then, and for
// 0, infinities and NaN.
template <bool EXACT>
GFN_DEV float quotient(float v, float d, float inv, bool& odd) {
  const float q = v * inv;
  if (!EXACT) return q;
  odd = odd || !(fminf(fabsf(v), fabsf(q)) >= 0x1p-100f && fabsf(q) <= 0x1p126f);
  return fmaf(fmaf(-q, d, v), inv, q);
}

// The penalties of one token with history word c.
template <bool EXACT>
GFN_DEV float penalise(float v, unsigned c, const RowTerms& r, bool& odd) {
  const float n = (float)(c & ~LOGITS_SEEN);
  bool strange = false;
  const float q = quotient<EXACT>(v, r.rep, r.inv_rep, strange), w = v > 0.f ? q : v * r.rep;
  odd = odd || (strange && c && v > 0.f);
  v = c ? w : v;
  return n > 0.f ? v - fmaf(r.freq, n, r.pres) : v;
}

template <bool EXACT>
GFN_DEV float finish_logit(float v, float bias, const RowTerms& r, bool& odd) {
  return quotient<EXACT>(v + bias, r.temp, r.inv_temp, odd);
}

// The whole of it by divisions.
GFN_DEV float shaped_logit(float v, unsigned c, float bias, const RowTerms& r) {
  const float n = (float)(c & ~LOGITS_SEEN);
  if (c) v = v > 0.f ? v / r.rep : v * r.rep;
  if (n > 0.f) v -= fmaf(r.freq, n, r.pres);
  return (v + bias) / r.temp;
}

// Token j of a row stands at place j + phase, where places that are multiples
// of VEC start on VEC elements of memory: rows of any length move in aligned
// groups of VEC, and only a row's first and last places go one by one.  A
// block owns THREADS * VEC * UNROLL places of one row.  Its logits, biases and
// mask words are on their way to registers while it counts the history.
// Without history four blocks per SM are asked for (with a bias and a mask 34
// registers would leave three: 27 us against 29 at 256 x 50257 bfloat16).
// BIAS: 0 none, 1 in aligned groups too, 2 one by one.
template <typename T, int VEC, int UNROLL, bool HIST, int BIAS, bool MASK>
__global__ void __launch_bounds__(LOGITS_THREADS, HIST ? 0 : 4) logits_kernel(const LogitsArgs p) {
  constexpr bool EXACT = sizeof(T) == 4;
  constexpr int STEP = LOGITS_THREADS * VEC, RUN = STEP * UNROLL, HEAD = 2, CHUNK = 4;
  __shared__ __align__(16) unsigned counts[HIST ? RUN : 1];
  const long long row = blockIdx.y;
  const int phase = VEC > 1 ? (int)((row * p.V) % VEC) : 0;
  const int start = blockIdx.x * RUN, last = p.V + phase;  // the block's first place; the row's end
  // pointers by place
  const T* x = static_cast<const T*>(p.x) + row * p.xs - phase;
  T* y = static_cast<T*>(p.y) + row * p.V - phase;
  const float* bias = BIAS ? p.bias + row * p.bs - phase : nullptr;
  const unsigned* allowed = MASK ? p.allowed + row * p.as : nullptr;
  Group<T, VEC> xv[UNROLL];
  Group<float, VEC> bv[UNROLL];
  unsigned av[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int i = start + u * STEP + (int)threadIdx.x * VEC;
    if (i >= phase && i + VEC <= last) {
      xv[u] = *reinterpret_cast<const Group<T, VEC>*>(x + i);  // out may be the same buffer: read, then written
      if (BIAS == 1) bv[u] = *reinterpret_cast<const Group<float, VEC>*>(bias + i);
      if (BIAS == 2) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) bv[u].v[e] = bias[i + e];
      }
      if (MASK) {
        const int j = i - phase;
        av[u] = allowed[j >> 5] >> (j & 31);
        if (VEC > 1 && (j & 31) > 32 - VEC) av[u] |= allowed[(j >> 5) + 1] << (32 - (j & 31));
      }
    }
  }
  RowTerms r;
  r.rep = p.rep_rows ? p.rep_rows[row] : p.rep;
  r.inv_rep = 1.f / r.rep;
  r.freq = p.freq_rows ? p.freq_rows[row] : p.freq;
  r.pres = p.pres_rows ? p.pres_rows[row] : p.pres;
  r.temp = p.temp_rows ? p.temp_rows[row] : p.temp;
  r.inv_temp = 1.f / r.temp;
  r.divides = !reciprocal_serves(r.temp) || (HIST && !reciprocal_serves(r.rep));
  if (HIST) {
    const long long* tok = p.tokens + row * p.ts;
    long long ahead[HEAD];  // the first tokens, fetched beside the row's length
#pragma unroll
    for (int k = 0; k < HEAD; ++k) {
      const int i = threadIdx.x + k * LOGITS_THREADS;
      ahead[k] = i < p.T ? tok[i] : 0;
    }
    const int len = p.lengths ? (int)min(max(p.lengths[row], 0LL), (long long)p.T) : p.T;
    const long long pl = p.prompts ? p.prompts[row] : 0;
    for (int i = threadIdx.x * 4; i < RUN; i += LOGITS_THREADS * 4)
      *reinterpret_cast<uint4*>(counts + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    auto count = [&](int i, long long t) {
      const unsigned place = (unsigned)((int)t + phase - start);
      if (i >= len) return;
      if ((unsigned long long)t >= (unsigned)p.V) gfn_flag_error(kDevErrBadToken);
      else if (place < (unsigned)RUN) {
        if (i < pl) atomicOr(&counts[place], LOGITS_SEEN);
        else atomicAdd(&counts[place], 1u);
      }
    };
#pragma unroll
    for (int k = 0; k < HEAD; ++k) count((int)threadIdx.x + k * LOGITS_THREADS, ahead[k]);
    // the rest of a long history, CHUNK loads under way at once (a plain loop of
    // one token: 38 us against 20 at 8 x 50257 float32 with 30000 tokens)
    for (int from = HEAD * LOGITS_THREADS; from < len; from += CHUNK * LOGITS_THREADS) {
      const int i = from + (int)threadIdx.x;
      long long t[CHUNK];
#pragma unroll
      for (int k = 0; k < CHUNK; ++k) t[k] = i + k * LOGITS_THREADS < len ? tok[i + k * LOGITS_THREADS] : 0;
#pragma unroll
      for (int k = 0; k < CHUNK; ++k) count(i + k * LOGITS_THREADS, t[k]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int i = start + u * STEP + (int)threadIdx.x * VEC;
    if (i >= phase && i + VEC <= last && !r.divides) {
      bool odd = false;
      float v[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = to_f(xv[u].v[e]);
      if (HIST) {
        const Group<unsigned, VEC> c = *reinterpret_cast<const Group<unsigned, VEC>*>(counts + (i - start));
        unsigned any = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) any |= c.v[e];
        if (any) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = penalise<EXACT>(v[e], c.v[e], r, odd);
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = finish_logit<EXACT>(v[e], BIAS ? bv[u].v[e] : 0.f, r, odd);
      if (!EXACT || !odd) {
        Group<T, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = from_f<T>(!MASK || ((av[u] >> e) & 1u) ? v[e] : -INFINITY);
        *reinterpret_cast<Group<T, VEC>*>(y + i) = o;
        continue;
      }
    }
    // one by one: a group that the row's end cuts, or that needs divisions
#pragma unroll 1
    for (int k = max(i, phase); k < min(i + VEC, last); ++k) {
      const int j = k - phase;
      const float v = shaped_logit(to_f(x[k]), HIST ? counts[k - start] : 0u, BIAS ? bias[k] : 0.f, r);
      y[k] = from_f<T>(!MASK || ((allowed[j >> 5] >> (j & 31)) & 1u) ? v : -INFINITY);
    }
  }
}

template <typename T, int VEC, int UNROLL, bool HIST>
int logits_launch(const LogitsArgs& p, cudaStream_t s) {
  constexpr int RUN = LOGITS_THREADS * VEC * UNROLL;
  const dim3 grid((unsigned)((p.V + (p.V % VEC ? VEC - 1LL : 0LL) + RUN - 1) / RUN), (unsigned)p.B);  // up to VEC - 1: the phase
  const bool mask = p.allowed != nullptr;
  if (!p.bias) {
    if (mask) logits_kernel<T, VEC, UNROLL, HIST, 0, true><<<grid, LOGITS_THREADS, 0, s>>>(p);
    else logits_kernel<T, VEC, UNROLL, HIST, 0, false><<<grid, LOGITS_THREADS, 0, s>>>(p);
  } else if (VEC > 1 && p.bias_groups) {
    if (mask) logits_kernel<T, VEC, UNROLL, HIST, 1, true><<<grid, LOGITS_THREADS, 0, s>>>(p);
    else logits_kernel<T, VEC, UNROLL, HIST, 1, false><<<grid, LOGITS_THREADS, 0, s>>>(p);
  } else {
    if (mask) logits_kernel<T, VEC, UNROLL, HIST, 2, true><<<grid, LOGITS_THREADS, 0, s>>>(p);
    else logits_kernel<T, VEC, UNROLL, HIST, 2, false><<<grid, LOGITS_THREADS, 0, s>>>(p);
  }
  return launch_status("logits_kernel");
}

template <typename T, int VEC, int UNROLL>
int logits_history(const LogitsArgs& p, cudaStream_t s) {
  return p.T > 0 ? logits_launch<T, VEC, UNROLL, true>(p, s) : logits_launch<T, VEC, UNROLL, false>(p, s);
}

template <typename T>
int logits_dispatch(LogitsArgs p, cudaStream_t s) {
  constexpr int VEC = 4;
  const uintptr_t xy = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y);
  // in and out in one phase, row by row
  const bool vec = xy % (VEC * sizeof(T)) == 0 && (p.B == 1 || (p.xs - p.V) % VEC == 0);
  p.bias_groups = p.bias && aligned16(p.bias) && (p.B == 1 || (p.bs - p.V) % VEC == 0);
  // Few tokens: small blocks, to use more SMs.  Many: larger ones, since every
  // block of a row reads its whole history (at 256 x 50257 bfloat16 with 2048
  // tokens, when this was chosen: two groups a thread 39 us, four 43, one 49).
  const bool many = (long long)p.B * p.V > 592LL * LOGITS_THREADS * VEC;
  if (vec) return many ? logits_history<T, VEC, 2>(p, s) : logits_history<T, VEC, 1>(p, s);
  return many ? logits_history<T, 1, 8>(p, s) : logits_history<T, 1, 2>(p, s);
}

}  // namespace

namespace gfn_abi {
cudaError_t error_word_logits(int* v, int reset, cudaStream_t s) { return gfn_unit_error_word(v, reset, s); }
}  // namespace gfn_abi

extern "C" {

int gfn_process_logits(const void* logits, long long logits_row_stride, int dtype, int batch, int vocab,
                       const long long* tokens, long long tokens_row_stride, int history, const long long* lengths,
                       const long long* prompt_lengths, float repetition, const float* repetition_rows,
                       float frequency, const float* frequency_rows, float presence, const float* presence_rows,
                       float temperature, const float* temperature_rows, const float* bias,
                       long long bias_row_stride, const void* allowed, long long allowed_row_stride, void* out,
                       gfn_stream_t stream) {
  if (batch < 0 || vocab <= 0 || history < 0 || (batch > 0 && (!logits || !out)))
    return fail(GFN_ERR_INVALID, "process_logits: batch=%d vocab=%d history=%d or a NULL operand", batch, vocab,
                history);
  if (history > 0 && !tokens) return fail(GFN_ERR_INVALID, "process_logits: a history without tokens");
  if (batch > 65535) return fail(GFN_ERR_UNSUPPORTED, "process_logits: batch %d above 65535", batch);
  if (history > 1 << 30) return fail(GFN_ERR_UNSUPPORTED, "process_logits: history %d above 2^30", history);
  if ((!repetition_rows && !(repetition > 0.f)) || (!temperature_rows && !(temperature > 0.f)))
    return fail(GFN_ERR_INVALID, "process_logits: repetition penalty and temperature must be positive");
  if (batch == 0) return GFN_OK;
  LogitsArgs p = {};
  p.x = logits; p.y = out; p.tokens = tokens; p.lengths = lengths; p.prompts = prompt_lengths;
  p.rep_rows = repetition_rows; p.freq_rows = frequency_rows; p.pres_rows = presence_rows;
  p.temp_rows = temperature_rows; p.bias = bias; p.allowed = static_cast<const unsigned*>(allowed);
  p.xs = logits_row_stride; p.ts = tokens_row_stride; p.bs = bias_row_stride; p.as = allowed_row_stride;
  p.B = batch; p.V = vocab; p.T = history;
  p.rep = repetition; p.freq = frequency; p.pres = presence; p.temp = temperature;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == GFN_F32) return logits_dispatch<float>(p, s);
  if (dtype == GFN_BF16) return logits_dispatch<__nv_bfloat16>(p, s);
  if (dtype == GFN_F16) return logits_dispatch<__half>(p, s);
  return fail(GFN_ERR_UNSUPPORTED, "process_logits: element type %d", dtype);
}

}  // extern "C"
