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
#include "abi.h"
#include "lm_ops.cuh"

using namespace gfn;
using namespace gfn_abi;

namespace {

constexpr int LOGITS_THREADS = 256;
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
  int B, V, T, run;
  float rep, freq, pres, temp;
};

template <typename T>
__global__ void __launch_bounds__(LOGITS_THREADS) logits_kernel(const LogitsArgs p) {
  extern __shared__ unsigned counts[];
  const long long row = blockIdx.y;
  const int j0 = blockIdx.x * p.run, n = min(p.run, p.V - j0);
  const bool hist = p.T > 0;
  if (hist) {
    for (int i = threadIdx.x; i < n; i += LOGITS_THREADS) counts[i] = 0u;
    __syncthreads();
    const long long* tok = p.tokens + row * p.ts;
    const long long len = p.lengths ? min(max(p.lengths[row], 0LL), (long long)p.T) : p.T;
    const long long pl = p.prompts ? p.prompts[row] : 0;
    for (long long i = threadIdx.x; i < len; i += LOGITS_THREADS) {
      const long long t = tok[i];
      if (t < 0 || t >= p.V) {
        gfn_flag_error(kDevErrBadToken);
        continue;
      }
      if (t < j0 || t >= j0 + n) continue;
      if (i < pl) atomicOr(&counts[t - j0], LOGITS_SEEN);
      else atomicAdd(&counts[t - j0], 1u);
    }
    __syncthreads();
  }
  const float rep = p.rep_rows ? p.rep_rows[row] : p.rep;
  const float freq = p.freq_rows ? p.freq_rows[row] : p.freq;
  const float pres = p.pres_rows ? p.pres_rows[row] : p.pres;
  const float temp = p.temp_rows ? p.temp_rows[row] : p.temp;
  const T* x = static_cast<const T*>(p.x) + row * p.xs + j0;
  T* y = static_cast<T*>(p.y) + row * p.V + j0;
  for (int i = threadIdx.x; i < n; i += LOGITS_THREADS) {
    float v = to_f(x[i]);
    if (hist && counts[i]) {
      const unsigned c = counts[i] & ~LOGITS_SEEN;
      v = v > 0.f ? v / rep : v * rep;
      if (c) v -= freq * (float)c + pres;
    }
    const int j = j0 + i;
    if (p.bias) v += p.bias[row * p.bs + j];
    v /= temp;
    if (p.allowed && !((p.allowed[row * p.as + (j >> 5)] >> (j & 31)) & 1u)) v = -INFINITY;
    y[i] = from_f<T>(v);
  }
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
  if ((!repetition_rows && !(repetition > 0.f)) || (!temperature_rows && !(temperature > 0.f)))
    return fail(GFN_ERR_INVALID, "process_logits: repetition penalty and temperature must be positive");
  if (batch == 0) return GFN_OK;
  LogitsArgs p = {};
  p.x = logits; p.y = out; p.tokens = tokens; p.lengths = lengths; p.prompts = prompt_lengths;
  p.rep_rows = repetition_rows; p.freq_rows = frequency_rows; p.pres_rows = presence_rows;
  p.temp_rows = temperature_rows; p.bias = bias; p.allowed = static_cast<const unsigned*>(allowed);
  p.xs = logits_row_stride; p.ts = tokens_row_stride; p.bs = bias_row_stride; p.as = allowed_row_stride;
  p.B = batch; p.V = vocab; p.T = history; p.run = 4096;
  p.rep = repetition; p.freq = frequency; p.pres = presence; p.temp = temperature;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((vocab + p.run - 1) / p.run), (unsigned)batch);
  const size_t smem = history > 0 ? (size_t)p.run * sizeof(unsigned) : 0;
  if (dtype == GFN_F32) logits_kernel<float><<<grid, LOGITS_THREADS, smem, s>>>(p);
  else if (dtype == GFN_BF16) logits_kernel<__nv_bfloat16><<<grid, LOGITS_THREADS, smem, s>>>(p);
  else if (dtype == GFN_F16) logits_kernel<__half><<<grid, LOGITS_THREADS, smem, s>>>(p);
  else return fail(GFN_ERR_UNSUPPORTED, "process_logits: element type %d", dtype);
  return launch_status("logits_kernel");
}

}  // extern "C"
