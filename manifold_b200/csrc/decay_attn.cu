// Linear attention with a decay for each head: the entry points, and how
// sequences are cut.  The kernels are in decay_attn.cuh.
#include <initializer_list>

#include "decay_attn.h"
#include "lm_host.h"

using namespace gfn_abi;
using namespace gfn_attn;

namespace {

constexpr int SEG_UNIT = 64;  // tokens; every kernel's block divides it

int resident(Kind kind, int dtype, int kd, int vd) {
  return dtype == GFN_F32 ? resident_f32(kind, kd, vd) : dtype == GFN_BF16 ? resident_bf16(kind, kd, vd) : resident_f16(kind, kd, vd);
}

// Where sequences and heads are too few to fill the device, sequences are cut
// into as many segments as it holds thread blocks at once, of two units at least.
struct Cut {
  int seg_len, segments;
  long long floats(int batch, int heads, int kd, int vd) const {
    return segments > 1 ? (long long)batch * heads * segments * kd * vd : 0;
  }
};
Cut cut(Kind kind, int dtype, int batch, int length, int heads, int kd, int vd, int sms) {
  const long long units = ((long long)length + SEG_UNIT - 1) / SEG_UNIT;
  long long n = (long long)resident(kind, dtype, kd, vd) * sms / ((long long)batch * heads);
  if (n > units / 2) n = units / 2;
  if (n < 1) n = 1;
  const long long per = (units + n - 1) / n;
  return {(int)(per * SEG_UNIT), (int)((units + per - 1) / per)};
}

// The largest piece, up to 16 bytes, that rows of `v` divide into and start on.
int piece_of(const View& v, int dim, int size) {
  unsigned long long all = reinterpret_cast<uintptr_t>(v.p) | 16ull;
  for (const long long n : {(long long)dim, v.sb, v.sl, v.sh}) all |= (unsigned long long)(n < 0 ? -n : n) * size;
  return (int)(all & (~all + 1));
}
int smallest(std::initializer_list<int> pieces) {
  int n = 16;
  for (const int q : pieces) n = q < n ? q : n;
  return n;
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

View view(const void* p, const long long* strides) { return {p, strides[0], strides[1], strides[2]}; }

bool enough(const void* workspace, long long bytes, long long floats) {
  return floats == 0 || (workspace && aligned16(workspace) && bytes >= 4 * floats);
}

}  // namespace

extern "C" {

long long gfn_decay_attention_workspace_bytes(int backward, int dtype, int batch, int length, int heads, int kdim, int vdim) {
  if (batch <= 0 || heads <= 0 || length <= 0) return 0;
  int sms = 0;
  if (attn_check("decay_attention", dtype, batch, length, heads, kdim, vdim, false) != GFN_OK || sm_count(&sms) != GFN_OK)
    return -1;
  long long n = cut(OUTPUT, dtype, batch, length, heads, kdim, vdim, sms).floats(batch, heads, kdim, vdim);
  if (backward) {
    const long long m = cut(PAIR, dtype, batch, length, heads, kdim, vdim, sms).floats(batch, heads, kdim, vdim);
    n = m > n ? m : n;
  }
  return 4 * n;
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
  p.a = view(q, q_strides); p.b = view(k, k_strides); p.c = view(v, v_strides);
  p.o = o; p.decay = decay; p.state = state; p.state_out = state_out;
  p.lengths = lengths; p.lengths64 = lengths_are_64; p.B = batch; p.L = length; p.H = heads; p.KD = kdim; p.VD = vdim;
  p.sr = vdim; p.sc = 1; p.s_in = p.s_state = scale; p.s_update = 1.f;
  if (length == 1) return dtype == GFN_F32 ? step_f32(p, s) : dtype == GFN_BF16 ? step_bf16(p, s) : step_f16(p, s);
  const Cut c = cut(OUTPUT, dtype, batch, length, heads, kdim, vdim, sms);
  p.seg_len = c.seg_len; p.segments = c.segments;
  p.segs = static_cast<float*>(workspace); p.segs_sr = vdim; p.segs_sc = 1;
  if (!enough(workspace, workspace_bytes, c.floats(batch, heads, kdim, vdim)))
    return fail(GFN_ERR_INVALID, "decay_attention: a workspace of gfn_decay_attention_workspace_bytes is needed");
  const int size = dtype == GFN_F32 ? 4 : 2;
  p.piece = smallest({piece_of(p.a, kdim, size), piece_of(p.b, kdim, size), piece_of(p.c, vdim, size)});
  return dtype == GFN_F32 ? forward_f32(p, false, s) : dtype == GFN_BF16 ? forward_bf16(p, false, s) : forward_f16(p, false, s);
}

int gfn_decay_attention_backward(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
                                 const void* v, const long long* v_strides, const void* d_o, const long long* do_strides,
                                 const float* decay, const float* state, const float* d_state_out, const void* lengths,
                                 int lengths_are_64, int dtype, int batch, int length, int heads, int kdim, int vdim,
                                 float scale, const void* forward_workspace, void* dq, void* dk, void* dv, float* d_state,
                                 void* workspace, long long workspace_bytes, gfn_stream_t stream) {
  int st = attn_check("decay_attention backward", dtype, batch, length, heads, kdim, vdim,
                      !decay || (length > 0 && (!q || !k || !v || !d_o || !dq || !dk || !dv)));
  if (st != GFN_OK) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (batch == 0 || heads == 0) return GFN_OK;
  if (length == 0) return attn_copy_state(d_state_out, d_state, (long long)batch * heads * kdim * vdim, s);
  int sms = 0;
  if ((st = sm_count(&sms)) != GFN_OK) return st;
  const View vq = view(q, q_strides), vk = view(k, k_strides), vv = view(v, v_strides), vo = view(d_o, do_strides);
  PassArgs p = {};
  p.decay = decay; p.lengths = lengths; p.lengths64 = lengths_are_64; p.B = batch; p.L = length; p.H = heads;
  const int size = dtype == GFN_F32 ? 4 : 2;
  p.piece = smallest({piece_of(vq, kdim, size), piece_of(vk, kdim, size), piece_of(vv, vdim, size), piece_of(vo, vdim, size)});
  // dq, over the forward pass's segments: its states serve again, transposed
  const Cut cf = cut(OUTPUT, dtype, batch, length, heads, kdim, vdim, sms);
  const Cut cr = cut(PAIR, dtype, batch, length, heads, kdim, vdim, sms);
  const bool known = forward_workspace && length > 1;
  const long long nf = known ? 0 : cf.floats(batch, heads, kdim, vdim), nr = cr.floats(batch, heads, kdim, vdim);
  if (!enough(workspace, workspace_bytes, nf > nr ? nf : nr))
    return fail(GFN_ERR_INVALID, "decay_attention backward: a workspace of gfn_decay_attention_workspace_bytes is needed");
  PassArgs f = p;
  f.a = vo; f.b = vv; f.c = vk; f.o = dq; f.state = state; f.KD = vdim; f.VD = kdim; f.sr = 1; f.sc = vdim;
  f.s_in = f.s_state = scale; f.s_update = 1.f;
  f.seg_len = cf.seg_len; f.segments = cf.segments;
  f.segs = known ? static_cast<float*>(const_cast<void*>(forward_workspace)) : static_cast<float*>(workspace);
  f.segs_sr = known ? 1 : kdim; f.segs_sc = known ? vdim : 1;
  PassArgs r = p;  // dv and dk
  r.a = vq; r.b = vk; r.c = vv; r.d = vo; r.o = dv; r.o2 = dk; r.state = d_state_out; r.state_out = d_state;
  r.KD = kdim; r.VD = vdim; r.sr = vdim; r.sc = 1; r.s_in = r.s_update = scale; r.s_state = 1.f;
  r.seg_len = cr.seg_len; r.segments = cr.segments;
  r.segs = static_cast<float*>(workspace); r.segs_sr = vdim; r.segs_sc = 1;
  st = dtype == GFN_F32 ? forward_f32(f, known, s) : dtype == GFN_BF16 ? forward_bf16(f, known, s) : forward_f16(f, known, s);
  if (st != GFN_OK) return st;
  return dtype == GFN_F32 ? pair_f32(r, s) : dtype == GFN_BF16 ? pair_bf16(r, s) : pair_f16(r, s);
}

}  // extern "C"
