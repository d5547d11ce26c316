// C ABI of the gated scan and of the scan layer's recurrence with their
// backward passes (gated_scan.cuh).
#include "abi.h"
#include "gated_scan.cuh"

using namespace gfn;
using namespace gfn_abi;

namespace {

int check_sizes(const char* what, int B, int L, int D) {
  if (B < 0 || L < 0 || D < 0) return fail(GFN_ERR_INVALID, "%s: batch=%d length=%d dim=%d", what, B, L, D);
  if ((long long)B * D > (1LL << 36)) return fail(GFN_ERR_INVALID, "%s: batch * dim above 2^36", what);
  return GFN_OK;
}

int num_states(int L) { return (L + SCAN_CK - 1) / SCAN_CK; }

unsigned column_blocks(int B, int D) { return (unsigned)(((long long)B * D + 127) / 128); }

}  // namespace

namespace gfn_abi {
cudaError_t error_word_gated_scan(int* v, int reset, cudaStream_t s) { return gfn_unit_error_word(v, reset, s); }
}  // namespace gfn_abi

extern "C" {

long long gfn_gated_scan_states_floats(int batch, int length, int dim) {
  if (batch < 0 || length < 0 || dim < 0) return -1;
  return (long long)batch * num_states(length) * dim;
}

long long gfn_gated_scan_workspace_bytes(int batch, int length, int dim) {
  if (batch < 0 || length < 0 || dim < 0) return -1;
  return 0;
}

int gfn_gated_scan_forward(const void* a, long long a_batch_stride, long long a_step_stride, const void* x,
                           long long x_batch_stride, long long x_step_stride, const float* h0, int dtype,
                           int batch, int length, int dim, void* h, float* h_last, float* states,
                           void* workspace, long long workspace_bytes, gfn_stream_t stream) {
  int st = check_sizes("gated_scan_forward", batch, length, dim);
  if (st) return st;
  if (batch == 0 || dim == 0) return GFN_OK;
  if (length > 0 && (!x || !h)) return fail(GFN_ERR_INVALID, "gated_scan_forward: NULL x or h");
  GScanArgs p = {};
  p.a = a; p.x = x; p.h0 = h0; p.h = h; p.h_last = h_last; p.states = states;
  p.a_sb = a_batch_stride; p.a_st = a_step_stride; p.x_sb = x_batch_stride; p.x_st = x_step_stride;
  p.B = batch; p.L = length; p.D = dim; p.nck = num_states(length);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = column_blocks(batch, dim);
  if (dtype == GFN_F32) gscan_forward_seq_kernel<float><<<grid, 128, 0, s>>>(p);
  else if (dtype == GFN_BF16) gscan_forward_seq_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  else if (dtype == GFN_F16) gscan_forward_seq_kernel<__half><<<grid, 128, 0, s>>>(p);
  else return fail(GFN_ERR_UNSUPPORTED, "gated_scan_forward: element type %d", dtype);
  return launch_status("gscan_forward_seq_kernel");
}

int gfn_gated_scan_backward(const void* a, long long a_batch_stride, long long a_step_stride, const void* x,
                            long long x_batch_stride, long long x_step_stride, const float* states,
                            const void* dh, long long dh_batch_stride, long long dh_step_stride,
                            const float* dh_last, int dtype, int batch, int length, int dim, void* da, void* dx,
                            float* dh0, void* workspace, long long workspace_bytes, gfn_stream_t stream) {
  int st = check_sizes("gated_scan_backward", batch, length, dim);
  if (st) return st;
  if (batch == 0 || dim == 0) return GFN_OK;
  if (length > 0 && (!x || !states)) return fail(GFN_ERR_INVALID, "gated_scan_backward: NULL x or states");
  GScanArgs p = {};
  p.a = a; p.x = x; p.states = const_cast<float*>(states); p.dh = dh; p.dlast = dh_last;
  p.da = da; p.dx = dx; p.dh0 = dh0;
  p.a_sb = a_batch_stride; p.a_st = a_step_stride; p.x_sb = x_batch_stride; p.x_st = x_step_stride;
  p.g_sb = dh_batch_stride; p.g_st = dh_step_stride;
  p.B = batch; p.L = length; p.D = dim; p.nck = num_states(length);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = column_blocks(batch, dim);
  if (dtype == GFN_F32) gscan_backward_seq_kernel<float><<<grid, 128, 0, s>>>(p);
  else if (dtype == GFN_BF16) gscan_backward_seq_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  else if (dtype == GFN_F16) gscan_backward_seq_kernel<__half><<<grid, 128, 0, s>>>(p);
  else return fail(GFN_ERR_UNSUPPORTED, "gated_scan_backward: element type %d", dtype);
  return launch_status("gscan_backward_seq_kernel");
}

int gfn_layer_scan_forward(const float* z, const float* v0, const float* x0, int batch, int length, int dim,
                           int heads, float base_dt, float* x_seq, float* v_seq, float* x_last, float* v_last,
                           float* states, void* workspace, long long workspace_bytes, gfn_stream_t stream) {
  int st = check_sizes("layer_scan_forward", batch, length, dim);
  if (st) return st;
  if (heads <= 0 || dim % heads) return fail(GFN_ERR_INVALID, "layer_scan_forward: dim %d, heads %d", dim, heads);
  if (batch == 0 || dim == 0) return GFN_OK;
  if (length > 0 && (!z || !x_seq || !v_seq)) return fail(GFN_ERR_INVALID, "layer_scan_forward: NULL operand");
  LScanArgs p = {};
  p.z = z; p.v0 = v0; p.x0 = x0; p.xs = x_seq; p.vs = v_seq; p.x_last = x_last; p.v_last = v_last;
  p.states = states; p.B = batch; p.L = length; p.D = dim; p.H = heads; p.nck = num_states(length);
  p.base_dt = base_dt;
  lscan_forward_seq_kernel<<<column_blocks(batch, dim), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return launch_status("lscan_forward_seq_kernel");
}

int gfn_layer_scan_backward(const float* z, const float* states, const float* gx, const float* gv,
                            const float* gx_last, const float* gv_last, int batch, int length, int dim, int heads,
                            float base_dt, float* dz, float* dx0, float* dv0, void* workspace,
                            long long workspace_bytes, gfn_stream_t stream) {
  int st = check_sizes("layer_scan_backward", batch, length, dim);
  if (st) return st;
  if (heads <= 0 || dim % heads) return fail(GFN_ERR_INVALID, "layer_scan_backward: dim %d, heads %d", dim, heads);
  if (batch == 0 || dim == 0) return GFN_OK;
  if (length > 0 && (!z || !states || !dz)) return fail(GFN_ERR_INVALID, "layer_scan_backward: NULL operand");
  LScanArgs p = {};
  p.z = z; p.states = const_cast<float*>(states); p.gx = gx; p.gv = gv; p.gxl = gx_last; p.gvl = gv_last;
  p.dz = dz; p.dv0 = dv0; p.dx0 = dx0; p.B = batch; p.L = length; p.D = dim; p.H = heads;
  p.nck = num_states(length); p.base_dt = base_dt;
  lscan_backward_seq_kernel<<<column_blocks(batch, dim), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return launch_status("lscan_backward_seq_kernel");
}

}  // extern "C"
