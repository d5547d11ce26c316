// C ABI of the gated scan and of the scan layer's recurrence with their
// backward passes (gated_scan.cuh).
#include <cuda.h>
#include <cudaTypedefs.h>

#include "gated_scan.cuh"
#include "lm_host.h"

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

// Up to this length a thread walks its column alone.
constexpr int SEQ_STEPS = 8;
constexpr long long TICKET_BYTES = 256;  // the ticket, then the words

// The runs and tiles of a launch, and its words in the workspace (all ones).
template <class Args>
int set_tiles(const char* what, Args* p, int run, int ct, int words, int occ, void* workspace, long long bytes,
              cudaStream_t s, unsigned* grid) {
  p->nchunks = (p->L + run - 1) / run;
  p->ctiles = (p->D + ct - 1) / ct;
  const long long tiles = (long long)p->B * p->ctiles, blocks = tiles * p->nchunks;
  if (blocks > 0x7fffffffLL) return fail(GFN_ERR_UNSUPPORTED, "%s: %lld blocks", what, blocks);
  *grid = (unsigned)blocks;
  // The runs of one column tile that are under way at once wait for one another
  // once per group.  With at most one of them a chain of states is enough
  // (composing maps nobody waits for cost 12 of 154 instructions per element in
  // the layer's backward); with more a group covers them twice over.
  int sms = 0;
  const int st = sm_count(&sms);
  if (st) return st;
  const long long slots = (long long)sms * occ;
  p->group = 1;
  if (tiles < slots)
    while (p->group < SCAN_GROUP && tiles * p->group < 2 * slots) p->group *= 2;
  p->words = nullptr;
  p->ticket = nullptr;
  if (p->nchunks == 1) return GFN_OK;
  const long long need = TICKET_BYTES + blocks * ct * words * 8;
  if (!workspace || bytes < need)
    return fail(GFN_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", what, workspace ? bytes : 0, need);
  if (!aligned16(workspace)) return fail(GFN_ERR_ALIGN, "%s: workspace not 16-byte aligned", what);
  p->ticket = static_cast<unsigned*>(workspace);
  p->words = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + TICKET_BYTES);
  return cuda_status(cudaMemsetAsync(workspace, 0xff, (size_t)need, s), what);
}

// Whether every row of an operand starts on 16 bytes and no stride is zero, as
// a tensor copy needs it.
bool rows16(const void* ptr, long long sb, long long st, int B, int L, int size) {
  return !ptr || (aligned16(ptr) && (B == 1 || (sb > 0 && sb * size % 16 == 0 && sb * size < (1LL << 40))) &&
                  (L == 1 || (st > 0 && st * size % 16 == 0 && st * size < (1LL << 40))));
}

// cuTensorMapEncodeTiled from the driver (no link-time libcuda dependency).
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

CUtensorMapDataType map_type(const float*) { return CU_TENSOR_MAP_DATA_TYPE_FLOAT32; }
CUtensorMapDataType map_type(const __nv_bfloat16*) { return CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }
CUtensorMapDataType map_type(const __half*) { return CU_TENSOR_MAP_DATA_TYPE_FLOAT16; }

// One operand (NULL: none) as a [B][L][cols] tensor with `steps` x `ct` boxes;
// strides in elements.
template <typename T>
int operand_map(CUtensorMap* m, const T* base, long long sb, long long st, int B, int L, int cols, int steps, int ct) {
  if (!base) return GFN_OK;
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return fail(GFN_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t row = (cuuint64_t)(cols * (int)sizeof(T));
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)L, (cuuint64_t)B};
  // the stride of a dimension of one element is never used, but has to be valid
  const cuuint64_t strides[2] = {L > 1 ? (cuuint64_t)st * sizeof(T) : row, B > 1 ? (cuuint64_t)sb * sizeof(T) : row};
  const cuuint32_t box[3] = {(cuuint32_t)ct, (cuuint32_t)steps, 1}, unit[3] = {1, 1, 1};
  const CUresult r = enc(m, map_type(base), 3, const_cast<T*>(base), dims, strides, box, unit,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(GFN_ERR_CUDA, "scan: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return GFN_OK;
}

// A persistent launch: OCC blocks per SM, each with `stage` bytes for the next
// run's operands.
template <class Args>
int launch(const char* what, void (*kernel)(Args, ScanMaps), const Args& p, const ScanMaps& maps, unsigned blocks,
           int occ, int threads, int stage, std::atomic<unsigned long long>* done, cudaStream_t s) {
  int sms = 0, st = sm_count(&sms);
  if (!st && stage) st = shared_limit(kernel, stage, done, what);
  if (st) return st;
  const unsigned slots = (unsigned)(sms * occ);
  kernel<<<blocks < slots ? blocks : slots, threads, stage, s>>>(p, maps);
  return launch_status(what);
}

template <int MODE, typename T, int VEC, int S, int NW, int OCC>
int gscan_forward(GScanArgs p, void* ws, long long bytes, cudaStream_t s) {
  unsigned blocks;
  const int st = set_tiles("gated_scan_forward", &p, S * NW, 32 * VEC, 1, OCC, ws, bytes, s, &blocks);
  if (st) return st;
  ScanMaps maps = {};
  if (MODE == SCAN_TMA) {
    int e = operand_map(&maps.m[0], static_cast<const T*>(p.x), p.x_sb, p.x_st, p.B, p.L, p.D, S * NW, 32 * VEC);
    if (!e) e = operand_map(&maps.m[1], static_cast<const T*>(p.a), p.a_sb, p.a_st, p.B, p.L, p.D, S * NW, 32 * VEC);
    if (e) return e;
  }
  static std::atomic<unsigned long long> done{0};
  return launch("gscan_forward_kernel", gscan_forward_kernel<MODE, T, VEC, S, NW, OCC>, p, maps, blocks, OCC, NW * 32,
                MODE == SCAN_TMA ? 2 * Stage<T, VEC, S, NW>::OPERAND : 0, &done, s);
}

template <int MODE, typename T, int VEC, int S, int NW, int OCC>
int gscan_backward(GScanArgs p, void* ws, long long bytes, cudaStream_t s) {
  unsigned blocks;
  const int st = set_tiles("gated_scan_backward", &p, S * NW, 32 * VEC, 1, OCC, ws, bytes, s, &blocks);
  if (st) return st;
  ScanMaps maps = {};
  if (MODE == SCAN_TMA) {
    int e = operand_map(&maps.m[0], static_cast<const T*>(p.x), p.x_sb, p.x_st, p.B, p.L, p.D, S * NW, 32 * VEC);
    if (!e) e = operand_map(&maps.m[1], static_cast<const T*>(p.a), p.a_sb, p.a_st, p.B, p.L, p.D, S * NW, 32 * VEC);
    if (!e) e = operand_map(&maps.m[2], static_cast<const T*>(p.dh), p.g_sb, p.g_st, p.B, p.L, p.D, S * NW, 32 * VEC);
    if (e) return e;
  }
  static std::atomic<unsigned long long> done{0};
  return launch("gscan_backward_kernel", gscan_backward_kernel<MODE, T, VEC, S, NW, OCC>, p, maps, blocks, OCC, NW * 32,
                MODE == SCAN_TMA ? 3 * Stage<T, VEC, S, NW>::OPERAND : 0, &done, s);
}

template <typename T>
int gscan_run(const GScanArgs& p, bool backward, void* ws, long long bytes, cudaStream_t s) {
  constexpr int z = sizeof(T);
  if (!backward && p.L <= SEQ_STEPS) {
    gscan_forward_seq_kernel<T><<<column_blocks(p.B, p.D), 128, 0, s>>>(p);
    return launch_status("gscan_forward_seq_kernel");
  }
  const bool tma = p.D * z % 16 == 0 && rows16(p.a, p.a_sb, p.a_st, p.B, p.L, z) &&
                    rows16(p.x, p.x_sb, p.x_st, p.B, p.L, z) && rows16(p.dh, p.g_sb, p.g_st, p.B, p.L, z) &&
                    aligned16(p.h) && aligned16(p.da) && aligned16(p.dx);
  if (tma)
    return backward ? gscan_backward<SCAN_TMA, T, 2, z == 2 ? 16 : 8, 8, 2>(p, ws, bytes, s)
                    : gscan_forward<SCAN_TMA, T, 2, z == 2 ? 32 : 16, 8, 2>(p, ws, bytes, s);
  return backward ? gscan_backward<SCAN_PLAIN, T, 1, 8, 8, 4>(p, ws, bytes, s)
                  : gscan_forward<SCAN_PLAIN, T, 1, 16, 8, 3>(p, ws, bytes, s);
}

int gscan_dispatch(const GScanArgs& p, int dtype, bool backward, void* ws, long long bytes, cudaStream_t s) {
  if (dtype == GFN_F32) return gscan_run<float>(p, backward, ws, bytes, s);
  if (dtype == GFN_BF16) return gscan_run<__nv_bfloat16>(p, backward, ws, bytes, s);
  if (dtype == GFN_F16) return gscan_run<__half>(p, backward, ws, bytes, s);
  return fail(GFN_ERR_UNSUPPORTED, "gated_scan: element type %d", dtype);
}

template <int MODE>
int lscan_forward(LScanArgs p, void* ws, long long bytes, cudaStream_t s) {
  constexpr int VEC = 1, S = 16, NW = 8, OCC = 2;
  unsigned blocks;
  const int st = set_tiles("layer_scan_forward", &p, S * NW, 32 * VEC, 2, OCC, ws, bytes, s, &blocks);
  if (st) return st;
  ScanMaps maps = {};
  if (MODE == SCAN_TMA) {
    const long long D = p.D;
    int e = operand_map(&maps.m[0], p.z, 3 * D * p.L, 3 * D, p.B, p.L, 3 * p.D, S * NW, 32 * VEC);
    if (e) return e;
  }
  static std::atomic<unsigned long long> done{0};
  return launch("lscan_forward_kernel", lscan_forward_kernel<MODE, VEC, S, NW, OCC>, p, maps, blocks, OCC, NW * 32,
                MODE == SCAN_TMA ? 3 * Stage<float, VEC, S, NW>::OPERAND : 0, &done, s);
}

template <int MODE>
int lscan_backward(LScanArgs p, void* ws, long long bytes, cudaStream_t s) {
  constexpr int VEC = 1, S = 8, NW = 8, OCC = 2;
  unsigned blocks;
  const int st = set_tiles("layer_scan_backward", &p, S * NW, 32 * VEC, 2, OCC, ws, bytes, s, &blocks);
  if (st) return st;
  ScanMaps maps = {};
  if (MODE == SCAN_TMA) {
    const long long D = p.D;
    int e = operand_map(&maps.m[0], p.z, 3 * D * p.L, 3 * D, p.B, p.L, 3 * p.D, S * NW, 32 * VEC);
    if (!e) e = operand_map(&maps.m[1], p.gx, D * p.L, D, p.B, p.L, p.D, S * NW, 32 * VEC);
    if (!e) e = operand_map(&maps.m[2], p.gv, D * p.L, D, p.B, p.L, p.D, S * NW, 32 * VEC);
    if (e) return e;
  }
  static std::atomic<unsigned long long> done{0};
  return launch("lscan_backward_kernel", lscan_backward_kernel<MODE, VEC, S, NW, OCC>, p, maps, blocks, OCC, NW * 32,
                MODE == SCAN_TMA ? 5 * Stage<float, VEC, S, NW>::OPERAND : 0, &done, s);
}

// A state or its gradient handed through a sequence of no steps.
int pass_through(const char* what, float* dst, const float* src, int B, int D, cudaStream_t s) {
  if (!dst) return GFN_OK;
  const size_t n = (size_t)B * D * sizeof(float);
  return cuda_status(src ? cudaMemcpyAsync(dst, src, n, cudaMemcpyDeviceToDevice, s) : cudaMemsetAsync(dst, 0, n, s),
                     what);
}

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
  if (length <= SCAN_CK || batch == 0 || dim == 0) return 0;
  // the shortest runs (SCAN_CK steps), the widest tiles (128 columns), two words
  return TICKET_BYTES + (long long)batch * num_states(length) * ((dim + 127LL) / 128 * 128) * 16;
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
  return gscan_dispatch(p, dtype, false, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
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
  if (length == 0) return pass_through("gated_scan_backward", dh0, dh_last, batch, dim, s);
  return gscan_dispatch(p, dtype, true, workspace, workspace_bytes, s);
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
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (length <= SEQ_STEPS) {
    lscan_forward_seq_kernel<<<column_blocks(batch, dim), 128, 0, s>>>(p);
    return launch_status("lscan_forward_seq_kernel");
  }
  const bool tma = dim % 4 == 0 && aligned16(z) && aligned16(x_seq) && aligned16(v_seq);
  return tma ? lscan_forward<SCAN_TMA>(p, workspace, workspace_bytes, s)
              : lscan_forward<SCAN_PLAIN>(p, workspace, workspace_bytes, s);
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
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (length == 0) {
    st = pass_through("layer_scan_backward", dv0, gv_last, batch, dim, s);
    return st ? st : pass_through("layer_scan_backward", dx0, gx_last, batch, dim, s);
  }
  const bool tma = dim % 4 == 0 && aligned16(z) && aligned16(gx) && aligned16(gv) && aligned16(dz);
  return tma ? lscan_backward<SCAN_TMA>(p, workspace, workspace_bytes, s)
              : lscan_backward<SCAN_PLAIN>(p, workspace, workspace_bytes, s);
}

}  // extern "C"
