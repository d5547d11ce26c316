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
  int B, L, D, nck;
};

// One thread per column, one step after the other.
template <typename T>
__global__ void __launch_bounds__(128) gscan_forward_seq_kernel(const GScanArgs p) {
  const long long c = blockIdx.x * 128LL + threadIdx.x;
  if (c >= (long long)p.B * p.D) return;
  const long long b = c / p.D, j = c - b * p.D;
  const T* a = p.a ? static_cast<const T*>(p.a) + b * p.a_sb + j : nullptr;
  const T* x = static_cast<const T*>(p.x) + b * p.x_sb + j;
  T* h = static_cast<T*>(p.h) + b * p.L * (long long)p.D + j;
  float s = p.h0 ? p.h0[c] : 0.f;
  for (int t = 0; t < p.L; ++t) {
    if (p.states && t % SCAN_CK == 0) p.states[(b * p.nck + t / SCAN_CK) * (long long)p.D + j] = s;
    s = fmaf(a ? to_f(a[t * p.a_st]) : 1.f, s, to_f(x[t * p.x_st]));
    h[(long long)t * p.D] = from_f<T>(s);
  }
  if (p.h_last) p.h_last[c] = s;
}

template <typename T>
__global__ void __launch_bounds__(128) gscan_backward_seq_kernel(const GScanArgs p) {
  const long long c = blockIdx.x * 128LL + threadIdx.x;
  if (c >= (long long)p.B * p.D) return;
  const long long b = c / p.D, j = c - b * p.D;
  const T* a = p.a ? static_cast<const T*>(p.a) + b * p.a_sb + j : nullptr;
  const T* x = static_cast<const T*>(p.x) + b * p.x_sb + j;
  const T* dh = p.dh ? static_cast<const T*>(p.dh) + b * p.g_sb + j : nullptr;
  const long long o = b * p.L * (long long)p.D + j;
  T* da = static_cast<T*>(p.da);
  T* dx = static_cast<T*>(p.dx);
  float m = p.dlast ? p.dlast[c] : 0.f;
  for (int k = p.nck - 1; k >= 0; --k) {
    const int t0 = k * SCAN_CK, n = min(SCAN_CK, p.L - t0);
    float hp[SCAN_CK];  // h_{t-1}
    float s = p.states[(b * p.nck + k) * (long long)p.D + j];
    for (int u = 0; u < n; ++u) {
      hp[u] = s;
      s = fmaf(a ? to_f(a[(t0 + u) * p.a_st]) : 1.f, s, to_f(x[(t0 + u) * p.x_st]));
    }
    for (int u = n - 1; u >= 0; --u) {
      const float g = (dh ? to_f(dh[(t0 + u) * p.g_st]) : 0.f) + m;
      const long long e = o + (long long)(t0 + u) * p.D;
      if (dx) dx[e] = from_f<T>(g);
      if (da) da[e] = from_f<T>(g * hp[u]);
      m = (a ? to_f(a[(t0 + u) * p.a_st]) : 1.f) * g;
    }
  }
  if (p.dh0) p.dh0[c] = m;
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
  int B, L, D, H, nck;
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

__global__ void __launch_bounds__(128) lscan_forward_seq_kernel(const LScanArgs p) {
  const long long c = blockIdx.x * 128LL + threadIdx.x;
  if (c >= (long long)p.B * p.D) return;
  const long long b = c / p.D, j = c - b * p.D;
  const float hs = head_scale((int)j, p.D / p.H);
  float v = p.v0 ? p.v0[c] : 0.f, x = p.x0 ? p.x0[c] : 0.f;
  for (int t = 0; t < p.L; ++t) {
    if (p.states && t % SCAN_CK == 0) p.states[(b * p.nck + t / SCAN_CK) * (long long)p.D + j] = v;
    const float* z = p.z + (b * p.L + t) * 3 * p.D + j;
    const float dt = (softplus_f(z[p.D]) * p.base_dt) * hs;
    v = gate(z[0]) * v + z[2LL * p.D] * dt;
    x = x + v * dt;
    const long long e = (b * p.L + t) * p.D + j;
    p.vs[e] = v;
    p.xs[e] = x;
  }
  if (p.v_last) p.v_last[c] = v;
  if (p.x_last) p.x_last[c] = x;
}

__global__ void __launch_bounds__(128) lscan_backward_seq_kernel(const LScanArgs p) {
  const long long c = blockIdx.x * 128LL + threadIdx.x;
  if (c >= (long long)p.B * p.D) return;
  const long long b = c / p.D, j = c - b * p.D;
  const float hs = head_scale((int)j, p.D / p.H);
  float m = p.gvl ? p.gvl[c] : 0.f, X = p.gxl ? p.gxl[c] : 0.f;
  for (int k = p.nck - 1; k >= 0; --k) {
    const int t0 = k * SCAN_CK, n = min(SCAN_CK, p.L - t0);
    float vp[SCAN_CK];
    float v = p.states[(b * p.nck + k) * (long long)p.D + j];
    for (int u = 0; u < n; ++u) {
      const float* z = p.z + (b * p.L + t0 + u) * 3 * p.D + j;
      vp[u] = v;
      v = gate(z[0]) * v + z[2LL * p.D] * ((softplus_f(z[p.D]) * p.base_dt) * hs);
    }
    for (int u = n - 1; u >= 0; --u) {
      const long long r = b * p.L + t0 + u;
      const float* z = p.z + r * 3 * p.D + j;
      float* dz = p.dz + r * 3 * p.D + j;
      float nA;
      const float A = gate(z[0], &nA), dt = (softplus_f(z[p.D]) * p.base_dt) * hs;
      if (p.gx) X += p.gx[r * p.D + j];
      const float l = (p.gv ? p.gv[r * p.D + j] : 0.f) + dt * X + m;
      dz[0] = l * vp[u] * (A * nA);
      dz[p.D] = (l * z[2LL * p.D] + X * v) * (p.base_dt * hs) * gate(z[p.D]);
      dz[2LL * p.D] = l * dt;
      v = vp[u];
      m = A * l;
    }
  }
  if (p.dv0) p.dv0[c] = m;
  if (p.dx0) p.dx0[c] = X;
}

}  // namespace gfn
