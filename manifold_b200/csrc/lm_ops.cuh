// Element types of the language-model operators (layer norm, gated scan,
// logit shaping): float32, bfloat16 and float16 in memory, float32 in
// registers.  A value is rounded once, when it is stored.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace gfn {

GFN_DEV float to_f(float v) { return v; }
GFN_DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
GFN_DEV float to_f(__half v) { return __half2float(v); }

template <typename T> GFN_DEV T from_f(float v);
template <> GFN_DEV float from_f<float>(float v) { return v; }
template <> GFN_DEV __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> GFN_DEV __half from_f<__half>(float v) { return __float2half_rn(v); }

// Two float32 values in one 64-bit register pair: Blackwell's packed
// arithmetic does both in one instruction (each rounded as by itself), which
// halves the issue slots of kernels that instructions bind.
struct F2 {
  unsigned long long v;
};
GFN_DEV F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
GFN_DEV F2 f2(float both) { return f2(both, both); }
GFN_DEV void split(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
GFN_DEV F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
GFN_DEV F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
GFN_DEV F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

}  // namespace gfn
