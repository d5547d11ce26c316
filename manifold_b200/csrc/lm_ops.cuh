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

}  // namespace gfn
