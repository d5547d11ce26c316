// The attention with decay for bfloat16 operands.
#include "decay_attn.cuh"

namespace gfn_attn {
int forward_bf16(const PassArgs& p, bool known, cudaStream_t s) { return attn_dims<__nv_bfloat16, false, OUTPUT>(p, known, s); }
int pair_bf16(const PassArgs& p, cudaStream_t s) { return attn_dims<__nv_bfloat16, true, PAIR>(p, false, s); }
int step_bf16(const PassArgs& p, cudaStream_t s) { return attn_step<__nv_bfloat16>(p, s); }
int resident_bf16(Kind kind, int kd, int vd) { return attn_resident<__nv_bfloat16>(kind, kd, vd); }
}  // namespace gfn_attn
