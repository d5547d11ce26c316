// The attention with decay for float16 operands.
#include "decay_attn.cuh"

namespace gfn_attn {
int forward_f16(const PassArgs& p, bool known, cudaStream_t s) { return attn_dims<__half, false, OUTPUT>(p, known, s); }
int pair_f16(const PassArgs& p, cudaStream_t s) { return attn_dims<__half, true, PAIR>(p, false, s); }
int step_f16(const PassArgs& p, cudaStream_t s) { return attn_step<__half>(p, s); }
int resident_f16(Kind kind, int kd, int vd) { return attn_resident<__half>(kind, kd, vd); }
}  // namespace gfn_attn
