// The attention with decay for float32 operands.
#include "decay_attn.cuh"

namespace gfn_attn {
int forward_f32(const PassArgs& p, bool known, cudaStream_t s) { return attn_dims<float, false, OUTPUT>(p, known, s); }
int pair_f32(const PassArgs& p, cudaStream_t s) { return attn_dims<float, true, PAIR>(p, false, s); }
int step_f32(const PassArgs& p, cudaStream_t s) { return attn_step<float>(p, s); }
int resident_f32(Kind kind, int kd, int vd) { return attn_resident<float>(kind, kd, vd); }
}  // namespace gfn_attn
