// What the units of the attention with decay share: the operands of a pass and
// how its sequences are cut.  decay_attn.cu has the entry points; there is a
// unit for each element type.
#pragma once
#include <cuda_runtime.h>

namespace gfn_attn {

struct View {  // [batch][length][heads][dim], inner stride 1
  const void* p;
  long long sb, sl, sh;
};

struct PassArgs {
  View a, b, c, d;      // q, k, v; in the two-output pass also do (see attn_kernel)
  void* o;              // [B][L][H][c.dim]
  void* o2;
  const float* decay;
  const float* state;   // before the first token, or nullptr
  float* state_out;     // after the last, or nullptr
  float* segs;          // [B * H][segments]: states by segment, KD x VD each, or nullptr (one segment)
  long long segs_sr, segs_sc;  // strides of their rows and columns
  const void* lengths;
  int lengths64;
  int B, L, H, KD, VD;  // dims of the state's rows (keys) and columns (values)
  long long sr, sc;     // strides of the state's rows and columns
  int seg_len, segments;
  float s_in, s_state, s_update;  // factors of the products within a block, with the state, and of the state's update
  int piece;            // operands arrive in pieces of so many bytes (16, 8, 4), or by single 16-bit elements (2)
};

// What a launch does: a segment's output, its part of the state alone, or the
// two outputs of the backward pass.
enum Kind { OUTPUT, STATE, PAIR };

// The padded dims that a kernel is compiled for.
struct Dims {
  int k, v;
};
inline Dims padded(int kd, int vd) {
  const int d = kd > vd ? kd : vd;
  if (d <= 32) return {32, 32};
  return {kd <= 64 ? 64 : 128, vd <= 64 ? 64 : 128};
}

// Thread blocks of a kind that an SM holds at once.
int resident_f32(Kind kind, int kd, int vd);
int resident_bf16(Kind kind, int kd, int vd);
int resident_f16(Kind kind, int kd, int vd);

// One pass: with several segments the states before each are worked out first
// (into `segs`), unless `known`; then the outputs.
int forward_f32(const PassArgs& p, bool known, cudaStream_t s);
int forward_bf16(const PassArgs& p, bool known, cudaStream_t s);
int forward_f16(const PassArgs& p, bool known, cudaStream_t s);
int pair_f32(const PassArgs& p, cudaStream_t s);
int pair_bf16(const PassArgs& p, cudaStream_t s);
int pair_f16(const PassArgs& p, cudaStream_t s);
int step_f32(const PassArgs& p, cudaStream_t s);
int step_bf16(const PassArgs& p, cudaStream_t s);
int step_f16(const PassArgs& p, cudaStream_t s);

}  // namespace gfn_attn
