"""Linear attention with a decay for each head: the gated scan's recurrence
(scan.py, gfn/scan.py:11-104) with a matrix for a state.  CUDA tensors only."""
from ._lib import torch_ops


def decay_attention(q, k, v, decay, state=None, return_state=False, lengths=None, scale=1.0):
    """o_t = scale * q_t S_t with S_t = decay S_{t-1} + k_t^T v_t, for each sequence and head.

    q, k [batch, length, heads, kdim], v [batch, length, heads, vdim]: float32,
    bfloat16 or float16, dims up to 128, any strides with an inner one of 1 (views
    of one projection, [batch, heads, length, dim] transposed, and k or v expanded
    over the heads are read in place).  decay [heads] float32 in [0, 1], constant
    (a decay that wants a gradient is refused).  state [batch, heads, kdim, vdim]
    float32, or None (zero).  lengths [batch] int64 or int32: of a padded batch,
    the tokens of each sequence that count; the others are not read and get zeros.

    Returns o [batch, length, heads, vdim] of v's type, or (o, state behind the
    last token) with return_state: pass that as state to continue the sequence, one
    token at a time (a kernel of its own) or segment by segment.  Differentiable
    (once) in q, k, v and state.

    The state is float32 throughout.  Products run on the tensor cores: float32
    operands in two tf32 pieces each (2^-22 a product, results to 1e-6); of bfloat16 ones the scores and the state
    are rounded to bfloat16 where they are multiplied (not where they are kept), of
    float16 ones to tf32's 11 bits; the operands themselves are exact.  A NaN or an
    infinity reaches what the recurrence takes it to and nothing else; a sequence with
    one takes three to four times as long, with many up to 20 times.
    """
    return torch_ops().decay_attention(q, k, v, decay, state, lengths, scale, return_state)
