"""Linear attention with a decay for each head: the gated scan's recurrence
(scan.py, gfn/scan.py:11-104) with a matrix for a state.  CUDA tensors only."""
import torch

from ._lib import GfnError, dtype_code, same_device, torch_ops


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
    operands in two tf32 pieces each (2^-22), float16 ones exactly, and of bfloat16
    ones the scores and the state are rounded to bfloat16 where they are multiplied
    (not where they are kept).  Tokens are taken in blocks of up to 64, so that a
    NaN or infinity in k or v reaches the outputs of its block's earlier tokens too.
    """
    same_device("decay_attention", q, k, v, decay, state, lengths)
    dtype_code(q, "q")
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:3] != q.shape[:3]:
        raise GfnError("decay_attention: q, k must be [batch, length, heads, kdim] and v [batch, length, heads, vdim], "
                       f"got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise GfnError(f"decay_attention: q is {q.dtype}, k {k.dtype}, v {v.dtype}")
    B, L, H, K = q.shape
    V = v.shape[3]
    if not 0 < K <= 128 or not 0 < V <= 128:
        raise GfnError(f"decay_attention: head dims from 1 to 128 are implemented, got {K}, {V}")
    if decay.dtype != torch.float32 or decay.shape != (H,):
        raise GfnError(f"decay_attention: decay must be float32 [{H}], got {decay.dtype} {tuple(decay.shape)}")
    grad = torch.is_grad_enabled()
    if grad and decay.requires_grad:
        raise GfnError("decay_attention is not differentiable in decay: pass decay.detach()")
    if not decay.is_contiguous():
        decay = decay.contiguous()
    wants = q.requires_grad or k.requires_grad or v.requires_grad
    if state is not None:
        if state.dtype != torch.float32 or state.shape != (B, H, K, V):
            raise GfnError(f"decay_attention: state must be float32 {(B, H, K, V)}, got {state.dtype} "
                           f"{tuple(state.shape)}")
        wants = wants or state.requires_grad
    if lengths is not None:
        if lengths.shape != (B,) or (lengths.dtype != torch.int64 and lengths.dtype != torch.int32):
            raise GfnError(f"decay_attention: lengths must be int64 or int32 [{B}], got {lengths.dtype} "
                           f"{tuple(lengths.shape)}")
        if not lengths.is_contiguous():
            lengths = lengths.contiguous()
    if isinstance(scale, torch.Tensor):
        raise GfnError("decay_attention: scale must be a number")
    out = torch_ops().decay_attention(q, k, v, decay, state, lengths, scale, return_state, wants and grad)
    return out if return_state else out[0]
