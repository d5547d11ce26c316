"""gfn.scan mirror: y_t = a_t * y_{t-1} + x_t over dim 1 (gfn/scan.py:11-104),
as one work-efficient pass per column on the GPU (no Hillis-Steele passes),
and the gated scan: the same recurrence with gradients, a carried state and
16-bit operands."""
import torch

from ._lib import GfnError, dtype_code, same_device, torch_ops
from .cuda.ops import _grad_wanted, _has_tangent, parallel_scan_fused

CUDA_AVAILABLE = True


def parallel_scan(a, x):
    """a, x: [batch, seq_len, dim] float32 CUDA tensors -> y of the same shape.
    Differentiable.  With a gradient wanted it runs as gated_scan(a, x), and so
    it does where a has another shape than x (it is broadcast) or rows do not
    start on 16 bytes."""
    if _grad_wanted(a, x) or _has_tangent(a, x) or not _one_pass(a, x):
        if x.dtype != torch.float32:
            raise GfnError(f"x must be float32, got {x.dtype}")
        return gated_scan(a, x)
    return parallel_scan_fused(a, x)


def _one_pass(a, x):
    """Whether parallel_scan_fused takes the operands: one shape, whole and aligned rows of 4."""
    return (x.dim() == 3 and x.shape[2] % 4 == 0 and (a is None or a.shape == x.shape)
            and all(t is None or not t.is_contiguous() or t.data_ptr() % 16 == 0 for t in (a, x)))


def gated_scan(a, x, h0=None, return_state=False):
    """h_t = a_t * h_{t-1} + x_t over dim 1 of x [batch, length, dim], from h0.

    a: x's type, x's shape or broadcastable to it (a decay per channel is read
    in place, by the path of rows that do not start on 16 bytes; one whose last
    dimension is broadcast, per head or per step, is first copied to x's shape),
    or None (a running sum).  x: float32, bfloat16 or float16, any batch and step
    strides.  h0: [batch, dim] float32, or None (zero).  The state is float32
    throughout; h has x's type.  Returns h, or (h, last state [batch, dim]
    float32) with return_state: pass that as h0 to continue the sequence, one
    token at a time or segment by segment.  A gate of zero starts a new
    sequence, so packed sequences need no more than that.  Differentiable
    (once) in a, x and h0, a broadcast a included.

    The length axis is split: a state passes a whole run of steps as h * P + p.
    P, the product of the run's gates, has an exponent range of its own, so gates
    may decay and grow by any amounts for which h itself stays in float32's range.
    """
    same_device("gated_scan", x, a, h0)
    dtype_code(x, "x")
    if x.dim() != 3:
        raise GfnError(f"gated_scan: x must be [batch, length, dim], got {tuple(x.shape)}")
    wants = x.requires_grad
    if a is not None:
        if a.dtype != x.dtype:
            raise GfnError(f"gated_scan: a is {a.dtype}, x {x.dtype}")
        if a.shape != x.shape:
            try:
                a = a.expand(x.shape)
            except RuntimeError:
                raise GfnError(f"gated_scan: a {tuple(a.shape)} does not broadcast to {tuple(x.shape)}") from None
        wants = wants or a.requires_grad
    if h0 is not None:
        if h0.dtype != torch.float32 or h0.shape != (x.shape[0], x.shape[2]):
            raise GfnError(f"gated_scan: h0 must be float32 [{x.shape[0]}, {x.shape[2]}], got {h0.dtype} "
                           f"{tuple(h0.shape)}")
        wants = wants or h0.requires_grad
    out = torch_ops().gated_scan(a, x, h0, return_state, wants and torch.is_grad_enabled())
    return out if return_state else out[0]
