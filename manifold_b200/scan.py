"""gfn.scan mirror: y_t = a_t * y_{t-1} + x_t over dim 1 (gfn/scan.py:11-104),
as one work-efficient pass per column on the GPU (no Hillis-Steele passes),
and the gated scan: the same recurrence with gradients, a carried state and
16-bit operands."""
import torch

from . import _lib
from ._lib import GfnError, call_on, dtype_code, first_order, ptr, same_device
from .cuda.ops import _grad_wanted, parallel_scan_fused

CUDA_AVAILABLE = True


def parallel_scan(a, x):
    """a, x: [batch, seq_len, dim] float32 CUDA tensors -> y of the same shape.
    Differentiable: with a gradient wanted it runs as gated_scan(a, x)."""
    if _grad_wanted(a, x):
        if x.dtype != torch.float32:
            raise GfnError(f"x must be float32, got {x.dtype}")
        return gated_scan(a, x)
    return parallel_scan_fused(a, x)


def _operand(t):
    """t [B, L, D] with inner stride 1 (itself where it has one: strided and
    broadcast batches and steps are read in place)."""
    return t if t.is_contiguous() or t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _workspace(x, B, L, D):
    n = _lib.load().gfn_gated_scan_workspace_bytes(B, L, D) if L > 1 else 0
    return (x.new_empty(n, dtype=torch.uint8) if n else None), n


def _forward(a, x, h0, want_last, want_states):
    B, L, D = x.shape
    x = _operand(x)
    h0 = None if h0 is None else h0.contiguous()
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    last = x.new_empty((B, D), dtype=torch.float32) if want_last else None
    states = None
    if want_states:
        states = x.new_empty(_lib.load().gfn_gated_scan_states_floats(B, L, D), dtype=torch.float32)
    ws, n = _workspace(x, B, L, D)
    pa = sa = ta = 0
    if a is not None:
        a = _operand(a)
        pa, (sa, ta, _) = a.data_ptr(), a.stride()
    sx, tx, _ = x.stride()
    call_on(x, "gfn_gated_scan_forward", pa, sa, ta, x.data_ptr(), sx, tx, ptr(h0), _lib.DTYPES[x.dtype], B, L, D,
            h.data_ptr(), ptr(last), ptr(states), ptr(ws), n)
    return h, last, states


class GatedScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, x, h0, return_state):
        h, last, states = _forward(a, x, h0, return_state, True)
        ctx.save_for_backward(a, x, states)
        ctx.set_materialize_grads(False)
        return (h, last) if return_state else h

    @staticmethod
    @first_order
    def backward(ctx, dh, dlast=None):
        a, x, states = ctx.saved_tensors
        if dh is None and dlast is None:
            return None, None, None, None
        B, L, D = x.shape
        need_a, need_x, need_h0, _ = ctx.needs_input_grad
        x = _operand(x)
        dlast = None if dlast is None else dlast.contiguous()
        da = torch.empty_like(x, memory_format=torch.contiguous_format) if need_a else None
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
        dh0 = x.new_empty((B, D), dtype=torch.float32) if need_h0 else None
        ws, n = _workspace(x, B, L, D)
        pa = sa = ta = pg = sg = tg = 0
        if a is not None:
            a = _operand(a)
            pa, (sa, ta, _) = a.data_ptr(), a.stride()
        if dh is not None:
            dh = _operand(dh)
            pg, (sg, tg, _) = dh.data_ptr(), dh.stride()
        sx, tx, _ = x.stride()
        call_on(x, "gfn_gated_scan_backward", pa, sa, ta, x.data_ptr(), sx, tx, states.data_ptr(), pg, sg, tg,
                ptr(dlast), _lib.DTYPES[x.dtype], B, L, D, ptr(da), ptr(dx), ptr(dh0), ptr(ws), n)
        return da, dx, dh0, None


def gated_scan(a, x, h0=None, return_state=False):
    """h_t = a_t * h_{t-1} + x_t over dim 1 of x [batch, length, dim], from h0.

    a: x's type, x's shape or broadcastable to it (a decay per channel, per
    head or per step is read in place where its last dimension is whole), or
    None (a running sum).  x: float32, bfloat16 or float16, any batch and step
    strides.  h0: [batch, dim] float32, or None (zero).  The state is float32
    throughout; h has x's type.  Returns h, or (h, last state [batch, dim]
    float32) with return_state: pass that as h0 to continue the sequence, one
    token at a time or segment by segment.  A gate of zero starts a new
    sequence, so packed sequences need no more than that.  Differentiable
    (once) in a, x and h0, a broadcast a included.

    The length axis is split: a state passes a whole run of steps as h * P + p,
    P the product of the run's gates, so |P| must not overflow (gates up to
    1 in magnitude never do).
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
    if wants and torch.is_grad_enabled():
        return GatedScanFn.apply(a, x, h0, return_state)
    h, last, _ = _forward(a, x, h0, return_state, False)
    return (h, last) if return_state else h
