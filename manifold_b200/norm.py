"""Layer norm on the library's kernels, forward and backward.

The reference applies torch's nn.LayerNorm before the readout
(gfn/model.py:113,393) and inside every scan layer
(gfn/layers/parallel.py:27,90).  ``layer_norm`` and ``LayerNorm`` compute the
same function, y = (x - mean) / sqrt(var + eps) * weight + bias over the last
dimension, in float32 arithmetic on float32, bfloat16 or float16 tensors, and
return the gradients of x, weight and bias.  CUDA tensors only.
"""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import GfnError, call_on, dtype_code, ptr, same_device


def _rows(t, dim):
    """t as [rows, dim] with inner stride 1 (a view where one exists)."""
    t = t.reshape(-1, dim)
    return t if dim == 1 or t.stride(1) == 1 else t.contiguous()


def _row_stride(t, dim):
    return t.stride(0) if t.shape[0] > 1 else dim


def _forward(x, weight, bias, eps, want_stats):
    D = x.shape[-1]
    xr = _rows(x, D)
    if xr.shape[0] > 1 and xr.stride(0) < D:  # rows that overlap (an expanded input)
        xr = xr.contiguous()
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stats = torch.empty(xr.shape[0], 2, device=x.device, dtype=torch.float32) if want_stats else None
    w = weight if weight is not None else bias
    code = dtype_code(x, "x")
    call_on(x, "gfn_layer_norm_forward", ptr(xr), _row_stride(xr, D), ptr(weight), ptr(bias), code,
            code if w is None else dtype_code(w, "weight"), xr.shape[0], D, float(eps), ptr(y), ptr(stats))
    return y, xr, stats


class LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, xr, stats = _forward(x, weight, bias, eps, True)
        # the caller's own tensor where possible, so that a later in-place change of it is noticed
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_like = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        D = x.shape[-1]
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        xr, dr = _rows(x, D), _rows(dy, D)
        rows = xr.shape[0]
        if rows > 1 and xr.stride(0) < D:
            xr = xr.contiguous()
        if rows > 1 and dr.stride(0) < D:
            dr = dr.contiguous()
        wdt = weight.dtype if weight is not None else (ctx.bias_like or x.dtype)
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need_x else None
        dw = torch.empty(D, device=x.device, dtype=wdt) if need_w else None
        db = torch.empty(D, device=x.device, dtype=wdt) if need_b else None
        ws, n = None, 0
        if need_w or need_b:
            n = _lib.load().gfn_layer_norm_backward_workspace_floats(rows, D)
            ws = torch.empty(n, device=x.device, dtype=torch.float32)
        call_on(x, "gfn_layer_norm_backward", ptr(xr), _row_stride(xr, D), ptr(dr), _row_stride(dr, D),
                ptr(weight), ptr(stats), dtype_code(x, "x"), _lib.DTYPES[wdt], rows, D, ptr(dx), ptr(dw),
                ptr(db), ptr(ws), n)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x [..., dim] over its last dimension.

    x: float32, bfloat16 or float16, any strides (rows of a wider tensor are
    read in place when their inner stride is 1).  weight, bias [dim]: float32
    or x's type (both of one type), each optional.  Differentiable in x, weight
    and bias (once); the weight gradients are summed in float32 in a fixed
    order.  Returns a contiguous tensor of x's shape and type.
    """
    same_device("layer_norm", x, weight, bias)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise GfnError(f"layer_norm: x must have a last dimension of at least 1, got {tuple(x.shape)}")
    dtype_code(x, "x")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != (x.shape[-1],):
            raise GfnError(f"layer_norm: {name} must be [{x.shape[-1]}], got {tuple(t.shape)}")
        if t.dtype not in (torch.float32, x.dtype):
            raise GfnError(f"layer_norm: {name} must be float32 or {x.dtype}, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise GfnError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return LayerNormFn.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over one dimension (the same parameters and state_dict) on the kernels."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise GfnError("LayerNorm: one normalised dimension is implemented, got "
                           f"{tuple(self.normalized_shape)}")

    def forward(self, x):
        if x.shape[-1:] != tuple(self.normalized_shape):
            raise GfnError(f"LayerNorm: expected a last dimension of {self.normalized_shape[0]}, "
                           f"got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
