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

from . import _lib
from ._lib import GfnError, call_on, dtype_code, first_order, ptr, same_device


def _rows(t, dim):
    """(t or a copy of it, rows, row stride): rows of `dim` elements with inner
    stride 1, in place where t has them."""
    if t.is_contiguous():
        return t, t.numel() // dim, dim
    r = t.reshape(-1, dim)
    if (dim > 1 and r.stride(1) != 1) or (r.shape[0] > 1 and r.stride(0) < dim):  # rows that overlap are expanded ones
        r = r.contiguous()
    return r, r.shape[0], r.stride(0) if r.shape[0] > 1 else dim


def _forward(x, weight, bias, eps, want_stats):
    D = x.shape[-1]
    xr, rows, stride = _rows(x, D)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = x.new_empty((rows, 2), dtype=torch.float32) if want_stats else None
    w = weight if weight is not None else bias
    code = _lib.DTYPES[x.dtype]
    call_on(x, "gfn_layer_norm_forward", xr.data_ptr(), stride, ptr(weight), ptr(bias), code,
            code if w is None else _lib.DTYPES[w.dtype], rows, D, eps, y.data_ptr(), ptr(stats))
    return y, stats


class LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        # the caller's own tensor, so that a later in-place change of it is noticed
        ctx.save_for_backward(x, weight, stats)
        w = weight if weight is not None else bias
        ctx.wdt = x.dtype if w is None else w.dtype
        return y

    @staticmethod
    @first_order
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        D, wdt = x.shape[-1], ctx.wdt
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        xr, rows, xs = _rows(x, D)
        dr, _, ds = _rows(dy, D)
        dx = dw = db = ws = None
        n = 0
        if need_x:
            dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        if need_w:
            dw = x.new_empty(D, dtype=wdt)
        if need_b:
            db = x.new_empty(D, dtype=wdt)
        if need_w or need_b:
            n = _lib.load().gfn_layer_norm_backward_workspace_floats(rows, D)
            ws = x.new_empty(n, dtype=torch.float32)
        call_on(x, "gfn_layer_norm_backward", xr.data_ptr(), xs, dr.data_ptr(), ds, ptr(weight), stats.data_ptr(),
                _lib.DTYPES[x.dtype], _lib.DTYPES[wdt], rows, D, ptr(dx), ptr(dw), ptr(db), ptr(ws), n)
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
    grad = torch.is_grad_enabled()
    wants = grad and x.requires_grad
    if weight is not None:
        weight = _weight("weight", weight, x)
        wants = wants or (grad and weight.requires_grad)
    if bias is not None:
        bias = _weight("bias", bias, x)
        wants = wants or (grad and bias.requires_grad)
        if weight is not None and weight.dtype != bias.dtype:
            raise GfnError(f"layer_norm: weight is {weight.dtype}, bias {bias.dtype}")
    if wants:
        return LayerNormFn.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


def _weight(name, t, x):
    if t.dim() != 1 or t.shape[0] != x.shape[-1]:
        raise GfnError(f"layer_norm: {name} must be [{x.shape[-1]}], got {tuple(t.shape)}")
    if t.dtype != torch.float32 and t.dtype != x.dtype:
        raise GfnError(f"layer_norm: {name} must be float32 or {x.dtype}, got {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


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
