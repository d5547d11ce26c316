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

from ._lib import GfnError, dtype_code, same_device, torch_ops


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
    return torch_ops().layer_norm(x, weight, bias, eps, wants)


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
