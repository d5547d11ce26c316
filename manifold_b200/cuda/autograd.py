"""Autograd functions of the single-head operators (the reference's
gfn/cuda/autograd.py: ChristoffelFusedFn, LeapfrogFusedFn).  Forward and
backward both run the library's kernels; the backward of the leapfrog is a
reverse replay that returns the gradients of every operand, the friction
gate's weights included."""
import torch
from torch.autograd import Function

from .._lib import first_order
from . import ops


class ChristoffelFusedFn(Function):
    """gfn/cuda/autograd.py:17-36."""

    @staticmethod
    def forward(ctx, v, U, W, x, V_w, plasticity, sing_thresh, sing_strength, topology, R, r):
        ctx.save_for_backward(v, U, W, x)
        ctx.args = (plasticity, sing_thresh, sing_strength, topology, R, r)
        return ops._christoffel_forward(v, U, W, x, V_w, plasticity, sing_thresh, sing_strength,
                                        topology, R, r)

    @staticmethod
    def backward(ctx, grad_gamma):
        v, U, W, x = ctx.saved_tensors
        gv, gU, gW, gx, _ = ops.christoffel_backward(grad_gamma.contiguous(), v, U, W, x, None, *ctx.args)
        return gv, gU, gW, gx, None, None, None, None, None, None, None


def christoffel_fused_autograd(v, U, W, x=None, V_w=None, plasticity=0.0, sing_thresh=1.0,
                               sing_strength=1.0, topology=0, R=2.0, r=1.0):
    return ChristoffelFusedFn.apply(v, U, W, x, V_w, plasticity, sing_thresh, sing_strength, topology,
                                    R, r)


class LeapfrogFusedFn(Function):
    """gfn/cuda/autograd.py:74-101, with the friction gate (Wf, bf), the input
    gate (Wi) and a tensor dt_scale differentiated too."""

    @staticmethod
    def forward(ctx, x, v, f, U, W, dt, dt_scale, steps, topology, Wf, bf, plasticity, R, r, Wi):
        ctx.save_for_backward(x, v, f, U, W, Wf, bf, Wi)
        ctx.args = (dt, dt_scale, steps, topology, R, r)
        return ops._leapfrog_forward(x, v, f, U, W, dt, dt_scale, steps, topology, Wf, bf, plasticity,
                                     R, r, Wi)

    @staticmethod
    def backward(ctx, grad_xn, grad_vn):
        x, v, f, U, W, Wf, bf, Wi = ctx.saved_tensors
        dt, dt_scale, steps, topology, R, r = ctx.args
        want_dt = isinstance(dt_scale, torch.Tensor) and ctx.needs_input_grad[6]
        dts = dt_scale.detach() if isinstance(dt_scale, torch.Tensor) else dt_scale
        out = ops.leapfrog_backward(grad_xn, grad_vn, x, v, f, U, W, dt, dts, steps, topology, R,
                                    r, Wf=Wf, bf=bf, Wi=Wi, want_dt=want_dt)
        gdt = None
        if want_dt:
            gdt = out.pop().reshape(dt_scale.shape).to(dt_scale.dtype)
        gx, gv, gf, gU, gW = out[:5]
        rest = out[5:]
        gWf = gbf = gWi = None
        if Wf is not None:
            gWf, gbf = rest[0], rest[1]
            rest = rest[2:]
            if bf is None:
                gbf = None
        if Wi is not None:
            gWi = rest[0]
        return (gx, gv, gf, gU, gW, None, gdt, None, None, gWf, gbf, None, None, None, gWi)


def leapfrog_fused_autograd(x, v, f, U, W, dt, dt_scale, steps, topology=0, Wf=None, bf=None,
                            plasticity=0.0, R=2.0, r=1.0, Wi=None):
    return LeapfrogFusedFn.apply(x, v, f, U, W, dt, dt_scale, steps, topology, Wf, bf, plasticity, R,
                                 r, Wi)


class LayerScanFn(Function):
    """The scan layer's recurrence (gfn/layers/parallel.py:101-121) with the
    gradients of its pre-activations and of the carried state (v0, x0)."""

    @staticmethod
    def forward(ctx, z, v0, x0, heads, base_dt, return_state):
        xs, vs, vl, xl, states = ops.layer_scan_forward(z, v0, x0, heads, base_dt, return_state, True)
        ctx.save_for_backward(z, states)
        ctx.args = (heads, base_dt)
        ctx.set_materialize_grads(False)
        return (xs, vs, vl, xl) if return_state else (xs, vs)

    @staticmethod
    @first_order
    def backward(ctx, gx, gv, gvl=None, gxl=None):
        if gx is None and gv is None and gvl is None and gxl is None:
            return None, None, None, None, None, None
        z, states = ctx.saved_tensors
        dz, dv0, dx0 = ops.layer_scan_backward(z, states, gx, gv, gvl, gxl, *ctx.args, ctx.needs_input_grad[1],
                                               ctx.needs_input_grad[2])
        return dz, dv0, dx0, None, None, None
