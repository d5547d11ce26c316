"""Operator boundary: the reference's ``gfn.cuda.ops`` entry points on the
B200 kernels (through the C ABI of include/gfn_b200.h).

Names, arguments and return values follow gfn/cuda/ops.py.  There is no
Python fallback: CPU tensors and unsupported options raise ``GfnError``.
"""
import torch

from .. import _lib
from .._lib import GfnError, call, ptr, require_cuda

CUDA_AVAILABLE = True  # the library is required; import fails loudly otherwise


def _f32c(t, name):
    if t is None:
        return None
    if t.dtype != torch.float32:
        raise GfnError(f"{name} must be float32, got {t.dtype}")
    return t.contiguous()


def _stream(t):
    return _lib.stream_of(t.device)


def _grad_wanted(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _has_tangent(*ts):
    """Whether one carries a forward-mode tangent (torch.autograd.forward_ad), which the kernels would drop."""
    return any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in ts)


def christoffel_fused(v, U, W, x=None, V_w=None, plasticity=0.0, sing_thresh=1.0,
                      sing_strength=1.0, topology=0, R=2.0, r=1.0):
    """Gamma(v) for one head (gfn/cuda/ops.py:88-118).  topology 0: the low-rank
    form (gfn/geometry/lowrank.py:93-98,125-127); topology 1: the toroidal form
    (gfn/geometry/toroidal.py:70-108, needs x).  Differentiable when an input
    requires grad (backward: christoffel_backward)."""
    if _grad_wanted(v, U, W, x):
        from .autograd import christoffel_fused_autograd
        return christoffel_fused_autograd(v, U, W, x, V_w, plasticity, sing_thresh, sing_strength,
                                          topology, R, r)
    return _christoffel_forward(v, U, W, x, V_w, plasticity, sing_thresh, sing_strength, topology, R, r)


def _christoffel_forward(v, U, W, x, V_w, plasticity, sing_thresh, sing_strength, topology, R, r):
    require_cuda(v, U, W, x)
    v = _f32c(v, "v")
    gamma = torch.empty_like(v)
    if topology == 1:
        if x is None:
            raise GfnError("christoffel_fused: the toroidal form needs x")
        if V_w is not None or plasticity != 0.0:
            raise GfnError("christoffel_fused: active inference is not implemented on this build")
        x = _f32c(x, "x")
        call("gfn_christoffel_torus", ptr(v), ptr(x), ptr(gamma), v.shape[0], v.shape[1], float(R),
             float(r), _stream(v))
        return gamma
    U, W = _f32c(U, "U"), _f32c(W, "W")
    call("gfn_christoffel_fused", ptr(v), ptr(U), ptr(W), ptr(gamma), None,
         ptr(V_w) if V_w is not None else None, v.shape[0], v.shape[1], U.shape[1],
         float(plasticity), float(sing_thresh), float(sing_strength), int(topology), float(R),
         float(r), _stream(v))
    return gamma


def reactive_christoffel(v, U, W, x=None, V_w=None, plasticity=0.0, sing_thresh=1.0,
                         sing_strength=1.0, topology=0, R=2.0, r=1.0):
    """gfn/cuda/ops.py:120-129: the reactive geometry.  With plasticity 0 and
    no singularity potential (active inference off) it is christoffel_fused;
    the active-inference terms raise."""
    if plasticity != 0.0 or V_w is not None:
        raise GfnError("reactive_christoffel: plasticity / singularities are not implemented on this build")
    return christoffel_fused(v, U, W, x, None, 0.0, sing_thresh, sing_strength, topology, R, r)


def christoffel_backward(grad_gamma, v, U, W, x=None, V_w=None, plasticity=0.0, sing_thresh=1.0,
                         sing_strength=1.0, topology=0, R=2.0, r=1.0):
    """Backward of christoffel_fused (the gfn_cuda.christoffel_backward binding,
    gfn/cuda/cuda_kernels.cpp:139-148).  Returns [grad_v, grad_U, grad_W,
    grad_x, grad_V_w]; grad_x is None without x, grad_V_w always None."""
    require_cuda(grad_gamma, v, U, W, x)
    gg, v = _f32c(grad_gamma, "grad_gamma"), _f32c(v, "v")
    B, d = v.shape
    dev = v.device
    grad_v = torch.empty_like(v)
    grad_x = torch.empty_like(v) if x is not None else None
    if topology == 1:
        if x is None:
            raise GfnError("christoffel_backward: the toroidal form needs x")
        x = _f32c(x, "x")
        call("gfn_christoffel_backward", ptr(gg), ptr(v), None, None, ptr(x), None, ptr(grad_v), None,
             None, ptr(grad_x), None, B, d, 4, float(plasticity), float(sing_thresh),
             float(sing_strength), 1, float(R), float(r), None, 0, _stream(v))
        gU = torch.zeros_like(U) if U is not None else None
        gW = torch.zeros_like(W) if W is not None else None
        return [grad_v, gU, gW, grad_x, None]
    U, W = _f32c(U, "U"), _f32c(W, "W")
    rank = U.shape[1]
    grad_U = torch.empty_like(U)
    grad_W = torch.empty_like(W)
    n = _lib.load().gfn_christoffel_backward_workspace_floats(B, d, rank)
    ws = torch.empty(max(int(n), 1), device=dev, dtype=torch.float32)
    call("gfn_christoffel_backward", ptr(gg), ptr(v), ptr(U), ptr(W), ptr(x), ptr(V_w), ptr(grad_v),
         ptr(grad_U), ptr(grad_W), ptr(grad_x), None, B, d, rank, float(plasticity), float(sing_thresh),
         float(sing_strength), 0, float(R), float(r), ptr(ws), ws.numel(), _stream(v))
    return [grad_v, grad_U, grad_W, grad_x, None]


def _dt_scales(dt_scale, x):
    if not isinstance(dt_scale, torch.Tensor):
        dt_scale = torch.tensor([float(dt_scale)], device=x.device, dtype=torch.float32)
    return dt_scale.reshape(-1).to(device=x.device, dtype=torch.float32).contiguous()


def leapfrog_fused(x, v, f, U, W, dt, dt_scale, steps, topology=0, Wf=None, bf=None,
                   plasticity=0.0, R=2.0, r=1.0, Wi=None):
    """One head's leapfrog, `steps` times (gfn/cuda/ops.py:131-182;
    gfn/integrators/symplectic/leapfrog.py:50-114).  Returns (x_new, v_new).

    Wi (an addition to the reference signature): the input gate, friction
    mu = 5 sigmoid(x Wf^T + bf + f Wi^T) (gfn/geometry/lowrank.py:114-123).
    topology 1: the toroidal step (Wf [hd, 2 hd] over [sin x, cos x], x wrapped
    into [0, 2 pi)).  Differentiable when an input requires grad."""
    if _grad_wanted(x, v, f, U, W, Wf, bf, Wi):
        from .autograd import leapfrog_fused_autograd
        return leapfrog_fused_autograd(x, v, f, U, W, dt, dt_scale, steps, topology, Wf, bf,
                                       plasticity, R, r, Wi)
    return _leapfrog_forward(x, v, f, U, W, dt, dt_scale, steps, topology, Wf, bf, plasticity, R, r, Wi)


def _leapfrog_forward(x, v, f, U, W, dt, dt_scale, steps, topology, Wf, bf, plasticity, R, r, Wi):
    require_cuda(x, v, f, U, W, Wf, bf, Wi)
    x, v = _f32c(x, "x"), _f32c(v, "v")
    f, Wf, bf, Wi = _f32c(f, "f"), _f32c(Wf, "Wf"), _f32c(bf, "bf"), _f32c(Wi, "Wi")
    U = _f32c(U, "U") if U is not None else None
    W = _f32c(W, "W") if W is not None else None
    dts = _dt_scales(dt_scale, x)
    x_new = torch.empty_like(x)
    v_new = torch.empty_like(v)
    if Wi is not None or topology == 1:
        rank = U.shape[1] if U is not None else 4
        call("gfn_leapfrog_fused_gated", ptr(x), ptr(v), ptr(f), ptr(U), ptr(W), ptr(Wf), ptr(bf),
             ptr(Wi), ptr(x_new), ptr(v_new), float(dt), ptr(dts), dts.numel(), x.shape[0],
             x.shape[1], rank, int(steps), int(topology), float(plasticity), float(R), float(r),
             _stream(x))
        return x_new, v_new
    call("gfn_leapfrog_fused", ptr(x), ptr(v), ptr(f), ptr(U), ptr(W), ptr(Wf), ptr(bf),
         ptr(x_new), ptr(v_new), float(dt), ptr(dts), dts.numel(), x.shape[0], x.shape[1],
         U.shape[1], int(steps), int(topology), float(plasticity), float(R), float(r), _stream(x))
    return x_new, v_new


def leapfrog_backward(grad_x_new, grad_v_new, x, v, f, U, W, dt, dt_scale, steps, topology=0,
                      R=2.0, r=1.0, Wf=None, bf=None, Wi=None, want_dt=False):
    """Backward of leapfrog_fused (the gfn_cuda.leapfrog_backward binding,
    gfn/cuda/cuda_kernels.cpp:190-196), by reverse replay.  Returns
    [grad_x, grad_v, grad_f, grad_U, grad_W], followed by grad_Wf, grad_bf
    when Wf is given, grad_Wi when Wi is given, and (want_dt) the gradient of
    dt_scale in its own shape (one value or one per row)."""
    require_cuda(x, v, f, U, W, Wf, bf, Wi, grad_x_new, grad_v_new)
    x, v = _f32c(x, "x"), _f32c(v, "v")
    f, Wf, bf, Wi = _f32c(f, "f"), _f32c(Wf, "Wf"), _f32c(bf, "bf"), _f32c(Wi, "Wi")
    gxn = _f32c(grad_x_new, "grad_x_new") if grad_x_new is not None else None
    gvn = _f32c(grad_v_new, "grad_v_new") if grad_v_new is not None else None
    B, d = x.shape
    dev = x.device
    if topology == 0:
        U, W = _f32c(U, "U"), _f32c(W, "W")
        rank = U.shape[1]
    else:
        rank = 4
    fin = 2 * d if topology == 1 else d
    if Wf is not None and bf is None:
        bf = torch.zeros(d, device=dev, dtype=torch.float32)
    dts = _dt_scales(dt_scale, x)
    gx, gv = torch.empty_like(x), torch.empty_like(v)
    gf = torch.empty_like(x) if f is not None else None
    gU = torch.empty_like(U) if topology == 0 else None
    gW = torch.empty_like(W) if topology == 0 else None
    gWf = torch.empty(d, fin, device=dev, dtype=torch.float32) if Wf is not None else None
    gbf = torch.empty(d, device=dev, dtype=torch.float32) if Wf is not None else None
    gWi = torch.empty(d, d, device=dev, dtype=torch.float32) if Wi is not None else None
    n = _lib.load().gfn_leapfrog_step_backward_workspace_floats(B, d, rank, int(steps), int(topology))
    ws = torch.empty(max(int(n), 1), device=dev, dtype=torch.float32)
    gdt = torch.empty(B, device=dev, dtype=torch.float32) if want_dt else None
    call("gfn_leapfrog_backward", ptr(gxn), ptr(gvn), ptr(x), ptr(v), ptr(f), ptr(U), ptr(W), ptr(Wf),
         ptr(bf), ptr(Wi), ptr(gx), ptr(gv), ptr(gf), ptr(gU), ptr(gW), ptr(gWf), ptr(gbf), ptr(gWi),
         ptr(gdt), B, d, rank, float(dt), ptr(dts), dts.numel(), int(steps), int(topology), float(R), float(r),
         ptr(ws), ws.numel(), _stream(x))
    out = [gx, gv, gf, gU, gW]
    if Wf is not None:
        out += [gWf, gbf]
    if Wi is not None:
        out.append(gWi)
    if want_dt:
        out.append(gdt.sum().reshape(1) if dts.numel() == 1 else gdt)
    return out


def leapfrog_pack(U_stack, W_stack, Wf_stack, bf_stack, dt_params, mix=None):
    """Pack stacked layer parameters for leapfrog_sequence.

    U_stack/W_stack [NL*H, hd, r], Wf_stack [NL*H, hd, hd], bf_stack
    [NL*H, hd], dt_params [NL*H]; mix = (Wx, bx, gx, Wv, bv, gv) with
    Wx/Wv [NL, d, d] and the rest [NL, d], or None when heads == 1.
    """
    NLH, hd, r = U_stack.shape
    dev = U_stack.device
    args = [_f32c(t, "stack") for t in (U_stack, W_stack, Wf_stack, bf_stack, dt_params)]
    if mix is not None:
        Wx = _f32c(mix[0], "Wx")
        num_layers, d, _ = Wx.shape
        heads = d // hd
        mix = [_f32c(t, "mix") for t in mix]
    else:
        heads = 1
        num_layers = NLH
        d = hd
        mix = [None] * 6
    n = _lib.load().gfn_leapfrog_pack_floats(d, heads, r, num_layers)
    if n < 0:
        call("gfn_leapfrog_pack_floats", d, heads, r, num_layers)  # raises with the message
    packed = torch.empty(int(n), device=dev, dtype=torch.float32)
    call("gfn_leapfrog_pack", *[ptr(t) for t in args], ptr(mix[0]), ptr(mix[1]), ptr(mix[2]),
         ptr(mix[3]), ptr(mix[4]), ptr(mix[5]), d, heads, r, num_layers, ptr(packed), packed.numel(),
         _lib.stream_of(dev))
    return packed, dict(dim=d, heads=heads, rank=r, num_layers=num_layers)


def leapfrog_sequence(x0, v0, packed, meta, base_dt, forces=None, ids=None, table=None,
                      mask=None, want_x_seq=True, want_v_seq=True):
    """Whole-sequence fused leapfrog recurrence over all layers.

    x0/v0: [B, d] or [1, d] / [d] (broadcast).  Exactly one of forces
    ([B, L, d] float32 or bfloat16) or ids ([B, L] int64) + table ([V, d]).
    Returns (x_seq, v_seq, x_final, v_final); x_seq/v_seq None if not wanted.
    """
    require_cuda(x0, v0, packed, forces, ids, table, mask)
    d = meta["dim"]
    x0 = _f32c(x0, "x0")
    v0 = _f32c(v0, "v0")
    if forces is not None:
        B, L, _ = forces.shape
        forces = forces.contiguous()
    elif ids is not None:
        B, L = ids.shape
        ids = ids.to(torch.int64).contiguous()
        table = _f32c(table, "table")
    else:
        raise GfnError("leapfrog_sequence needs forces or ids")
    if x0.dim() == 1 or x0.shape[0] == 1:
        stride = 0
        if B > 1 and (v0.dim() != 1 and v0.shape[0] != 1):
            raise GfnError("x0 and v0 must both broadcast or both be [B, d]")
    else:
        if x0.shape != (B, d) or v0.shape != (B, d):
            raise GfnError(f"state must be [B={B}, d={d}]")
        stride = d
    dev = x0.device
    x_seq = torch.empty(B, L, d, device=dev, dtype=torch.float32) if want_x_seq else None
    v_seq = torch.empty(B, L, d, device=dev, dtype=torch.float32) if want_v_seq else None
    x_f = torch.empty(B, d, device=dev, dtype=torch.float32)
    v_f = torch.empty(B, d, device=dev, dtype=torch.float32)
    f32 = forces if (forces is not None and forces.dtype == torch.float32) else None
    fbf = forces if (forces is not None and forces.dtype == torch.bfloat16) else None
    if forces is not None and f32 is None and fbf is None:
        raise GfnError(f"forces must be float32 or bfloat16, got {forces.dtype}")
    if mask is not None:
        mask = mask.to(torch.float32).contiguous()
    call("gfn_leapfrog_sequence_forward", ptr(x0), ptr(v0), stride, ptr(f32), ptr(fbf), ptr(ids),
         ptr(table), table.shape[0] if table is not None else 0, ptr(mask), ptr(packed),
         packed.numel(), B, L, d, meta["heads"], meta["rank"], meta["num_layers"],
         float(base_dt), ptr(x_seq), ptr(v_seq), ptr(x_f), ptr(v_f), _lib.stream_of(dev))
    return x_seq, v_seq, x_f, v_f


def leapfrog_layered_pack(U_stack, W_stack, Wf_stack, bf_stack, dt_params, mix):
    """Pack stacked layer parameters for leapfrog_layered_sequence (heads > 1).

    Same operands as leapfrog_pack; the layout keeps each head's weights
    contiguous and the mixing matrices [out][in] for the batched GEMM.
    """
    NLH, hd, r = U_stack.shape
    dev = U_stack.device
    args = [_f32c(t, "stack") for t in (U_stack, W_stack, Wf_stack, bf_stack, dt_params)]
    if mix is None:
        raise GfnError("the layered path needs head mixing (heads > 1)")
    mix = [_f32c(t, "mix") for t in mix]
    num_layers, d, _ = mix[0].shape
    heads = d // hd
    n = _lib.load().gfn_leapfrog_layered_pack_floats(d, heads, r, num_layers)
    if n < 0:
        raise GfnError(f"layered pack: unsupported shape d={d} heads={heads} rank={r}")
    packed = torch.empty(int(n), device=dev, dtype=torch.float32)
    call("gfn_leapfrog_layered_pack", *[ptr(t) for t in args], *[ptr(t) for t in mix], d, heads, r,
         num_layers, ptr(packed), packed.numel(), _lib.stream_of(dev))
    return packed, dict(dim=d, heads=heads, rank=r, num_layers=num_layers, layered=True)


def leapfrog_layered_sequence(x0, v0, packed, meta, base_dt, forces=None, ids=None, table=None,
                              mask=None, want_x_seq=True, want_v_seq=True, workspace=None):
    """leapfrog_sequence computed layer by layer (head step kernel + fp32
    cuBLAS mixing GEMM per layer); the choice for large batches."""
    require_cuda(x0, v0, packed, forces, ids, table, mask)
    d = meta["dim"]
    x0 = _f32c(x0, "x0")
    v0 = _f32c(v0, "v0")
    if forces is not None:
        B, L, _ = forces.shape
        forces = forces.contiguous()
    elif ids is not None:
        B, L = ids.shape
        ids = ids.to(torch.int64).contiguous()
        table = _f32c(table, "table")
    else:
        raise GfnError("leapfrog_layered_sequence needs forces or ids")
    if x0.dim() == 1 or x0.shape[0] == 1:
        stride = 0
    else:
        if x0.shape != (B, d) or v0.shape != (B, d):
            raise GfnError(f"state must be [B={B}, d={d}]")
        stride = d
    dev = x0.device
    x_seq = torch.empty(B, L, d, device=dev, dtype=torch.float32) if want_x_seq else None
    v_seq = torch.empty(B, L, d, device=dev, dtype=torch.float32) if want_v_seq else None
    x_f = torch.empty(B, d, device=dev, dtype=torch.float32)
    v_f = torch.empty(B, d, device=dev, dtype=torch.float32)
    f32 = forces if (forces is not None and forces.dtype == torch.float32) else None
    fbf = forces if (forces is not None and forces.dtype == torch.bfloat16) else None
    if forces is not None and f32 is None and fbf is None:
        raise GfnError(f"forces must be float32 or bfloat16, got {forces.dtype}")
    if mask is not None:
        mask = mask.to(torch.float32).contiguous()
    nws = _lib.load().gfn_leapfrog_layered_workspace_floats(B, d)
    if workspace is None or workspace.numel() < nws:
        workspace = torch.empty(int(nws), device=dev, dtype=torch.float32)
    call("gfn_leapfrog_layered_forward", ptr(x0), ptr(v0), stride, ptr(f32), ptr(fbf), ptr(ids),
         ptr(table), table.shape[0] if table is not None else 0, ptr(mask), ptr(packed),
         packed.numel(), B, L, d, meta["heads"], meta["rank"], meta["num_layers"],
         float(base_dt), ptr(x_seq), ptr(v_seq), ptr(x_f), ptr(v_f), ptr(workspace),
         workspace.numel(), _lib.stream_of(dev))
    return x_seq, v_seq, x_f, v_f


def recurrent_manifold_fused(x, v, f, U_stack, W_stack, dt, dt_scales, forget_rates, num_heads,
                             plasticity=0.0, sing_thresh=1.0, sing_strength=1.0,
                             mix_x=None, mix_v=None, Wf=None, Wi=None, bf=None,
                             Wp=None, bp=None, topology=0, R=2.0, r=1.0):
    """Whole-sequence recurrence with the reference's stacked operands
    (gfn/cuda/ops.py:224-236, arguments as gfn/model.py:222-375 builds them).
    Returns (x_final, v_final, x_seq, reg_loss).

    The reference sends leapfrog models to its per-token loop instead
    (gfn/model.py:207), so this entry computes that loop's leapfrog MLayer
    recurrence (gfn/layers/base.py:198-338) on the library's fused sequence
    kernel, for the operands given here:
      x, v [B, d]; f [B, L, d]; U_stack / W_stack [NL*H, hd, r];
      Wf [NL*H, hd, hd] and bf [NL*H, hd] (friction; None: no friction);
      dt_scales [H]: softplus(dt_params) of the first layer, used by every
      layer (as the reference's dispatch passes it);
      mix_x / mix_v: [d, d] (one matrix for every layer, as the reference
      passes layer 0's) or [NL, d, d]; the mixing biases are 0 and the
      RMSNorm gains 1, since the reference's argument list carries neither.
    forget_rates and Wi are accepted and unused (the leapfrog friction reads
    the forget stack only, gfn/integrators/symplectic/leapfrog.py:72-81);
    reg_loss is 0.  Active inference (plasticity, singularities) and the
    torus raise.  Inference only (no autograd)."""
    require_cuda(x, v, f, U_stack, W_stack, Wf, bf, mix_x, mix_v)
    if plasticity != 0.0 or sing_strength != 1.0 or topology != 0:
        raise GfnError("recurrent_manifold_fused: only the Euclidean leapfrog without active inference")
    if Wp is not None and bool((Wp != 0).any()):
        raise GfnError("recurrent_manifold_fused: singularity potentials are not implemented")
    H = int(num_heads)
    NLH, hd, rank = U_stack.shape
    NL = NLH // H
    d = hd * H
    dev = x.device
    if Wf is None:
        # no friction: sigmoid(-inf) = 0 through a bias far below the gate's range
        Wf = torch.zeros(NLH, hd, hd, device=dev, dtype=torch.float32)
        bf = torch.full((NLH, hd), -1e30, device=dev, dtype=torch.float32)
    elif bf is None:
        bf = torch.zeros(NLH, hd, device=dev, dtype=torch.float32)
    if not isinstance(dt_scales, torch.Tensor):
        dt_scales = torch.full((H,), float(dt_scales), device=dev, dtype=torch.float32)
    s = dt_scales.reshape(-1).to(device=dev, dtype=torch.float32)
    if s.numel() == 1:
        s = s.expand(H)
    # dt_params whose softplus is the given scale (the pack applies softplus)
    dtp = torch.where(s > 20.0, s, torch.log(torch.expm1(s.double())).float())
    dt_params = dtp.repeat(NL).contiguous()
    mix = None
    if H > 1:
        if mix_x is None or mix_v is None or mix_x.numel() == 0:
            raise GfnError("recurrent_manifold_fused: heads > 1 needs mix_x and mix_v")
        mx = mix_x.reshape(-1, d, d).expand(NL, d, d).contiguous()
        mv = mix_v.reshape(-1, d, d).expand(NL, d, d).contiguous()
        zeros = torch.zeros(NL, d, device=dev, dtype=torch.float32)
        ones = torch.ones(NL, d, device=dev, dtype=torch.float32)
        mix = (mx, zeros, ones, mv, zeros, ones)
    packed, meta = leapfrog_pack(U_stack, W_stack, Wf.reshape(NLH, hd, hd), bf.reshape(NLH, hd),
                                 dt_params, mix)
    with torch.no_grad():
        x_seq, _, xf, vf = leapfrog_sequence(x, v, packed, meta, float(dt), forces=f, want_v_seq=False)
    reg_loss = torch.zeros((), device=dev, dtype=torch.float32)
    return xf, vf, x_seq, reg_loss


MIX_SPLIT_BF16, MIX_FP32_SIMT, MIX_SPLIT_F16, MIX_UMMA_F16 = 0, 1, 2, 3


def set_layered_mixing(mode):
    """Mixing-GEMM arithmetic of the layered path: MIX_UMMA_F16 (default; the
    two-piece fp16 split computed by the library's own tcgen05 kernel, three
    MMAs per K step), MIX_SPLIT_F16 (the same split as one cuBLAS GEMM,
    K = 3 dim; both need activations below 2^15), MIX_SPLIT_BF16 (three-piece bf16 split, K = 6 dim, full fp32 range)
    or MIX_FP32_SIMT (fp32 SGEMM).  Returns the previous mode."""
    prev = _lib.load().gfn_leapfrog_layered_set_mixing(int(mode))
    if prev < 0:
        _lib.check(-prev, "gfn_leapfrog_layered_set_mixing")
    return prev


def get_layered_mixing():
    return _lib.load().gfn_leapfrog_layered_set_mixing(-1)


def leapfrog_plan(batch, dim, heads, rank, num_layers):
    import ctypes
    out = (ctypes.c_int * 8)()
    call("gfn_leapfrog_plan", batch, dim, heads, rank, num_layers, out)
    return dict(cluster=out[0], rows_per_cluster=out[1], clusters=out[2], smem=out[3],
                k_chunk=out[4], ring=out[5], max_active_clusters=out[6], k_split=out[7])


def parallel_scan_fused(a, x, workspace=True):
    """y_t = a_t y_{t-1} + x_t over dim 1 of [B, L, D] (gfn/scan.py:11-104).
    a None means a == 1."""
    require_cuda(a, x)
    x = _f32c(x, "x")
    a = _f32c(a, "a")
    if x.dim() != 3 or (a is not None and a.numel() != x.numel()):
        raise GfnError(f"parallel_scan_fused: a {None if a is None else tuple(a.shape)} and x {tuple(x.shape)} must "
                       "be [batch, length, dim]")
    B, L, D = x.shape
    y = torch.empty_like(x)
    ws = None
    if workspace:
        n = _lib.load().gfn_parallel_scan_workspace_floats(B, L, D)
        ws = torch.empty(int(n), device=x.device, dtype=torch.float32)
    call("gfn_parallel_scan", ptr(a), ptr(x), ptr(y), ptr(ws), ws.numel() if ws is not None else 0,
         B, L, D, _stream(x))
    return y


def parallel_layer_scan(z, heads, base_dt=0.1, state=None, return_state=False):
    """ParallelMLayer recurrence from z = [zA | zdt | zB] ([B, L, 3D]).
    Returns (x_seq, v_seq).

    state: (v, x), each [B, D] float32, where the sequence continues from
    (None: zero); with return_state the result is (x_seq, v_seq, (v, x)), the
    state after the last step.  Differentiable in z and the state.  Calls with
    a state, return_state or a gradient split the length axis when the columns
    alone do not fill the GPU; so do those whose rows do not start on 16 bytes,
    as the one-pass kernel of the others needs it."""
    require_cuda(z)
    if state is not None or return_state or _grad_wanted(z) or _has_tangent(z) or z.dim() != 3 or z.shape[2] % 12:
        return _layer_scan(z, heads, base_dt, state, return_state)
    z = _f32c(z, "z")
    if z.data_ptr() % 16:
        return _layer_scan(z, heads, base_dt, state, return_state)
    B, L, D3 = z.shape
    D = D3 // 3
    x_seq = torch.empty(B, L, D, device=z.device, dtype=torch.float32)
    v_seq = torch.empty_like(x_seq)
    call("gfn_parallel_layer_scan", ptr(z), ptr(x_seq), ptr(v_seq), B, L, D, int(heads),
         float(base_dt), _stream(z))
    return x_seq, v_seq


def _layer_scan(z, heads, base_dt, state, return_state):
    v0, x0 = (None, None) if state is None else state
    _lib.same_device("parallel_layer_scan", z, v0, x0)
    z = _f32c(z, "z")
    if z.dim() != 3 or z.shape[2] % 3:
        raise GfnError(f"parallel_layer_scan: z must be [batch, length, 3 dim], got {tuple(z.shape)}")
    for name, t in (("v", v0), ("x", x0)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (z.shape[0], z.shape[2] // 3)):
            raise GfnError(f"parallel_layer_scan: state {name} must be float32 [{z.shape[0]}, {z.shape[2] // 3}], "
                           f"got {t.dtype} {tuple(t.shape)}")
    out = _lib.torch_ops().layer_scan(z, v0, x0, int(heads), float(base_dt), return_state, _grad_wanted(z, v0, x0))
    return (out[0], out[1], (out[2], out[3])) if return_state else out


def functional_embedding(ids, W0, b0, W1, b1, W2, b2, Wo, bo, impulse, omega0=30.0,
                         out_dtype=torch.float32):
    """FunctionalEmbedding(mode='binary') forward (gfn/embeddings.py:171-206)."""
    require_cuda(ids, Wo)
    ids = ids.to(torch.int64).contiguous()
    ws = [_f32c(t, "siren weight") for t in (W0, b0, W1, b1, W2, b2, Wo, bo)]
    imp = _f32c(impulse.reshape(1), "impulse")
    d = Wo.shape[0]
    out = torch.empty(*ids.shape, d, device=ids.device, dtype=out_dtype)
    f32 = out if out_dtype == torch.float32 else None
    bf = out if out_dtype == torch.bfloat16 else None
    if f32 is None and bf is None:
        raise GfnError("functional_embedding: out_dtype must be float32 or bfloat16")
    call("gfn_functional_embedding", ptr(ids), ids.numel(), *[ptr(t) for t in ws], ptr(imp),
         float(omega0), d, ptr(f32), ptr(bf), _stream(ids))
    return out


def device_error(reset=True):
    return _lib.device_error(reset)


SCHEMES = {"euler": 0, "heun": 1, "rk4": 2, "verlet": 3, "yoshida": 4, "forest_ruth": 5,
           "omelyan": 6, "dormand_prince": 7, "rk45": 7, "leapfrog": 8}


def integrator_heads(scheme, x, v, f, U, W, dt, dt_scale, steps=1, topology=0, Wf=None, bf=None,
                     Wi=None, heads=1, R=2.0, r=1.0, plasticity=0.0, V=None, V_bias=None,
                     singularity=0, sing_thresh=1.0, sing_strength=1.0):
    """One launch of integrator `scheme` (a SCHEMES name or id) over every head.

    x, v, f: [B, heads * hd]; U, W: [heads, hd, rank] (or [hd, rank] for one
    head; unused on the torus); Wf [heads, hd, fin], bf [heads, hd], Wi
    [heads, hd, hd] (the friction gate, optional); dt_scale: a number, one
    value per head (heads > 1), per row (heads == 1) or [B, heads].  Active
    inference: plasticity, and singularity 1 (soft) / 2 (hard) with the
    potential weights V [heads, fin] and V_bias [heads].  Returns (x_new, v_new).
    """
    sid = SCHEMES[scheme] if isinstance(scheme, str) else int(scheme)
    require_cuda(x, v, f, U, W, Wf, bf, Wi)
    if _grad_wanted(x, v, f, U, W, Wf, bf, Wi):
        raise GfnError("integrator backward is implemented for the leapfrog only")
    x, v = _f32c(x, "x"), _f32c(v, "v")
    f, Wf, bf, Wi = _f32c(f, "f"), _f32c(Wf, "Wf"), _f32c(bf, "bf"), _f32c(Wi, "Wi")
    B, d = x.shape
    hd = d // heads
    if topology == 0:
        U, W = _f32c(U, "U"), _f32c(W, "W")
        rank = U.shape[-1]
    else:
        U = W = None
        rank = 4
    dts = _dt_scales(dt_scale, x)
    V, V_bias = _f32c(V, "V"), _f32c(V_bias, "V_bias")
    x_new, v_new = torch.empty_like(x), torch.empty_like(v)
    call("gfn_integrator_heads", sid, ptr(x), ptr(v), ptr(f), ptr(U), ptr(W), ptr(Wf), ptr(bf), ptr(Wi),
         ptr(x_new), ptr(v_new), float(dt), ptr(dts), dts.numel(), B, int(heads), hd, rank, int(steps),
         int(topology), float(R), float(r), float(plasticity), ptr(V), ptr(V_bias), int(singularity),
         float(sing_thresh), float(sing_strength), _stream(x))
    return x_new, v_new


def _integrator_op(name):
    def fn(x, v, f, U, W, dt, dt_scale, steps, topology=0, R=2.0, r=1.0, Wf=None, bf=None, Wi=None):
        return integrator_heads(name, x, v, f, U, W, dt, dt_scale, steps, topology, Wf, bf, Wi, 1, R, r)
    fn.__name__ = f"{name}_fused"
    fn.__doc__ = (f"One head's {name} integrator, `steps` times (the reference's gfn.cuda.ops."
                  f"{name}_fused signature, gfn/cuda/ops.py:184-222), with the optional friction "
                  "gate (Wf, bf, Wi) the reference's Christoffel applies in its combined form.")
    return fn


euler_fused = _integrator_op("euler")
heun_fused = _integrator_op("heun")
rk4_fused = _integrator_op("rk4")
verlet_fused = _integrator_op("verlet")
yoshida_fused = _integrator_op("yoshida")
forest_ruth_fused = _integrator_op("forest_ruth")
omelyan_fused = _integrator_op("omelyan")
dormand_prince_fused = _integrator_op("dormand_prince")
