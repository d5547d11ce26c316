"""Gates whose products leave float32's range: decay then growth, growth that
meets a tiny state, zeros behind large products, huge states that decay.

Tolerances as in tests/test_gpu_gated_scan.py (S_t = |a| S_{t-1} + |x_t|,
u = 2^-24), with the roundings near float32's smallest value counted too, each
at most the value itself or that smallest value: e_t = |a| e_{t-1} + 16 u S_t +
min(S_t, 2^-149).  (16 rather than 8: a product beyond 2^+-100 carries 20 bits.)
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from oracle import lm_ops as O

DEV = "cuda:0"
U, TINY = 2.0 ** -24, 2.0 ** -149
UO = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUB = {torch.float32: TINY, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # smallest values


def _np(t):
    return t.detach().double().cpu().numpy()


def _envelope(a, x, h0):
    S, _ = O.gated_scan(np.abs(a), np.abs(x), np.abs(h0))
    e, _ = O.gated_scan(np.abs(a), 16 * U * S + np.minimum(S, TINY), None)
    return S, e


def _check(got, want, tol, what):
    bad = ~(np.abs(_np(got) - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:3].tolist(), _np(got)[bad][:3], want[bad][:3], tol[bad][:3])


def _run(a, x, h0, dh, dl):
    """a, x, dh [B, L, D], h0, dl [B, D] against the definition, both ways."""
    dt = x.dtype
    leaves = [t.detach().clone().requires_grad_(True) for t in (a, x, h0)]
    h, last = gfn.gated_scan(*leaves, return_state=True)
    da, dx, dh0 = torch.autograd.grad((h, last), leaves, (dh, dl))
    an, xn, h0n, dhn, dln = map(_np, (a, x, h0, dh, dl))
    want, wl = O.gated_scan(an, xn, h0n)
    S, e = _envelope(an, xn, h0n)
    _check(h, want, SUB[dt] + UO[dt] * np.abs(want) + e, "h")
    _check(last, wl, TINY + U * np.abs(wl) + e[:, -1], "last")
    rda, rdx, rdh0 = O.gated_scan_backward(an, xn, h0n, dhn, dln)
    ar = an[:, ::-1]
    G, eg = _envelope(np.concatenate([np.ones_like(ar[:, :1]), ar[:, :-1]], 1), dhn[:, ::-1], dln)
    G, eg = G[:, ::-1], eg[:, ::-1]
    hp = np.concatenate([h0n[:, None], want[:, :-1]], 1)
    ehp = np.concatenate([np.zeros_like(h0n[:, None]), e[:, :-1]], 1)
    _check(dx, rdx, SUB[dt] + UO[dt] * np.abs(rdx) + eg, "dx")
    _check(da, rda, SUB[dt] + (UO[dt] + 2 * U) * np.abs(rda) + eg * np.abs(hp) + (G + eg) * ehp, "da")
    _check(dh0, rdh0, TINY + 2 * U * np.abs(rdh0) + np.abs(an[:, 0]) * eg[:, 0], "dh0")
    assert gfn.cuda.ops.device_error() == 0


def _flat(L, D, dtype, value=0.0):
    return torch.full((1, L, D), value, device=DEV).to(dtype)


def _state(D, value):
    return torch.full((1, D), value, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 61])
@pytest.mark.parametrize("down,up,half", [(0.5, 1.9, 256), (0.5, 1.9, 700), (0.25, 3.0, 90), (1e-3, 800.0, 40)])
def test_gates_that_decay_and_then_grow(D, dtype, down, up, half):
    a = _flat(2 * half, D, dtype, down)
    a[:, half:] = up
    z = _flat(2 * half, D, dtype)
    _run(a, z, _state(D, 1.0), z, _state(D, 0.0))
    _run(a.flip(1), z, _state(D, 0.0), z, _state(D, 1.0))  # the messages' direction
    x = z.clone()
    x[:, ::7] = 1.0
    a[:, half:] = 1.0
    _run(a, x, _state(D, 1.0), x, _state(D, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 61])
@pytest.mark.parametrize("at", [0, 5, 100, 128, 200])
def test_growing_gates_that_meet_a_tiny_state(D, at):
    a, x = _flat(400, D, torch.float32, 1.0), _flat(400, D, torch.float32)
    a[:, at:at + 70] = 4.0  # 2^140 in all
    _run(a, x, _state(D, 1e-30), x, _state(D, 0.0))
    _run(a.flip(1), x, _state(D, 0.0), x, _state(D, 1e-30))
    a[:, at + 90] = 0.0  # a new sequence behind it
    x[:, at + 90] = 3.0
    _run(a, x, _state(D, 1e-30), x, _state(D, 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 61])
def test_a_zero_state_stays_zero_through_overflowing_products(D):
    a, x = _flat(800, D, torch.float32, 4.0), _flat(800, D, torch.float32)
    a[:, 500] = 0.0
    _run(a, x, _state(D, 0.0), x, _state(D, 0.0))
    x[:, 510] = 1e-30
    a[:, 511:] = 1.0
    _run(a, x, _state(D, 0.0), x, _state(D, 0.0))
    a = torch.full_like(a, 0.5)  # empty stretches between packed sequences
    a[:, ::200], x[:, ::200] = 0.0, 1.0
    a[:, 300:420] = 0.0
    _run(a, x, _state(D, 3.0), x, _state(D, 3.0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 61])
def test_huge_states_decay_to_the_end(D):
    a, z = _flat(500, D, torch.float32, 0.5), _flat(500, D, torch.float32)
    _run(a, z, _state(D, 1e38), z, _state(D, 1e38))
    a[:, ::2] = -1e-20
    a[:, 1::2] = 9e19
    _run(a, z, _state(D, 1e10), z, _state(D, 1e10))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("D", [64, 61])
def test_products_that_wander(D, seed):
    # the state's exponent walks within +-100 while the gates' runs reach far beyond
    g = torch.Generator().manual_seed(seed)
    w = torch.cumsum(torch.randint(-9, 10, (2, 1500, D), generator=g), 1)
    w = ((w + 100) % 400 - 200).abs() - 100  # reflected
    a = torch.exp2(torch.diff(w, dim=1, prepend=torch.zeros(2, 1, D).long()).double())
    a *= torch.where(torch.rand(a.shape, generator=g) < 0.5, -1.0, 1.0) * (0.9 + 0.2 * torch.rand(a.shape, generator=g))
    a = a.float().to(DEV)
    z = torch.zeros_like(a)
    _run(a, z, torch.full((2, D), 1.5, device=DEV), z, torch.full((2, D), 0.0, device=DEV))
    _run(a, z, torch.full((2, D), 0.0, device=DEV), z, torch.full((2, D), 1e-28, device=DEV))


@pytest.mark.gpu
def test_parallel_scan_with_a_gradient_has_the_same_domain():
    a, x = torch.ones(1, 300, 64, device=DEV), torch.zeros(1, 300, 64, device=DEV)
    a[:, 130:200] = 4.0
    x[:, 0] = 1e-30
    y = gfn.parallel_scan(a, x.requires_grad_(True))
    want, _ = O.gated_scan(_np(a), _np(x), None)
    assert np.isfinite(want).all() and want.max() > 1e12
    assert (np.abs(_np(y) - want) <= 300 * 16 * U * want).all()
    g, = torch.autograd.grad(y.sum(), x)  # sums of products up to 2^140 of ones
    assert not torch.isnan(g).any()


@pytest.mark.gpu
@pytest.mark.parametrize("D,heads", [(64, 4), (33, 1)])
def test_layer_states_decay_to_the_end(D, heads):
    z = torch.zeros(1, 600, 3 * D, device=DEV)
    z[..., :D] = -3.0  # gates of 0.047
    v0, x0 = _state(D, 1e30), _state(D, 2.0)
    xs, vs, (vl, xl) = gfn.cuda.ops.parallel_layer_scan(z, heads, state=(v0, x0), return_state=True)
    wx, wv, _, _ = O.layer_scan(_np(z), heads, 0.1, _np(v0), _np(x0))
    A, _, dt, _, _ = O.layer_scan_terms(_np(z), heads, 0.1)
    S, e = O.gated_scan(A, np.zeros_like(wv), _np(v0))[0], None
    e, _ = O.gated_scan(A, 48 * U * S + np.minimum(S, TINY), None)
    _check(vs, wv, TINY + e, "v")
    _check(vl, wv[:, -1], TINY + e[:, -1], "last v")
    ex, _ = O.gated_scan(None, 48 * U * S * dt + e * dt + 8 * U * np.abs(wx), None)
    _check(xs, wx, ex, "x")
