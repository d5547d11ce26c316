"""GPU parity of the gated scan and of the stateful scan layer, with their
gradients, against the float64 step-by-step definitions (oracle/lm_ops.py).

Tolerances, with u = 2^-24 and uo the rounding of the output type.  A scan of
|a|, |x| from |h0| bounds every partial sum: S_t = |a| S_{t-1} + |x_t|.  Each
step rounds a few times at u S_t, a run of n steps passed as (P, p) carries n
roundings more of the same terms, and an error e_{t-1} arrives as |a| e_{t-1}:
  e_t = |a| e_{t-1} + 8 u S_t.
Gradients follow the same rule on the reversed recurrence, and a product of
two such quantities carries e1 |q2| + |q1| e2 + e1 e2.  The scan layer's gates
come from exp / log1p / a division: 16 u relative on A, dt and their slopes.
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from manifold_b200 import _lib
from oracle import lm_ops as O

DEV = "cuda:0"
U = 2.0 ** -24
UO = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-36, torch.bfloat16: 1e-36, torch.float16: 2.0 ** -24}


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _check(got, want, tol, what):
    got = _np(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(),
                           float(np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300))))


def _rev(t):
    return t[:, ::-1]


def _envelope(a, x, h0):
    """(S, e): the magnitude bound and the error bound of the recurrence."""
    S, _ = O.gated_scan(np.abs(a), np.abs(x), None if h0 is None else np.abs(h0))
    e, _ = O.gated_scan(np.abs(a), 8 * U * S, None)
    return S, e


def _prev(h, h0):
    first = np.zeros_like(h[:, :1]) if h0 is None else h0[:, None]
    return np.concatenate([first, h[:, :-1]], 1)


def _check_scan(a, x, h0, h, last, dh=None, dlast=None, grads=None):
    """a, x, ...: torch tensors; grads: (da, dx, dh0), entries may be None."""
    dt = x.dtype
    an, xn, h0n = _np(a), _np(x), _np(h0)
    an = np.ones_like(xn) if an is None else np.broadcast_to(an, xn.shape)
    want, wl = O.gated_scan(an, xn, h0n)
    if xn.shape[1] == 0:
        S = e = want
        el = np.zeros_like(wl)
    else:
        S, e = _envelope(an, xn, h0n)
        el = e[:, -1]
    _check(h, want, TINY[dt] + UO[dt] * np.abs(want) + e, "h")
    if last is not None:
        assert last.dtype == torch.float32
        _check(last, wl, 1e-36 + U * np.abs(wl) + el, "last")
    if grads is None:
        return
    dhn, dln = _np(dh), _np(dlast)
    rda, rdx, rdh0 = O.gated_scan_backward(an, xn, h0n, dhn, dln)
    src = np.zeros_like(xn) if dhn is None else dhn
    # the message recurrence m_t = a_t (dh_t + m_{t+1}) run backwards
    anr = _rev(an)
    shifted = np.concatenate([np.ones_like(anr[:, :1]), anr[:, :-1]], 1)
    if xn.shape[1]:
        G, eg = _envelope(shifted, _rev(src), dln)
        G, eg = _rev(G), _rev(eg)
        hp = np.abs(_prev(want, h0n))
        ehp = _prev(e, None)
        da, dx, dh0 = grads
        if dx is not None:
            _check(dx, rdx, TINY[dt] + UO[dt] * np.abs(rdx) + eg, "dx")
        if da is not None:
            _check(da, rda, TINY[dt] + UO[dt] * np.abs(rda) + eg * hp + (G + eg) * ehp + 2 * U * np.abs(rda), "da")
        if dh0 is not None:
            _check(dh0, rdh0, 1e-36 + 2 * U * np.abs(rdh0) + np.abs(an[:, 0]) * eg[:, 0], "dh0")
    elif grads[2] is not None:
        _check(grads[2], rdh0, 1e-36, "dh0")


def _inputs(B, L, D, dtype, seed, lo=0.0):
    g = torch.Generator().manual_seed(seed)
    a = (lo + (1 - lo) * torch.rand(B, L, D, generator=g)).to(dtype).to(DEV)
    x = torch.randn(B, L, D, generator=g).to(dtype).to(DEV)
    h0 = torch.randn(B, D, generator=g).to(DEV)
    dh = torch.randn(B, L, D, generator=g).to(dtype).to(DEV)
    dl = torch.randn(B, D, generator=g).to(DEV)
    return a, x, h0, dh, dl


def _run(a, x, h0, dh, dl):
    with torch.no_grad():
        h_inf, last_inf = gfn.gated_scan(a, x, h0, return_state=True)
    leaves = [t.detach().requires_grad_(True) for t in (a, x, h0) if t is not None]
    it = iter(leaves)
    av, xv = (None if a is None else next(it)), next(it)
    hv = None if h0 is None else next(it)
    h, last = gfn.gated_scan(av, xv, hv, return_state=True)
    assert h.dtype == x.dtype and h.shape == x.shape
    assert torch.equal(h, h_inf) and torch.equal(last, last_inf)
    outs, gos = [], []
    if dh is not None:
        outs.append(h), gos.append(dh)
    if dl is not None:
        outs.append(last), gos.append(dl)
    grads = list(torch.autograd.grad(outs, leaves, gos, retain_graph=True))
    again = torch.autograd.grad(outs, leaves, gos)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # no order-dependent sums
    da = None if a is None else grads.pop(0)
    dx = grads.pop(0)
    dh0 = grads.pop(0) if h0 is not None else None
    _check_scan(a, x, h0, h, last, dh, dl, (da, dx, dh0))
    assert gfn.cuda.ops.device_error() == 0


SHAPES = [(1, 1, 1), (2, 1, 64), (3, 2, 33), (1, 7, 256), (2, 63, 32), (2, 64, 100), (1, 65, 128), (3, 127, 40),
          (1, 128, 8), (2, 129, 130), (1, 255, 64), (1, 256, 192), (2, 257, 3), (5, 300, 72), (1, 1000, 513),
          (1, 5003, 24), (2, 2048, 96), (40, 150, 512), (300, 70, 64), (1, 9001, 5), (700, 3, 257)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gated_scan_matches_definition(shape, dtype):
    _run(*_inputs(*shape, dtype, seed=sum(shape), lo=0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("lo", [0.0, 0.95, 1.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_scan_gate_ranges(dtype, lo):
    # fast decay, slow decay, no decay
    _run(*_inputs(2, 700, 68, dtype, seed=3, lo=lo))


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,D", [(2, 300, 96), (1, 1500, 33)])
def test_gated_scan_optional_operands(B, L, D):
    a, x, h0, dh, dl = _inputs(B, L, D, torch.float32, 11, 0.7)
    _run(a, x, None, dh, None)
    _run(a, x, h0, None, dl)
    _run(None, x, h0, dh, dl)
    _run(-a, x, h0, dh, dl)  # signs alternate


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_scan_zero_gates_start_new_sequences(dtype):
    a, x, h0, dh, dl = _inputs(2, 600, 40, dtype, 5, 0.9)
    for t in (0, 1, 130, 256, 257, 511, 599):
        a[:, t] = 0
    _run(a, x, h0, dh, dl)
    h = gfn.gated_scan(a, x, h0)
    assert torch.equal(h[:, 256], x[:, 256])
    seg = gfn.gated_scan(a[:, 257:511].contiguous(), x[:, 257:511].contiguous())
    tol = 8 * 40 * UO[dtype]
    torch.testing.assert_close(seg.float(), h[:, 257:511].float(), rtol=tol, atol=tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_scan_growing_gates(dtype):
    a, x, h0, dh, dl = _inputs(2, 400, 48, dtype, 17, 0.95)
    _run((a * 1.06).to(dtype), x, h0, dh, dl)


@pytest.mark.gpu
def test_gated_scan_calls_on_two_streams_at_once():
    # blocks of one call wait for one another, never for another call's
    args = [_inputs(1, 20000, 96, torch.bfloat16, 30 + i, 0.9)[:3] for i in range(2)]
    want = [gfn.gated_scan(*t) for t in args]
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(gfn.gated_scan(*args[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)
    assert gfn.cuda.ops.device_error() == 0


@pytest.mark.gpu
def test_gated_scan_underflowing_products():
    # the product of a run's gates is below float32; the state is not lost to NaN
    a = torch.full((1, 900, 64), 1e-3, device=DEV)
    x = torch.randn(1, 900, 64, device=DEV)
    h0 = torch.full((1, 64), 1e30, device=DEV)
    _run(a, x, h0, torch.randn_like(x), torch.full((1, 64), 1e30, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("L", [40, 1000])
def test_gated_scan_non_finite_values_follow_the_definition(L):
    g = torch.Generator().manual_seed(2)
    a = (0.5 + 0.5 * torch.rand(2, L, 48, generator=g)).to(DEV)
    x = torch.randn(2, L, 48, generator=g).to(DEV)
    x[0, 5, 3], x[0, 9, 7], x[1, 20, 0] = float("inf"), float("nan"), float("-inf")
    h = gfn.gated_scan(a, x)
    ref = torch.empty_like(h)
    s = torch.zeros(2, 48, device=DEV)
    for t in range(L):
        s = a[:, t] * s + x[:, t]
        ref[:, t] = s
    assert torch.equal(torch.isnan(h), torch.isnan(ref))
    assert torch.equal(torch.isposinf(h), torch.isposinf(ref))
    assert torch.equal(torch.isneginf(h), torch.isneginf(ref))
    # a sequence that starts afresh after the non-finite one: 0 * inf is NaN in the definition, so the
    # state is dropped by h0 of the next call instead
    ok = torch.isfinite(ref)
    torch.testing.assert_close(h[ok], ref[ok], rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_scan_strides_and_broadcast_gates(dtype):
    g = torch.Generator().manual_seed(9)
    base = torch.randn(3, 210, 3 * 56 + 1, generator=g).to(dtype).to(DEV)
    gate = torch.rand(3, 210, 3 * 56 + 1, generator=g).to(dtype).to(DEV)
    dh = torch.randn(3, 210, 56, generator=g).to(dtype).to(DEV)
    h0, dl = torch.randn(3, 56, generator=g).to(DEV), torch.randn(3, 56, generator=g).to(DEV)
    for a, x in ((gate[..., :56], base[..., 56:112]), (gate[..., 1:57], base[..., 111:167]),
                 (gate[..., ::3][..., :56], base[..., 3:59]),
                 (gate[:, 100:101, 1:57].expand(-1, 210, -1), base.transpose(0, 1)[:3, :3, :56].transpose(0, 1)
                  .repeat(1, 70, 1))):
        _run(a, x, h0, dh, dl)
    # gradients of broadcast gates are summed over what they were broadcast over
    x = base[..., :56]
    for shape in ((56,), (1, 210, 1), (3, 1, 56), (3, 210, 1)):
        av = torch.rand(shape, generator=g).to(dtype).to(DEV).requires_grad_(True)
        full = av.detach().expand(3, 210, 56)
        h = gfn.gated_scan(av, x, h0)
        da, = torch.autograd.grad(h, av, dh)
        assert da.shape == shape
        rda, _, _ = O.gated_scan_backward(_np(full), _np(x), _np(h0), _np(dh), None)
        axes = tuple(i for i in range(3) if ((1,) * (3 - len(shape)) + shape)[i] == 1)
        want = rda.sum(axes).reshape(shape)
        # a sum of n rounded terms: the type's rounding of each, in a root-mean-square sense times 8, plus its own
        n = rda.size / want.size
        tol = 8 * UO[dtype] * np.sqrt((rda ** 2).sum(axes)).reshape(shape) + 4 * UO[dtype] * np.abs(want) \
            + n * 64 * U * np.abs(rda).max()
        assert (np.abs(_np(da) - want) <= tol).all()
    dh_t = dh.transpose(1, 2).contiguous().transpose(1, 2)  # inner stride not 1
    dh_e = dh[:, :1, :1].expand(3, 210, 56)
    a = gate[..., :56]
    _run(a, x, h0, dh_t, dl)
    _run(a, x, h0, dh_e, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 61])
def test_gated_scan_other_orders_of_batch_and_time(dtype, D):
    g = torch.Generator().manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    gate = lambda *s: torch.rand(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    h0 = torch.randn(5, D, generator=g).to(DEV)
    # time-major storage: the batch stride is the smaller one
    a, x, dh = gate(270, 5, D).transpose(0, 1), r(270, 5, D).transpose(0, 1), r(270, 5, D).transpose(0, 1)
    _run(a, x, h0, dh, None)
    # windows that overlap: a step stride below the width, a batch stride below the sequence
    base = r(5 * 8 + 270 * 8 + D)
    x = base.as_strided((5, 270, D), (8, 8, 1))
    with torch.no_grad():
        h, last = gfn.gated_scan(a, x, h0, return_state=True)
    _check_scan(a, x, h0, h, last)
    # every second step, every second row
    a, x, dh = gate(10, 540, D)[::2, ::2], r(10, 540, D)[::2, 1::2], r(10, 540, D)[1::2, ::2]
    _run(a, x, h0, dh, None)
    # each operand in an order of its own
    _run(gate(270, 5, D).transpose(0, 1), r(5, 270, D), h0, r(5, 270, 2 * D)[..., D:], None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_scan_segments_and_single_tokens_continue_the_state(dtype):
    a, x, h0, _, _ = _inputs(2, 333, 70, dtype, 21, 0.8)
    h, last = gfn.gated_scan(a, x, h0, return_state=True)
    s, out = h0, []
    for lo, hi in ((0, 1), (1, 2), (2, 130), (130, 131), (131, 333), (333, 333)):
        o, s = gfn.gated_scan(a[:, lo:hi], x[:, lo:hi], s, return_state=True)
        out.append(o)
    seg = torch.cat(out, 1)
    _check_scan(a, x, h0, seg, s)
    torch.testing.assert_close(s, last, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_gated_scan_empty_sizes():
    for B, L, D in ((2, 0, 8), (0, 5, 8), (2, 5, 0)):
        x = torch.zeros(B, L, D, device=DEV, requires_grad=True)
        a = torch.zeros(B, L, D, device=DEV, requires_grad=True)
        h0 = torch.randn(B, D, device=DEV, requires_grad=True)
        h, last = gfn.gated_scan(a, x, h0, return_state=True)
        assert h.shape == (B, L, D) and last.shape == (B, D)
        if L == 0:
            assert torch.equal(last, h0)
        da, dx, dh0 = torch.autograd.grad((h, last), (a, x, h0), (torch.zeros_like(h), torch.ones_like(last)))
        assert da.shape == dx.shape == (B, L, D)
        if L == 0:
            assert torch.equal(dh0, torch.ones_like(h0))
    z = torch.zeros(2, 0, 24, device=DEV)
    v0, x0 = torch.randn(2, 8, device=DEV), torch.randn(2, 8, device=DEV)
    xs, vs, (v, x) = gfn.cuda.ops.parallel_layer_scan(z, 2, state=(v0, x0), return_state=True)
    assert xs.shape == vs.shape == (2, 0, 8) and torch.equal(v, v0) and torch.equal(x, x0)


@pytest.mark.gpu
def test_gated_scan_large_offsets():
    # a view whose steps lie more than 2^31 elements apart: 64-bit offsets
    base = torch.zeros(2 ** 31 + 4096, device=DEV, dtype=torch.float16)
    x = base.as_strided((1, 2, 64), (0, 2 ** 31 + 128, 1))
    x.normal_()
    a = torch.full((1, 2, 64), 0.5, device=DEV, dtype=torch.float16)
    _run(a, x, None, torch.randn(1, 2, 64, device=DEV).half(), None)


@pytest.mark.gpu
def test_parallel_scan_gradient():
    a, x, _, dh, _ = _inputs(2, 130, 40, torch.float32, 4, 0.5)
    for gate in (a, None):
        xv = x.clone().requires_grad_(True)
        av = None if gate is None else gate.clone().requires_grad_(True)
        y = gfn.parallel_scan(av, xv)
        torch.testing.assert_close(y.detach(), gfn.parallel_scan(gate, x), rtol=1e-5, atol=1e-5)
        leaves = [xv] if av is None else [av, xv]
        grads = torch.autograd.grad(y, leaves, dh)
        _check_scan(gate, x, None, y, None, dh, None, (grads[0] if av is not None else None, grads[-1], None))


@pytest.mark.gpu
def test_gated_scan_side_stream_and_graph():
    a, x, h0, _, _ = _inputs(1, 3000, 64, torch.float32, 6, 0.9)
    ref = gfn.gated_scan(a, x, h0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = gfn.gated_scan(a, x, h0)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = gfn.gated_scan(a, x, h0)
    for _ in range(3):
        z.zero_()
        g.replay()
        assert torch.equal(z, ref)


# ------------------------------------------------------------ the scan layer
def _layer_check(z, heads, base_dt, v0, x0, xs, vs, vl, xl, g=None, grads=None):
    zn, v0n, x0n = _np(z), _np(v0), _np(x0)
    D = zn.shape[-1] // 3
    A, nA, dt, sdt, hs = O.layer_scan_terms(zn, heads, base_dt)
    zb = zn[..., 2 * D:]
    wx, wv, wxl, wvl = O.layer_scan(zn, heads, base_dt, v0n, x0n)
    S, _ = O.gated_scan(A, np.abs(zb * dt), None if v0n is None else np.abs(v0n))
    ev, _ = O.gated_scan(A, 48 * U * S, None)
    SX, _ = O.gated_scan(None, S * dt, None if x0n is None else np.abs(x0n))
    ex, _ = O.gated_scan(None, 48 * U * S * dt + ev * dt + 8 * U * SX, None)
    _check(vs, wv, 1e-36 + ev, "v")
    _check(xs, wx, 1e-36 + ex, "x")
    if vl is not None:
        _check(vl, wvl, 1e-36 + ev[:, -1], "v last")
        _check(xl, wxl, 1e-36 + ex[:, -1], "x last")
    if grads is None:
        return
    gx, gv, gvl, gxl = (_np(t) for t in g)
    dz, dv0, dx0 = O.layer_scan_backward(zn, heads, base_dt, v0n, gx, gv, gxl, gvl)
    zero = np.zeros_like(wv)
    ax = zero if gx is None else np.abs(gx)
    X, _ = O.gated_scan(None, _rev(ax), None if gxl is None else np.abs(gxl))
    eX = _rev(O.gated_scan(None, 8 * U * X, None)[0])
    X = _rev(X)
    src = (zero if gv is None else np.abs(gv)) + dt * X
    Ar = np.concatenate([np.ones_like(A[:, :1]), _rev(A)[:, :-1]], 1)
    Lm, _ = O.gated_scan(Ar, _rev(src), None if gvl is None else np.abs(gvl))
    el = _rev(O.gated_scan(Ar, _rev(48 * U * src + dt * eX) + 48 * U * Lm, None)[0])
    Lm = _rev(Lm)
    vp, evp = np.abs(_prev(wv, v0n)), _prev(ev, None)
    tA = (el * vp + (Lm + el) * evp + 48 * U * Lm * vp) * A * nA
    tD = (el * np.abs(zb) + eX * np.abs(wv) + (X + eX) * ev + 48 * U * (Lm * np.abs(zb) + X * np.abs(wv))) * hs * sdt
    tB = (el + 48 * U * Lm) * dt
    _check(grads[0], dz, 1e-36 + np.concatenate([tA, tD, tB], -1), "dz")
    if grads[1] is not None:
        _check(grads[1], dv0, 1e-36 + A[:, 0] * el[:, 0] + 48 * U * A[:, 0] * Lm[:, 0], "dv0")
    if grads[2] is not None:
        _check(grads[2], dx0, 1e-36 + eX[:, 0], "dx0")


def _layer_run(B, L, D, heads, seed, state=True, use=("gx", "gv", "gvl", "gxl"), base_dt=0.1, zscale=1.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen).to(DEV)  # noqa: E731
    z = r(B, L, 3 * D) * zscale
    v0, x0 = (r(B, D), r(B, D)) if state else (None, None)
    g = [r(B, L, D) if "gx" in use else None, r(B, L, D) if "gv" in use else None,
         r(B, D) if "gvl" in use else None, r(B, D) if "gxl" in use else None]
    with torch.no_grad():
        inf = gfn.cuda.ops.parallel_layer_scan(z, heads, base_dt, state=(v0, x0), return_state=True)
    leaves = [t.detach().requires_grad_(True) for t in (z, v0, x0) if t is not None]
    st = tuple(leaves[1:]) if state else None
    xs, vs, (vl, xl) = gfn.cuda.ops.parallel_layer_scan(leaves[0], heads, base_dt, state=st, return_state=True)
    assert torch.equal(xs, inf[0]) and torch.equal(vs, inf[1])
    assert torch.equal(vl, inf[2][0]) and torch.equal(xl, inf[2][1])
    pairs = [(o, q) for o, q in zip((xs, vs, vl, xl), g) if q is not None]
    grads = torch.autograd.grad([p[0] for p in pairs], leaves, [p[1] for p in pairs], allow_unused=True)
    _layer_check(z, heads, base_dt, v0, x0, xs, vs, vl, xl, g, (*grads, None, None)[:3])
    assert gfn.cuda.ops.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,D,heads", [(1, 1, 4, 1), (2, 1, 64, 8), (3, 5, 33, 3), (1, 64, 32, 4), (2, 65, 40, 2),
                                         (1, 127, 96, 4), (2, 128, 7, 1), (1, 129, 128, 8), (4, 300, 130, 2),
                                         (1, 1000, 64, 8), (1, 5001, 20, 4), (32, 140, 256, 8), (600, 4, 64, 4)])
def test_layer_scan_matches_definition(B, L, D, heads):
    _layer_run(B, L, D, heads, seed=B + L + D)


@pytest.mark.gpu
@pytest.mark.parametrize("use", [("gx",), ("gv",), ("gvl",), ("gxl",), ("gx", "gv")])
@pytest.mark.parametrize("state", [True, False])
def test_layer_scan_partial_gradients(use, state):
    _layer_run(2, 290, 48, 4, seed=7, state=state, use=use)


@pytest.mark.gpu
def test_layer_scan_extreme_preactivations():
    # gates at exactly 0 and 1, steps at 0 and far above softplus's linear threshold
    _layer_run(2, 260, 32, 2, seed=3, zscale=40.0)


@pytest.mark.gpu
def test_layer_scan_agrees_with_the_stateless_kernel_and_segments():
    z = torch.randn(2, 400, 3 * 64, device=DEV)
    with torch.no_grad():
        x0, v0 = gfn.cuda.ops.parallel_layer_scan(z, 4)
        x1, v1, (vl, xl) = gfn.cuda.ops.parallel_layer_scan(z, 4, return_state=True)
        _layer_check(z, 4, 0.1, None, None, x0, v0, None, None)
        _layer_check(z, 4, 0.1, None, None, x1, v1, vl, xl)
        st, xs, vs = None, [], []
        for lo, hi in ((0, 1), (1, 200), (200, 201), (201, 400)):
            a, b, st = gfn.cuda.ops.parallel_layer_scan(z[:, lo:hi], 4, state=st, return_state=True)
            xs.append(a), vs.append(b)
        _layer_check(z, 4, 0.1, None, None, torch.cat(xs, 1), torch.cat(vs, 1), *st)


# -------------------------------------------------------------- refusals, CPU
@pytest.mark.gpu
def test_scan_refusals_on_the_gpu():
    x = torch.zeros(2, 5, 8, device=DEV)
    for a, y, h0 in ((x[:, :4], x, None), (x.bfloat16(), x, None), (x, x.double(), None), (x, x[0], None),
                     (x, x, torch.zeros(2, 7, device=DEV)), (x, x, torch.zeros(2, 8, device=DEV).half()),
                     (x.cpu(), x, None), (x, x, torch.zeros(2, 8))):
        with pytest.raises(gfn.GfnError):
            gfn.gated_scan(a, y, h0)
    z = torch.zeros(2, 5, 24, device=DEV)
    scan = gfn.cuda.ops.parallel_layer_scan
    for args, kw in (((z[..., :23], 1), {}), ((z, 3), {}), ((z, 0), {}), ((z.half(), 2), {}),
                     ((z, 2), dict(state=(x[:, 0], torch.zeros(2, 4, device=DEV)))),
                     ((z, 2), dict(state=(x[:, 0].half(), x[:, 0])))):
        with pytest.raises(gfn.GfnError):
            scan(*args, return_state=True, **kw)
    xg = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(gfn.gated_scan(x, xg).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        g.sum().backward()


def test_scan_refusals():
    with pytest.raises(gfn.GfnError):  # no CPU path
        gfn.gated_scan(torch.ones(1, 4, 4), torch.ones(1, 4, 4))
    lib = _lib.load()
    assert lib.gfn_gated_scan_states_floats(2, 65, 8) == 2 * 2 * 8
    assert lib.gfn_gated_scan_workspace_bytes(-1, 4, 4) == -1
    args = [None, 0, 0, None, 0, 0, None, 0, 2, 3, 4, None, None, None, None, 0, None]
    assert lib.gfn_gated_scan_forward(*args) == 1           # NULL x, h
    args[8] = -1
    assert lib.gfn_gated_scan_forward(*args) == 1           # negative batch
    args[8] = 0
    assert lib.gfn_gated_scan_forward(*args) == 0           # nothing to do
    assert lib.gfn_layer_scan_forward(None, None, None, 1, 1, 8, 3, 0.1, None, None, None, None, None, None, 0,
                                      None) == 1            # heads do not divide dim


def test_scan_definition_gradients_against_differences():
    rng = np.random.default_rng(1)
    a, x, h0 = rng.uniform(0.2, 1, (2, 5, 3)), rng.standard_normal((2, 5, 3)), rng.standard_normal((2, 3))
    dh, dl = rng.standard_normal((2, 5, 3)), rng.standard_normal((2, 3))
    z, v0, x0 = rng.standard_normal((2, 5, 12)), rng.standard_normal((2, 4)), rng.standard_normal((2, 4))
    gx, gv, gxl, gvl = (rng.standard_normal(s) for s in ((2, 5, 4), (2, 5, 4), (2, 4), (2, 4)))

    def f(a, x, h0):
        h, last = O.gated_scan(a, x, h0)
        return (h * dh).sum() + (last * dl).sum()

    def q(z, v0, x0):
        xs, vs, xl, vl = O.layer_scan(z, 2, 0.1, v0, x0)
        return (xs * gx).sum() + (vs * gv).sum() + (xl * gxl).sum() + (vl * gvl).sum()

    for fn, args, grads in ((f, (a, x, h0), O.gated_scan_backward(a, x, h0, dh, dl)),
                            (q, (z, v0, x0), O.layer_scan_backward(z, 2, 0.1, v0, gx, gv, gxl, gvl))):
        for k, g in enumerate(grads):
            for i in range(0, g.size, 3):
                hi, lo = [t.copy() for t in args], [t.copy() for t in args]
                hi[k].reshape(-1)[i] += 1e-6
                lo[k].reshape(-1)[i] -= 1e-6
                assert abs((fn(*hi) - fn(*lo)) / 2e-6 - g.reshape(-1)[i]) < 1e-7
