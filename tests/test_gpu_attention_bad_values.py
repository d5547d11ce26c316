"""NaN and infinities in the operands of decay_attention: they reach what the
recurrence takes them to and nothing else, token by token and element by element,
as the float64 recurrence (oracle/lm_ops.py) has it.

What stays finite has the tolerances of test_gpu_decay_attention.py: relative to
the sums over magnitudes, 2^-18 for states, and for outputs one rounding and the
operands' own (2^-8 bfloat16, 2^-11 float16).
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from oracle import lm_ops as O

DEV = "cuda:0"
UO = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
OPERAND = {torch.float32: 2.0 ** -18, torch.bfloat16: 2.0 ** -8 + 2.0 ** -18, torch.float16: 2.0 ** -11 + 2.0 ** -18}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAN, INF = float("nan"), float("inf")


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _reach(name, got, want, tol, signs=False):
    """Finite where the definition is, and close there; signs: the same infinities and NaN elsewhere too."""
    assert got.shape == want.shape, name
    fine = np.isfinite(want)
    wrong = np.isfinite(got) != fine
    assert not wrong.any(), (name, int(wrong.sum()), np.argwhere(wrong)[0])
    bad = ~(np.abs(got - want)[fine] <= tol[fine])
    assert not bad.any(), (name, int(bad.sum()), np.abs(got - want)[fine][bad].max())
    if signs:
        other = ~fine & ~((got == want) | (np.isnan(got) & np.isnan(want)))
        assert not other.any(), (name, int(other.sum()), got[other][0], want[other][0])


def _check(ts, clean, decay, st, lengths, scale, do, dl, what):
    """ts: q, k, v with bad values; clean: the same without, for the tolerances."""
    leaves = [t.clone().requires_grad_(True) for t in (*ts, st)]
    o, last = gfn.decay_attention(*leaves[:3], decay, state=leaves[3], return_state=True, lengths=lengths, scale=scale)
    grads = torch.autograd.grad((o, last), leaves, (do, dl))
    dt = ts[0].dtype
    uo, op = UO[dt], OPERAND[dt]
    n = [_np(t) for t in (*ts, decay, st)]
    m = [np.abs(_np(t)) for t in (*clean, decay, st)]
    m[4][~np.isfinite(m[4])] = 1.0
    d = np.abs(_np(do))
    d[~np.isfinite(d)] = 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        wo, ws = O.decay_attention(*n, _np(lengths), scale)
        wg = O.decay_attention_backward(*n, _np(lengths), scale, _np(do), _np(dl))
        bo, bs = O.decay_attention(*m, _np(lengths), scale)
        bg = O.decay_attention_backward(*m, _np(lengths), scale, d, np.abs(_np(dl)))
        _reach(what + ": o", _np(o), wo, uo * np.abs(wo) + op * bo + 2.0 ** -24)
        _reach(what + ": state", _np(last), ws, 2.0 ** -18 * bs, signs=True)
        for name, g, w, b in zip(("dq", "dk", "dv"), grads, wg, bg):
            _reach(what + ": " + name, _np(g), w, uo * np.abs(w) + op * b + 2.0 ** -24)
        _reach(what + ": dstate", _np(grads[3]), wg[3], 2.0 ** -18 * bg[3], signs=True)


def _case(B, L, H, K, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = (r(B, L, H, d).to(dtype).to(DEV) for d in (K, K, V))
    decay = (1 - 2.0 ** -(1 + 6 * torch.arange(H).float() / max(H - 1, 1))).to(DEV)
    return q, k, v, decay, r(B, H, K, V).to(DEV), r(B, L, H, V).to(dtype).to(DEV), r(B, H, K, V).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("L,K,V", [(150, 24, 40), (150, 64, 64), (90, 32, 32), (70, 100, 128), (700, 16, 24)])
def test_bad_values_reach_what_the_recurrence_takes_them_to(L, K, V, bad, dtype):
    """One element of a token of one head in each sequence: of q, k, v or the outputs' gradient; first, inner, last of tiles."""
    places = [(name, t) for name in ("q", "k", "v", "do") for t in (0, 37, 47, L // 2, L - 1)]
    q, k, v, decay, st, do, dl = _case(len(places), L, 2, K, V, dtype, seed=L)
    ts = dict(q=q.clone(), k=k.clone(), v=v.clone(), do=do.clone())
    for b, (name, t) in enumerate(places):
        ts[name][b, t, 1, 3] = bad if b % 2 else -bad
    _check([ts[n] for n in "qkv"], (q, k, v), decay, st, None, K ** -0.5, ts["do"], dl, "all")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_several_bad_tokens_of_a_padded_batch(dtype):
    q, k, v, decay, st, do, dl = _case(3, 400, 2, 40, 64, dtype)
    lengths = torch.tensor([400, 257, 30], device=DEV)
    ts, d = [q.clone(), k.clone(), v.clone()], do.clone()
    ts[2][0, 5, 0, 7], ts[2][0, 9, 0, 8], ts[2][0, 300, 0, 9] = INF, NAN, -INF
    ts[1][1, 250, 1, 2], ts[1][1, 20, 0, 39], ts[0][1, 100, 0, 1] = NAN, INF, INF
    ts[2][2, 29], d[2, 11, 1, 4], ts[1][2, 31], ts[2][2, 30] = INF, NAN, NAN, NAN
    _check(ts, (q, k, v), decay, st, lengths, 0.2, d, dl, "several")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [NAN, INF])
def test_bad_values_under_decays_that_fade_at_once(bad, dtype):
    """Decays of 0 and of powers that leave float32's range within a tile: 0 x NaN is NaN, an infinity that fades is one."""
    for L in (200, 600):
        places = [(name, t) for name in ("q", "k", "v", "do") for t in (3, 60, 130)]
        q, k, v, _, st, do, dl = _case(len(places), L, 4, 16, 24, dtype, seed=L)
        decay = torch.tensor([0.0, 1e-30, 0.1, 1.0], device=DEV)
        ts = dict(q=q.clone(), k=k.clone(), v=v.clone(), do=do.clone())
        for b, (name, t) in enumerate(places):
            ts[name][b, t, :, 3] = bad
        _check([ts[n] for n in "qkv"], (q, k, v), decay, st, None, 0.25, ts["do"], dl, "all")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_bad_states(dtype):
    """NaN and infinities in the state that is carried in, and in the gradient of the one that is handed on."""
    for L in (1, 100, 900):
        q, k, v, decay, st, do, dl = _case(2, L, 2, 24, 32, dtype, seed=L)
        bad, d = st.clone(), dl.clone()
        bad[0, 1, 3, 4], bad[1, 0, 5, 6], d[1, 1, 7, 8], d[0, 0, 9, 10] = NAN, INF, -INF, NAN
        _check((q, k, v), (q, k, v), decay, bad, None, 0.2, do, dl, "state of %d" % L)
        _check((q, k, v), (q, k, v), decay, st, None, 0.2, do, d, "gradient of %d" % L)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_bad_values_in_a_sequence_of_many_segments(dtype):
    """125 segments, whose parts are joined by eight warps."""
    q, k, v, _, st, do, dl = _case(2, 16000, 2, 8, 8, dtype)
    decay = torch.tensor([0.1, 0.99], device=DEV)
    ts, s0 = [q.clone(), k.clone(), v.clone()], st.clone()
    ts[1][0, 9000, :, 1], ts[2][0, 12345, 0, 2], s0[0, 1, 5, 6], s0[1, 0, 3, 3] = INF, NAN, -INF, INF
    _check(ts, (q, k, v), decay, s0, None, 0.3, do, dl, "many")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,K,V", [(140, 24, 32), (90, 64, 64), (600, 16, 24)])
def test_the_largest_finite_values(L, K, V, dtype):
    """finfo.min and finfo.max are values like others where scores, sums (before the factor) and results are in range."""
    q, k, v, decay, st, do, dl = _case(5, L, 2, K, V, dtype, seed=L)
    # all others below 1: 3.4e38 times one above (v d_o is a score of dq) is no float32, nor 65504 times one a float16
    q, k, v, st, do, dl = q * 2.0 ** -12, k * 2.0 ** -6, *(t * 2.0 ** -4 for t in (v, st, do, dl))
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    v[0, 20, 1, 3], v[1, 70, 0, 4], q[2, 50, 1, 5] = low, high, low
    k[3, 61, 0, 2], v[3, 61, 0] = high, v[3, 61, 0] * 2.0 ** -10
    do[4, 33, 1, 7] = high
    _check((q, k, v), (q, k, v), decay, st, None, 2.0 ** -8, do, dl, "largest")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_bad_values_in_a_replayed_graph(dtype):
    """A captured training step meets a NaN and an infinity in one replay and none in the next."""
    q, k, v, decay, _, do, _ = _case(2, 1500, 3, 64, 64, dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step(ts):
        o = gfn.decay_attention(*ts, decay)
        return (o, *torch.autograd.grad(o, ts, do))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.detach().clone().requires_grad_(True) for t in leaves])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(leaves)
    for bad in (False, True, False):
        with torch.no_grad():
            k[0, 700, 1, 3] = NAN if bad else 1.0
            v[1, 10, 2, 5] = INF if bad else 1.0
        graph.replay()
        want = step([t.detach().clone().requires_grad_(True) for t in leaves])
        for a, b in zip(outs, want):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
        assert torch.isfinite(outs[0]).all().item() != bad
