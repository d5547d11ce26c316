"""GPU parity of decay_attention and its gradients against the float64
recurrence (oracle/lm_ops.py).

Tolerances are relative to the same sums over magnitudes (|q|, |k|, |v|): the
state and its gradient are float32 sums of products whose operands are exact or
split (float32: 2^-22 a product, twice; powers of the decay: a few 2^-23 each;
sums: 2^-24 a term over blocks of 64 and one addition a block), 2^-18 in all.
Outputs add the operand roundings: scores and state to bfloat16 (2^-8 each) for
bfloat16, to tf32's 11 bits (2^-11 each) for float16, and one rounding (uo) of
the result.
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


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _close(name, got, want, tol):
    assert got.shape == want.shape, name
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (name, int(bad.sum()), np.abs(got - want)[bad].max(), np.argwhere(bad)[0])


def _run(q, k, v, decay, state=None, lengths=None, scale=1.0, seed=0, train=True):
    n = [_np(t) for t in (q, k, v, decay, state, lengths)]
    ab = [None if t is None else np.abs(t) for t in n[:5]]
    uo, op, f32 = UO[q.dtype], OPERAND[q.dtype], 2.0 ** -18
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 1e-30
    with torch.no_grad():
        o, last = gfn.decay_attention(q, k, v, decay, state=state, return_state=True, lengths=lengths, scale=scale)
        alone = gfn.decay_attention(q, k, v, decay, state=state, lengths=lengths, scale=scale)
    assert torch.equal(o, alone) and o.dtype == q.dtype and last.dtype == torch.float32
    wo, ws = O.decay_attention(*n[:4], n[4], n[5], scale)
    bo, bs = O.decay_attention(*ab[:4], ab[4], n[5], abs(scale))
    _close("o", _np(o), wo, uo * np.abs(wo) + op * bo + tiny)
    _close("state", _np(last), ws, f32 * bs + 1e-30)
    if not train:
        return o, last
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, v, state)]
    o2, last2 = gfn.decay_attention(*leaves[:3], decay, state=leaves[3], return_state=True, lengths=lengths, scale=scale)
    if q.shape[1] != 1:  # one token without gradients has a kernel of its own
        assert torch.equal(o, o2) and torch.equal(last, last2)
    g = torch.Generator().manual_seed(seed)
    do = torch.randn(v.shape, generator=g).to(v.dtype).to(DEV)
    dl = torch.randn(last.shape, generator=g).to(DEV)
    some = [t for t in leaves if t is not None]
    grads = torch.autograd.grad((o2, last2), some, (do, dl))
    want = O.decay_attention_backward(*n[:4], n[4], n[5], scale, _np(do), _np(dl))
    big = O.decay_attention_backward(*ab[:4], ab[4], n[5], abs(scale), np.abs(_np(do)), np.abs(_np(dl)))
    for name, got, w, b in zip(("dq", "dk", "dv", "dstate"), grads, want, big):
        if name == "dstate":
            _close(name, _np(got), w, f32 * b + 1e-30)
        else:
            _close(name, _np(got), w, uo * np.abs(w) + op * b + tiny)
    return o, last


def _case(B, L, H, K, V, dtype, seed=0, state=True, ragged=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = (r(B, L, H, d).to(dtype).to(DEV) for d in (K, K, V))
    decay = (1 - 2.0 ** -(1 + 7 * torch.arange(H).float() / max(H - 1, 1))).to(DEV)
    st = r(B, H, K, V).to(DEV) if state else None
    lengths = torch.randint(0, L + 1, (B,), generator=g).to(DEV) if ragged else None
    return q, k, v, decay, st, lengths


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,H,K,V", [(1, 1, 1, 1, 1), (2, 1, 3, 64, 64), (1, 1, 2, 100, 128), (2, 2, 2, 16, 8),
                                       (1, 63, 2, 32, 32), (2, 64, 1, 64, 64), (1, 65, 2, 64, 32), (1, 33, 1, 128, 128),
                                       (2, 130, 3, 40, 72), (1, 129, 2, 7, 9), (1, 257, 1, 128, 64), (1, 200, 2, 33, 65)])
def test_outputs_state_and_gradients(B, L, H, K, V, dtype):
    q, k, v, decay, st, _ = _case(B, L, H, K, V, dtype, seed=L)
    _run(q, k, v, decay, st, None, K ** -0.5)
    _run(q, k, v, decay, None, None, 1.0, seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,H,K,V", [(1, 1100, 2, 64, 64), (3, 700, 1, 20, 24), (1, 1030, 1, 128, 96), (2, 2500, 2, 32, 16),
                                       (1, 16000, 1, 24, 9)])
def test_sequences_cut_into_segments(B, L, H, K, V, dtype):
    q, k, v, decay, st, lengths = _case(B, L, H, K, V, dtype, seed=L, ragged=True)
    _run(q, k, v, decay, st, None, K ** -0.5)
    _run(q, k, v, decay, st, lengths, K ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 64, 100, 600])
def test_padded_batches(L, dtype):
    """Lengths of zero, one and all; NaN and infinities behind them are not read."""
    q, k, v, decay, st, _ = _case(5, L, 2, 32, 40, dtype, seed=L)
    lengths = torch.tensor([0, 1, L, L // 2, max(L - 1, 0)], device=DEV)
    o, last = _run(q, k, v, decay, st, lengths)
    assert torch.equal(last[0], st[0]) and not o[0].any()
    behind = torch.arange(L, device=DEV) >= lengths.unsqueeze(1)
    for t in (q, k, v):
        t[behind] = float("nan")
    o2, last2 = gfn.decay_attention(q, k, v, decay, state=st, return_state=True, lengths=lengths.int())
    assert torch.equal(o, o2) and torch.equal(last, last2)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, st)]
    o2, last2 = gfn.decay_attention(*leaves[:3], decay, state=leaves[3], return_state=True, lengths=lengths)
    do = torch.ones_like(o2)
    do[behind] = float("nan")
    for g, t in zip(torch.autograd.grad((o2, last2), leaves, (do, torch.ones_like(last2))), leaves):
        assert torch.isfinite(g).all()
        assert t is leaves[3] or not g[behind].any()
    long = torch.tensor([-5, 1, L + 9, L // 2, max(L - 1, 0)], device=DEV)  # clamped
    assert torch.equal(gfn.decay_attention(q, k, v, decay, state=st, lengths=long)[1:], o[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_how_far_a_bad_token_reaches(bad, dtype):
    """Up to 15 tokens against the order of the pass, one sequence, one head."""
    q, k, v, decay, st, _ = _case(2, 300, 2, 24, 40, dtype)
    do = torch.randn(v.shape, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)

    def both(*ts):
        leaves = [t.clone().requires_grad_(True) for t in ts]
        o = gfn.decay_attention(*leaves, decay, state=st)
        return (o, *torch.autograd.grad(o, leaves, do))
    want = both(q, k, v)
    for i in range(3):
        for t in (70, 127, 128, 200):
            ts = [q.clone(), k.clone(), v.clone()]
            ts[i][1, t, 1] = bad
            got = both(*ts)
            for a, b in zip(got, want):
                assert torch.equal(a[0], b[0]) and torch.equal(a[1, :, 0], b[1, :, 0])  # other sequences, other heads
            early, late = slice(0, t - 15), slice(t + 16, None)
            if i == 0:  # q: its own output; dk and dv before it, and up to 15 tokens behind
                assert torch.equal(got[0][1, :t], want[0][1, :t]) and torch.equal(got[0][1, t + 1:], want[0][1, t + 1:])
                for g, w in zip(got[2:], want[2:]):
                    assert torch.equal(g[1, late], w[1, late])
                assert torch.equal(got[1], want[1])
            else:  # k, v: outputs from the token on, and up to 15 before
                assert torch.equal(got[0][1, early], want[0][1, early])
                assert not torch.isfinite(got[0][1, t, 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_decays_from_0_to_1(dtype):
    q, k, v, _, st, _ = _case(1, 150, 6, 16, 24, dtype)
    decay = torch.tensor([0.0, 1e-30, 1e-3, 0.5, 1 - 2.0 ** -20, 1.0], device=DEV)
    _run(q, k, v, decay, st, None, 0.25)
    q, k, v, _, st, _ = _case(2, 1, 6, 16, 24, dtype)
    _run(q, k, v, decay, st, None, 0.25)
    outside = torch.tensor([-3.0, 1e-30, 1e-3, 0.5, 1 - 2.0 ** -20, 7.0], device=DEV)
    assert torch.equal(gfn.decay_attention(q, k, v, outside, state=st), gfn.decay_attention(q, k, v, decay, state=st))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,V", [(64, 64), (24, 40), (13, 27)])
def test_a_sequence_in_segments_and_single_tokens(K, V, dtype):
    """Segment by segment and token by token from the carried state: within both runs' tolerances."""
    q, k, v, decay, st, _ = _case(2, 140, 2, K, V, dtype)
    o, last = _run(q, k, v, decay, st, None, 0.3, train=False)
    n = [_np(t) for t in (q, k, v, decay, st)]
    bo, bs = O.decay_attention(*[np.abs(t) for t in n], None, 0.3)
    s, parts = st, []
    for a, b in ((0, 70), (70, 71), (71, 72), (72, 140)):
        y, s = gfn.decay_attention(q[:, a:b], k[:, a:b], v[:, a:b], decay, state=s, return_state=True, scale=0.3)
        parts.append(y)
    y = torch.cat(parts, 1)
    _close("o", _np(y), _np(o), 2 * UO[dtype] * np.abs(_np(o)) + 2 * OPERAND[dtype] * bo)
    _close("state", _np(s), _np(last), 2.0 ** -17 * bs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_of_operands(dtype):
    """Views of one projection, [batch, heads, length, dim], rows off 16 bytes, k and v shared by the heads."""
    q, k, v, decay, st, _ = _case(2, 90, 4, 32, 32, dtype)
    o, last = _run(q, k, v, decay, st)
    same = lambda a, b, c: torch.equal(gfn.decay_attention(a, b, c, decay, state=st), o)  # noqa: E731
    z = torch.stack([q, k, v], 3)
    assert same(z[..., 0, :], z[..., 1, :], z[..., 2, :])
    assert same(*[t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)])
    assert same(*[t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)])
    wide = torch.zeros(2, 90, 4, 37, device=DEV, dtype=dtype)
    wide[..., 3:35] = k
    assert same(q, wide[..., 3:35], v)
    one_k, one_v = k[:, :, :1].detach().requires_grad_(True), v[:, :, :1].detach().requires_grad_(True)
    y = gfn.decay_attention(q, one_k.expand_as(k), one_v.expand_as(v), decay, state=st)
    _run(q, one_k.detach().expand_as(k), one_v.detach().expand_as(v), decay, st)
    do = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    gk, gv = torch.autograd.grad(y, [one_k, one_v], do)
    n = [_np(t) for t in (q, one_k.expand_as(k), one_v.expand_as(v), decay, st)]
    w = O.decay_attention_backward(*n, None, 1.0, _np(do))
    b = O.decay_attention_backward(*[np.abs(t) for t in n], None, 1.0, np.abs(_np(do)))
    for got, i in ((gk, 1), (gv, 2)):  # rounded per head, then summed and rounded by PyTorch
        _close("shared", _np(got), w[i].sum(2, keepdims=True),
               (OPERAND[dtype] + 4 * UO[dtype]) * b[i].sum(2, keepdims=True) + 1e-6)
    leaf = q.clone().requires_grad_(True)
    g, = torch.autograd.grad(gfn.decay_attention(leaf, k, v, decay).sum(), leaf)  # a broadcast gradient
    assert torch.isfinite(g).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_single_gradients_and_absent_ones(dtype):
    q, k, v, decay, st, _ = _case(1, 80, 2, 16, 16, dtype)
    do, dl = torch.randn(v.shape, device=DEV).to(dtype), torch.randn(st.shape, device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, st)]
    o, last = gfn.decay_attention(*leaves[:3], decay, state=leaves[3], return_state=True)
    want = torch.autograd.grad((o, last), leaves, (do, dl))
    for i in range(4):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v, st))]
        o, last = gfn.decay_attention(*some[:3], decay, state=some[3], return_state=True)
        g, = torch.autograd.grad((o, last), [some[i]], (do, dl))
        assert torch.equal(g, want[i])
    o, last = gfn.decay_attention(*leaves[:3], decay, state=leaves[3], return_state=True)
    n = [_np(t) for t in (q, k, v, decay, st)]
    w = O.decay_attention_backward(*n, None, 1.0, None, _np(dl))
    b = O.decay_attention_backward(*[np.abs(t) for t in n], None, 1.0, None, np.abs(_np(dl)))
    grads = torch.autograd.grad(last, leaves, dl, allow_unused=True)  # the state alone
    for got, x, y in zip(grads, w, b):
        assert got is not None
        _close("state alone", _np(got), x, UO[dtype] * np.abs(x) + OPERAND[dtype] * y + 1e-7)


@pytest.mark.gpu
def test_float16_beyond_its_range_inside():
    """Scores and states above 65504 whose outputs are not."""
    q = torch.full((1, 200, 1, 32), 60.0, device=DEV, dtype=torch.float16)
    k = torch.full((1, 200, 1, 32), 60.0, device=DEV, dtype=torch.float16)
    v = torch.full((1, 200, 1, 32), 2.0 ** -12, device=DEV, dtype=torch.float16)
    _run(q, k, v, torch.ones(1, device=DEV), None, None, 2.0 ** -4, train=False)
    v[:] = 100.0
    _run(q * 2.0 ** -12, k * 20, v, torch.ones(1, device=DEV), None, None, 2.0 ** -13, train=False)


@pytest.mark.gpu
def test_empty_sequences_and_batches():
    q, k, v, decay, st, _ = _case(2, 4, 3, 16, 8, torch.float32)
    leaves = [t[:, :0].clone().requires_grad_(True) for t in (q, k, v)] + [st.clone().requires_grad_(True)]
    o, last = gfn.decay_attention(*leaves[:3], decay, state=leaves[3], return_state=True)
    assert o.shape == (2, 0, 3, 8) and torch.equal(last, st)
    g, = torch.autograd.grad(last, leaves[3], st * 2)
    assert torch.equal(g, st * 2)
    o, last = gfn.decay_attention(q[:, :0], k[:, :0], v[:, :0], decay, return_state=True)
    assert not last.any()
    assert gfn.decay_attention(q[:0], k[:0], v[:0], decay).shape == (0, 4, 3, 8)


@pytest.mark.gpu
def test_repeats_bit_for_bit():
    q, k, v, decay, st, lengths = _case(2, 3000, 3, 64, 64, torch.bfloat16, ragged=True)
    leaves = [t.requires_grad_(True) for t in (q, k, v, st)]

    def once():
        o, last = gfn.decay_attention(*leaves[:3], decay, state=leaves[3], return_state=True, lengths=lengths)
        return (o, last, *torch.autograd.grad((o, last), leaves, (torch.ones_like(o), torch.ones_like(last))))
    first = once()
    for _ in range(3):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_far_apart_tokens_and_offsets_past_32_bits(dtype):
    """Views whose batch or token stride passes 2^31 elements, in and behind the same allocation."""
    size = 2 if dtype != torch.float32 else 4
    base = torch.zeros(2 ** 31 // 2 * 3, device=DEV, dtype=dtype)  # 2^31 elements lie between the first and the last third
    q, k, v, decay, st, _ = _case(3, 5, 2, 16, 16, dtype)
    far = lambda t, at: base.as_strided(t.shape, (2 ** 30 + 8 * size, 64, 16, 1), at).copy_(t)  # noqa: E731
    a, b, c = far(q, 0), far(k, 1024), far(v, 2048)
    o, last = gfn.decay_attention(q, k, v, decay, state=st, return_state=True)
    o2, last2 = gfn.decay_attention(a, b, c, decay, state=st, return_state=True)
    assert torch.equal(o, o2) and torch.equal(last, last2)
    del base, a, b, c


@pytest.mark.gpu
def test_a_million_tokens():
    """One long sequence: the state behind 2^20 tokens against float64 sums (a decay of 1 adds them all)."""
    n = 2 ** 20 + 37
    g = torch.Generator(device=DEV).manual_seed(0)
    q, k, v = (torch.randn(1, n, 1, 8, device=DEV, generator=g).bfloat16() for _ in range(3))
    for gam in (1.0, 1 - 2.0 ** -10):
        decay = torch.tensor([gam], device=DEV)
        o, last = gfn.decay_attention(q, k, v, decay, return_state=True)
        w = gam ** torch.arange(n - 1, -1, -1, device=DEV, dtype=torch.float64)
        want = torch.einsum("t,tk,tv->kv", w, k[0, :, 0].double(), v[0, :, 0].double())
        big = torch.einsum("t,tk,tv->kv", w, k[0, :, 0].double().abs(), v[0, :, 0].double().abs())
        assert ((last[0, 0] - want).abs() <= 2.0 ** -18 * big).all()
        tail = (q[0, -1, 0].double() @ want)
        bound = 2.0 ** -8 * (q[0, -1, 0].double().abs() @ want.abs()) + 2.0 ** -8 * tail.abs() + 2.0 ** -8 * 64 * 8 * 16
        assert ((o[0, -1, 0] - tail).abs() <= bound).all()
