"""GPU parity of token_logprobs and its gradient against the float64 row-by-row
definition (oracle/lm_ops.py).

Tolerances, with u = 2^-24 and c = vocab / 256 + 40 terms in a chain of sums: an
exponential is off by 2^-22 of itself plus u times its argument's size (twice, for
the difference and the product by log2 e), Z by that and c u.  Terms that matter
have arguments below 32, which makes 2^-18 + c u of Z; log Z and the differences
add u of their own size.  The entropy carries the same on sums no larger than
log V + 1 times as large, the gradient on p (|sum of g| + |g_H| (|log p| + H)),
plus one rounding to the logits' type (uo).
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from oracle import lm_ops as O

DEV = "cuda:0"
U = 2.0 ** -24
UO = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _close(got, want, tol):
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # the results are float32: lowest - highest = -6.8e38 is -inf there (rounding to nearest goes to
    # infinity from (2 - 2^-24) 2^127 = 3.4028236e38 on)
    want = np.where(np.abs(want) >= (2 - 2.0 ** -24) * 2.0 ** 127, np.copysign(np.inf, want), want)
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    ok = ~(inf | np.isnan(want))
    bad = ~(np.abs(got - want)[ok] <= np.broadcast_to(tol, want.shape)[ok])
    assert not bad.any(), (int(bad.sum()), np.abs(got - want)[ok].max())


def _check(logits, tokens, top, seed=0, ignore=-100, parts=("lp", "ent", "top")):
    """Forward (with and without gradients) and backward of the asked parts."""
    N, V = logits.shape
    x = _np(logits)
    lp, ent, tlp, tid = O.token_logprobs(x, _np(tokens), top, ignore)
    with np.errstate(invalid="ignore"):
        m = x.max(-1)
    eps = 2.0 ** -18 + (V / 256 + 40) * U
    span = np.log(V) + 1
    leaf = logits.detach().requires_grad_(True)
    r = gfn.token_logprobs(leaf, tokens, top=top, entropy=True, ignore_index=ignore)
    with torch.no_grad():
        again = gfn.token_logprobs(logits, tokens, top=top, entropy=True, ignore_index=ignore)
    for a, b in zip(r, again):
        assert (a is None) == (b is None) and (a is None or torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)))
    with np.errstate(invalid="ignore"):
        _close(_np(r.logprobs), lp, eps + 4 * U * (np.abs(lp) + span))
        _close(_np(r.entropy), ent, 2 * eps * span)
    if top:
        assert np.array_equal(_np(r.top_tokens), tid)
        with np.errstate(invalid="ignore"):
            _close(_np(r.top_logprobs), tlp, eps + 4 * U * (np.abs(tlp) + span))
    g = torch.Generator().manual_seed(seed)
    glp, gent, gtop = torch.randn(N, generator=g), torch.randn(N, generator=g), torch.randn(N, max(top, 1), generator=g)
    outs, grads = [], []
    if "lp" in parts:
        outs.append(r.logprobs), grads.append(glp.to(DEV))
    if "ent" in parts:
        outs.append(r.entropy), grads.append(gent.to(DEV))
    if "top" in parts and top:
        outs.append(r.top_logprobs), grads.append(gtop.to(DEV))
    d, = torch.autograd.grad(outs, leaf, grads)
    rows = np.isfinite(m) | (x == -np.inf).all(-1)  # rows without NaN or +inf
    assert np.isnan(_np(d)[~rows]).all()
    pick = lambda name, t: _np(t)[rows] if name in parts else None  # noqa: E731
    gt = pick("top", gtop) if top else None
    want = O.token_logprobs_backward(x[rows], _np(tokens)[rows], tid[rows], pick("lp", glp), pick("ent", gent), gt, ignore)
    p = np.exp(x[rows] - np.where(np.isfinite(m[rows]), m[rows], 0)[:, None])
    p /= np.maximum(p.sum(-1, keepdims=True), 1e-300)
    total = (np.abs(_np(glp)[rows]) + np.abs(_np(gtop)[rows]).sum(-1) + 2 * span * np.abs(_np(gent)[rows]))[:, None]
    with np.errstate(divide="ignore"):
        big = p * total * (1 + np.minimum(-np.log(np.maximum(p, 1e-300)), 100))
    direct = np.abs(_np(glp)[rows]) + np.abs(_np(gtop)[rows]).sum(-1)
    uo = UO[logits.dtype]
    _close(_np(d)[rows], want, uo * np.abs(want) + 4 * eps * big + 8 * U * direct[:, None] * (want != 0) + 2.0 ** -24)
    assert d.dtype == logits.dtype
    return r, d


def _case(N, V, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(N, V, generator=g)).to(dtype).to(DEV)
    return x, torch.randint(0, V, (N,), generator=g).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (2, 32, 32), (5, 33, 20), (1, 100, 32), (9, 1000, 1),
                                     (4, 1025, 32), (2, 4099, 5), (300, 515, 8), (1, 32000, 20), (2, 50257, 32),
                                     (700, 2049, 4), (5, 131071, 32)])
def test_logprobs_entropy_top_and_gradient(N, V, top, dtype):
    x, t = _case(N, V, dtype, seed=V)
    _check(x, t, top, seed=N)
    assert gfn.cuda.ops.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [64, 5000, 50257])
def test_masked_logits(V, dtype):
    """Rows that a grammar leaves many, few, one and no tokens; given tokens inside and outside the mask."""
    x, t = _case(8, V, dtype, seed=V)
    keep = torch.rand(8, V, generator=torch.Generator().manual_seed(1)).to(DEV)
    x = x.masked_fill(keep > torch.tensor([1.0, 0.5, 20 / V, 5 / V, 0, 0, 0, 0.1], device=DEV).unsqueeze(1), -float("inf"))
    x[4, V // 3] = 2.0
    x[5, V - 1] = -1e4
    t[4], t[5] = V // 3, V - 1
    r, d = _check(x, t, 20)
    assert r.logprobs[4] == 0 and r.entropy[4] == 0 and r.logprobs[5] == 0
    assert r.logprobs[6] == -float("inf") and r.entropy[6] == 0 and not d[6].any()
    assert r.top_tokens[6].tolist() == list(range(20))
    assert (d[x == -float("inf")] == 0).logical_or((t.unsqueeze(1) == torch.arange(V, device=DEV))[x == -float("inf")]).logical_or(
        (r.top_tokens.unsqueeze(2) == torch.arange(V, device=DEV)).any(1)[x == -float("inf")]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [2, 700])
def test_ties_nan_and_infinities(N, dtype):
    """Constant rows, -0 against 0, large logits all in one thread's part, NaN and +inf."""
    V = 4096 * 3 + 5
    x, t = _case(N, V, dtype, seed=3)
    x[0] = 1.25
    _check(x, t, 32)
    x[0] = 0.0
    x[0, ::2] = -0.0
    x[1, 5::256 * 16 // x.element_size()] = 50.0
    _check(x, t, 32)
    x[1] = torch.arange(V, device=DEV).to(dtype)  # rising, ties in 16 bits
    _check(x, t, 9)
    x[0, 0:16 // x.element_size()] = 60.0
    x[0, 256 * 16 // x.element_size() * torch.arange(1, 20, device=DEV) % V] = 61.0
    x[0] = torch.where(torch.arange(V, device=DEV) // (16 // x.element_size()) % 256 < 4, 40.0 + x[0].float() / 8, -40.0).to(dtype)
    _check(x, t, 32)
    x[0, V // 2] = float("nan")
    x[0, 7] = float("nan")
    x[1, 9] = float("inf")
    r, _ = _check(x, t, 5)
    assert r.top_tokens[0, :2].tolist() == [7, V // 2] and r.top_tokens[1, 0] == 9
    assert gfn.cuda.ops.device_error() == 0


@pytest.mark.gpu
def test_logits_of_any_size():
    for shift in (1e4, -1e4, 3e30):
        x, t = _case(3, 999, torch.float32)
        if abs(shift) < 1e10:
            x += shift
            x = x.round()  # differences that float32 holds
        else:
            x[:, 5] = shift
        _check(x, t, 4)
    x, t = _case(3, 999, torch.float16, spread=1.0)
    x[:, 3] = 65504.0
    x[1, 4] = -65504.0
    _check(x, t, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [3, 700])
def test_masks_of_the_types_lowest_value(N, dtype):
    """A mask of finfo.min instead of -inf: probability 0 beside others, and a uniform row where it is all there is."""
    V, low = 1003, torch.finfo(dtype).min
    x, t = _case(N, V, dtype)
    x[0] = low
    x[1, 5:] = low
    x[2, ::2] = torch.finfo(dtype).max
    x[2, 1::2] = low
    t[1] = 3
    r, d = _check(x, t, 7)
    assert abs(r.entropy[0].item() - np.log(V)) < 1e-5 and r.top_tokens[0].tolist() == list(range(7))
    assert r.top_tokens[1].tolist()[5:] == [5, 6] and torch.isfinite(d).all()


@pytest.mark.gpu
@pytest.mark.parametrize("parts", [("lp",), ("ent",), ("top",), ("lp", "ent"), ("lp", "top"), ("ent", "top")])
def test_each_result_alone_and_its_gradient(parts):
    x, t = _case(40, 777, torch.float32)
    t[::5] = -100
    full, _ = _check(x, t, 6, parts=parts)
    r = gfn.token_logprobs(x, t if "lp" in parts else None, top=6 if "top" in parts else 0, entropy="ent" in parts)
    assert [v is not None for v in r] == ["lp" in parts, "ent" in parts, "top" in parts, "top" in parts]
    for a, b in zip(r, full):
        assert a is None or torch.equal(a, b)
    leaf = x.clone().requires_grad_(True)
    r = gfn.token_logprobs(leaf, t, top=6, entropy=True)
    assert not r.top_tokens.requires_grad and r.entropy.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_and_strides_of_operands(dtype):
    x, t = _case(12, 300, dtype)
    base, d0 = _check(x, t, 5)
    wide = torch.randn(12, 311, device=DEV).to(dtype)
    wide[:, 7:307] = x
    r, d = _check(wide[:, 7:307], t, 5)
    for a, b in zip(r, base):
        assert (a == b).all() or (a - b).abs().max() < 1e-5
    assert d.shape == d0.shape
    _check(x.t().contiguous().t(), t, 5)
    _check(x[:1].expand(12, 300), t, 5)
    lead = x.view(3, 4, 300).requires_grad_(True)
    r = gfn.token_logprobs(lead, t.view(3, 4).int(), top=5, entropy=True)
    assert r.logprobs.shape == (3, 4) and r.top_tokens.shape == (3, 4, 5)
    assert torch.equal(r.logprobs.flatten(), base.logprobs)
    g, = torch.autograd.grad(r.top_logprobs[..., 1:3].sum() + r.logprobs.mean(), lead)  # broadcast and sliced gradients
    assert g.shape == lead.shape and torch.isfinite(g).all()
    one = gfn.token_logprobs(x[0].detach(), t[0], top=2)
    assert one.logprobs.shape == () and one.top_tokens.shape == (2,)
    none = gfn.token_logprobs(x[:0], t[:0], top=2, entropy=True)
    assert none.top_logprobs.shape == (0, 2)


@pytest.mark.gpu
def test_given_tokens_ignored_and_outside():
    x, t = _case(20, 90, torch.float32)
    t[3], t[4] = -100, 0
    _check(x, t, 3)
    _check(x, t.clamp(min=0), 3, ignore=0)  # a token of the vocabulary may be the ignored one
    assert gfn.cuda.ops.device_error() == 0
    t[3] = 90
    leaf = x.clone().requires_grad_(True)
    r = gfn.token_logprobs(leaf, t)
    assert torch.isnan(r.logprobs[3]) and torch.isfinite(r.logprobs[4:]).all()
    assert gfn.cuda.ops.device_error() == 2
    g, = torch.autograd.grad(r.logprobs.sum(), leaf)
    assert torch.isnan(g[3]).all() and torch.isfinite(g[4:]).all() and torch.isfinite(g[:3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 300, 2000])
def test_a_given_token_among_the_alternatives_has_the_same_bits(N):
    x, _ = _case(N, 3001, torch.float32)
    r = gfn.token_logprobs(x, x.argmax(-1), top=3)
    assert torch.equal(r.logprobs, r.top_logprobs[:, 0]) and torch.equal(r.top_tokens[:, 0], x.argmax(-1))
    assert (r.top_logprobs <= 0).all()


@pytest.mark.gpu
def test_generate_with_logprobs():
    torch.manual_seed(0)
    m = gfn.Manifold(vocab_size=17, dim=16, depth=1, heads=2, use_scan=True).to(DEV)
    prompt = torch.tensor([[1, 2, 3]], device=DEV)
    plain = m.generate(prompt, max_new_tokens=5)
    ids, info = m.generate(prompt, max_new_tokens=5, logprobs=3)
    assert ids == plain and len(info) == 5
    seen = torch.tensor([ids], device=DEV)
    for i, step in enumerate(info):
        logits = m(seen[:, :3 + i])[0][0, -1].double() if i == 0 else m(seen[:, 2 + i:3 + i])[0][0, -1].double()
        want = torch.log_softmax(logits, -1)
        assert step["token"] == ids[3 + i] and abs(step["logprob"] - want[ids[3 + i]].item()) < 1e-4
        assert step["top_tokens"][0] == ids[3 + i] and len(step["top_logprobs"]) == 3 and step["entropy"] > 0
