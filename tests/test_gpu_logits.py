"""GPU parity of process_logits against the float64 row-by-row definition
(oracle/lm_ops.py), its masks and refusals, and generate() with them.

Tolerance: the penalty, the bias and the division round once each in float32
(u = 2^-24) on terms no larger than |x| max(rep, 1) + freq c + pres + |bias|;
the result is rounded once to the logits' type (uo).
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from oracle import lm_ops as O

DEV = "cuda:0"
U = 2.0 ** -24
UO = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _np(t):
    return t.detach().double().cpu().numpy() if torch.is_tensor(t) and t.is_floating_point() else (
        t.detach().cpu().numpy() if torch.is_tensor(t) else t)


def _compare(logits, out, **kw):
    n = {k: _np(v) for k, v in kw.items()}
    want = O.process_logits(_np(logits), **n)
    col = lambda k, d: np.broadcast_to(np.asarray(n.get(k, d), np.float64), (logits.shape[0],))[:, None]  # noqa: E731
    bias = np.abs(n["bias"]) if n.get("bias") is not None else 0.0
    T = 0 if n.get("tokens") is None else n["tokens"].shape[1]
    big = (np.abs(_np(logits)) * np.maximum(col("rep", 1.0), 1 / col("rep", 1.0)) + np.abs(col("freq", 0.0)) * T
           + np.abs(col("pres", 0.0)) + bias) / col("temperature", 1.0)
    got = _np(out)
    assert got.shape == want.shape and out.dtype == logits.dtype
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    tol = 2.0 ** -24 + UO[logits.dtype] * np.abs(want) + 8 * U * big
    bad = ~(np.abs(got - want)[~inf] <= tol[~inf])
    assert not bad.any(), (int(bad.sum()), np.abs(got - want)[~inf].max())


def _case(B, V, T, dtype, seed, per_row=True, bias=None, mask=None):
    g = torch.Generator().manual_seed(seed)
    logits = (4 * torch.randn(B, V, generator=g)).to(dtype).to(DEV)
    # few distinct tokens: every history repeats some
    tokens = (torch.rand(B, T, generator=g) ** 3 * min(V, 50)).long().clamp_(max=V - 1).to(DEV)
    lengths = torch.randint(0, T + 1, (B,), generator=g).to(DEV)
    prompts = (torch.rand(B, generator=g) * (lengths.cpu() + 1)).long().to(DEV)
    par = [1 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g),
           0.5 + torch.rand(B, generator=g)]
    par = [p.to(DEV) for p in par] if per_row else [float(p[0]) for p in par]
    bt = None
    if bias == "shared":
        bt = torch.randn(V, generator=g).to(DEV)
    elif bias == "row":
        bt = torch.randn(B, V, generator=g).to(DEV)
    mt = None
    if mask == "shared":
        mt = (torch.rand(V, generator=g) < 0.3).to(DEV)
    elif mask == "row":
        mt = (torch.rand(B, V, generator=g) < torch.rand(B, 1, generator=g)).to(DEV)
    return logits, tokens, lengths, prompts, par, bt, mt


def _run(logits, tokens, lengths, prompts, par, bt, mt, packed=True):
    rep, freq, pres, temp = par
    out = gfn.process_logits(logits, tokens, lengths, prompts, rep, freq, pres, bt, temp,
                             gfn.pack_token_mask(mt) if mt is not None and packed else mt)
    _compare(logits, out, tokens=tokens, lengths=lengths, prompt_lengths=prompts, rep=rep, freq=freq, pres=pres,
             bias=bt, temperature=temp, allowed=mt)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,V,T,bias,mask", [(1, 1, 1, None, None), (1, 7, 3, "shared", "row"),
                                             (3, 32, 40, "row", "shared"), (2, 33, 9, None, "row"),
                                             (5, 1000, 64, "row", "row"), (2, 4097, 300, "shared", None),
                                             (1, 32000, 50, None, None), (9, 8200, 1, "row", "row"),
                                             (4, 50257, 200, "row", "row"), (70, 515, 17, "shared", "shared")])
def test_process_logits_matches_definition(B, V, T, bias, mask, dtype):
    _run(*_case(B, V, T, dtype, B + V + T, True, bias, mask))
    _run(*_case(B, V, T, dtype, B + V + T + 1, False, bias, mask), packed=False)


@pytest.mark.gpu
def test_process_logits_optional_operands():
    lg, tok, ln, pr, par, bt, mt = _case(4, 777, 30, torch.float32, 3, True, "row", "row")
    _run(lg, tok, None, None, par, None, None)
    _run(lg, tok, ln, None, par, None, mt)
    _run(lg, tok, None, pr, par, bt, None)
    _run(lg, None, None, None, par, bt, mt)
    _run(lg, tok[:, :0], None, None, par, bt, mt)
    assert torch.equal(gfn.process_logits(lg), lg)
    out = gfn.process_logits(lg, tok.int(), ln.int(), pr.int(), *par[:3], bt, par[3], mt)
    assert torch.equal(out, _run(lg, tok, ln, pr, par, bt, mt))
    assert gfn.process_logits(lg[:0]).shape == (0, 777)


@pytest.mark.gpu
def test_process_logits_long_history_of_one_token():
    # every count in one word: 5000 increments of one shared-memory counter
    lg = torch.randn(2, 9000, device=DEV)
    tok = torch.full((2, 5000), 8999, device=DEV, dtype=torch.int64)
    out = gfn.process_logits(lg, tok, frequency_penalty=0.25, presence_penalty=0.5)
    assert torch.equal(out[:, :-1], lg[:, :-1])
    torch.testing.assert_close(out[:, -1], lg[:, -1] - 1250.5)


@pytest.mark.gpu
def test_process_logits_empty_masks_and_special_values():
    lg = torch.randn(3, 100, device=DEV)
    lg[0, 1], lg[0, 2], lg[0, 3] = float("-inf"), float("inf"), float("nan")
    lg[1] = torch.finfo(torch.float32).min  # masked by the type's lowest value
    tok = torch.tensor([[1, 2, 3], [4, 5, 6], [7, 8, 9]], device=DEV)
    mask = torch.ones(3, 100, device=DEV, dtype=torch.bool)
    mask[2] = False
    out = gfn.process_logits(lg, tok, repetition_penalty=2.0, allowed=mask)
    assert out[0, 1] == float("-inf") and out[0, 2] == float("inf") and torch.isnan(out[0, 3])
    assert (out[1, 4:7] == float("-inf")).all()  # twice the lowest value
    assert (out[1, 7:] == lg[1, 7:]).all()
    assert (out[2] == float("-inf")).all()       # a mask that leaves nothing
    mask[0, 1:4] = False                         # masked places hold -inf whatever was there
    assert (gfn.process_logits(lg, tok, repetition_penalty=2.0, allowed=mask)[0, 1:4] == float("-inf")).all()


@pytest.mark.gpu
def test_process_logits_bits_past_the_vocabulary_are_ignored():
    lg = torch.randn(2, 40, device=DEV)
    words = torch.tensor([[0, -256], [5, -1]], device=DEV, dtype=torch.int32)  # row 0 allows tokens >= 40 only
    out = gfn.process_logits(lg, allowed=words)
    assert (out[0] == float("-inf")).all()
    keep = [0, 2] + list(range(32, 40))
    assert torch.equal(out[1, keep], lg[1, keep]) and int(torch.isinf(out[1]).sum()) == 30


@pytest.mark.gpu
def test_process_logits_tokens_outside_the_vocabulary():
    gfn.cuda.ops.device_error()
    lg = torch.randn(1, 64, device=DEV)
    tok = torch.tensor([[3, 64, -1, 2 ** 40, 3]], device=DEV)
    out = gfn.process_logits(lg, tok, frequency_penalty=1.0)
    want = lg.clone()
    want[0, 3] -= 2.0
    assert torch.equal(out, want)
    assert gfn.cuda.ops.device_error() & 2
    # beyond a row's length anything may stand
    gfn.process_logits(lg, tok, torch.tensor([1], device=DEV), frequency_penalty=1.0)
    assert gfn.cuda.ops.device_error() == 0
    out = gfn.process_logits(lg, tok[:, :1], torch.tensor([9], device=DEV), torch.tensor([-4], device=DEV),
                             frequency_penalty=1.0)  # lengths are clamped to the history
    want[0, 3] = lg[0, 3] - 1.0
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_process_logits_strides(dtype):
    lg, tok, ln, pr, par, bt, mt = _case(4, 999, 20, dtype, 8, True, "row", "row")
    wide = torch.zeros(4, 3, 1001, device=DEV, dtype=dtype)
    wide[:, 1, 1:1000] = lg
    words = gfn.pack_token_mask(mt)
    big_w = torch.zeros(4, words.shape[1] + 3, device=DEV, dtype=torch.int32)
    big_w[:, 2:-1] = words
    ref = _run(lg, tok, ln, pr, par, bt, mt)
    for x in (wide[:, 1, 1:1000], lg.t().contiguous().t()):
        out = gfn.process_logits(x, torch.stack([tok, tok], -1)[..., 0], ln, pr, *par[:3],
                                 torch.cat([bt, bt], 1)[:, 999:], par[3], big_w[:, 2:-1])
        assert torch.equal(out, ref)


@pytest.mark.gpu
def test_process_logits_refusals_on_the_gpu():
    lg = torch.zeros(2, 64, device=DEV)
    tok = torch.zeros(2, 3, device=DEV, dtype=torch.int64)
    two = torch.ones(2, device=DEV)
    for kw in (dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(temperature=0.0),
               dict(temperature=float("nan")), dict(bias=torch.zeros(63, device=DEV)),
               dict(tokens=tok.float()), dict(tokens=tok[:1]), dict(lengths=tok[:, 0]),
               dict(tokens=tok, lengths=tok), dict(temperature=two.double()), dict(temperature=torch.ones(3, device=DEV)),
               dict(allowed=torch.ones(64, device=DEV)), dict(allowed=torch.ones(65, device=DEV, dtype=torch.bool)),
               dict(allowed=torch.ones(3, device=DEV, dtype=torch.int32)), dict(temperature=two.cpu()),
               dict(tokens=tok.cpu())):
        with pytest.raises(gfn.GfnError):
            gfn.process_logits(lg, **kw)
    for bad in (lg[0], lg.double(), lg.clone().requires_grad_(True), lg[:, :0]):
        with pytest.raises(gfn.GfnError):
            gfn.process_logits(bad)


@pytest.mark.gpu
@pytest.mark.parametrize("name,shape", [("bias", (64,)), ("repetition_penalty", (2,)), ("frequency_penalty", (2,)),
                                        ("presence_penalty", (2,)), ("temperature", (2,))])
def test_process_logits_refuses_to_cut_a_gradient(name, shape):
    """No operand that wants a gradient is silently detached."""
    lg, t = torch.zeros(2, 64, device=DEV), torch.ones(shape, device=DEV, requires_grad=True)
    with pytest.raises(gfn.GfnError):
        gfn.process_logits(lg, **{name: t})
    with torch.no_grad():
        gfn.process_logits(lg, **{name: t})
    gfn.process_logits(lg, **{name: t.detach()})


def test_process_logits_refusals():
    with pytest.raises(gfn.GfnError):  # no CPU path
        gfn.process_logits(torch.zeros(1, 8))
    with pytest.raises(gfn.GfnError):
        gfn.pack_token_mask(torch.zeros(4))
    lib = gfn._lib.load()
    tail = [1.0, None, 0.0, None, 0.0, None, 1.0, None, None, 0, None, 0]
    assert lib.gfn_process_logits(None, 8, 0, 1, 8, None, 0, 0, None, None, *tail, None, None) == 1
    assert lib.gfn_process_logits(16, 8, 0, 1, 8, None, 0, 3, None, None, *tail, 16, None) == 1  # no tokens
    assert lib.gfn_process_logits(16, 8, 9, 1, 8, None, 0, 0, None, None, *tail, 16, None) == 2  # element type
    tail[6] = 0.0
    assert lib.gfn_process_logits(16, 8, 0, 1, 8, None, 0, 0, None, None, *tail, 16, None) == 1  # temperature


def test_pack_token_mask():
    m = torch.zeros(2, 70, dtype=torch.bool)
    m[0, 0] = m[0, 31] = m[0, 33] = m[1, 69] = True
    w = gfn.pack_token_mask(m)
    assert w.tolist() == [[1 - 2 ** 31, 2, 0], [0, 0, 32]] and w.dtype == torch.int32


# ----------------------------------------------------- in a model's hands
def _scan_model(vocab=50, dim=64, depth=2, heads=4):
    torch.manual_seed(0)
    return gfn.Manifold(vocab_size=vocab, dim=dim, depth=depth, heads=heads, use_scan=True).to(DEV)


@pytest.mark.gpu
def test_scan_model_streams_like_one_pass():
    m = _scan_model().eval()
    ids = torch.randint(0, 50, (3, 40), device=DEV)
    with torch.no_grad():
        whole, end = m.stream(ids)
        torch.testing.assert_close(whole, m(ids)[0], rtol=1e-4, atol=1e-4)
        st, parts = None, []
        for lo, hi in ((0, 17), (17, 18), (18, 19), (19, 40)):
            lg, st = m.stream(ids[:, lo:hi], st)
            parts.append(lg)
        torch.testing.assert_close(torch.cat(parts, 1), whole, rtol=1e-4, atol=1e-4)
        for (v, x), (v1, x1) in zip(st, end):
            torch.testing.assert_close(v, v1, rtol=1e-4, atol=1e-4)
            torch.testing.assert_close(x, x1, rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
def test_scan_model_trains_end_to_end():
    # every parameter's gradient against torch's autograd of the same layer in float64
    m = _scan_model(vocab=20, dim=32, depth=2, heads=2).use_library_norm()
    ids = torch.randint(0, 20, (2, 30), device=DEV)
    tgt = torch.randint(0, 20, (2, 30), device=DEV)
    gfn.cross_entropy(m(ids)[0], tgt).backward()
    sd = {k: v.detach().double().cpu().requires_grad_(v.is_floating_point()) for k, v in m.named_parameters()}
    cur = sd["embedding.weight"][ids.cpu()]
    F = torch.nn.functional
    for i in range(2):
        q = f"layers.{i}."
        f = F.layer_norm(cur, (32,), sd[q + "norm_x.weight"], sd[q + "norm_x.bias"])
        A = torch.sigmoid(F.linear(f, sd[q + "to_A.0.weight"], sd[q + "to_A.0.bias"]))
        hs = 0.1 * 1.5 ** torch.arange(2).double().repeat_interleave(16)
        dt = F.softplus(F.linear(f, sd[q + "to_dt.0.weight"], sd[q + "to_dt.0.bias"])) * hs
        Bv = F.linear(f, sd[q + "to_B.weight"], sd[q + "to_B.bias"]) * dt
        v, x, xs = torch.zeros(2, 32).double(), torch.zeros(2, 32).double(), []
        for t in range(30):
            v = A[:, t] * v + Bv[:, t]
            x = x + v * dt[:, t]
            xs.append(x)
        cur = torch.stack(xs, 1)
    out = F.layer_norm(cur, (32,), sd["readout_norm.weight"], sd["readout_norm.bias"])
    loss = F.cross_entropy(F.linear(out, sd["readout.weight"], sd["readout.bias"]).view(-1, 20), tgt.cpu().view(-1))
    loss.backward()
    seen = 0
    for k, p in m.named_parameters():
        ref = sd[k].grad
        if ref is None:
            assert p.grad is None or not p.grad.any(), k
            continue
        seen += 1
        # float32 forward and backward through ten products and two scans: 1e-4 of the largest entry
        assert (p.grad.double().cpu() - ref).abs().max() <= 1e-4 * ref.abs().max() + 1e-9, k
    assert seen >= 2 * 8 + 5


@pytest.mark.gpu
def test_library_norm_matches_torch_norm_in_a_leapfrog_model():
    torch.manual_seed(1)
    m = gfn.Manifold(vocab_size=30, dim=64, depth=1, rank=16, heads=4, integrator_type="leapfrog").to(DEV)
    ids = torch.randint(0, 30, (2, 6), device=DEV)
    grads = []
    for on in (False, True):
        m.use_library_norm(on).zero_grad()
        m(ids)[0].square().mean().backward()
        grads.append({k: p.grad.clone() for k, p in m.named_parameters() if p.grad is not None})
    for k, g in grads[0].items():
        torch.testing.assert_close(grads[1][k], g, rtol=1e-4, atol=1e-4 * float(g.abs().max()) + 1e-9)


@pytest.mark.gpu
@pytest.mark.parametrize("scan", [True, False])
def test_generate_with_penalties_and_masks(scan):
    torch.manual_seed(2)
    m = (_scan_model() if scan else
         gfn.Manifold(vocab_size=50, dim=64, depth=1, rank=16, heads=4, integrator_type="leapfrog").to(DEV))
    prompt = torch.tensor([[3, 4, 5]], device=DEV)
    kw = dict(max_new_tokens=8, carry_state=scan)
    plain = m.generate(prompt, **kw)
    assert m.generate(prompt, repetition_penalty=1.0 + 1e-7, **kw) == plain
    even = torch.arange(50, device=DEV) % 2 == 0
    assert all(t % 2 == 0 for t in m.generate(prompt, allowed=even, **kw)[3:])
    # a grammar: the next token is the last one plus one
    step = lambda toks: torch.arange(50, device=DEV) == (toks[-1] + 1) % 50  # noqa: E731
    assert m.generate(prompt, allowed=step, **kw)[3:] == list(range(6, 14))
    out = m.generate(prompt, presence_penalty=1e6, **kw)[3:]
    assert len(set(out)) == len(out)  # no token twice
    out = m.generate(prompt, allowed=even, top_k=5, temperature=0.7, **kw)[3:]
    assert all(t % 2 == 0 for t in out)
    with pytest.raises(gfn.GfnError):
        m.generate(prompt, allowed=torch.zeros(50, device=DEV, dtype=torch.bool), top_k=3, **kw)
    bias = torch.zeros(50, device=DEV)
    bias[7] = 1e4
    assert set(m.generate(prompt, logit_bias=bias, **kw)[3:]) == {7}


@pytest.mark.gpu
def test_generate_carries_the_scan_state():
    m = _scan_model()
    prompt = torch.tensor([[1, 2, 3, 4]], device=DEV)
    out = m.generate(prompt, max_new_tokens=6, carry_state=True)
    seq = prompt
    with torch.no_grad():
        for _ in range(6):  # the whole sequence again for every token
            seq = torch.cat([seq, m(seq)[0][:, -1:].argmax(-1)], 1)
    assert out == seq[0].tolist()


def test_stream_is_the_scan_paths():
    m = gfn.Manifold(vocab_size=4, dim=32, depth=1, heads=2, integrator_type="leapfrog")
    with pytest.raises(gfn.GfnError):
        m.stream(torch.zeros(1, 2, dtype=torch.long))
    m = gfn.Manifold(vocab_size=4, dim=32, depth=1, heads=2, use_scan=True)
    with pytest.raises(gfn.GfnError):  # no CPU path
        m.stream(torch.zeros(1, 2, dtype=torch.long))
