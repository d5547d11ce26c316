"""Refusals of the embedding, log probability and attention
calls, and their float64 gradients (oracle/lm_ops.py) against differences."""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from oracle import lm_ops as O


def test_cpu_tensors_are_refused():
    f, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    q = torch.zeros(1, 2, 2, 8)
    for call in (lambda: gfn.embed_tokens(i, f), lambda: gfn.token_logprobs(f, i),
                 lambda: gfn.decay_attention(q, q, q, torch.ones(2))):
        with pytest.raises(gfn.GfnError, match="CUDA"):
            call()


def _differences(f, x, h=1e-5):
    g = np.zeros(x.shape)
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        g[i] = (f(a) - f(b)) / (2 * h)
    return g


def test_embedding_gradient_against_differences():
    r = np.random.default_rng(0)
    ids, w, dy = np.array([2, 0, 2, 4, 1, 2]), r.standard_normal((5, 3)), r.standard_normal((6, 3))
    got = O.embed_tokens_backward(ids, dy, 5, 1.5)
    np.testing.assert_allclose(got, _differences(lambda x: (dy * O.embed_tokens(ids, x, 1.5)).sum(), w), atol=1e-8)


def test_logprob_gradient_against_differences():
    r = np.random.default_rng(1)
    x, t = r.standard_normal((3, 6)), np.array([4, -100, 0])
    g = [r.standard_normal(3), r.standard_normal(3), r.standard_normal((3, 2))]
    top = O.token_logprobs(x, t, 2)[3]

    def value(y):
        lp, ent, tlp, tid = O.token_logprobs(y, t, 2)
        assert np.array_equal(tid, top)
        return (g[0] * lp).sum() + (g[1] * ent).sum() + (g[2] * tlp).sum()
    np.testing.assert_allclose(O.token_logprobs_backward(x, t, top, *g), _differences(value, x), atol=1e-8)


def test_attention_gradient_against_differences():
    r = np.random.default_rng(2)
    q, k, v = r.standard_normal((2, 4, 2, 3)), r.standard_normal((2, 4, 2, 3)), r.standard_normal((2, 4, 2, 2))
    decay, s, lengths = np.array([0.9, 0.3]), r.standard_normal((2, 2, 3, 2)), [4, 2]
    do, dl = r.standard_normal(v.shape), r.standard_normal(s.shape)
    got = O.decay_attention_backward(q, k, v, decay, s, lengths, 0.7, do, dl)
    args = [q, k, v, s]
    for i in range(4):
        def value(x):
            a = [x if j == i else t for j, t in enumerate(args)]
            o, last = O.decay_attention(*a[:3], decay, a[3], lengths, 0.7)
            return (do * o).sum() + (dl * last).sum()
        np.testing.assert_allclose(got[i], _differences(value, args[i]), atol=1e-8)


def test_host_entries_refuse_what_they_do_not_take():
    from manifold_b200 import _lib
    lib = _lib.load()
    assert lib.gfn_token_embed_backward_workspace_bytes(-1, 5, 5) == -1
    assert lib.gfn_token_embed_backward_workspace_bytes(2 ** 31, 5, 5) == -1
    assert lib.gfn_token_embed_backward_workspace_bytes(100, 50257, 64) >= 16 * 100
    assert lib.gfn_token_embed_forward(None, 1, 3, None, 4, 0, 5, 4, 1.0, None, None) == 1
    assert lib.gfn_token_embed_backward(None, 1, 3, None, 4, 0, 5, 4, 1.0, -1, None, None, 0, None) == 1
    assert lib.gfn_token_logprobs_forward(None, 4, 0, 3, 4, None, -100, 0, None, None, None, None, None, None) == 1
    assert lib.gfn_token_logprobs_forward(1, 4, 0, 3, 4, None, -100, 5, None, None, 1, 1, None, None) == 2
    assert lib.gfn_token_logprobs_forward(1, 99, 0, 3, 99, None, -100, 33, None, None, 1, 1, None, None) == 2
    z = [None] * 9
    assert lib.gfn_decay_attention_forward(*z, 0, 0, 1, 4, 2, 129, 8, 1.0, None, None, None, 0, None) == 1
    one = [1, 1, 1, 1, 1, 1, 1, None, None]
    assert lib.gfn_decay_attention_forward(*one, 0, 0, 1, 4, 2, 129, 8, 1.0, 1, None, None, 0, None) == 2
    assert lib.gfn_decay_attention_forward(*one, 0, 9, 1, 4, 2, 8, 8, 1.0, 1, None, None, 0, None) == 2
    assert lib.gfn_decay_attention_forward(*one, 0, 0, 70000, 4, 2, 8, 8, 1.0, 1, None, None, 0, None) == 2


@pytest.mark.gpu
def test_refusals_of_the_embedding():
    dev = "cuda:0"
    w, i = torch.zeros(5, 3, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    for call in (lambda: gfn.embed_tokens(i.float(), w), lambda: gfn.embed_tokens(i, w[0]), lambda: gfn.embed_tokens(i, w.double()),
                 lambda: gfn.embed_tokens(i, w[:0]), lambda: gfn.embed_tokens(i, w[:, :0]), lambda: gfn.embed_tokens(i.cpu(), w),
                 lambda: gfn.embed_tokens(i, w, padding_idx=5), lambda: gfn.embed_tokens(i, w, padding_idx=-6),
                 lambda: gfn.embed_tokens(i, w, scale=torch.ones((), device=dev)), lambda: gfn.embed_tokens(None, w),
                 lambda: gfn.embed_tokens(i, None), lambda: gfn.embed_tokens(i.bool(), w)):
        with pytest.raises(gfn.GfnError):
            call()


@pytest.mark.gpu
def test_refusals_of_the_log_probabilities():
    dev = "cuda:0"
    x, t = torch.zeros(4, 40, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    f = gfn.token_logprobs
    for call in (lambda: f(x), lambda: f(x, t[:3]), lambda: f(x, t.float()), lambda: f(x, t, top=33), lambda: f(x, t, top=-1),
                 lambda: f(x[:, :4], t, top=5), lambda: f(x.double(), t), lambda: f(x, t.cpu()), lambda: f(x[:, :0], t),
                 lambda: f(x[0, 0], t), lambda: f(None, t), lambda: f(x, t.view(2, 2)), lambda: f(x.long(), t)):
        with pytest.raises(gfn.GfnError):
            call()
    with pytest.raises(TypeError):
        f(x, t, top=1.5)


@pytest.mark.gpu
def test_refusals_of_the_attention():
    dev = "cuda:0"
    q, g, s = torch.zeros(2, 3, 4, 8, device=dev), torch.ones(4, device=dev), torch.zeros(2, 4, 8, 8, device=dev)
    n = torch.ones(2, dtype=torch.int64, device=dev)
    wide = torch.zeros(2, 3, 4, 129, device=dev)
    f = gfn.decay_attention
    for call in (lambda: f(q[0], q[0], q[0], g), lambda: f(q, q[:, :2], q, g), lambda: f(q, q, q[:, :, :2], g),
                 lambda: f(q, q.bfloat16(), q, g), lambda: f(q.double(), q.double(), q.double(), g), lambda: f(q, q, wide, g),
                 lambda: f(wide, wide, q, g), lambda: f(q[..., :0], q[..., :0], q, g), lambda: f(q, q, q, g[:3]),
                 lambda: f(q, q, q, g.double()), lambda: f(q, q, q, 0.9), lambda: f(q, q, q, g, state=s[:1]),
                 lambda: f(q, q, q, g, state=s.bfloat16()), lambda: f(q, q, q, g, lengths=n[:1]),
                 lambda: f(q, q, q, g, lengths=n.float()), lambda: f(q, q, q, g, lengths=[1, 2]), lambda: f(q, q, q, g.cpu()),
                 lambda: f(q, q, q, g, scale=torch.ones((), device=dev)), lambda: f(q, q, q, g.clone().requires_grad_(True))):
        with pytest.raises(gfn.GfnError):
            call()
    with torch.no_grad():  # no gradient wanted: the decay may be a parameter
        f(q, q, q, g.clone().requires_grad_(True))


@pytest.mark.gpu
def test_forward_mode_is_refused_and_second_derivatives_raise():
    import torch.autograd.forward_ad as fwd
    dev = "cuda:0"
    w, i = torch.randn(5, 8, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    q, g = torch.randn(1, 3, 2, 8, device=dev), torch.ones(2, device=dev)
    with fwd.dual_level():
        d = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: gfn.embed_tokens(i, d(w)), lambda: gfn.token_logprobs(d(w[:4]), i),
                     lambda: gfn.decay_attention(d(q), q, q, g), lambda: gfn.decay_attention(q, q, q, d(g))):
            with pytest.raises(gfn.GfnError):
                call()
    for call, t in ((lambda x: gfn.embed_tokens(i, x), w), (lambda x: gfn.token_logprobs(x, i[:4] % 4).logprobs, w[:4]),
                    (lambda x: gfn.decay_attention(x, x, x, g), q)):
        x = t.clone().requires_grad_(True)
        first, = torch.autograd.grad((call(x) ** 2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), x)
