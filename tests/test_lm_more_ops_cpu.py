"""Without a GPU: refusals of the embedding, log probability and attention
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
