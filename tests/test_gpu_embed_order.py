"""The gradient of the embedding's table adds the tokens of a row in their order,
however many blocks, parts and digits the sort takes (rows of up to 33 tokens
lie in two runs of 32 sorted ones and are one chain of float32 additions); and
lookups in rows that stand off 16 bytes.
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn

DEV = "cuda:0"


def _chain(ids, dy, vocab, back=False):
    """Row by row, the float32 sum of dy in the order of the tokens (or the opposite one)."""
    if back:
        ids, dy = ids[::-1], dy[::-1]
    at = np.argsort(ids, kind="stable")
    key = ids[at]
    first = np.searchsorted(key, key)
    rank = np.arange(len(key)) - first
    acc = np.zeros((vocab, dy.shape[1]), np.float32)
    for r in range(rank.max() + 1):
        now = at[rank == r]
        acc[ids[now]] += dy[now]
    return acc


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [4, 3])
@pytest.mark.parametrize("rows,each,vocab", [(60, 33, 61), (300, 13, 300), (400, 12, 70000), (4000, 20, 262145),
                                             (20000, 15, 20000), (20000, 30, 40000)])
def test_sums_run_in_the_order_of_the_tokens(rows, each, vocab, dim):
    """1980 tokens (one block sorts them) to 600000 (several parts to a block), one to three digits, rows far apart."""
    r = np.random.default_rng(rows)
    ids = r.permutation(np.repeat(r.permutation(vocab)[:rows], each))
    # magnitudes over 2^12: nearly every order rounds to something else
    dy = (r.standard_normal((len(ids), dim)) * 2.0 ** r.integers(0, 12, (len(ids), dim))).astype(np.float32)
    want = _chain(ids, dy, vocab)
    assert (want != _chain(ids, dy, vocab, back=True)).mean() > 0.5 * rows / vocab
    w = torch.zeros(vocab, dim, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(gfn.embed_tokens(torch.from_numpy(ids).to(DEV), w), w, torch.from_numpy(dy).to(DEV))
    assert np.array_equal(g.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 3000])
def test_wide_rows_off_16_bytes(n, dtype):
    """Rows of a wider table at every offset, the last one at the end of its allocation."""
    dim, vocab = 133, 37
    ids = (torch.arange(n, device=DEV) * 7 + vocab - 1) % vocab
    w = torch.randn(vocab, dim, device=DEV).to(dtype)
    want = gfn.embed_tokens(ids, w, 1.5)
    assert torch.equal(want, (1.5 * w[ids].float()).to(dtype))
    for gap in (0, 1, 3, 8, 11):
        for front in range(9):
            wide = torch.full((front + vocab * (dim + gap) - gap,), float("nan"), device=DEV, dtype=dtype)
            view = wide.as_strided((vocab, dim), (dim + gap, 1), front)
            view.copy_(w)
            assert torch.equal(gfn.embed_tokens(ids, view, 1.5), want), (gap, front)
