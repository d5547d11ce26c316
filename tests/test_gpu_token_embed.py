"""GPU parity of embed_tokens and its table's gradient against the float64
definitions (oracle/lm_ops.py).

Tolerances: the factor and the product round once each in float32 (u = 2^-24),
the result once to its type (uo); a row of the gradient sums n terms, each sum
off by at most u times the terms' magnitude, and is rounded once.  float16 has
a smallest step of 2^-24.
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
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _close(got, want, tol):
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.abs(got - want)[bad].max())


def _check(ids, w, scale, padding=None, seed=0, dy=None):
    leaf = w.detach().requires_grad_(True)
    y = gfn.embed_tokens(ids, leaf, scale, padding)
    uo = UO[w.dtype]
    want = O.embed_tokens(_np(ids), _np(w), scale)
    assert y.dtype == w.dtype and y.is_contiguous()
    _close(_np(y), want, (2 * U + uo) * np.abs(want) + 2.0 ** -24)
    if dy is None:
        dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(seed)).to(w.dtype).to(DEV)
    g, = torch.autograd.grad(y, leaf, dy)
    n = np.bincount(np.clip(_np(ids).reshape(-1), 0, w.shape[0] - 1), minlength=w.shape[0])[:, None]
    want = O.embed_tokens_backward(_np(ids), _np(dy), w.shape[0], scale, padding)
    big = O.embed_tokens_backward(_np(ids), np.abs(_np(dy)), w.shape[0], abs(scale), padding)
    assert g.dtype == w.dtype and g.shape == w.shape
    _close(_np(g), want, uo * np.abs(want) + (n + 3) * U * big + 2.0 ** -24)
    return y, g


def _ids(n, vocab, seed=0, power=4):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(n, generator=g) ** power * vocab).long().clamp_(max=vocab - 1).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (1, 7, 3), (5, 300, 16), (31, 512, 8), (32, 511, 7), (33, 40, 64),
                                         (64, 1000, 130), (2047, 600, 24), (2048, 513, 17), (2049, 70000, 5),
                                         (4100, 300, 40), (9000, 20, 33), (6000, 262145, 4), (3000, 2, 1001)])
def test_embedding_and_its_gradient(n, vocab, dim, dtype):
    w = torch.randn(vocab, dim, generator=torch.Generator().manual_seed(n)).to(dtype).to(DEV)
    _check(_ids(n, vocab, seed=vocab), w, 0.7)
    assert gfn.cuda.ops.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 70, 3000, 70000])
def test_one_token_everywhere_and_all_different(n):
    """A row summed by every group of tokens, and rows of one token each in falling order."""
    w = torch.randn(n, 20, device=DEV)
    _check(torch.full((n,), 3, device=DEV), w, 1.0)
    _check(torch.arange(n - 1, -1, -1, device=DEV), w, 1.0)
    _check((torch.arange(n, device=DEV) // 37) % n, w, 1.0)


@pytest.mark.gpu
def test_order_of_sums_is_the_order_of_tokens():
    """Terms that cancel only in order: 2^24, 1, -2^24 gives 0 in float32, any other order 1."""
    ids = torch.tensor([5, 1, 5, 1, 5], device=DEV)
    w = torch.zeros(9, 1, device=DEV, requires_grad=True)
    dy = torch.tensor([[2.0 ** 24], [3.0], [1.0], [4.0], [-(2.0 ** 24)]], device=DEV)
    g, = torch.autograd.grad(gfn.embed_tokens(ids, w), w, dy)
    assert g[5].item() == 0.0 and g[1].item() == 7.0


@pytest.mark.gpu
def test_repeats_bit_for_bit_and_more_than_a_tile_per_block():
    n, vocab = 600000, 50000  # several parts of tokens to a block
    ids, w = _ids(n, vocab), torch.randn(vocab, 4, device=DEV, requires_grad=True)
    dy = torch.randn(n, 4, device=DEV)
    first = torch.autograd.grad(gfn.embed_tokens(ids, w), w, dy)[0]
    for _ in range(3):
        assert torch.equal(first, torch.autograd.grad(gfn.embed_tokens(ids, w), w, dy)[0])
    want = torch.zeros(vocab, 4, device=DEV, dtype=torch.float64).index_add_(0, ids, dy.double())
    big = torch.zeros(vocab, 4, device=DEV, dtype=torch.float64).index_add_(0, ids, dy.double().abs())
    n = torch.bincount(ids, minlength=vocab).unsqueeze(1)
    assert ((first - want).abs() <= U * want.abs() + (n + 3) * U * big).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_types_and_strides_of_operands(dtype):
    w = torch.randn(50, 24, device=DEV).to(dtype)
    ids = _ids(60, 50).view(3, 4, 5)
    base, grad = _check(ids, w, 2.5)
    for same in (ids.int(), ids.transpose(0, 2).contiguous().transpose(0, 2)):
        y, g = _check(same, w, 2.5)
        assert torch.equal(y, base) and torch.equal(g, grad)
    wide = torch.randn(50, 40, device=DEV).to(dtype)
    wide[:, 3:27] = w  # rows of a wider table, off 16 bytes
    assert torch.equal(gfn.embed_tokens(ids, wide[:, 3:27], 2.5), base)
    wide[:, 8:32] = w
    assert torch.equal(gfn.embed_tokens(ids, wide[:, 8:32], 2.5), base)
    assert torch.equal(gfn.embed_tokens(ids, w.t().contiguous().t(), 2.5), base)
    dy = torch.randn(60, 1, device=DEV).to(dtype)
    _check(ids, w, 2.5, dy=dy.expand(60, 24).view(3, 4, 5, 24))  # a broadcast gradient
    _check(ids, w, 2.5, dy=torch.randn(3, 4, 5, 30, device=DEV).to(dtype)[..., 1:25])
    assert gfn.embed_tokens(ids[:0], w).shape == (0, 4, 5, 24)
    leaf = w.clone().requires_grad_(True)
    g, = torch.autograd.grad(gfn.embed_tokens(ids[:0], leaf).sum(), leaf)
    assert not g.any()
    assert gfn.embed_tokens(torch.tensor(7, device=DEV), w).shape == (24,)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [50, 5000])
def test_padding_and_tokens_outside_the_table(n):
    w = torch.randn(30, 12, device=DEV)
    ids = _ids(n, 30, power=1)
    y, g = _check(ids, w, 1.5, padding=4)
    assert not g[4].any() and y[ids == 4].any()
    assert torch.equal(g, _check(ids, w, 1.5, padding=4)[1])
    leaf = w.clone().requires_grad_(True)
    m = gfn.Embedding(30, 12, padding_idx=-2, scale=1.5).to(DEV)
    with torch.no_grad():
        m.weight.copy_(w)
    m(ids).sum().backward()
    assert not m.weight.grad[28].any() and m.weight.grad[27].any()
    assert gfn.cuda.ops.device_error() == 0
    ids[::7] = 30
    ids[1::9] = -1
    y = gfn.embed_tokens(ids, leaf, 1.5)
    bad = (ids < 0) | (ids >= 30)
    assert not y[bad].any() and gfn.cuda.ops.device_error() == 2
    g, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    want = 1.5 * torch.bincount(ids[~bad], minlength=30).float().unsqueeze(1).expand(30, 12)
    assert torch.equal(g, want) and gfn.cuda.ops.device_error() == 2


@pytest.mark.gpu
def test_the_library_embedding_of_a_model():
    """use_library_embedding: the model's own results, in training and without gradients."""
    for scan in (False, True):
        torch.manual_seed(0)
        model = gfn.Manifold(vocab_size=40, dim=32, depth=1, heads=2, rank=4, use_scan=scan,
                             integrator_type="leapfrog", base_dt=0.1).to(DEV)
        ids = _ids(60, 40).view(2, 30)
        ref = torch.nn.functional.embedding(ids, model.embedding.weight)
        grads = []
        for on in (False, True):
            assert model.use_library_embedding(on) is model
            assert torch.equal(model._forces(ids, None), ref)
            model.zero_grad(set_to_none=True)
            model(ids)[0].square().sum().backward()
            grads.append(model.embedding.weight.grad.clone())
        n = torch.bincount(ids.flatten(), minlength=40).max().item()
        big = grads[0].abs().max().item()
        assert (grads[1] - grads[0]).abs().max().item() <= 4 * (n + 4) * 2.0 ** -24 * n * big


@pytest.mark.gpu
def test_a_model_with_a_scaled_embedding():
    """A gfn.Embedding with a factor in a model's place: the fused lookup, which knows no factor, is not taken."""
    for scan in (False, True):
        torch.manual_seed(0)
        model = gfn.Manifold(vocab_size=40, dim=32, depth=1, heads=2, rank=4, use_scan=scan,
                             integrator_type="leapfrog", base_dt=0.1).to(DEV)
        ids = _ids(60, 40).view(2, 30)
        scaled = gfn.Embedding(40, 32, scale=3.0).to(DEV)
        with torch.no_grad():
            scaled.weight.copy_(model.embedding.weight)
            want = model(force_manual=3.0 * model.embedding(ids))[0]
            model.embedding = scaled
            for on in (False, True):
                model.use_library_embedding(on)
                # the products of 3 and the weights round once on either side
                assert torch.equal(model(ids)[0], want)
