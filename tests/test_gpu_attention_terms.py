"""Every term of decay_attention's sums, one by one.

Whole numbers: with decays of 1 and 0 all scores, states and outputs are whole
numbers that every operand type holds (256 for bfloat16, 2048 for float16's
scores and states), so that results are exact up to the one rounding at the end;
a lost, doubled or misplaced token shows.  Normal numbers: the error of a token's
outputs against the root of the sum of its terms' squares instead of the sum of
their magnitudes: scores, state and result are rounded to the operands' step, at
most 2^-8 (bfloat16) or 2^-11 (float16) relative, independently of one another,
with a standard deviation of that over sqrt(3); 2.5 steps are more than four of
them.  One lost token is far outside, which is shown on the definition itself.
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn

DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
STEP = {torch.float32: 2.0 ** -18, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _scores(q, k, decay):
    """[B, H, L, L] of g^(i-j) q_i k_j in float64, and the powers."""
    n = q.shape[1]
    i = torch.arange(n, device=q.device)
    gap = (i[:, None] - i).double()
    w = torch.where(gap >= 0, decay.double()[:, None, None] ** gap.clamp(min=0), 0.0)
    return torch.einsum("bihk,bjhk->bhij", q.double(), k.double()) * w, w


def _whole(B, L, H, K, V, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randint(-1, 2, s, generator=g).to(DEV)  # noqa: E731
    return r(B, L, H, K), r(B, L, H, K), r(B, L, H, V), r(B, L, H, V), r(B, H, K, V), r(B, H, K, V)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,H,K,V", [(1, 64, 2, 32, 32), (2, 150, 2, 64, 64), (1, 333, 2, 64, 128), (1, 260, 2, 128, 64),
                                       (1, 150, 2, 128, 128), (1, 1500, 2, 128, 128), (1, 1300, 2, 64, 128), (1, 1400, 2, 64, 64),
                                       (1, 1100, 2, 31, 17), (1, 900, 2, 40, 72), (1, 97, 2, 9, 120)])
def test_whole_numbers_are_exact(B, L, H, K, V, dtype):
    q, k, v, do, st, dl = _whole(B, L, H, K, V, seed=L)
    decay = torch.tensor([1.0, 0.0], device=DEV)
    leaves = [t.to(dtype).requires_grad_(True) for t in (q, k, v)] + [st.float().requires_grad_(True)]
    o, last = gfn.decay_attention(*leaves[:3], decay, state=leaves[3], return_state=True)
    dq, dk, dv, ds = torch.autograd.grad((o, last), leaves, (do.to(dtype), dl.float()))
    q, k, v, do, st, dl = (t.double() for t in (q, k, v, do, st, dl))
    p, w = _scores(q, k, decay)
    on = decay.double().view(1, H, 1, 1)  # 1: the state lasts, 0: it is gone with the first token
    held = torch.cumsum(k[..., :, None] * v[..., None, :], 1)[:, :, 0] + st[:, None, 0]
    after = torch.flip(torch.cumsum(torch.flip(q[..., :, None] * do[..., None, :], [1]), 1), [1])[:, :, 0] + dl[:, None, 0]
    limit = {torch.float32: 2.0 ** 22, torch.bfloat16: 256, torch.float16: 2048}[dtype]
    assert max(held.abs().max(), after.abs().max(), p.abs().max()) <= limit  # the premise, of the inputs alone
    d, _ = _scores(do, v, decay)  # do_i v_j
    first = st * on
    want = dict(
        o=torch.einsum("bhij,bjhv->bihv", p, v) + torch.einsum("bihk,bhkv->bihv", q, first),
        last=torch.einsum("bjhk,bjhv,hj->bhkv", k, v, w[:, -1]) + first,
        dq=torch.einsum("bhij,bjhk->bihk", d, k) + torch.einsum("bihv,bhkv->bihk", do, first),
        dk=torch.einsum("bhij,bihk->bjhk", d, q) + torch.einsum("hj,bhkv,bjhv->bjhk", w[:, -1], dl, v),
        dv=torch.einsum("bhij,bihv->bjhv", p, do) + torch.einsum("hj,bhkv,bjhk->bjhv", w[:, -1], dl, k),
        ds=on * (after[:, 0, None] if H == 1 else torch.stack([after[:, 0], torch.zeros_like(after[:, 0])], 1)))
    for name, got in dict(o=o, last=last, dq=dq, dk=dk, dv=dv, ds=ds).items():
        assert torch.equal(got, want[name].to(got.dtype)), (name, (got.double() - want[name]).abs().max())


def _normal(B, L, H, K, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    decay = (1 - 2.0 ** -(3 + 4 * torch.arange(H).float() / max(H - 1, 1))).to(DEV)
    return r(B, L, H, K), r(B, L, H, K), r(B, L, H, V), r(B, L, H, V), decay


def _rows(got, want, square, step):
    """The error of each token's outputs in units of what is allowed."""
    err = (got.double() - want).norm(dim=-1)
    return err / (step * want.norm(dim=-1) + 2.5 * step * square.sqrt() + 1e-30)


def _terms(rows, keys, values, w):
    """sum_j p_ij values_j, and the sum of its terms' squares, once by scores and once by the products in them."""
    p = torch.einsum("bihk,bjhk->bhij", rows.double(), keys.double()) * w
    size = torch.einsum("bihk,bjhk->bhij", rows.double() ** 2, keys.double() ** 2) * w ** 2
    norm = (values.double() ** 2).sum(-1)
    return torch.einsum("bhij,bjhv->bihv", p, values.double()), torch.einsum("bhij,bjh->bih", p ** 2 + size, norm), p


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,H,K,V", [(2, 300, 3, 64, 64), (1, 1000, 2, 64, 64), (1, 900, 2, 128, 128), (1, 700, 2, 64, 128),
                                       (2, 200, 2, 40, 72), (1, 1200, 2, 32, 32)])
def test_no_term_is_lost_among_normal_numbers(B, L, H, K, V, dtype):
    q, k, v, do, decay = _normal(B, L, H, K, V, dtype, seed=L)
    step = STEP[dtype]
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = gfn.decay_attention(*leaves, decay)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    _, w = _scores(q, k, decay)
    back = w.transpose(-1, -2)
    for name, got, args in (("o", o, (q, k, v, w)), ("dq", dq, (do, v, k, w)), ("dv", dv, (k, q, do, back)),
                            ("dk", dk, (v, do, q, back))):
        want, square, p = _terms(*args)
        assert (_rows(got, want, square, step) <= 1).all(), (name, _rows(got, want, square, step).max())
        # the definition without one token: some outputs of every sequence and head show it
        j = L // 2
        lost = want - torch.einsum("bhi,bhv->bihv", p[:, :, :, j], args[2].double()[:, j])
        assert (_rows(lost.to(got.dtype), want, square, step).amax(1) > 1).all(), name
