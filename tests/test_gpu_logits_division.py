"""Quotients of process_logits: exact roundings, and penalties and temperatures
at the ends of float32's range.

Without penalties and bias the only operation is one float32 division: the
result is IEEE's correctly rounded quotient, compared bit for bit with numpy's.
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from oracle import lm_ops as O

DEV = "cuda:0"
U, TINY = 2.0 ** -24, 2.0 ** -149


def _rows(params):
    return torch.tensor(params, dtype=torch.float32, device=DEV)


def _logits(B, V, seed, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = 4 * torch.randn(B, V, generator=g) * torch.exp2(spread * (2 * torch.rand(B, V, generator=g) - 1))
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = 0.0, -0.0, float("inf"), float("-inf")
    return x.to(DEV)


ENDS = [1.0, 0.7, 1.3, 3.0, 1e-3, 1e3, 1e-30, 1e30, 3e-38, 1e-38, 2.8e-39, 1e-40, 1.4e-45, 8.6e37, 3.4e38]


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1003, 8192])
@pytest.mark.parametrize("spread", [0.0, 20.0, 125.0])
def test_temperature_divides_with_one_rounding(V, spread):
    t = _rows(ENDS)
    x = _logits(len(ENDS), V, V, spread)
    with np.errstate(over="ignore", under="ignore"):
        want = x.cpu().numpy() / t.cpu().numpy()[:, None]
    got = gfn.process_logits(x, temperature=t).cpu().numpy()
    assert np.array_equal(got, want)
    for k in (1, 2, 10, 11):  # the same as a number
        assert np.array_equal(gfn.process_logits(x[k:k + 1], temperature=float(t[k])).cpu().numpy(), want[k:k + 1])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1003, 8192])
@pytest.mark.parametrize("spread", [0.0, 20.0, 125.0])
def test_repetition_penalty_divides_with_one_rounding(V, spread):
    rep = _rows(ENDS)
    x = _logits(len(ENDS), V, V + 1, spread)
    tok = torch.arange(V, device=DEV).expand(len(ENDS), V)  # every token was seen, in the prompt
    prompt = torch.full((len(ENDS),), V, device=DEV)
    xn, rn = x.cpu().numpy(), rep.cpu().numpy()[:, None]
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        want = np.where(xn > 0, xn / rn, xn * rn)
    assert np.array_equal(gfn.process_logits(x, tok, None, prompt, repetition_penalty=rep).cpu().numpy(), want)


@pytest.mark.gpu
def test_smallest_temperature_and_penalty_keep_zeros_and_signs():
    x = torch.tensor([[0.0, -0.0, 1e-44, -1e-44, 1.0, -1.0, float("inf"), float("-inf"), float("nan")]], device=DEV)
    y = gfn.process_logits(x, temperature=1e-40)
    assert y[0, 0] == 0 and y[0, 1] == 0
    assert 0.9e-4 < y[0, 2] < 1.1e-4 and -1.1e-4 < y[0, 3] < -0.9e-4
    assert (y[0, [4, 6]] == float("inf")).all() and (y[0, [5, 7]] == float("-inf")).all() and torch.isnan(y[0, 8])
    tok = torch.arange(9, device=DEV).unsqueeze(0)
    y = gfn.process_logits(x, tok, repetition_penalty=1e-40, frequency_penalty=0.25)
    assert y[0, 0] == -0.25 and y[0, 1] == -0.25 and torch.isnan(y[0, 8])
    assert y[0, 4] == float("inf") and y[0, 5] == -0.25


@pytest.mark.gpu
@pytest.mark.parametrize("B,V,T", [(1, 32000, 50), (40, 5003, 2000)])
def test_shaped_logits_round_once_per_operation(B, V, T):
    g = torch.Generator().manual_seed(T)
    x = (4 * torch.randn(B, V, generator=g)).to(DEV)
    tok = (torch.rand(B, T, generator=g) ** 2 * V).long().to(DEV)
    rep, temp = (1 + torch.rand(B, generator=g)).to(DEV), (0.5 + torch.rand(B, generator=g)).to(DEV)
    got = gfn.process_logits(x, tok, repetition_penalty=rep, temperature=temp).double().cpu().numpy()
    want = O.process_logits(x.double().cpu().numpy(), tok.cpu().numpy(), rep=rep.double().cpu().numpy(),
                            temperature=temp.double().cpu().numpy())
    # two roundings of relative size u: the penalty's and the temperature's
    assert (np.abs(got - want) <= 2.001 * U * np.abs(want)).all()
