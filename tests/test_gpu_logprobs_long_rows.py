"""The gradient of log probabilities over rows of nearly 2^31 logits, the longest
that are taken: every place of the row is written, the given token and the
alternatives at its end get their terms, and nothing behind it is touched.
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from manifold_b200 import _lib

DEV = "cuda:0"
LONGEST = 0x7fffff00  # vocabulary
GUARD, TAIL, TOP = 16384, 9000, 4


def test_longer_rows_are_refused():
    lib = _lib.load()
    assert lib.gfn_token_logprobs_backward(1, 4, 1, 1, LONGEST + 1, 1, -100, 0, None, 1, None, 1, None, None, 1, None) == 2
    assert lib.gfn_token_logprobs_forward(1, 4, 1, 1, LONGEST + 1, 1, -100, 0, 1, None, None, None, None, None) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shift", [(torch.bfloat16, 0), (torch.bfloat16, 1), (torch.bfloat16, 8), (torch.float32, 4)])
def test_gradient_at_the_end_of_the_longest_rows(dtype, shift):
    """shift: places between the logits' alignment and the gradient's (1: single elements instead of groups of 16 bytes).

    Tolerance: the given terms are 1 and below, probabilities below 1e-3 and float32 to 2^-18, rounded once.
    """
    lib, code = _lib.load(), {torch.float32: 0, torch.bfloat16: 1}[dtype]
    x = torch.full((LONGEST + 8,), -40.0, device=DEV, dtype=dtype)[:LONGEST]
    x[-TAIL:] = torch.randn(TAIL, generator=torch.Generator().manual_seed(0)).to(dtype).to(DEV)
    best = torch.tensor([LONGEST - 1, LONGEST - 2, LONGEST - 700, LONGEST - 8200], device=DEV)
    x[best] = torch.tensor([6.0, 5.5, 5.0, 4.5], device=DEV, dtype=dtype)
    token = torch.tensor([LONGEST - 5], device=DEV)
    lp, ent, top_lp, stats = (torch.empty(n, device=DEV) for n in (1, 1, TOP, 2))
    top = torch.empty(TOP, device=DEV, dtype=torch.int64)
    out = torch.full((LONGEST + 2 * GUARD,), 7.0, device=DEV, dtype=dtype)
    dx = out[GUARD + shift:GUARD + shift + LONGEST]
    glp, gent = torch.tensor([1.0], device=DEV), torch.tensor([0.5], device=DEV)
    gtop = torch.tensor([0.25, -0.5, 0.125, 1.0], device=DEV)
    p = lambda t: t.data_ptr()  # noqa: E731
    assert lib.gfn_token_logprobs_forward(p(x), LONGEST, code, 1, LONGEST, p(token), -100, TOP, p(lp), p(ent), p(top_lp),
                                          p(top), p(stats), torch.cuda.current_stream().cuda_stream) == 0
    assert lib.gfn_token_logprobs_backward(p(x), LONGEST, code, 1, LONGEST, p(token), -100, TOP, p(top), p(stats), p(ent),
                                           p(glp), p(gent), p(gtop), p(dx), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert top.tolist() == best.tolist()
    tail = x[-TAIL:].double().cpu().numpy()
    rest = (LONGEST - TAIL) * np.exp(-40.0)
    z = np.exp(tail).sum() + rest
    logp = tail - np.log(z)
    prob = np.exp(logp)
    entropy = -(prob * logp).sum() - rest / z * (-40.0 - np.log(z))
    want = -(1.0 + gtop.sum().item()) * prob - 0.5 * prob * (logp + entropy)
    for t, g in zip([token.item()] + best.tolist(), [1.0] + gtop.tolist()):
        want[t - (LONGEST - TAIL)] += g
    got = dx[-TAIL:].double().cpu().numpy()
    uo = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    assert (np.abs(got - want) <= uo * np.abs(want) + 2.0 ** -16 * (prob + 2.0 ** -8 * np.abs(want))).all()
    assert abs(ent.item() - entropy) <= 2.0 ** -16 * entropy
    head = dx[:-TAIL]
    assert (head == head[0]).all() and 0 < abs(head[0].item()) < 1e-15  # each of probability e^-40 / z
    assert (out[:GUARD + shift] == 7).all() and (out[GUARD + shift + LONGEST:] == 7).all()
