"""The error of float32 decay_attention as a whole: its root mean square relative to
the results', against float64.

Sums that stay on the tensor cores are cut, not rounded: at most 24 cuts a block of
tokens for the state (heads up to 32; 12 for others), each of at most 2^-23 of the
part summed so far, on average half of that of half of the sum, 7.2e-7 in all and of
one sign.  Outputs add three cuts of a step's own sum (0.9e-7), products in two tf32
pieces (2^-23 root mean square) and rounded additions: below 1e-6.  Cuts over all
steps of an output, three each, would add half of 3 (K + 32) / 8 2^-24 or more.
"""
import pytest
import torch

import manifold_b200 as gfn

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,H,K,V", [(2, 1000, 4, 128, 128), (1, 1500, 4, 64, 64), (2, 1200, 5, 40, 72), (2, 1500, 4, 32, 32),
                                       (2, 500, 2, 128, 16)])
def test_float32_as_a_whole(B, L, H, K, V):
    g = torch.Generator().manual_seed(L)
    q, k, v, do = (torch.randn(B, L, H, d, generator=g).to(DEV) for d in (K, K, V, V))
    decay = 1 - 2.0 ** (-5 - 4 * torch.arange(H, device=DEV).float() / (H - 1))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = gfn.decay_attention(*leaves, decay)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    gap = torch.arange(L, device=DEV)[:, None] - torch.arange(L, device=DEV)
    w = torch.where(gap >= 0, decay.double()[:, None, None] ** gap.clamp(min=0).double(), 0.0)
    p = torch.einsum("bihk,bjhk->bhij", q, k) * w
    d = torch.einsum("bihv,bjhv->bhij", do, v) * w
    want = dict(o=torch.einsum("bhij,bjhv->bihv", p, v), dq=torch.einsum("bhij,bjhk->bihk", d, k),
                dk=torch.einsum("bhij,bihk->bjhk", d, q), dv=torch.einsum("bhij,bihv->bjhv", p, do))
    for name, got in dict(o=o, dq=dq, dk=dk, dv=dv).items():
        err = ((got - want[name]).norm() / want[name].norm()).item()
        assert err <= 1e-6, (name, err)
