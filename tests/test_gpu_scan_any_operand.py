"""The scans take without a gradient what they take with one: any dim, alignment
and broadcast gates; what does not fit is refused before a kernel reads it."""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from oracle import lm_ops as O

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,D,heads", [(2, 50, 33, 3), (1, 700, 66, 2), (3, 9, 7, 1), (2, 0, 6, 2), (2, 5, 1, 1)])
def test_layer_scan_without_a_gradient_takes_any_dim(B, L, D, heads):
    z = torch.randn(B, L, 3 * D, device=DEV)
    with torch.no_grad():
        xs, vs = gfn.cuda.ops.parallel_layer_scan(z, heads)
        want = gfn.cuda.ops.parallel_layer_scan(z, heads, return_state=True)
    assert torch.equal(xs, want[0]) and torch.equal(vs, want[1])


@pytest.mark.gpu
def test_layer_scan_without_a_gradient_takes_any_alignment():
    base = torch.randn(1 + 2 * 40 * 3 * 32, device=DEV)
    z = base[1:].view(2, 40, 96)
    with torch.no_grad():
        xs, vs = gfn.cuda.ops.parallel_layer_scan(z, 4)
        xa, va = gfn.cuda.ops.parallel_layer_scan(z.clone(), 4)
    torch.testing.assert_close(xs, xa, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(vs, va, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [33, 66])
def test_scan_model_of_any_width_trains_and_is_evaluated(dim):
    torch.manual_seed(0)
    m = gfn.Manifold(vocab_size=11, dim=dim, depth=2, heads=3, use_scan=True).to(DEV)
    ids = torch.randint(0, 11, (2, 30), device=DEV)
    trained = m(ids)[0]
    trained.square().mean().backward()
    with torch.no_grad():
        torch.testing.assert_close(m.eval()(ids)[0], trained.detach(), rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(m.stream(ids)[0], trained.detach(), rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,D", [(2, 50, 33), (1, 300, 6), (2, 0, 6)])
def test_parallel_scan_without_a_gradient_takes_any_dim_and_alignment(B, L, D):
    a, x = torch.rand(B, L, D, device=DEV), torch.randn(B, L, D, device=DEV)
    for gate in (a, None):
        y = gfn.parallel_scan(gate, x)
        assert torch.equal(y, gfn.gated_scan(gate, x))
    base = torch.randn(1 + 2 * 40 * 32, device=DEV)
    x = base[1:].view(2, 40, 32)
    a = torch.rand(2, 40, 32, device=DEV)
    want, _ = O.gated_scan(a.double().cpu().numpy(), x.double().cpu().numpy())
    assert np.abs(gfn.parallel_scan(a, x).double().cpu().numpy() - want).max() < 1e-4


@pytest.mark.gpu
def test_scans_refuse_operands_that_do_not_fit_without_a_gradient():
    x = torch.zeros(2, 5, 8, device=DEV)
    for a in (torch.zeros(2, 5, 4, device=DEV), torch.zeros(2, 4, 8, device=DEV), torch.zeros(3, 5, 8, device=DEV),
              x.half()):
        with pytest.raises(gfn.GfnError):
            gfn.parallel_scan(a, x)
        with pytest.raises(gfn.GfnError):
            gfn.cuda.ops.parallel_scan_fused(a, x)
    for z, heads in ((torch.zeros(2, 5, 25, device=DEV), 1), (torch.zeros(5, 24, device=DEV), 2),
                     (torch.zeros(2, 5, 24, device=DEV), 3), (torch.zeros(2, 5, 24, device=DEV), 0)):
        with pytest.raises(gfn.GfnError):
            gfn.cuda.ops.parallel_layer_scan(z, heads)


@pytest.mark.gpu
def test_parallel_scan_without_a_gradient_broadcasts_its_gate():
    x, a = torch.randn(2, 30, 8, device=DEV), torch.rand(8, device=DEV)
    y = gfn.parallel_scan(a, x)
    torch.testing.assert_close(y, gfn.parallel_scan(a.expand(2, 30, 8).contiguous(), x), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(y, gfn.parallel_scan(a, x.clone().requires_grad_(True)).detach(), rtol=1e-5, atol=1e-5)
