"""Forward-mode differentiation and vmap: refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import manifold_b200 as gfn

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused_not_dropped(grad):
    """A dual tensor comes back with its tangent or not at all; the operators have no forward mode."""
    x, w = torch.randn(2, 6, 8, device=DEV), torch.ones(8, device=DEV)
    z, s = torch.randn(2, 6, 24, device=DEV), torch.zeros(2, 8, device=DEV)
    scan, lg = gfn.cuda.ops.parallel_layer_scan, torch.randn(2, 8, device=DEV)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        d = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: gfn.layer_norm(d(x)), lambda: gfn.layer_norm(x, d(w)), lambda: gfn.layer_norm(x, w, d(w)),
                 lambda: gfn.gated_scan(d(x), x), lambda: gfn.gated_scan(x, d(x)), lambda: gfn.gated_scan(x, x, d(s)),
                 lambda: gfn.gated_scan(None, d(x)), lambda: gfn.parallel_scan(x, d(x)), lambda: gfn.parallel_scan(d(x), x),
                 lambda: scan(d(z), 2), lambda: scan(z, 2, state=(d(s), s)), lambda: scan(z, 2, state=(s, d(s))),
                 lambda: gfn.process_logits(d(lg)), lambda: gfn.process_logits(lg, bias=d(w)),
                 lambda: gfn.process_logits(lg, temperature=d(torch.ones(2, device=DEV)))]
        for i, call in enumerate(calls):
            with pytest.raises(gfn.GfnError):
                call()
                pytest.fail(f"call {i} returned")
        gfn.layer_norm(x), gfn.gated_scan(x, x), scan(z, 2)  # tensors without a tangent still run
    v = torch.vmap(lambda t: t * 2)(x)
    with pytest.raises(RuntimeError):  # no batching rule either
        torch.vmap(gfn.layer_norm)(v)
