"""A failure inside a backward pass raises GfnError, as one of the forward does."""
import ctypes

import pytest
import torch

import manifold_b200 as gfn
from manifold_b200 import _lib

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("entry", ["gfn_layer_norm_backward", "gfn_gated_scan_backward", "gfn_layer_scan_backward"])
def test_a_failing_backward_raises_the_librarys_error(entry):
    ops, lib = _lib.torch_ops(), _lib.load()
    x, z = torch.randn(2, 6, 8, device=DEV), torch.randn(2, 6, 24, device=DEV)
    call = {"gfn_layer_norm_backward": (lambda t: gfn.layer_norm(t), x),
            "gfn_gated_scan_backward": (lambda t: gfn.gated_scan(None, t), x),
            "gfn_layer_scan_backward": (lambda t: gfn.cuda.ops.parallel_layer_scan(t, 2)[0], z)}[entry]
    leaf = call[1].clone().requires_grad_(True)
    y = call[0](leaf)
    addresses = [ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _lib.TORCH_ENTRIES]
    fail = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: 5)  # the launch that a device refuses
    broken = list(addresses)
    broken[_lib.TORCH_ENTRIES.index(entry)] = ctypes.cast(fail, ctypes.c_void_p).value
    try:
        ops.bind(tuple(broken), gfn.GfnError)
        with pytest.raises(gfn.GfnError, match=entry):
            torch.autograd.grad(y.sum(), leaf, retain_graph=True)
    finally:
        ops.bind(tuple(addresses), gfn.GfnError)
    g, = torch.autograd.grad(y.sum(), leaf)  # the graph survived, and so did the binding
    assert torch.isfinite(g).all()
