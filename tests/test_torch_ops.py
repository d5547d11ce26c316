"""The C++ host side of the language-model operators: its binding to the
library, and the autograd machinery around it (checkpointing, graphs kept for
a second backward, CUDA graphs, threads, hooks on saved tensors)."""
import ctypes
import threading

import pytest
import torch

import manifold_b200 as gfn
from manifold_b200 import _lib

DEV = "cuda"


def test_binding_loads_once_and_checks_its_arguments():
    ops = _lib.torch_ops()
    assert ops is _lib.torch_ops()
    assert set(_lib.TORCH_ENTRIES) <= set(_lib.EXPORTED)
    for name, n in (("layer_norm", 5), ("gated_scan", 5), ("layer_scan", 7), ("process_logits", 17)):
        with pytest.raises(TypeError):
            getattr(ops, name)(*[None] * (n - 1))
        with pytest.raises((gfn.GfnError, TypeError)):
            getattr(ops, name)(*[1] * n)
    with pytest.raises(TypeError):
        ops.bind((1, 2), gfn.GfnError)
    lib = _lib.load()
    addresses = [ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _lib.TORCH_ENTRIES]
    with pytest.raises(ValueError):
        ops.bind(tuple([0] + addresses[1:]), gfn.GfnError)


def _case(op, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    if op == "norm":
        return (lambda x, w, b: gfn.layer_norm(x, w, b)), [r(300, 96), r(96), r(96)]
    if op == "scan":
        return (lambda a, x, h0: gfn.gated_scan(a, x, h0)), [torch.sigmoid(r(2, 300, 40)), r(2, 300, 40), r(2, 40)]
    return (lambda z, v, x: gfn.cuda.ops.parallel_layer_scan(z, 2, state=(v, x))[0]), [r(2, 300, 120), r(2, 40), r(2, 40)]


def _leaves(ts):
    return [t.clone().requires_grad_(True) for t in ts]


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["norm", "scan", "layer"])
def test_checkpointed_twice_and_hooked_gradients_are_the_same(op):
    f, ts = _case(op)
    leaves = _leaves(ts)
    y = f(*leaves)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for a, b in zip(want, torch.autograd.grad(y, leaves, dy)):  # the graph serves twice
        assert torch.equal(a, b)
    leaves = _leaves(ts)
    y = torch.utils.checkpoint.checkpoint(f, *leaves, use_reentrant=False)
    for a, b in zip(want, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(a, b)
    leaves = _leaves(ts)
    with torch.autograd.graph.save_on_cpu():
        y = f(*leaves)
    for a, b in zip(want, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(a, b)
    for i in range(len(ts)):  # one operand at a time
        some = [t.clone().requires_grad_(k == i) for k, t in enumerate(ts)]
        g, = torch.autograd.grad(f(*some), [some[i]], dy)
        assert torch.equal(g, want[i])


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["norm", "scan", "layer"])
def test_training_step_in_a_cuda_graph(op):
    f, ts = _case(op)
    leaves = _leaves(ts)
    dy = torch.randn(f(*leaves).shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(f(*leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = f(*leaves)
        grads = torch.autograd.grad(y, leaves, dy)
    _, new = _case(op, seed=5)
    with torch.no_grad():
        for t, n in zip(leaves, new):
            t.copy_(n)
    graph.replay()
    torch.cuda.synchronize()
    fresh = _leaves(new)
    want = f(*fresh)
    assert torch.equal(y, want)
    for a, b in zip(grads, torch.autograd.grad(want, fresh, dy)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_from_several_threads():
    f, ts = _case("scan")
    leaves = _leaves(ts)
    want = torch.autograd.grad(f(*leaves).sum(), leaves)
    torch.cuda.synchronize()
    out, errors = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    mine = _leaves(ts)
                    out[i] = torch.autograd.grad(f(*mine).sum(), mine)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for grads in out:
        for a, b in zip(grads, want):
            assert torch.equal(a, b)
