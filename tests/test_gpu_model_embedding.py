"""use_library_embedding with an embedding that a user has put in the model's
place: hooks, options and forward methods of its own take effect as they do without.
"""
import pytest
import torch

import manifold_b200 as gfn

DEV = "cuda:0"


def _model(embedding=None):
    torch.manual_seed(0)
    model = gfn.Manifold(vocab_size=40, dim=32, depth=1, heads=2, rank=4, use_scan=True).to(DEV)
    if embedding is not None:
        model.embedding = embedding.to(DEV)
    return model


def _ids():
    return (torch.arange(60, device=DEV) ** 2 % 40).view(2, 30)


@pytest.mark.gpu
@pytest.mark.parametrize("options", [dict(max_norm=0.1), dict(scale_grad_by_freq=True), dict(sparse=True),
                                     dict(padding_idx=4)])
def test_options_of_the_embedding(options):
    ids, seen = _ids(), []
    for on in (False, True):
        torch.manual_seed(1)
        model = _model(torch.nn.Embedding(40, 32, **options)).use_library_embedding(on)
        y = model._forces(ids, None)
        y.backward(torch.arange(1, 61, device=DEV).view(2, 30, 1).expand_as(y) / 64)
        g = model.embedding.weight.grad
        seen.append((y.detach(), g.is_sparse, g.to_dense(), model.embedding.weight.detach()))
    for a, b in zip(*seen):
        assert a == b if isinstance(a, bool) else torch.equal(a, b)


@pytest.mark.gpu
def test_hooks_of_the_embedding():
    for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook"):
        model, calls = _model().use_library_embedding(), []
        getattr(model.embedding, register)(lambda *a: calls.append(1) and None)
        model(_ids())[0].sum().backward()
        assert len(calls) == 1, register
    model = _model().use_library_embedding()
    handle = model.embedding.register_forward_hook(lambda m, i, y: 2 * y)
    doubled = model._forces(_ids(), None)
    handle.remove()
    assert torch.equal(doubled, 2 * model._forces(_ids(), None))


@pytest.mark.gpu
def test_hooks_of_every_module():
    model, calls = _model().use_library_embedding(), []
    handle = torch.nn.modules.module.register_module_forward_hook(
        lambda m, i, y: calls.append(m) if m is model.embedding else None)
    try:
        model(_ids())
    finally:
        handle.remove()
    assert len(calls) == 1


@pytest.mark.gpu
def test_an_embedding_with_a_forward_of_its_own():
    class Shifted(torch.nn.Embedding):
        def forward(self, ids):
            return super().forward(ids) + 1

    model, ids = _model(Shifted(40, 32)), _ids()
    want = model._forces(ids, None)
    assert torch.equal(model.use_library_embedding()._forces(ids, None), want)


@pytest.mark.gpu
def test_the_plain_embedding_takes_the_kernels():
    model, ids = _model().use_library_embedding(), _ids()
    assert "EmbedNode" in model._forces(ids, None).grad_fn.name()
    model.embedding = gfn.Embedding(40, 32, scale=2.0).to(DEV)
    assert "EmbedNode" in model._forces(ids, None).grad_fn.name()
