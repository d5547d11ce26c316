"""gfn.Embedding as a module: its constructors, what it shows and keeps."""
import copy
import pickle

import pytest
import torch

import manifold_b200 as gfn

DEV = "cuda:0"


def test_from_a_given_table():
    w = torch.randn(7, 5)
    m = gfn.Embedding.from_pretrained(w)
    assert type(m) is gfn.Embedding and m.scale == 1.0 and m.padding_idx is None
    assert m.weight.data_ptr() == w.data_ptr() and not m.weight.requires_grad
    m = gfn.Embedding.from_pretrained(w.bfloat16(), freeze=False, padding_idx=-2, scale=2.5)
    assert (m.num_embeddings, m.embedding_dim, m.padding_idx, m.scale) == (7, 5, 5, 2.5)
    assert m.weight.requires_grad and m.weight.dtype == torch.bfloat16
    assert torch.equal(m.weight, w.bfloat16())  # the row of padding_idx as it was given
    for bad in (torch.zeros(3), torch.zeros(2, 3, 4)):
        with pytest.raises(gfn.GfnError):
            gfn.Embedding.from_pretrained(bad)
    with pytest.raises(TypeError):  # not an option of this module's
        gfn.Embedding.from_pretrained(w, max_norm=1.0)
    with pytest.raises(TypeError):  # nn.Embedding's third positional is no factor
        gfn.Embedding.from_pretrained(w, True, None, 2.0)


def test_the_factor_is_shown_and_travels():
    m = gfn.Embedding(7, 5, padding_idx=2, scale=2.5)
    assert repr(m) == "Embedding(7, 5, padding_idx=2, scale=2.5)"
    assert repr(gfn.Embedding(7, 5)) == "Embedding(7, 5)"
    assert copy.deepcopy(m).scale == 2.5 and pickle.loads(pickle.dumps(m)).scale == 2.5
    assert list(m.state_dict()) == ["weight"]


@pytest.mark.gpu
def test_a_given_table_looked_up_and_trained():
    w = torch.randn(9, 6, device=DEV)
    ids = torch.tensor([[1, 8, 3], [3, 3, 0]], device=DEV)
    m = gfn.Embedding.from_pretrained(w, freeze=False, padding_idx=8, scale=0.5)
    y = m(ids)
    assert torch.equal(y, 0.5 * w[ids])
    y.sum().backward()
    n = torch.bincount(ids.flatten(), minlength=9).float()
    n[8] = 0
    assert torch.equal(m.weight.grad, 0.5 * n.unsqueeze(1).expand(9, 6))
