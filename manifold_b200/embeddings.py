"""Token -> force embeddings (mirror of gfn/embeddings.py).

FunctionalEmbedding (the one the LM-shaped configuration uses) runs as one
fused SIREN kernel over all [B, L] tokens; ImplicitEmbedding keeps the
reference's module and evaluates with torch GPU ops (it is not on any
benchmarked path).  embed_tokens and Embedding look a table up on the
library's kernels and sum its gradient by sorted tokens.
"""
import numpy as np
import torch
import torch.nn as nn

from ._lib import GfnError, require_cuda, torch_ops
from .cuda import ops


def embed_tokens(ids, weight, scale=1.0, padding_idx=None):
    """scale * weight[ids], of shape [*ids.shape, dim] and the weight's type.

    ids: int64 or int32 of any shape.  weight [vocab, dim]: float32, bfloat16 or
    float16; rows of a wider table are read in place.  scale: a number.
    Differentiable (once) in weight: the rows of every token are summed in
    float32 in a fixed order (the tokens are sorted; no atomics), so that results
    repeat bit for bit; tokens equal to padding_idx take no part.  A
    token outside the vocabulary gives a row of zeros, takes no part in the
    gradient and sets a device error bit (gfn.cuda.ops.device_error).
    """
    return torch_ops().embed_tokens(ids, weight, scale, padding_idx)


class Embedding(nn.Embedding):
    """nn.Embedding (the same parameters and state_dict) on the kernels, with a factor."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale = scale

    @classmethod
    def from_pretrained(cls, embeddings, freeze=True, padding_idx=None, *, scale=1.0):
        """A module on the table `embeddings` [vocab, dim], which it shares; freeze: the table is not trained."""
        if embeddings.dim() != 2:
            raise GfnError(f"Embedding.from_pretrained: embeddings must be [vocab, dim], got {tuple(embeddings.shape)}")
        module = cls(*embeddings.shape, padding_idx=padding_idx, scale=scale, device="meta", dtype=embeddings.dtype)
        module.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return module

    def extra_repr(self):
        return super().extra_repr() + ("" if self.scale == 1.0 else f", scale={self.scale}")

    def forward(self, input_ids):
        return embed_tokens(input_ids, self.weight, self.scale, self.padding_idx)


class SineLayer(nn.Module):
    """sin(omega_0 * Linear(x)) with SIREN init (gfn/embeddings.py:24-49)."""

    def __init__(self, in_features, out_features, bias=True, is_first=False, omega_0=30.0):
        super().__init__()
        self.omega_0 = omega_0
        self.is_first = is_first
        self.linear = nn.Linear(in_features, out_features, bias=bias)
        self.init_weights()

    def init_weights(self):
        with torch.no_grad():
            if self.is_first:
                bound = 1 / self.linear.weight.size(1)
            else:
                bound = np.sqrt(6 / self.linear.weight.size(1)) / self.omega_0
            self.linear.weight.uniform_(-bound, bound)

    def forward(self, x):
        return torch.sin(self.omega_0 * self.linear(x))


class ImplicitEmbedding(nn.Module):
    """Coordinate table -> SIREN -> Linear, x1.5 (gfn/embeddings.py:52-119)."""

    def __init__(self, vocab_size, emb_dim, coord_dim=16, hidden_dim=64, layers=2):
        super().__init__()
        self.vocab_size = vocab_size
        self.emb_dim = emb_dim
        self.coord_dim = coord_dim
        self.coords = nn.Embedding(vocab_size, coord_dim)
        nn.init.uniform_(self.coords.weight, -1.0, 1.0)
        net = [SineLayer(coord_dim, hidden_dim, is_first=True, omega_0=30.0)]
        for _ in range(layers):
            net.append(SineLayer(hidden_dim, hidden_dim, is_first=False, omega_0=30.0))
        self.net = nn.Sequential(*net)
        self.out_proj = nn.Linear(hidden_dim, emb_dim)
        with torch.no_grad():
            nn.init.xavier_uniform_(self.out_proj.weight)
            nn.init.zeros_(self.out_proj.bias)

    def forward(self, input_ids):
        require_cuda(input_ids)
        return self.out_proj(self.net(self.coords(input_ids))) * 1.5


class FunctionalEmbedding(nn.Module):
    """Zero-lookup embedding: id -> bits -> SIREN -> force
    (gfn/embeddings.py:121-206).  Mode 'binary' runs on the fused kernel."""

    def __init__(self, vocab_size, emb_dim, coord_dim=16, hidden_dim=64, layers=2, mode="binary",
                 impulse_scale=1.0, omega_0=30.0):
        super().__init__()
        self.mode = mode
        self.coord_dim = coord_dim
        self.omega_0 = omega_0
        self.impulse_scale = nn.Parameter(torch.tensor(impulse_scale), requires_grad=True)
        if self.mode == "linear":
            self.net = nn.Identity()
            self.out_proj = nn.Linear(self.coord_dim, emb_dim)
            with torch.no_grad():
                nn.init.constant_(self.out_proj.weight, 1.0)
                nn.init.zeros_(self.out_proj.bias)
        else:
            net = [SineLayer(self.coord_dim, hidden_dim, is_first=True, omega_0=self.omega_0)]
            for _ in range(layers):
                net.append(SineLayer(hidden_dim, hidden_dim, is_first=False, omega_0=self.omega_0))
            self.net = nn.Sequential(*net)
            self.out_proj = nn.Linear(hidden_dim, emb_dim)
            with torch.no_grad():
                self.out_proj.weight.data *= 1.5
                nn.init.zeros_(self.out_proj.bias)
        if self.mode == "sinusoidal":
            if coord_dim % 2 != 0:
                self.coord_dim += 1
            freqs = torch.exp(torch.arange(0, self.coord_dim, 2).float()
                              * -(np.log(10000.0) / self.coord_dim))
            self.register_buffer("freqs", freqs)
        self.hidden_dim = hidden_dim
        self.n_layers = layers
        self.out_dtype = torch.float32

    def _fused_ok(self):
        return (self.mode == "binary" and self.coord_dim == 16 and self.hidden_dim == 64
                and self.n_layers == 2)

    def forward(self, input_ids, out_dtype=None):
        require_cuda(input_ids)
        if not self._fused_ok():
            raise GfnError(f"FunctionalEmbedding mode={self.mode!r} coord_dim={self.coord_dim} "
                           "is not implemented on this build (binary/16/64/2 is)")
        n = self.net
        return ops.functional_embedding(
            input_ids, n[0].linear.weight, n[0].linear.bias, n[1].linear.weight, n[1].linear.bias,
            n[2].linear.weight, n[2].linear.bias, self.out_proj.weight, self.out_proj.bias,
            self.impulse_scale, self.omega_0, out_dtype=out_dtype or self.out_dtype)
