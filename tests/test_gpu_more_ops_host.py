"""The host side of the embedding, log probabilities and attention: the
autograd machinery, CUDA graphs, streams and threads, and a run of the three
together as a small language model uses them."""
import threading

import pytest
import torch

import manifold_b200 as gfn

DEV = "cuda"


def _case(op, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    if op == "embed":
        ids = (torch.rand(3000, generator=torch.Generator().manual_seed(7)) ** 3 * 200).long().to(DEV)
        return (lambda w: gfn.embed_tokens(ids, w, 1.5, 3)), [r(200, 40)]
    if op == "logprob":
        t = torch.arange(60, device=DEV) % 500
        t[::7] = -100

        def call(x):
            out = gfn.token_logprobs(x, t, top=4, entropy=True)
            return torch.cat([out.logprobs, out.entropy, out.top_logprobs.flatten()])
        return call, [r(60, 500)]
    decay = torch.tensor([0.9, 0.99], device=DEV)

    def call(q, k, v, s):  # noqa: F811
        o, last = gfn.decay_attention(q, k, v, decay, state=s, return_state=True, scale=0.3)
        return torch.cat([o.flatten(), last.flatten()])
    return call, [r(2, 700, 2, 24), r(2, 700, 2, 24), r(2, 700, 2, 40), r(2, 2, 24, 40)]


OPS = ["embed", "logprob", "attn"]


def _leaves(ts):
    return [t.clone().requires_grad_(True) for t in ts]


def _dy(y):
    return torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_checkpointed_twice_and_hooked_gradients_are_the_same(op):
    f, ts = _case(op)
    leaves = _leaves(ts)
    y = f(*leaves)
    dy = _dy(y)
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


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_two_training_steps_in_cuda_graphs(op):
    """Two graphs of the same call, replayed in turn with other data: neither disturbs the other."""
    f, ts = _case(op)
    sets = [_leaves(ts), _leaves(ts)]
    dy = _dy(f(*sets[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(f(*sets[0]), sets[0], dy)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for leaves in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = f(*leaves)
            outs.append((y, *torch.autograd.grad(y, leaves, dy)))
        graphs.append(graph)
    for i, leaves in enumerate(sets):
        with torch.no_grad():
            for t, n in zip(leaves, _case(op, seed=5 + i)[1]):
                t.copy_(n)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        fresh = _leaves(_case(op, seed=5 + i)[1])
        y = f(*fresh)
        for a, b in zip(out, (y, *torch.autograd.grad(y, fresh, dy))):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_two_streams_and_several_threads(op):
    f, ts = _case(op)
    leaves = _leaves(ts)
    y = f(*leaves)
    dy = _dy(y)
    want = (y, *torch.autograd.grad(y, leaves, dy))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            mine = _leaves(ts)
            y = f(*mine)
            got.append((y, *torch.autograd.grad(y, mine, dy)))
    torch.cuda.synchronize()
    errors = []

    def run():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    mine = _leaves(ts)
                    y = f(*mine)
                    got.append((y, *torch.autograd.grad(y, mine, dy)))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(got) == 36
    for out in got:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_operands_changed_in_place_before_the_backward_pass_are_noticed(op):
    f, ts = _case(op)
    leaves = _leaves(ts)
    inner = [t * 1.0 for t in leaves]
    y = f(*inner)
    if op == "embed":
        ids = torch.zeros(4, dtype=torch.int64, device=DEV)
        y = gfn.embed_tokens(ids, inner[0])
        ids += 1
    else:
        inner[0].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


class _Model(torch.nn.Module):
    """Embedding, one mixing layer of attention with decay, readout: the calls in the order they are used."""

    def __init__(self, vocab, dim, heads):
        super().__init__()
        self.heads = heads
        self.embedding = gfn.Embedding(vocab, dim, padding_idx=0, scale=dim ** 0.5)
        self.norm, self.out_norm = gfn.LayerNorm(dim), gfn.LayerNorm(dim)
        self.qkv, self.out, self.readout = (torch.nn.Linear(dim, n) for n in (3 * dim, dim, vocab))
        self.register_buffer("decay", 1 - 2.0 ** -torch.linspace(2, 6, heads))

    def forward(self, ids, state=None, lengths=None):
        x = self.embedding(ids)
        q, k, v = self.qkv(self.norm(x)).view(*ids.shape, 3, self.heads, -1).unbind(2)
        o, state = gfn.decay_attention(q, k, v, self.decay, state=state, return_state=True, lengths=lengths,
                                       scale=q.shape[-1] ** -0.5)
        return self.readout(self.out_norm(x + self.out(o.flatten(2)))), state


def _plain(model, ids, lengths):
    """The same in elementary float64 operations."""
    d = {n: p.detach().double().requires_grad_(True) for n, p in model.named_parameters()}
    B, L = ids.shape
    norm = lambda x, n: torch.nn.functional.layer_norm(x, x.shape[-1:], d[n + ".weight"], d[n + ".bias"])  # noqa: E731
    lin = lambda x, n: x @ d[n + ".weight"].t() + d[n + ".bias"]  # noqa: E731
    x = torch.nn.functional.embedding(ids, d["embedding.weight"], padding_idx=0) * model.embedding.scale
    q, k, v = lin(norm(x, "norm"), "qkv").view(B, L, 3, model.heads, -1).unbind(2)
    gam = model.decay.double().view(1, -1, 1, 1)
    s, o = 0.0, []
    for t in range(L):
        live = (t < lengths).view(B, 1, 1, 1)
        s = torch.where(live, gam * s + k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2), s)
        o.append(torch.where(live[..., 0], (q[:, t].unsqueeze(-2) @ s).squeeze(-2) * q.shape[-1] ** -0.5, 0.0))
    return lin(norm(x + lin(torch.stack(o, 1).flatten(2), "out"), "out_norm"), "readout"), d


@pytest.mark.gpu
def test_the_three_together_train_and_stream():
    """A training step's gradients against float64, and a padded prompt continued token by token."""
    torch.manual_seed(0)
    vocab, B, L = 61, 3, 150
    model = _Model(vocab, 48, 4).to(DEV)
    ids = torch.randint(1, vocab, (B, L), device=DEV)
    lengths = torch.tensor([L, 97, 1], device=DEV)
    pad = torch.arange(L, device=DEV) >= lengths.unsqueeze(1)
    ids[pad] = 0
    target = torch.roll(ids, -1, 1).masked_fill(pad.roll(-1, 1) | (torch.arange(L, device=DEV) == L - 1), -100)
    logits, state = model(ids, lengths=lengths)
    r = gfn.token_logprobs(logits, target, top=3, entropy=True)
    keep = (~pad).float()
    loss = -(r.logprobs.sum() + 0.1 * (r.entropy * keep).sum() + 0.01 * (r.top_logprobs[..., 2] * keep).sum()) / B
    loss.backward()
    wl, d = _plain(model, ids, lengths)
    lp = torch.log_softmax(wl, -1)
    given = torch.where(target >= 0, lp.gather(-1, target.clamp(min=0).unsqueeze(-1)).squeeze(-1), 0.0)
    ent = -(lp.exp() * lp).sum(-1)
    third = lp.gather(-1, r.top_tokens[..., 2:]).squeeze(-1)
    want = -(given.sum() + 0.1 * (ent * keep).sum() + 0.01 * (third * keep).sum()) / B
    want.backward()
    # everything is float32: products of 48 to 61 terms, sums over up to 248 tokens, 2^-24 a step and some 2^-22
    assert abs(loss.item() - want.item()) <= 1e-4 * abs(want.item())
    for n, p in model.named_parameters():
        err = (p.grad - d[n].grad).norm() / d[n].grad.norm()
        assert err < 1e-4, (n, err)
    assert not model.embedding.weight.grad[0].any()
    # serving: every sequence goes on from its own length, one token at a time
    with torch.no_grad():
        more = torch.randint(1, vocab, (B, 5), device=DEV)
        steps = []
        for t in range(5):
            lg, state = model(more[:, t:t + 1], state=state)
            steps.append(lg)
        for i, n in enumerate(lengths.tolist()):
            whole, _ = model(torch.cat([ids[i:i + 1, :n], more[i:i + 1]], 1))
            for t in range(5):
                assert (steps[t][i, 0] - whole[0, n + t]).abs().max() < 1e-4
                a, b = (gfn.token_logprobs(x, top=4, entropy=True) for x in (steps[t][i], whole[0, n + t:n + t + 1]))
                assert (a.entropy - b.entropy).abs().max() < 1e-4
    assert gfn.cuda.ops.device_error() == 0
