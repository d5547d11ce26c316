"""Measured cases of what a recurrent language model reads, mixes and answers
with: the embedding of its tokens and that table's gradient, linear attention
with a decay for each head, and the log probabilities of given tokens with the
entropy and the top alternatives.

Each case can run in two forms: the plain form (elementary torch operations
in float32, rounded once at the end) and, with ``own = True``, the calls a
user makes of manifold_b200.  ``exact`` evaluates the definitions in float64.
"""
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100


def listed():
    return [
        # the next token of 64 streams: all latency
        dict(name="embed_step", op="embed", tokens=64, vocab=32000, dim=1024, dtype="f32", train=False),
        # the prompts of a batch, 64 x 1024 tokens, 16-bit table
        dict(name="embed_prompt_bf16", op="embed", tokens=65536, vocab=50257, dim=1024, dtype="bf16", train=False),
        # a training step of 64 sequences of 1024 tokens, dim 512
        dict(name="embed_train", op="embed", tokens=65536, vocab=32000, dim=512, dtype="f32", train=True),
        # training with an odd width and a ragged number of tokens
        dict(name="embed_train_odd", op="embed", tokens=20011, vocab=50257, dim=1001, dtype="bf16", train=True),
        # one token of 64 streams with the carried states: latency, and the states' bytes
        dict(name="attn_step", op="attn", batch=64, length=1, heads=8, kdim=64, vdim=64, dtype="bf16", state=True,
             ragged=False, train=False),
        # one long document read in at once: few heads, a long axis
        dict(name="attn_prompt_bf16", op="attn", batch=1, length=65536, heads=8, kdim=64, vdim=64, dtype="bf16",
             state=True, ragged=False, train=False),
        # a training batch of 32 sequences, dim 512 in 8 heads
        dict(name="attn_train_bf16", op="attn", batch=32, length=2048, heads=8, kdim=64, vdim=64, dtype="bf16",
             state=False, ragged=False, train=True),
        # training on odd sizes in float32: padded sequences, the state carried between segments
        dict(name="attn_train_odd", op="attn", batch=3, length=5003, heads=5, kdim=40, vdim=72, dtype="f32",
             state=True, ragged=True, train=True),
        # one stream's next token: its log probability, the entropy and 5 alternatives
        dict(name="logprob_one", op="logprob", rows=1, vocab=32000, dtype="f32", top=5, entropy=True, masked=False,
             train=False),
        # a served batch under a grammar: 20 alternatives, some rows allow fewer tokens than that
        dict(name="logprob_batch", op="logprob", rows=256, vocab=50257, dtype="bf16", top=20, entropy=True,
             masked=True, train=False),
        # policy training on 8 sequences of 1024 tokens: log probabilities and an entropy bonus
        dict(name="logprob_train", op="logprob", rows=8192, vocab=32000, dtype="f32", top=0, entropy=True,
             masked=False, train=True),
        # a ragged number of rows, 16-bit logits, gradients through the alternatives as in distillation
        dict(name="logprob_train_odd", op="logprob", rows=4099, vocab=50257, dtype="bf16", top=8, entropy=False,
             masked=False, train=True),
    ]


_MOST = {}


def _affordable(case):
    """Whether no more is read, written or computed than in the largest listed case of the operator."""
    if not _MOST:
        for c in listed():
            for unit, n in work(c).items():
                _MOST[c["op"], unit] = max(_MOST.get((c["op"], unit), 0), n)
    return all(n <= _MOST[case["op"], unit] for unit, n in work(case).items())


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]; half of them odd or ragged as they fall,
    half rounded to a multiple of 8 where that fits."""
    n = max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))
    return n - n % 8 if n >= 16 and rng.random() < 0.5 else n


def draw(rng):
    while True:
        op = rng.choice(["embed", "attn", "logprob"])
        dtype = rng.choice(["f32", "bf16", "f16"])
        if op == "embed":
            case = dict(op=op, tokens=_log_int(rng, 1, 65536), vocab=_log_int(rng, 256, 65536),
                        dim=_log_int(rng, 16, 4096), dtype=dtype, train=rng.random() < 0.6)
        elif op == "attn":
            length = 1 if rng.random() < 0.15 else _log_int(rng, 1, 65536)
            case = dict(op=op, batch=_log_int(rng, 1, 64), length=length, heads=_log_int(rng, 1, 16),
                        kdim=_log_int(rng, 8, 128), vdim=_log_int(rng, 8, 128), dtype=dtype,
                        state=rng.random() < 0.5, ragged=rng.random() < 0.4, train=rng.random() < 0.5)
        else:
            case = dict(op=op, rows=_log_int(rng, 1, 8192), vocab=_log_int(rng, 64, 131072), dtype=dtype,
                        top=rng.choice([0, 1, 5, 20, 32]), entropy=rng.random() < 0.6, masked=rng.random() < 0.4,
                        train=rng.random() < 0.5)
        if _affordable(case):
            return case


def _distinct(tokens, vocab):
    """Expected number of distinct ids among `tokens` draws of vocab * rand ** 4."""
    edge = (torch.arange(vocab + 1, dtype=torch.float64) / vocab) ** 0.25
    return float(-torch.expm1(tokens * torch.log1p(-(edge[1:] - edge[:-1]).clamp(max=1 - 1e-12))).sum())


def work(case):
    op, s = case["op"], BYTES[case["dtype"]]
    if op == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        out = {"bytes": int(8 * n + (n + _distinct(n, v)) * d * s), "flops": n * d}
        if case["train"]:  # the gradient of the rows in, that of the whole table out
            out = {"bytes": out["bytes"] + (n + v) * d * s, "flops": 2 * n * d}
        return out
    if op == "attn":
        bh, kd, vd = case["batch"] * case["heads"], case["kdim"], case["vdim"]
        n = bh * case["length"]
        if case["ragged"]:  # lengths spread evenly over the upper half
            n = n * 3 // 4
        st = 4 * bh * kd * vd if case["state"] else 0
        if case["train"]:  # q, k, v, do in; o, dq, dk, dv out; the states and their gradients
            return {"bytes": (4 * kd + 4 * vd) * n * s + 4 * st, "flops": 14 * kd * vd * n}
        return {"bytes": (2 * kd + 2 * vd) * n * s + 2 * st, "flops": 4 * kd * vd * n}
    n, v, k = case["rows"], case["vocab"], case["top"]
    small = n * (12 + (4 if case["entropy"] else 0) + 12 * k)
    if case["train"]:  # logits in, their gradient out; the small outputs' gradients
        return {"bytes": 2 * n * v * s + 2 * small, "flops": 12 * n * v}
    return {"bytes": n * v * s + small, "flops": 6 * n * v}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device=dev, generator=gen)

    op, dt = case["op"], DTYPES[case["dtype"]]
    st = dict(case=case)
    if op == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        # token frequencies fall off like a power law
        st["ids"] = (rand(n) ** 4 * v).long().clamp_(max=v - 1)
        st["weight"] = (0.02 * randn(v, d)).to(dt)
        st["scale"] = d ** 0.5
        if case["train"]:
            st["dy"] = randn(n, d).to(dt)
    elif op == "attn":
        b, n, h = case["batch"], case["length"], case["heads"]
        st["q"] = randn(b, n, h, case["kdim"]).to(dt)
        st["k"] = randn(b, n, h, case["kdim"]).to(dt)
        st["v"] = randn(b, n, h, case["vdim"]).to(dt)
        # half lives from 22 tokens on, longer from head to head
        st["decay"] = 1.0 - 2.0 ** (-5.0 - 7.0 * torch.arange(h, device=dev, dtype=torch.float32) / max(h - 1, 1))
        st["scale"] = case["kdim"] ** -0.5
        if case["state"]:
            st["state"] = randn(b, h, case["kdim"], case["vdim"])
        if case["ragged"]:
            lengths = n - (rand(b) * ((n + 1) // 2)).long()
            lengths[0] = n
            st["lengths"] = lengths
        if case["train"]:
            st["do"] = randn(b, n, h, case["vdim"]).to(dt)
            if case["state"]:
                st["dlast"] = randn(b, h, case["kdim"], case["vdim"])
    else:
        n, v = case["rows"], case["vocab"]
        x = 3.0 * randn(n, v)
        tokens = (rand(n) * v).long().clamp_(max=v - 1)
        if case["masked"]:
            # a grammar lets through many tokens of some rows and few of others; the given one always
            share = rand(n, 1)
            share[::3] = 8.0 / v
            x.masked_fill_(rand(n, v) >= share, float("-inf"))
            x.scatter_(1, tokens.unsqueeze(1), 3.0 * randn(n, 1))
        if case["train"]:
            tokens[::16] = IGNORE  # padding
            st["glp"] = randn(n)
            if case["entropy"]:
                st["gent"] = randn(n)
            if case["top"]:
                st["gtop"] = randn(n, case["top"])
        st["logits"] = x.to(dt)
        st["tokens"] = tokens
    return st


# -------------------------------------------------------------- plain forms
def _embed_plain(st):
    c, w = st["case"], st["weight"]
    y = (w[st["ids"]].float() * st["scale"]).to(w.dtype)
    if not c["train"]:
        return y
    dw = torch.zeros(w.shape, device=w.device, dtype=torch.float32)
    dw.index_add_(0, st["ids"], st["dy"].float())
    return y, (dw * st["scale"]).to(w.dtype)


_CHUNK = 64


def _decay_pass(q, k, v, decay, lengths, state, dlast_len):
    """o_t = q_t S_t with S_t = decay S_{t-1} + k_t v_t^T in chunks, and the state after `lengths` tokens.
    q, k [B, H, L, K], v [B, H, L, V] float32, zero from `lengths` on; dlast_len: whether the state is wanted."""
    b, h, n, kd = q.shape
    c = min(_CHUNK, n)
    m = (n + c - 1) // c
    pad = m * c - n
    if pad:
        q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)) for t in (q, k, v))
    q, k, v = (t.reshape(b, h, m, c, t.shape[-1]) for t in (q, k, v))
    lg = torch.log(decay.double()).view(1, h, 1, 1)
    i = torch.arange(c, device=q.device, dtype=torch.float64)
    gap = i[:, None] - i
    mask = torch.where(gap >= 0, torch.exp(gap.clamp(min=0) * lg[0]), 0.0).float()  # [H, C, C]
    o = ((q @ k.transpose(-1, -2)) * mask[:, None]) @ v
    local = (k * torch.exp((c - 1 - i) * lg[0, :, 0]).float()[:, None, :, None]).transpose(-1, -2) @ v
    j = torch.arange(m + 1, device=q.device, dtype=torch.float64)
    hop = j[:, None] - 1 - j[:m]
    carry = torch.where(hop >= 0, torch.exp(c * hop.clamp(min=0) * lg[0]), 0.0).float()  # [H, M + 1, M]
    before = (carry @ local.flatten(-2)).unflatten(-1, local.shape[-2:])  # the state before each chunk, and the last
    if state is not None:
        before = before + torch.exp(c * j * lg[0, :, 0]).float()[:, :, None, None] * state.unsqueeze(2)
    o = o + (q @ before[:, :, :m]) * torch.exp((i + 1) * lg[0, :, 0]).float()[:, None, :, None]
    o = o.reshape(b, h, m * c, -1)[:, :, :n]
    last = None
    if dlast_len:
        # keys from `lengths` on are zero: the state has only decayed since, which is taken back from its terms
        t = torch.arange(n, device=q.device)
        left = lengths.view(b, 1, 1).double() - 1 - t
        wgt = torch.where(left >= 0, torch.exp(left.clamp(min=0) * lg[:, :, 0]), 0.0).float()  # [B, H, L]
        kk, vv = k.reshape(b, h, m * c, kd)[:, :, :n], v.reshape(b, h, m * c, -1)[:, :, :n]
        last = (kk * wgt.unsqueeze(-1)).transpose(-1, -2) @ vv
        if state is not None:
            last = last + torch.exp(lengths.view(b, 1).double() * lg[:, :, 0, 0]).float()[:, :, None, None] * state
    return o, last


def _from_end(t, lengths):
    """Rows in the opposite order within each sequence of [B, H, L, D]; zero rows stay behind it."""
    n = t.shape[2]
    at = (lengths.view(-1, 1) - 1 - torch.arange(n, device=t.device)).clamp(min=0)
    keep = torch.arange(n, device=t.device) < lengths.view(-1, 1)
    r = t.gather(2, at[:, None, :, None].expand(-1, t.shape[1], -1, t.shape[3]))
    return r * keep[:, None, :, None]


def _attn_plain(st):
    c, dt = st["case"], st["q"].dtype
    b, n = c["batch"], c["length"]
    dev = st["q"].device
    lengths = st.get("lengths", torch.full((b,), n, device=dev))
    keep = (torch.arange(n, device=dev) < lengths.view(b, 1))[:, None, :, None]
    rows = lambda t: torch.where(keep, t.transpose(1, 2).float(), 0.0)  # noqa: E731
    back = lambda t: t.transpose(1, 2).to(dt).contiguous()  # noqa: E731
    q, k, v, s0 = rows(st["q"]) * st["scale"], rows(st["k"]), rows(st["v"]), st.get("state")
    o, last = _decay_pass(q, k, v, st["decay"], lengths, s0, c["state"])
    out = [back(o)] + ([last] if c["state"] else [])
    if c["train"]:
        do = rows(st["do"])
        dq, _ = _decay_pass(do, v, k, st["decay"], lengths, None if s0 is None else s0.transpose(-1, -2), False)
        r = {name: _from_end(t, lengths) for name, t in (("q", q), ("k", k), ("v", v), ("do", do))}
        # the gradient of the last state stands one step behind the last token
        gam = st["decay"].view(1, -1, 1, 1)
        gl = None if not c["state"] else st["dlast"] / gam
        dv, first = _decay_pass(r["k"], r["q"], r["do"], st["decay"], lengths, gl, c["state"])
        dk, _ = _decay_pass(r["v"], r["do"], r["q"], st["decay"], lengths,
                            None if gl is None else gl.transpose(-1, -2), False)
        out += [back(dq * st["scale"]), back(_from_end(dk, lengths)), back(_from_end(dv, lengths))]
        if c["state"]:
            out.append(first * gam)
    return tuple(out)


def _logprob_plain(st):
    c, x = st["case"], st["logits"].float()
    m = x.max(-1, keepdim=True).values
    d = x - m
    e = torch.exp(d)
    z = e.sum(-1, keepdim=True)
    lp = d - torch.log(z)
    tok = st["tokens"]
    valid = tok != IGNORE
    at = tok.clamp(min=0).unsqueeze(1)
    out = [torch.where(valid, lp.gather(1, at)[:, 0], 0.0)]
    p = e / z
    plp = torch.where(p > 0, p * lp, 0.0) if c["entropy"] else None
    if c["entropy"]:
        ent = -plp.sum(-1)
        out.append(ent)
    if c["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]].clone()
        out += [lp.gather(1, order), order]
    if c["train"]:
        g = torch.where(valid, st["glp"], 0.0).unsqueeze(1)
        total = g
        if c["top"]:
            total = g + st["gtop"].sum(-1, keepdim=True)
        dx = -p * total
        if c["entropy"]:
            dx -= st["gent"].unsqueeze(1) * (plp + p * ent.unsqueeze(1))
        dx.scatter_add_(1, at, g)
        if c["top"]:
            dx.scatter_add_(1, order, st["gtop"])
        out.append(dx.to(st["logits"].dtype))
    return tuple(out)


# ---------------------------------------------------------- the framework's
def _own(st):
    import manifold_b200 as gfn
    c, op = st["case"], st["case"]["op"]
    if op == "embed":
        if not c["train"]:
            return gfn.embed_tokens(st["ids"], st["weight"], scale=st["scale"])
        w = st["weight"].detach().requires_grad_(True)
        y = gfn.embed_tokens(st["ids"], w, scale=st["scale"])
        return (y.detach(), *torch.autograd.grad(y, w, st["dy"]))
    if op == "attn":
        kw = dict(lengths=st.get("lengths"), scale=st["scale"])
        if not c["train"]:
            if c["state"]:
                return gfn.decay_attention(st["q"], st["k"], st["v"], st["decay"], state=st["state"],
                                           return_state=True, **kw)
            return (gfn.decay_attention(st["q"], st["k"], st["v"], st["decay"], **kw),)
        leaves = [st[n].detach().requires_grad_(True) for n in ("q", "k", "v")]
        if not c["state"]:
            o = gfn.decay_attention(*leaves, st["decay"], **kw)
            return (o.detach(), *torch.autograd.grad(o, leaves, st["do"]))
        leaves.append(st["state"].detach().requires_grad_(True))
        o, last = gfn.decay_attention(*leaves[:3], st["decay"], state=leaves[3], return_state=True, **kw)
        return (o.detach(), last.detach(), *torch.autograd.grad((o, last), leaves, (st["do"], st["dlast"])))
    kw = dict(top=c["top"], entropy=c["entropy"], ignore_index=IGNORE)
    if not c["train"]:
        return tuple(t for t in gfn.token_logprobs(st["logits"], st["tokens"], **kw) if t is not None)
    x = st["logits"].detach().requires_grad_(True)
    r = gfn.token_logprobs(x, st["tokens"], **kw)
    outs, grads = [r.logprobs], [st["glp"]]
    if c["entropy"]:
        outs.append(r.entropy)
        grads.append(st["gent"])
    if c["top"]:
        outs.append(r.top_logprobs)
        grads.append(st["gtop"])
    return (*[t.detach() for t in r if t is not None], *torch.autograd.grad(outs, x, grads))


def run(state):
    if own:
        return _own(state)
    return {"embed": _embed_plain, "attn": _attn_plain, "logprob": _logprob_plain}[state["case"]["op"]](state)


# ------------------------------------------------------- definitions, 64 bits
def _exact_attn(case, st):
    """One token after the other, forward and back."""
    b, n, h = case["batch"], case["length"], case["heads"]
    q, k, v = (st[x].double() for x in ("q", "k", "v"))
    gam = st["decay"].double().view(1, h, 1, 1)
    lengths = st.get("lengths", torch.full((b,), n, device=q.device)).tolist()
    shape = (b, h, case["kdim"], case["vdim"])
    s = st["state"].double() if case["state"] else torch.zeros(shape, device=q.device, dtype=torch.float64)
    o, dq, dk, dv = torch.zeros_like(v), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    train = case["train"]
    do = st["do"].double() if train else None
    live = torch.tensor([[t < m for m in lengths] for t in range(n)], device=q.device).view(n, b, 1, 1, 1)
    same = min(lengths) == n
    for t in range(n):
        new = gam * s + k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2)
        s = new if same else torch.where(live[t], new, s)
        o[:, t] = st["scale"] * (q[:, t].unsqueeze(-2) @ s).squeeze(-2)
        if train:
            dq[:, t] = st["scale"] * (s @ do[:, t].unsqueeze(-1)).squeeze(-1)
    out = [o] + ([s] if case["state"] else [])
    if train:
        r = st["dlast"].double() if case["state"] else torch.zeros_like(s)
        for t in range(n - 1, -1, -1):
            new = r + st["scale"] * q[:, t].unsqueeze(-1) * do[:, t].unsqueeze(-2)
            dk[:, t] = (new @ v[:, t].unsqueeze(-1)).squeeze(-1)
            dv[:, t] = (k[:, t].unsqueeze(-2) @ new).squeeze(-2)
            r = gam * new if same else torch.where(live[t], gam * new, r)
        out += [dq, dk, dv] + ([r] if case["state"] else [])
    if not same:
        for i, m in enumerate(lengths):
            for x in (o, dq, dk, dv):
                x[i, m:] = 0.0
    return tuple(out)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "embed":
        w = st["weight"].double()
        y = w.index_select(0, st["ids"]) * st["scale"]
        if not case["train"]:
            return y
        dw = torch.zeros_like(w).index_put_((st["ids"],), st["dy"].double() * st["scale"], accumulate=True)
        return y, dw
    if case["op"] == "attn":
        return _exact_attn(case, st)
    x = st["logits"].double()
    lp = x - torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(lp)
    rows = torch.arange(case["rows"], device=x.device)
    valid = st["tokens"] != IGNORE
    out = [torch.zeros_like(p[:, 0]).index_put_((rows[valid],), lp[rows[valid], st["tokens"][valid]])]
    if case["entropy"]:
        ent = torch.special.entr(p).sum(-1)
        out.append(ent)
    if case["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]].clone()
        out += [lp.gather(1, order), order]
    if case["train"]:
        direct = torch.zeros_like(x)
        direct[rows[valid], st["tokens"][valid]] = st["glp"].double()[valid]
        if case["top"]:
            direct.scatter_add_(1, order, st["gtop"].double())
        dx = direct - p * direct.sum(-1, keepdim=True)
        if case["entropy"]:  # d H / d x_j = -p_j (log p_j + H)
            dx += st["gent"].double().unsqueeze(1) * (torch.special.entr(p) - p * ent.unsqueeze(1))
        out.append(dx)
    return tuple(out)
