"""Measured cases of the language-model operators: layer norm, the gated scan,
the scan layer's recurrence, and the shaping of logits before sampling.

Each case can run in two forms: the plain form (elementary torch operations
in float32, rounded once at the end) and, with ``own = True``, the calls a
user makes of manifold_b200.  ``exact`` evaluates the definitions in float64.
"""
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
BASE_DT = 0.1


def listed():
    return [
        # the readout's norm for one token of 64 streams: all latency
        dict(name="norm_decode", op="norm", rows=64, dim=256, dtype="f32", wdtype="f32", train=False),
        # the readout's norm over a batch of prompts (20 x 1024 tokens), 16-bit activations
        dict(name="norm_prompt_bf16", op="norm", rows=20480, dim=1024, dtype="bf16", wdtype="bf16", train=False),
        # the readout's norm in a training step of 64 sequences of 1024 tokens, dim 512
        dict(name="norm_train", op="norm", rows=65536, dim=512, dtype="f32", wdtype="f32", train=True),
        # training with an odd width and a ragged number of rows, float32 weights beside 16-bit activations
        dict(name="norm_train_odd", op="norm", rows=20011, dim=1001, dtype="bf16", wdtype="f32", train=True),
        # one token of 64 streams with the carried state: all latency
        dict(name="scan_step", op="scan", batch=64, length=1, dim=256, dtype="f32", state=True, train=False),
        # one long document read in at once: few columns, a long axis
        dict(name="scan_prompt_bf16", op="scan", batch=1, length=65536, dim=512, dtype="bf16", state=True,
             train=False),
        # a training batch of 16 sequences
        dict(name="scan_train", op="scan", batch=16, length=2048, dim=512, dtype="f32", state=False, train=True),
        # training on odd sizes with the state carried between segments
        dict(name="scan_train_odd", op="scan", batch=3, length=5003, dim=1001, dtype="bf16", state=True, train=True),
        # a scan layer streaming a 20,000-token prompt in one call
        dict(name="layer_prompt", op="layer", batch=1, length=20000, dim=256, heads=8, state=True, train=False,
             vgrad=False),
        # a scan layer's training step; the next layer reads x only
        dict(name="layer_train", op="layer", batch=32, length=2048, dim=512, heads=8, state=False, train=True,
             vgrad=False),
        # one stream's next token after 50 tokens: repetition penalty and temperature
        dict(name="logits_one", op="logits", batch=1, vocab=32000, history=50, dtype="f32", counts=False,
             bias="none", mask=False),
        # a served batch: every penalty, a bias per request, a grammar mask, ragged histories
        dict(name="logits_batch", op="logits", batch=256, vocab=50257, history=2048, dtype="bf16", counts=True,
             bias="row", mask=True),
    ]


_MAX_BYTES = {}


def _max_bytes(op):
    if not _MAX_BYTES:
        for c in listed():
            _MAX_BYTES[c["op"]] = max(_MAX_BYTES.get(c["op"], 0), work(c)["bytes"])
    return _MAX_BYTES[op]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]; half of them odd or ragged as they fall,
    half rounded to a multiple of 8 where that fits."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    n = max(lo, min(hi, n))
    if n >= 16 and rng.random() < 0.5:
        n -= n % 8
    return n if n != 3072 else 3080


def draw(rng):
    while True:
        op = rng.choice(["norm", "norm", "scan", "scan", "scan", "layer", "layer", "logits"])
        if op == "norm":
            dtype = rng.choice(["f32", "bf16", "f16"])
            case = dict(op=op, rows=_log_int(rng, 1, 65536), dim=_log_int(rng, 64, 8192), dtype=dtype,
                        wdtype=rng.choice([dtype, "f32"]), train=rng.random() < 0.6)
        elif op == "scan":
            case = dict(op=op, batch=_log_int(rng, 1, 256), length=_log_int(rng, 1, 65536),
                        dim=_log_int(rng, 64, 2048), dtype=rng.choice(["f32", "bf16", "f16"]),
                        state=rng.random() < 0.5, train=rng.random() < 0.6)
        elif op == "layer":
            heads = rng.choice([1, 2, 4, 8])
            case = dict(op=op, batch=_log_int(rng, 1, 256), length=_log_int(rng, 1, 20000),
                        dim=4 * heads * _log_int(rng, 4, 31), heads=heads, state=rng.random() < 0.5,
                        train=rng.random() < 0.6, vgrad=rng.random() < 0.5)
        else:
            case = dict(op=op, batch=_log_int(rng, 1, 256), vocab=_log_int(rng, 256, 65536),
                        history=_log_int(rng, 1, 4096), dtype=rng.choice(["f32", "bf16", "f16"]),
                        counts=rng.random() < 0.7, bias=rng.choice(["none", "shared", "row"]),
                        mask=rng.random() < 0.5)
        if work(case)["bytes"] <= _max_bytes(op):
            return case


def work(case):
    op = case["op"]
    if op == "norm":
        n, s, ws = case["rows"] * case["dim"], BYTES[case["dtype"]], BYTES[case["wdtype"]]
        if case["train"]:  # x, dy in; y, dx out; weight, bias in; their gradients out
            return {"bytes": 4 * n * s + 4 * case["dim"] * ws, "flops": 21 * n}
        return {"bytes": 2 * n * s + 2 * case["dim"] * ws, "flops": 8 * n}
    if op == "scan":
        n, s = case["batch"] * case["length"] * case["dim"], BYTES[case["dtype"]]
        st = case["batch"] * case["dim"] * 4 if case["state"] else 0
        if case["train"]:  # a, x, dh in; h, da, dx out; the states and their gradients
            return {"bytes": 6 * n * s + 4 * st, "flops": 5 * n}
        return {"bytes": 3 * n * s + 2 * st, "flops": 2 * n}
    if op == "layer":
        n = case["batch"] * case["length"] * case["dim"]
        st = 2 * case["batch"] * case["dim"] * 4 if case["state"] else 0
        if case["train"]:  # z, gx, (gv) in; x, v, dz out; the states and their gradients
            return {"bytes": (36 + (4 if case["vgrad"] else 0)) * n + 4 * st, "flops": 50 * n}
        return {"bytes": 20 * n + 2 * st, "flops": 20 * n}
    b, v = case["batch"], case["vocab"]
    nbytes = 2 * b * v * BYTES[case["dtype"]] + 8 * b * case["history"]
    nbytes += {"none": 0, "shared": 4 * v, "row": 4 * b * v}[case["bias"]]
    if case["mask"]:
        nbytes += 4 * b * ((v + 31) // 32)
    return {"bytes": nbytes, "flops": 6 * b * v}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device=dev, generator=gen)

    op = case["op"]
    st = dict(case=case)
    if op == "norm":
        dt, wdt = DTYPES[case["dtype"]], DTYPES[case["wdtype"]]
        n, d = case["rows"], case["dim"]
        # activations with a per-row offset and scale, as a residual stream has them
        st["x"] = (randn(n, d) * (0.5 + rand(n, 1)) + 0.3 * randn(n, 1)).to(dt)
        st["w"] = (1.0 + 0.1 * randn(d)).to(wdt)
        st["b"] = (0.1 * randn(d)).to(wdt)
        if case["train"]:
            st["dy"] = randn(n, d).to(dt)
    elif op == "scan":
        dt = DTYPES[case["dtype"]]
        b, n, d = case["batch"], case["length"], case["dim"]
        a = torch.sigmoid(randn(b, n, d) + 2.0)
        st["x"] = (randn(b, n, d) * (1.0 - a)).to(dt)
        st["a"] = a.to(dt)
        del a
        if case["state"]:
            st["h0"] = 0.5 * randn(b, d)
        if case["train"]:
            st["dh"] = randn(b, n, d).to(dt)
            if case["state"]:
                st["dlast"] = randn(b, d)
    elif op == "layer":
        b, n, d = case["batch"], case["length"], case["dim"]
        # pre-activations [zA | zdt | zB] of the three projections of a normalised input
        z = randn(b, n, 3 * d)
        z[..., :d] += 1.0
        st["z"] = z
        if case["state"]:
            st["v0"], st["x0"] = 0.5 * randn(b, d), randn(b, d)
        if case["train"]:
            st["gx"] = randn(b, n, d) / n
            if case["vgrad"]:
                st["gv"] = randn(b, n, d)
            if case["state"]:
                st["gvl"], st["gxl"] = randn(b, d), randn(b, d)
    else:
        b, v, h = case["batch"], case["vocab"], case["history"]
        st["logits"] = (3.0 * randn(b, v)).to(DTYPES[case["dtype"]])
        # token frequencies fall off like a power law: histories repeat their tokens
        st["tokens"] = (rand(b, h) ** 4 * v).long().clamp_(max=v - 1)
        lengths = 1 + (rand(b) * h).long()
        lengths[0] = h
        st["lengths"] = lengths.clamp_(max=h)
        st["prompt"] = (rand(b) * (st["lengths"] + 1)).long()
        st["rep"] = 1.0 + 0.5 * rand(b)
        st["temp"] = 0.5 + rand(b)
        if case["counts"]:
            st["freq"], st["pres"] = 0.5 * rand(b), 0.5 * rand(b)
        if case["bias"] == "shared":
            st["bias"] = randn(v)
        elif case["bias"] == "row":
            st["bias"] = randn(b, v)
        if case["mask"]:
            # 32 tokens a word, bit i of word j for token 32 j + i; some rows allow few tokens
            words = torch.randint(-2**31, 2**31, (b, (v + 31) // 32), device=dev, generator=gen)
            tight = torch.randint(-2**31, 2**31, words.shape, device=dev, generator=gen)
            tight &= torch.randint(-2**31, 2**31, words.shape, device=dev, generator=gen)
            words[::2] &= tight[::2]
            st["allowed"] = words.to(torch.int32)
    return st


# -------------------------------------------------------------- plain forms
def _norm_plain(st):
    c, x, w, b = st["case"], st["x"].float(), st["w"].float(), st["b"].float()
    mu = x.mean(-1, keepdim=True)
    xc = x - mu
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xh = xc * rstd
    y = (xh * w + b).to(st["x"].dtype)
    if not c["train"]:
        return y
    dy = st["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return (y, dx.to(st["x"].dtype), (dy * xh).sum(0).to(st["w"].dtype), dy.sum(0).to(st["b"].dtype))


def _doubling(a, x):
    """h_t = a_t h_{t-1} + x_t from zero over dim 1, by log2(L) doubling passes."""
    n, s = x.shape[1], 1
    a, h = a, x.clone()
    while s < n:
        h[:, s:] += a[:, s:] * h[:, :-s]
        s2 = 2 * s
        if s2 < n:
            a = torch.cat([a[:, :s], a[:, s:] * a[:, :-s]], 1)
        s = s2
    return h


def _scan_f32(a, x, h0):
    if h0 is not None:
        x = x.clone()
        x[:, 0] += a[:, 0] * h0
    return _doubling(a, x)


def _reverse_scan_f32(a, g, last):
    """g_t + a_{t+1} (...)_{t+1}, with `last` arriving behind the final step."""
    g = g.flip(1)
    an = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    if last is not None:
        g = g.clone()
        g[:, 0] += last
    return _doubling(an, g).flip(1)


def _scan_plain(st):
    c, dt = st["case"], st["x"].dtype
    a, x, h0 = st["a"].float(), st["x"].float(), st.get("h0")
    h = _scan_f32(a, x, h0)
    out = [h.to(dt)]
    if c["state"]:
        out.append(h[:, -1].clone())
    if c["train"]:
        g = _reverse_scan_f32(a, st["dh"].float(), st.get("dlast"))
        first = h0 if h0 is not None else torch.zeros_like(h[:, 0])
        hp = torch.cat([first.unsqueeze(1), h[:, :-1]], 1)
        out += [(g * hp).to(dt), g.to(dt)]
        if c["state"]:
            out.append(a[:, 0] * g[:, 0])
    return tuple(out)


def _head_scale(d, heads, dev, dtype):
    return BASE_DT * 1.5 ** torch.arange(heads, device=dev, dtype=dtype).repeat_interleave(d // heads)


def _softplus(z):
    return z.clamp(min=0.0) + torch.log1p(torch.exp(-z.abs()))


def _layer_plain(st):
    c, z = st["case"], st["z"]
    d = c["dim"]
    za, zd, zb = z[..., :d], z[..., d:2 * d], z[..., 2 * d:]
    hs = _head_scale(d, c["heads"], z.device, torch.float32)
    A = torch.sigmoid(za)
    dt = _softplus(zd) * hs
    v = _scan_f32(A, zb * dt, st.get("v0"))
    xs = torch.cumsum(v * dt, 1)
    if c["state"]:
        xs = xs + st["x0"].unsqueeze(1)
    out = [xs, v]
    if c["state"]:
        out += [v[:, -1].clone(), xs[:, -1].clone()]
    if c["train"]:
        gx = st["gx"]
        if c["state"]:
            gx = gx.clone()
            gx[:, -1] += st["gxl"]
        X = torch.cumsum(gx.flip(1), 1).flip(1)
        g = dt * X
        if c["vgrad"]:
            g = g + st["gv"]
        lam = _reverse_scan_f32(A, g, st.get("gvl"))
        first = st["v0"] if c["state"] else torch.zeros_like(v[:, 0])
        vp = torch.cat([first.unsqueeze(1), v[:, :-1]], 1)
        dz = torch.cat([lam * vp * A * (1.0 - A), (lam * zb + X * v) * hs * torch.sigmoid(zd), lam * dt], -1)
        out.append(dz)
        if c["state"]:
            out += [A[:, 0] * lam[:, 0], X[:, 0].clone()]
    return tuple(out)


def _logits_form(st, dtype):
    """The definition in `dtype`: penalties, bias, temperature, mask."""
    c, x = st["case"], st["logits"].to(dtype)
    b, v = x.shape
    pos = torch.arange(c["history"], device=x.device)
    valid = pos < st["lengths"].unsqueeze(1)
    gen = valid & (pos >= st["prompt"].unsqueeze(1))
    seen = torch.zeros(b, v, device=x.device, dtype=torch.int32).scatter_add_(1, st["tokens"], valid.int())
    rep = st["rep"].to(dtype).unsqueeze(1)
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    if c["counts"]:
        cnt = torch.zeros(b, v, device=x.device, dtype=torch.int32).scatter_add_(1, st["tokens"], gen.int())
        x = x - (st["freq"].to(dtype).unsqueeze(1) * cnt + st["pres"].to(dtype).unsqueeze(1) * (cnt > 0))
    if "bias" in st:
        x = x + st["bias"].to(dtype)
    x = x / st["temp"].to(dtype).unsqueeze(1)
    if "allowed" in st:
        bits = (st["allowed"].unsqueeze(-1) >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bits.reshape(b, -1)[:, :v] != 0, x, float("-inf"))
    return x


# ---------------------------------------------------------- the framework's
def _own(st):
    import manifold_b200 as gfn
    c, op = st["case"], st["case"]["op"]
    if op == "norm":
        if not c["train"]:
            return gfn.layer_norm(st["x"], st["w"], st["b"], EPS)
        leaves = [st[k].detach().requires_grad_(True) for k in ("x", "w", "b")]
        y = gfn.layer_norm(*leaves, EPS)
        return (y.detach(), *torch.autograd.grad(y, leaves, st["dy"]))
    if op == "scan":
        if not c["train"]:
            if c["state"]:
                return gfn.gated_scan(st["a"], st["x"], st["h0"], return_state=True)
            return (gfn.gated_scan(st["a"], st["x"]),)
        keys = ("a", "x", "h0") if c["state"] else ("a", "x")
        leaves = [st[k].detach().requires_grad_(True) for k in keys]
        if c["state"]:
            h, last = gfn.gated_scan(*leaves, return_state=True)
            return (h.detach(), last.detach(), *torch.autograd.grad((h, last), leaves, (st["dh"], st["dlast"])))
        h = gfn.gated_scan(*leaves)
        return (h.detach(), *torch.autograd.grad(h, leaves, st["dh"]))
    if op == "layer":
        scan = gfn.cuda.ops.parallel_layer_scan
        if not c["train"]:
            if c["state"]:
                xs, v, (vl, xl) = scan(st["z"], c["heads"], BASE_DT, state=(st["v0"], st["x0"]), return_state=True)
                return xs, v, vl, xl
            return scan(st["z"], c["heads"], BASE_DT)
        leaves = [st[k].detach().requires_grad_(True) for k in (("z", "v0", "x0") if c["state"] else ("z",))]
        outs, gouts = [], []
        if c["state"]:
            xs, v, (vl, xl) = scan(leaves[0], c["heads"], BASE_DT, state=tuple(leaves[1:]), return_state=True)
            res, outs, gouts = [xs, v, vl, xl], [xs, vl, xl], [st["gx"], st["gvl"], st["gxl"]]
        else:
            xs, v = scan(leaves[0], c["heads"], BASE_DT)
            res, outs, gouts = [xs, v], [xs], [st["gx"]]
        if c["vgrad"]:
            outs.append(v)
            gouts.append(st["gv"])
        return (*[r.detach() for r in res], *torch.autograd.grad(outs, leaves, gouts))
    return gfn.process_logits(st["logits"], st["tokens"], st["lengths"], st["prompt"],
                              repetition_penalty=st["rep"], frequency_penalty=st.get("freq", 0.0),
                              presence_penalty=st.get("pres", 0.0), bias=st.get("bias"),
                              temperature=st["temp"], allowed=st.get("allowed"))


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "norm":
        return _norm_plain(state)
    if op == "scan":
        return _scan_plain(state)
    if op == "layer":
        return _layer_plain(state)
    return _logits_form(state, torch.float32).to(state["logits"].dtype)


# ------------------------------------------------------- definitions, 64 bits
def _seq(a, x, h):
    """The recurrence, one step after the other, in float64."""
    out = torch.empty_like(x)
    for t in range(x.shape[1]):
        torch.addcmul(x[:, t], a[:, t], h, out=out[:, t])
        h = out[:, t]
    return out


def _seq_back(a, g, m):
    """l_t = g_t + m_{t+1}, m_t = a_t l_t; returns (l, m_0)."""
    out = torch.empty_like(g)
    for t in range(g.shape[1] - 1, -1, -1):
        torch.add(g[:, t], m, out=out[:, t])
        m = a[:, t] * out[:, t]
    return out, m


def exact(case, seed):
    st = prepare(case, seed)
    d64 = {k: t.double() for k, t in st.items() if torch.is_tensor(t) and t.is_floating_point()}
    op = case["op"]
    if op == "norm":
        x = d64["x"]
        var, mu = torch.var_mean(x, -1, correction=0, keepdim=True)
        sd = (var + EPS).sqrt()
        xh = (x - mu) / sd
        y = xh * d64["w"] + d64["b"]
        if not case["train"]:
            return y
        dy = d64["dy"]
        g = dy * d64["w"]
        proj = (g * xh).mean(-1, keepdim=True)
        return y, (g - g.mean(-1, keepdim=True) - xh * proj) / sd, torch.einsum("nd,nd->d", dy, xh), dy.sum(0)
    if op == "scan":
        a, x = d64["a"], d64["x"]
        h0 = d64.get("h0", torch.zeros_like(x[:, 0]))
        h = _seq(a, x, h0)
        out = [h] + ([h[:, -1]] if case["state"] else [])
        if case["train"]:
            g, m = _seq_back(a, d64["dh"], d64.get("dlast", torch.zeros_like(h0)))
            out += [torch.cat([(g[:, 0] * h0).unsqueeze(1), g[:, 1:] * h[:, :-1]], 1), g]
            if case["state"]:
                out.append(m)
        return tuple(out)
    if op == "layer":
        d, z = case["dim"], d64["z"]
        za, zd, zb = z.split(d, -1)
        hs = _head_scale(d, case["heads"], z.device, torch.float64)
        A, dt = 1.0 / (1.0 + torch.exp(-za)), torch.logaddexp(zd, torch.zeros_like(zd)) * hs
        zero = torch.zeros_like(za[:, 0])
        v0, x0 = d64.get("v0", zero), d64.get("x0", zero)
        v = _seq(A, zb * dt, v0)
        one = torch.ones_like(zero).unsqueeze(1).expand_as(A)
        xs = _seq(one, v * dt, x0)
        out = [xs, v] + ([v[:, -1], xs[:, -1]] if case["state"] else [])
        if case["train"]:
            X, X0 = _seq_back(one, d64["gx"], d64.get("gxl", zero))
            lam, m = _seq_back(A, dt * X + d64.get("gv", 0.0), d64.get("gvl", zero))
            vp = torch.cat([v0.unsqueeze(1), v[:, :-1]], 1)
            out.append(torch.cat([lam * vp * A * (1 - A), (lam * zb + X * v) * hs / (1 + torch.exp(-zd)),
                                  lam * dt], -1))
            if case["state"]:
                out += [m, X0]
        return tuple(out)
    return _exact_logits(case, st, d64)


def _exact_logits(case, st, d64):
    """Row by row from the token counts, in float64."""
    x = d64["logits"].clone()
    v = case["vocab"]
    for i, (n, p) in enumerate(zip(st["lengths"].tolist(), st["prompt"].tolist())):
        row, tok = x[i], st["tokens"][i, :n]
        hit = torch.unique(tok)
        row[hit] = torch.where(row[hit] > 0, row[hit] / d64["rep"][i], row[hit] * d64["rep"][i])
        if case["counts"]:
            cnt = torch.bincount(tok[p:], minlength=v)
            row -= d64["freq"][i] * cnt + d64["pres"][i] * (cnt > 0)
    if "bias" in st:
        x += d64["bias"]
    x /= d64["temp"].unsqueeze(1)
    if "allowed" in st:
        col = torch.arange(v, device=x.device)
        bit = (st["allowed"].long()[:, col // 32] >> (col % 32)) & 1
        x[bit == 0] = float("-inf")
    return x
