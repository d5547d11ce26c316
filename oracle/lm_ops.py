"""Float64 definitions of the language-model operators and their gradients
(layer norm, gated scan, the scan layer's recurrence, logit shaping, token embedding, log
probabilities, attention with decay): plain
numpy, one step after the other, the yardstick of the kernels' tests."""
import numpy as np


def layer_norm(x, w=None, b=None, eps=1e-5):
    x = np.asarray(x, np.float64)
    mu = x.mean(-1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mu) ** 2).mean(-1, keepdims=True) + eps)
    y = (x - mu) * rstd
    if w is not None:
        y = y * w
    return y if b is None else y + b


def layer_norm_backward(x, dy, w=None, eps=1e-5):
    """(dx, dweight, dbias) of sum(dy * layer_norm(x))."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    mu = x.mean(-1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mu) ** 2).mean(-1, keepdims=True) + eps)
    xh = (x - mu) * rstd
    g = dy if w is None else dy * w
    dx = rstd * (g - g.mean(-1, keepdims=True) - xh * (g * xh).mean(-1, keepdims=True))
    axes = tuple(range(x.ndim - 1))
    return dx, (dy * xh).sum(axes), dy.sum(axes)


def gated_scan(a, x, h0=None):
    """h_t = a_t h_{t-1} + x_t over axis 1 of [B, L, D]; returns (h, last state)."""
    x = np.asarray(x, np.float64)
    a = np.ones_like(x) if a is None else np.broadcast_to(np.asarray(a, np.float64), x.shape)
    h = np.zeros_like(x[:, :1].sum(1)) if h0 is None else np.asarray(h0, np.float64)
    out = np.empty_like(x)
    for t in range(x.shape[1]):
        h = a[:, t] * h + x[:, t]
        out[:, t] = h
    return out, h


def gated_scan_backward(a, x, h0, dh, dlast):
    """(da, dx, dh0) of sum(dh * h) + sum(dlast * last)."""
    h, _ = gated_scan(a, x, h0)
    a = np.ones_like(h) if a is None else np.broadcast_to(np.asarray(a, np.float64), h.shape)
    first = np.zeros_like(h[:, :1].sum(1)) if h0 is None else np.asarray(h0, np.float64)
    m = np.zeros_like(first) if dlast is None else np.asarray(dlast, np.float64)
    da, dx = np.empty_like(h), np.empty_like(h)
    for t in range(h.shape[1] - 1, -1, -1):
        g = m if dh is None else dh[:, t] + m
        dx[:, t] = g
        da[:, t] = g * (h[:, t - 1] if t else first)
        m = a[:, t] * g
    return da, dx, m


def _sigmoid(z):
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1.0, e) / (1.0 + e)


def layer_scan_terms(z, heads, base_dt):
    """(A, 1 - A, dt, sigma(zdt), head scale) of the scan layer's pre-activations [zA | zdt | zB];
    1 - A = sigma(-zA) keeps its digits where A rounds to 1."""
    z = np.asarray(z, np.float64)
    D = z.shape[-1] // 3
    hs = base_dt * np.repeat(1.5 ** np.arange(heads), D // heads)
    return _sigmoid(z[..., :D]), _sigmoid(-z[..., :D]), np.logaddexp(0.0, z[..., D:2 * D]) * hs, _sigmoid(z[..., D:2 * D]), hs


def layer_scan(z, heads, base_dt, v0=None, x0=None):
    """v_t = A_t v_{t-1} + zB_t dt_t, x_t = x_{t-1} + v_t dt_t; returns (x, v, last x, last v)."""
    z = np.asarray(z, np.float64)
    D = z.shape[-1] // 3
    A, _, dt, _, _ = layer_scan_terms(z, heads, base_dt)
    v, vl = gated_scan(A, z[..., 2 * D:] * dt, v0)
    x, xl = gated_scan(None, v * dt, x0)
    return x, v, xl, vl


def layer_scan_backward(z, heads, base_dt, v0, gx, gv, gxl=None, gvl=None):
    """(dz, dv0, dx0) of sum(gx x) + sum(gv v) + sum(gxl x_last) + sum(gvl v_last)."""
    z = np.asarray(z, np.float64)
    D = z.shape[-1] // 3
    A, nA, dt, sdt, hs = layer_scan_terms(z, heads, base_dt)
    zb = z[..., 2 * D:]
    v, _ = gated_scan(A, zb * dt, v0)
    zero = np.zeros((z.shape[0], D))
    first = zero if v0 is None else np.asarray(v0, np.float64)
    X = zero if gxl is None else np.asarray(gxl, np.float64)
    m = zero if gvl is None else np.asarray(gvl, np.float64)
    dz = np.empty_like(z)
    for t in range(z.shape[1] - 1, -1, -1):
        if gx is not None:
            X = X + gx[:, t]
        lam = dt[:, t] * X + m
        if gv is not None:
            lam = lam + gv[:, t]
        vp = v[:, t - 1] if t else first
        dz[:, t, :D] = lam * vp * A[:, t] * nA[:, t]
        dz[:, t, D:2 * D] = (lam * zb[:, t] + X * v[:, t]) * hs * sdt[:, t]
        dz[:, t, 2 * D:] = lam * dt[:, t]
        m = A[:, t] * lam
    return dz, m, X


def process_logits(logits, tokens=None, lengths=None, prompt_lengths=None, rep=1.0, freq=0.0, pres=0.0,
                   bias=None, temperature=1.0, allowed=None):
    """Row by row: repetition penalty on every token of the history, frequency and presence
    penalties on the generated part, bias, temperature, mask (bool [V] or [B, V])."""
    x = np.array(logits, np.float64)
    B, V = x.shape
    per_row = lambda p: np.broadcast_to(np.asarray(p, np.float64), (B,))  # noqa: E731
    rep, freq, pres, temperature = map(per_row, (rep, freq, pres, temperature))
    for i in range(B):
        if tokens is not None:
            n = tokens.shape[1] if lengths is None else int(lengths[i])
            p = 0 if prompt_lengths is None else int(prompt_lengths[i])
            hist = [int(t) for t in tokens[i, :n]]
            for t in set(t for t in hist if 0 <= t < V):
                x[i, t] = x[i, t] / rep[i] if x[i, t] > 0 else x[i, t] * rep[i]
                c = sum(1 for u in hist[p:] if u == t)
                if c:
                    x[i, t] -= freq[i] * c + pres[i]
        if bias is not None:
            x[i] += np.broadcast_to(np.asarray(bias, np.float64), (B, V))[i]
        x[i] /= temperature[i]
        if allowed is not None:
            x[i] = np.where(np.broadcast_to(allowed, (B, V))[i], x[i], -np.inf)
    return x


def embed_tokens(ids, weight, scale=1.0):
    """scale * weight[ids], zeros for ids outside the table."""
    w, ids = np.asarray(weight, np.float64), np.asarray(ids)
    y = np.zeros(ids.shape + (w.shape[1],))
    ok = (ids >= 0) & (ids < w.shape[0])
    y[ok] = scale * w[ids[ok]]
    return y


def embed_tokens_backward(ids, dy, vocab, scale=1.0, padding_idx=None):
    """dweight of sum(dy * embed_tokens)."""
    dy = np.asarray(dy, np.float64)
    dw = np.zeros((vocab, dy.shape[-1]))
    for i, g in zip(np.asarray(ids).reshape(-1), dy.reshape(-1, dy.shape[-1])):
        if 0 <= i < vocab and i != padding_idx:
            dw[i] += scale * g
    return dw


def token_logprobs(logits, tokens=None, top=0, ignore_index=-100):
    """Row by row (logprobs, entropy, top_logprobs, top_tokens): of equal logits the lower token first, NaN above all."""
    x = np.asarray(logits, np.float64)
    N, V = x.shape
    lp, ent = np.zeros(N), np.zeros(N)
    top_lp, top_id = np.zeros((N, top)), np.zeros((N, top), np.int64)
    for i in range(N):
        if np.isnan(x[i]).any() or (x[i] == np.inf).any():
            logp = np.full(V, np.nan)
            ent[i] = np.nan
        elif (x[i] == -np.inf).all():
            logp = np.full(V, -np.inf)
        else:
            m = x[i].max()
            logp = (x[i] - m) - np.log(np.exp(x[i] - m).sum())
            live = logp > -np.inf
            ent[i] = -(np.exp(logp[live]) * logp[live]).sum()
        key = np.where(np.isnan(x[i]), np.inf, x[i])
        order = np.lexsort((np.arange(V), -key, ~np.isnan(x[i])))[:top]
        top_id[i], top_lp[i] = order, logp[order]
        if tokens is not None and tokens[i] != ignore_index:
            lp[i] = logp[tokens[i]] if 0 <= tokens[i] < V else np.nan
    return lp, ent, top_lp, top_id


def token_logprobs_backward(logits, tokens, top_tokens, g_lp, g_ent, g_top, ignore_index=-100):
    """dlogits of sum(g_lp logprobs) + sum(g_ent entropy) + sum(g_top top_logprobs); each g may be None."""
    x = np.asarray(logits, np.float64)
    N, V = x.shape
    dx = np.zeros((N, V))
    for i in range(N):
        if (x[i] == -np.inf).all():
            continue
        m = x[i].max()
        logp = (x[i] - m) - np.log(np.exp(x[i] - m).sum())
        p = np.exp(logp)
        pairs = [] if g_lp is None or tokens[i] == ignore_index else [(tokens[i], g_lp[i])]
        pairs += [] if g_top is None else list(zip(top_tokens[i], g_top[i]))
        for t, g in pairs:
            dx[i] -= g * p
            dx[i, t] += g
        if g_ent is not None:
            live = p > 0
            H = -(p[live] * logp[live]).sum()
            dx[i, live] -= g_ent[i] * p[live] * (logp[live] + H)
    return dx


def decay_attention(q, k, v, decay, state=None, lengths=None, scale=1.0):
    """S_t = decay S_{t-1} + k_t v_t^T, o_t = scale q_t S_t on [B, L, H, .]; returns (o, last state)."""
    q, k, v, decay = (np.asarray(t, np.float64) for t in (q, k, v, decay))
    B, L, H, K = q.shape
    S = np.zeros((B, H, K, v.shape[3])) if state is None else np.array(state, np.float64)
    o = np.zeros(v.shape)
    for b in range(B):
        for t in range(L if lengths is None else min(max(int(lengths[b]), 0), L)):
            S[b] = decay[:, None, None] * S[b] + k[b, t][:, :, None] * v[b, t][:, None, :]
            o[b, t] = scale * np.einsum("hk,hkv->hv", q[b, t], S[b])
    return o, S


def decay_attention_backward(q, k, v, decay, state, lengths, scale, do, dlast=None):
    """(dq, dk, dv, dstate) of sum(do * o) + sum(dlast * last state)."""
    q, k, v, decay = (np.asarray(t, np.float64) for t in (q, k, v, decay))
    B, L, H, K = q.shape
    S = np.zeros((B, H, K, v.shape[3])) if state is None else np.array(state, np.float64)
    R = np.zeros_like(S) if dlast is None else np.array(dlast, np.float64)
    do = np.zeros(v.shape) if do is None else np.asarray(do, np.float64)
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        for t in range(n):
            S[b] = decay[:, None, None] * S[b] + k[b, t][:, :, None] * v[b, t][:, None, :]
            dq[b, t] = scale * np.einsum("hv,hkv->hk", do[b, t], S[b])
        for t in range(n - 1, -1, -1):
            G = R[b] + scale * q[b, t][:, :, None] * do[b, t][:, None, :]
            dk[b, t] = np.einsum("hkv,hv->hk", G, v[b, t])
            dv[b, t] = np.einsum("hkv,hk->hv", G, k[b, t])
            R[b] = decay[:, None, None] * G
    return dq, dk, dv, R
