"""Logits before sampling: penalties for the tokens of a row's history, a
bias, the temperature and a grammar mask, in one kernel (the reference samples
from bare logits, gfn/model.py:404-469).  CUDA tensors only."""
import torch

from . import _lib
from ._lib import GfnError, call_on, dtype_code, ptr, same_device


def pack_token_mask(mask):
    """bool [..., vocab] -> int32 words [..., ceil(vocab / 32)], bit i of word w
    for token 32 w + i (the form process_logits reads)."""
    if mask.dtype != torch.bool:
        raise GfnError(f"pack_token_mask: mask must be bool, got {mask.dtype}")
    words = (mask.shape[-1] + 31) // 32
    m = torch.nn.functional.pad(mask, (0, 32 * words - mask.shape[-1]))
    bits = m.reshape(*mask.shape[:-1], words, 32).long() << torch.arange(32, device=mask.device)
    w = bits.sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _per_row(v, name, B, positive):
    """(number, per-row tensor or None) of a parameter given as either."""
    if not torch.is_tensor(v):
        if positive and not v > 0:
            raise GfnError(f"process_logits: {name} must be positive, got {v}")
        return float(v), None
    if v.dtype != torch.float32 or v.shape != (B,):
        raise GfnError(f"process_logits: {name} must be a number or float32 [{B}], got {v.dtype} {tuple(v.shape)}")
    return 1.0, v.contiguous()


def _rows_or_shared(t, name, B, n):
    """t [n] or [B, n] with inner stride 1, and its row stride (0: shared)."""
    if t.shape != (n,) and t.shape != (B, n):
        raise GfnError(f"process_logits: {name} must be [{n}] or [{B}, {n}], got {tuple(t.shape)}")
    if t.stride(-1) != 1 and n > 1:
        t = t.contiguous()
    return t, (t.stride(0) if t.dim() == 2 else 0)


def _index(t, name, shape):
    if t.dtype not in (torch.int64, torch.int32) or t.shape != shape:
        raise GfnError(f"process_logits: {name} must be int64 {list(shape)}, got {t.dtype} {tuple(t.shape)}")
    return t.to(torch.int64)


def process_logits(logits, tokens=None, lengths=None, prompt_lengths=None, repetition_penalty=1.0,
                   frequency_penalty=0.0, presence_penalty=0.0, bias=None, temperature=1.0, allowed=None):
    """New logits [batch, vocab] for sampling, of the logits' type, from

      s = x > 0 ? x / repetition_penalty : x * repetition_penalty   (token in the history)
      s = s - (frequency_penalty * count + presence_penalty)        (count > 0)
      out = (s + bias) / temperature, -inf where not allowed

    tokens [batch, T] int64: each row's history; of a row the first
    lengths[row] tokens count (None: all), and those from prompt_lengths[row]
    on (None: all) are the generated ones that `count` counts.  A token outside
    the vocabulary is skipped and sets a device error bit
    (gfn.cuda.ops.device_error).  Each penalty and the temperature: a number,
    or a float32 tensor [batch]; repetition penalty and temperature are
    positive.  bias: [vocab] or [batch, vocab].  allowed: bool [vocab] or
    [batch, vocab], or its packed int32 words (pack_token_mask).  A row whose
    mask leaves nothing comes back all -inf.  Not differentiable.
    """
    same_device("process_logits", logits, tokens, lengths, prompt_lengths, bias, allowed)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise GfnError(f"process_logits: logits must be [batch, vocab], got {tuple(logits.shape)}")
    if torch.is_grad_enabled() and logits.requires_grad:
        raise GfnError("process_logits is not differentiable: call it under torch.no_grad() or on logits.detach()")
    code = dtype_code(logits, "logits")
    B, V = logits.shape
    x = logits if V == 1 or logits.stride(1) == 1 else logits.contiguous()
    T = 0
    if tokens is not None:
        tokens = _index(tokens, "tokens", (B, tokens.shape[-1]))
        T = tokens.shape[1]
        if T > 1 and tokens.stride(1) != 1:
            tokens = tokens.contiguous()
        lengths = None if lengths is None else _index(lengths, "lengths", (B,)).contiguous()
        if prompt_lengths is not None:
            prompt_lengths = _index(prompt_lengths, "prompt_lengths", (B,)).contiguous()
    elif lengths is not None or prompt_lengths is not None:
        raise GfnError("process_logits: lengths need tokens")
    rep, rep_rows = _per_row(repetition_penalty, "repetition_penalty", B, True)
    freq, freq_rows = _per_row(frequency_penalty, "frequency_penalty", B, False)
    pres, pres_rows = _per_row(presence_penalty, "presence_penalty", B, False)
    temp, temp_rows = _per_row(temperature, "temperature", B, True)
    same_device("process_logits", logits, rep_rows, freq_rows, pres_rows, temp_rows)
    bs = ms = 0
    if bias is not None:
        bias, bs = _rows_or_shared(bias.to(torch.float32), "bias", B, V)
    if allowed is not None:
        if allowed.dtype == torch.bool:
            if allowed.shape[-1:] != (V,):
                raise GfnError(f"process_logits: allowed must cover {V} tokens, got {tuple(allowed.shape)}")
            allowed = pack_token_mask(allowed)
        if allowed.dtype != torch.int32:
            raise GfnError(f"process_logits: allowed must be bool or int32 words, got {allowed.dtype}")
        allowed, ms = _rows_or_shared(allowed, "allowed", B, (V + 31) // 32)
    out = torch.empty(B, V, device=logits.device, dtype=logits.dtype)
    call_on(logits, "gfn_process_logits", ptr(x), x.stride(0) if B > 1 else V, code, B, V, ptr(tokens),
            tokens.stride(0) if T else 0, T, ptr(lengths), ptr(prompt_lengths), rep, ptr(rep_rows), freq,
            ptr(freq_rows), pres, ptr(pres_rows), temp, ptr(temp_rows), ptr(bias), bs, ptr(allowed), ms, ptr(out))
    return out
