"""Logits before sampling: penalties for the tokens of a row's history, a
bias, the temperature and a grammar mask, in one kernel (the reference samples
from bare logits, gfn/model.py:404-469); and what the logits say of given
tokens: log probabilities, the entropy and the top alternatives, with their
gradient.  CUDA tensors only."""
from typing import NamedTuple, Optional

import torch

from ._lib import GfnError, dtype_code, same_device, torch_ops


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


_CUT = "process_logits is not differentiable: call it under torch.no_grad() or on detached tensors"


def _per_row(v, name, B, x, grad, positive):
    """(number, tensor or None) of a parameter given as a number or per row of x."""
    if not isinstance(v, torch.Tensor):
        if positive and not v > 0:
            raise GfnError(f"process_logits: {name} must be positive, got {v}")
        return v, None
    if v.dtype != torch.float32 or v.dim() != 1 or v.shape[0] != B or v.get_device() != x.get_device():
        raise GfnError(f"process_logits: {name} must be a number or float32 [{B}] on {x.device}, got "
                       f"{v.dtype} {tuple(v.shape)} on {v.device}")
    if grad and v.requires_grad:
        raise GfnError(_CUT)
    return 1.0, v if v.is_contiguous() else v.contiguous()


def _rows_or_shared(t, name, B, n):
    """t [n] or [B, n] with inner stride 1, and its row stride (0: shared)."""
    if t.shape != (n,) and t.shape != (B, n):
        raise GfnError(f"process_logits: {name} must be [{n}] or [{B}, {n}], got {tuple(t.shape)}")
    if t.stride(-1) != 1 and n > 1:
        t = t.contiguous()
    return t, (t.stride(0) if t.dim() == 2 else 0)


def _lengths(t, name, B):
    if t.dim() != 1 or t.shape[0] != B or (t.dtype != torch.int64 and t.dtype != torch.int32):
        raise GfnError(f"process_logits: {name} must be int64 [{B}], got {t.dtype} {tuple(t.shape)}")
    t = t if t.dtype == torch.int64 else t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


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
    grad = torch.is_grad_enabled()
    if grad and (logits.requires_grad or (bias is not None and bias.requires_grad)):
        raise GfnError(_CUT)
    dtype_code(logits, "logits")
    B, V = logits.shape
    x = logits if logits.is_contiguous() or V == 1 or logits.stride(1) == 1 else logits.contiguous()
    ts = 0
    if tokens is not None:
        if tokens.dim() != 2 or tokens.shape[0] != B or (tokens.dtype != torch.int64 and tokens.dtype != torch.int32):
            raise GfnError(f"process_logits: tokens must be int64 [{B}, T], got {tokens.dtype} {tuple(tokens.shape)}")
        T = tokens.shape[1]
        if tokens.dtype != torch.int64:
            tokens = tokens.to(torch.int64)
        ts, step = tokens.stride()
        if T > 1 and step != 1:
            tokens = tokens.contiguous()
            ts = T
        lengths = None if lengths is None else _lengths(lengths, "lengths", B)
        prompt_lengths = None if prompt_lengths is None else _lengths(prompt_lengths, "prompt_lengths", B)
    elif lengths is not None or prompt_lengths is not None:
        raise GfnError("process_logits: lengths need tokens")
    rep, rep_rows = _per_row(repetition_penalty, "repetition_penalty", B, logits, grad, True)
    freq, freq_rows = _per_row(frequency_penalty, "frequency_penalty", B, logits, grad, False)
    pres, pres_rows = _per_row(presence_penalty, "presence_penalty", B, logits, grad, False)
    temp, temp_rows = _per_row(temperature, "temperature", B, logits, grad, True)
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
    return torch_ops().process_logits(x, tokens, ts, lengths, prompt_lengths, rep, freq, pres, temp, rep_rows, freq_rows,
                                      pres_rows, temp_rows, bias, bs, allowed, ms)


class TokenLogprobs(NamedTuple):
    """Float32 of the logits' leading shape (the last two: [..., top], int64 tokens); None where not asked for."""
    logprobs: Optional[torch.Tensor]
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def token_logprobs(logits, tokens=None, top=0, entropy=False, ignore_index=-100):
    """TokenLogprobs of logits [..., vocab]: the log probability of each row's
    token, the row's entropy, and its `top` most probable tokens (at most 32,
    largest first, the lowest token first where logits are equal).

    logits: float32, bfloat16 or float16; rows of a wider tensor are read in
    place.  tokens: int64 or int32 of the logits' leading shape, or None.  A token
    equal to ignore_index has log probability 0 and no gradient; another one
    outside the vocabulary gives NaN and sets a device error bit
    (gfn.cuda.ops.device_error).  Logits of -inf (masked tokens) have probability
    0.  A row that has none above -inf gives -inf, entropy 0 and a gradient of
    zeros; one with NaN or +inf gives NaN.  Differentiable (once) in the logits,
    through every float result.
    """
    return TokenLogprobs(*torch_ops().token_logprobs(logits, tokens, top, entropy, ignore_index))
