"""Penalties, biases and masks on logits before sampling (``nl_process_logits``).

The reference samples the raw logits (nlearn/model.py:440-444); a serving
loop first discourages tokens that were used, adds per-request biases and
rules out what a grammar does not allow.
"""
from __future__ import annotations

import torch

from .._lib import BF16, F32, check, lib, stream_handle
from ..paged import _cuda, _ints, _no_grad, _on

_DT = {torch.float32: F32, torch.bfloat16: BF16}


def _per_row(name: str, t, B: int, dev) -> int:
    if t is None:
        return 0
    _cuda(name, t, dev)
    if t.dtype != torch.float32 or t.shape != (B,) or (B > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape ({B},)")
    return t.data_ptr()


def process_logits(logits: torch.Tensor, *, tokens: torch.Tensor | None = None, lens: torch.Tensor | None = None,
                   prompt_lens: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   mask: torch.Tensor | None = None, mask_rows: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """logits [B, V] (f32 or bf16, any row pitch) -> processed logits of the same type.

    In this order, each part left out where its arguments are:
      * penalties: row b's tokens are tokens[b, :lens[b]] (int32), the first
        prompt_lens[b] (default 0) its prompt.  A token that occurs: x / r where x > 0,
        else x * r, with r = repetition[b]; one generated c > 0 times after the
        prompt: x - frequency[b] * c - presence[b].
      * bias: bias[b, i] (f32) is added to column bias_ids[b, i] (int32).
      * mask: int32 words [rows, >= ceil(V / 32)]; a column whose bit (v % 32 of
        word v // 32) is 0 becomes -inf.  Row b uses mask row b, or
        mask_rows[b] (int32) where given; below 0 or past the last: no mask.
    Ids outside [0, V) are ignored.  ``out`` may be ``logits`` (in place).
    """
    _cuda("logits", logits)
    dev = logits.device
    _no_grad("process_logits", logits, bias)
    if logits.dtype not in _DT:
        raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [batch, vocab] with contiguous rows")
    B, V = logits.shape
    if B > 65535 or V == 0:
        raise ValueError(f"logits must have at most 65535 rows and at least one column, got {tuple(logits.shape)}")
    if out is None:
        # rows on 16-byte boundaries, whatever the vocabulary
        per = 16 // logits.element_size()
        out = torch.empty(B, (V + per - 1) // per * per, device=dev, dtype=logits.dtype)[:, :V]
    else:
        _cuda("out", out, dev)
        if out.shape != logits.shape or out.dtype != logits.dtype or (V > 1 and out.stride(1) != 1):
            raise ValueError("out must have the shape and type of logits and contiguous rows")
        if out.data_ptr() != logits.data_ptr() and _overlap(out, logits):
            raise ValueError("out must be logits itself or not overlap it")
        if out.data_ptr() == logits.data_ptr() and B > 1 and out.stride(0) != logits.stride(0):
            raise ValueError("out must be logits itself or not overlap it")
    if B > 1 and (out.stride(0) < V or logits.stride(0) < V):
        raise ValueError("rows of logits and out must not overlap")
    tp = tl = L = lp = pp = 0
    if tokens is not None:
        if lens is None:
            raise ValueError("tokens come with lens")
        _ints("tokens", tokens, (B, None), dev)
        _ints("lens", lens, (B,), dev)
        if prompt_lens is not None:
            pp = _ints("prompt_lens", prompt_lens, (B,), dev).data_ptr()
        L = tokens.shape[1]
        if L:
            tp, tl, lp = tokens.data_ptr(), max(tokens.stride(0), L), lens.data_ptr()
    elif any(t is not None for t in (lens, prompt_lens, repetition, frequency, presence)):
        raise ValueError("penalties and lengths come with tokens")
    rp, fp, ap = (_per_row(n, t, B, dev) for n, t in (("repetition", repetition), ("frequency", frequency),
                                                      ("presence", presence)))
    n_bias = ip = bp = ldb = 0
    if (bias is None) != (bias_ids is None):
        raise ValueError("bias and bias_ids come together")
    if bias is not None:
        _ints("bias_ids", bias_ids, (B, None), dev)
        _cuda("bias", bias, dev)
        if bias.dtype != torch.float32 or bias.shape != bias_ids.shape:
            raise ValueError("bias must be float32 and of bias_ids' shape")
        if bias.stride() != bias_ids.stride():
            bias, bias_ids = bias.contiguous(), bias_ids.contiguous()
        n_bias = bias.shape[1]
        ip, bp, ldb = bias_ids.data_ptr(), bias.data_ptr(), max(bias.stride(0), n_bias)
    mp = ldm = n_masks = mr = 0
    if mask is not None:
        _ints("mask", mask, (None, None), dev)
        n_masks, words = mask.shape
        if words < (V + 31) // 32:
            raise ValueError(f"mask must have {(V + 31) // 32} words a row, got {words}")
        if mask_rows is not None:
            mr = _ints("mask_rows", mask_rows, (B,), dev).data_ptr()
        elif n_masks != B:
            raise ValueError(f"mask must have {B} rows, or come with mask_rows")
        if n_masks:
            mp, ldm = mask.data_ptr(), max(mask.stride(0), words)
    elif mask_rows is not None:
        raise ValueError("mask_rows come with mask")
    if B == 0:
        return out
    with _on(dev):
        check(lib.nl_process_logits(logits.data_ptr(), max(logits.stride(0), V), _DT[logits.dtype], out.data_ptr(),
                                    max(out.stride(0), V), tp, tl, lp, pp, L, rp, fp, ap, ip, bp, ldb, n_bias, mp,
                                    ldm, n_masks, mr, B, V, stream_handle()), "nl_process_logits")
    return out


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two row-major matrices meet."""
    def span(t):
        lo = t.data_ptr()
        return lo, lo + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size()
    if a.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


__all__ = ["process_logits"]
