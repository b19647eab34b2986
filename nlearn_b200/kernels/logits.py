"""Penalties, biases and masks on logits before sampling (``nl_process_logits``).

The reference samples the raw logits (nlearn/model.py:440-444); a serving
loop first discourages tokens that were used, adds per-request biases and
rules out what a grammar does not allow.
"""
from __future__ import annotations

import torch

from .._lib import BF16, F32
from ..paged import _ints1, _ints2, _launch, _no_grad, _refuse_place

_DT = {torch.float32: F32, torch.bfloat16: BF16}


def _per_row(name: str, t, B: int, index: int) -> int:
    if t is None:
        return 0
    if t.dtype is torch.float32 and t.dim() == 1 and t.numel() == B and t.is_contiguous() and t.get_device() == index:
        return t.data_ptr()
    if t.get_device() != index:
        _refuse_place(name, t, index)
    raise ValueError(f"{name} must be a contiguous float32 tensor of shape ({B},)")


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
    index = logits.get_device()
    if index < 0:
        _refuse_place("logits", logits, index)
    _no_grad("process_logits", logits, bias)
    dt = _DT.get(logits.dtype)
    if dt is None:
        raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    if logits.dim() != 2:
        raise ValueError("logits must be [batch, vocab]")
    B, V = logits.shape
    ldx, unit = logits.stride()
    if (V > 1 and unit != 1) or (B > 1 and ldx < V):
        raise ValueError("rows of logits must be contiguous and not overlap")
    if B > 65535 or V == 0:
        raise ValueError(f"logits must have at most 65535 rows and at least one column, got {(B, V)}")
    if out is None:
        # rows on 16-byte boundaries, whatever the vocabulary
        ldy = (V + 7) // 8 * 8 if dt == BF16 else (V + 3) // 4 * 4
        out = logits.new_empty_strided((B, V), (ldy, 1))
    else:
        if out.get_device() != index:
            _refuse_place("out", out, index)
        if out.shape != (B, V) or out.dtype is not logits.dtype:
            raise ValueError("out must have the shape and type of logits")
        ldy, unit = out.stride()
        if (V > 1 and unit != 1) or (B > 1 and ldy < V):
            raise ValueError("rows of out must be contiguous and not overlap")
        same = out.data_ptr() == logits.data_ptr() and (ldy == ldx or B <= 1)
        if not same and _overlap(out, logits):
            raise ValueError("out must be logits itself or not overlap it")
    tp = tl = L = lp = pp = 0
    if tokens is not None:
        if lens is None:
            raise ValueError("tokens come with lens")
        _, L, tl = _ints2("tokens", tokens, B, index)
        lp = _ints1("lens", lens, B, index)
        if prompt_lens is not None:
            pp = _ints1("prompt_lens", prompt_lens, B, index)
        tp = tokens.data_ptr() if L else 0
    elif lens is not None or prompt_lens is not None or repetition is not None or frequency is not None \
            or presence is not None:
        raise ValueError("penalties and lengths come with tokens")
    rp, fp = _per_row("repetition", repetition, B, index), _per_row("frequency", frequency, B, index)
    ap = _per_row("presence", presence, B, index)
    n_bias = ip = bp = ldb = 0
    if bias is not None or bias_ids is not None:
        if bias is None or bias_ids is None:
            raise ValueError("bias and bias_ids come together")
        _, n_bias, ldb = _ints2("bias_ids", bias_ids, B, index)
        if bias.get_device() != index:
            _refuse_place("bias", bias, index)
        if bias.dtype is not torch.float32 or bias.shape != (B, n_bias):
            raise ValueError("bias must be float32 and of bias_ids' shape")
        if bias.stride() != bias_ids.stride():
            bias, bias_ids, ldb = bias.contiguous(), bias_ids.contiguous(), n_bias
        ip, bp = bias_ids.data_ptr(), bias.data_ptr()
    mp = ldm = n_masks = mr = 0
    if mask is not None:
        n_masks, words, ldm = _ints2("mask", mask, None, index)
        if words < (V + 31) // 32:
            raise ValueError(f"mask must have {(V + 31) // 32} words a row, got {words}")
        if mask_rows is not None:
            mr = _ints1("mask_rows", mask_rows, B, index)
        elif n_masks != B:
            raise ValueError(f"mask must have {B} rows, or come with mask_rows")
        mp = mask.data_ptr() if n_masks else 0
    elif mask_rows is not None:
        raise ValueError("mask_rows come with mask")
    if B == 0:
        return out
    _launch("nl_process_logits", index, logits.data_ptr(), out.data_ptr(), tp, lp, pp, rp, fp, ap, ip, bp, mp, mr,
            max(ldx, V), max(ldy, V), tl, ldb, ldm, dt, L, n_bias, n_masks, B, V)
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
