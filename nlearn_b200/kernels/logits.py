"""Penalties, biases and masks on logits before sampling (``nl_process_logits``).

The reference samples the raw logits (nlearn/model.py:440-444); a serving
loop first discourages tokens that were used, adds per-request biases and
rules out what a grammar does not allow.
"""
from __future__ import annotations

import torch

from ..paged import _host


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
    return _host.process_logits(logits, tokens, lens, prompt_lens, repetition, frequency, presence, bias_ids, bias,
                                mask, mask_rows, out)


__all__ = ["process_logits"]
