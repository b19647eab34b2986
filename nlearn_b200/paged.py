"""Paged key-value caches: decode attention, writes into pages, block tables.

A sequence's keys and values lie in pages of ``page_size`` tokens that belong
to it one by one, so sequences of any lengths share one cache.  A layer has a
key cache and a value cache of logical shape

    [n_pages, kv_heads, page_size, head_dim]        (bf16, or float8_e4m3fn)

with any strides whose rows are contiguous and 16-byte aligned (a token-major
cache [n_pages, page_size, kv_heads, head_dim] is passed as its
``transpose(1, 2)``).  ``block_table`` (int32 [batch, max_blocks]) lists each
sequence's pages in order, ``slot = page * page_size + row``.

* ``update_block_tables``   lengths -> pages, block tables, slots (one launch)
* ``paged_kv_write``        keys and values of many tokens into their slots
* ``paged_decode_attention`` attention of one new token per sequence, which may
                            also append that token's key and value

All run on the current CUDA stream of the tensors' device, read lengths and
tables on the device (no host copy: a step can be captured into a CUDA graph),
and have no backward.  The reference has no counterpart (nlearn/model.py:
417-465 recomputes the whole sequence for every token).
"""
from __future__ import annotations

from typing import NamedTuple

import torch


class _Ops:
    """The compiled host side of these operators (csrc/host/ops_py.cpp), loaded on first use."""

    def __getattr__(self, name):
        try:
            from . import _ops
        except ImportError as e:
            raise ImportError(f"nlearn_b200._ops is missing ({e}): build it with `python -m nlearn_b200.build`") from e
        for fn in ("paged_decode_attention", "paged_kv_write", "update_block_tables", "process_logits"):
            setattr(self, fn, getattr(_ops, fn))
        return getattr(_ops, name)


_host = _Ops()


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                           lens: torch.Tensor, k_new: torch.Tensor | None = None, v_new: torch.Tensor | None = None,
                           *, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                           scale: float | None = None, out: torch.Tensor | None = None,
                           lse: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale * q k^T) v of one new token per sequence over its pages.

    q [B, Hq, d] bf16 (d 64 or 128; Hq a multiple of the caches' head count, query
    head h reads kv head h // (Hq / Hk)); lens int32 [B] counts the keys, the
    new token's included (0: the row's output is 0 and its lse -inf, as where every
    score is -inf).  With k_new and v_new [B, Hk, d], key lens - 1 comes from
    there and is written into its slot in the caches (the page that takes it
    stands in no other place of the tables); without them it is in the cache
    already.  An infinite element of v_cache gives NaN in its column.  scale
    defaults to d**-0.5; k_scale, v_scale (f32 [Hk]) multiply an e4m3
    cache's values.  lse (f32 [B, Hq]), if given, is filled with the log of the sum of
    exp(scaled scores).  -> out [B, Hq, d] bf16; an ``out`` that is given may
    be q itself and shares no other memory with the operands.
    """
    return _host.paged_decode_attention(q, k_cache, v_cache, block_table, lens, k_new, v_new, k_scale, v_scale, scale,
                                        out, lse)


def paged_kv_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slots: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None) -> None:
    """Write k, v [T, kv_heads, head_dim] (bf16; strided views of a fused qkv
    projection are read in place) into slots[t] (int32 [T]) of the caches.
    Negative slots are padding; no slot may occur twice, and k and v lie in none
    of them.  An e4m3 cache holds round(x / scale), saturating at 448."""
    _host.paged_kv_write(k, v, k_cache, v_cache, slots, k_scale, v_scale)


class BlockPlan(NamedTuple):
    """What one serving step writes and where (all int32, on the device).  The tensors
    that the call made are parts of one allocation, which lives as long as any of them."""
    slots: torch.Tensor      # [n_tokens] slot of each token of the flat list, -1: none
    positions: torch.Tensor  # [n_tokens] its position in its sequence, -1: none
    cu: torch.Tensor         # [batch + 1] first token of each row
    lens: torch.Tensor       # [batch] lengths after the step
    n_free: torch.Tensor     # [1] free pages after the step
    status: torch.Tensor     # [batch] 0, or why the row was refused (ROW_*)


ROW_OK, ROW_NO_PAGES, ROW_TOO_LONG, ROW_NO_SLOTS, ROW_INVALID = range(5)
MAX_ROWS = 8192


def update_block_tables(block_table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor,
                        free_pages: torch.Tensor, n_free: torch.Tensor, page_size: int, n_tokens: int, *,
                        done: torch.Tensor | None = None, lens_out: torch.Tensor | None = None,
                        n_free_out: torch.Tensor | None = None) -> BlockPlan:
    """One serving step of the block tables, on the device and in one launch
    (at most MAX_ROWS rows).

    Rows with done != 0 give their pages back and restart at length 0; then
    every row grows by new_lens tokens, taking the pages that needs from the stack
    free_pages[:n_free] (its size is the number of pages of the cache).
    block_table and free_pages are updated in place; lens and n_free too where
    lens_out=lens and n_free_out=n_free are passed.  A row that cannot be
    served (see ``BlockPlan.status``: ROW_NO_PAGES, ROW_TOO_LONG, ROW_NO_SLOTS,
    ROW_INVALID) keeps its length and gets no slots; rows are served in order,
    and after one that finds no pages no later row gets any.  n_tokens is
    the length of the flat token list that slots and positions cover.
    """
    return BlockPlan._make(_host.update_block_tables(block_table, lens, new_lens, free_pages, n_free, page_size,
                                                     n_tokens, done, lens_out, n_free_out))


__all__ = ["paged_decode_attention", "paged_kv_write", "update_block_tables", "BlockPlan", "ROW_OK", "ROW_NO_PAGES",
           "ROW_TOO_LONG", "ROW_NO_SLOTS", "ROW_INVALID", "MAX_ROWS"]
