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

from contextlib import nullcontext
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib, stream_handle

_CACHE_DT = {torch.bfloat16: _lib.BF16, torch.float8_e4m3fn: _lib.E4M3}
HEAD_DIMS = (64, 128)


def _cuda(name: str, t: torch.Tensor, device=None) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name}: nlearn_b200 paged operators run on CUDA tensors only (no CPU fallback)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _on(device: torch.device):
    """Context in which `device` is current (entry points launch on the current device)."""
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _ints(name: str, t: torch.Tensor, shape: tuple, device) -> torch.Tensor:
    """An int32 tensor of `shape` (None: any size) with unit stride along its last dim."""
    _cuda(name, t, device)
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != len(shape) or any(want is not None and have != want for have, want in zip(t.shape, shape)):
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")
    return t


def _no_grad(name: str, *ts) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError(f"{name} has no backward: call it under torch.no_grad()")


def _rows(name: str, t: torch.Tensor) -> torch.Tensor:
    """bf16 [n, heads, d] with contiguous 16-byte aligned rows (copied only when needed)."""
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        return t.contiguous()
    return t


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, device):
    """Checks both caches; -> (dtype code, page, head, token strides)."""
    _cuda("k_cache", k_cache, device)
    _cuda("v_cache", v_cache, device)
    dt = _CACHE_DT.get(k_cache.dtype)
    if dt is None or v_cache.dtype != k_cache.dtype:
        raise TypeError(f"caches must both be bfloat16 or float8_e4m3fn, got {k_cache.dtype} and {v_cache.dtype}")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("caches must be [n_pages, kv_heads, page_size, head_dim], both of one shape, got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    st = k_cache.stride()
    if v_cache.stride() != st:
        raise ValueError(f"caches must have the same strides, got {st} and {v_cache.stride()}")
    per = 16 // k_cache.element_size()
    if st[3] != 1 or any(s % per for s in st[:3]) or k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16:
        raise ValueError("cache rows must be contiguous and lie on 16-byte boundaries")
    n_pages, heads, page, d = k_cache.shape
    if n_pages * page > 2**31 - 1:
        raise ValueError(f"cache has {n_pages * page} slots, over the limit of 2**31 - 1")
    return dt, st[0], st[1], st[2]


def _scale(name: str, t, heads: int, cache: torch.Tensor):
    if t is None:
        return 0
    if cache.dtype == torch.bfloat16:
        raise ValueError(f"{name} goes with a float8_e4m3fn cache")
    _cuda(name, t, cache.device)
    if t.dtype != torch.float32 or t.shape != (heads,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape ({heads},)")
    return t.data_ptr()


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                           lens: torch.Tensor, k_new: torch.Tensor | None = None, v_new: torch.Tensor | None = None,
                           *, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                           scale: float | None = None, out: torch.Tensor | None = None,
                           lse: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale * q k^T) v of one new token per sequence over its pages.

    q [B, Hq, d] bf16 (d 64 or 128; Hq a multiple of the caches' head count, query
    head h reads kv head h // (Hq / Hk)); lens int32 [B] counts the keys, the
    new token's included (0: the row's output is 0 and its lse -inf).  With k_new
    and v_new [B, Hk, d], key lens - 1 comes from there and is written into
    its slot in the caches; without them it is in the cache already.  scale
    defaults to d**-0.5; k_scale, v_scale (f32 [Hk]) multiply an e4m3
    cache's values.  lse (f32 [B, Hq]), if given, is filled with the log of the sum of
    exp(scaled scores).  -> out [B, Hq, d] bf16.
    """
    _cuda("q", q)
    dev = q.device
    _no_grad("paged_decode_attention", q, k_new, v_new)
    if q.dim() != 3:
        raise ValueError(f"q must be [batch, heads, head_dim], got {tuple(q.shape)}")
    dt, page_s, head_s, tok_s = _caches(k_cache, v_cache, dev)
    B, Hq, d = q.shape
    n_pages, Hk, page, dk = k_cache.shape
    if d != dk or d not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} and the caches', got {d} and {dk}")
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads do not share {Hk} kv heads evenly")
    q = _rows("q", q)
    _ints("block_table", block_table, (B, None), dev)
    _ints("lens", lens, (B,), dev)
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new come together")
    n_b = n_h = kn = vn = 0
    if k_new is not None:
        for name, t in (("k_new", k_new), ("v_new", v_new)):
            _cuda(name, t, dev)
            if t.shape != (B, Hk, d):
                raise ValueError(f"{name} must have shape {(B, Hk, d)}, got {tuple(t.shape)}")
        k_new, v_new = _rows("k_new", k_new), _rows("v_new", v_new)
        if k_new.stride() != v_new.stride():
            k_new, v_new = k_new.contiguous(), v_new.contiguous()
        n_b, n_h, kn, vn = k_new.stride(0), k_new.stride(1), k_new.data_ptr(), v_new.data_ptr()
    ks, vs = _scale("k_scale", k_scale, Hk, k_cache), _scale("v_scale", v_scale, Hk, v_cache)
    if out is None:
        out = torch.empty(B, Hq, d, device=dev, dtype=torch.bfloat16)
    else:
        _cuda("out", out, dev)
        if out.shape != (B, Hq, d) or out.dtype != torch.bfloat16 or out.stride(2) != 1:
            raise ValueError(f"out must be bfloat16 {(B, Hq, d)} with contiguous rows")
    lp = ls = 0
    if lse is not None:
        _cuda("lse", lse, dev)
        if lse.shape != (B, Hq) or lse.dtype != torch.float32 or (Hq > 1 and lse.stride(1) != 1):
            raise ValueError(f"lse must be float32 {(B, Hq)} with contiguous rows")
        lp, ls = lse.data_ptr(), lse.stride(0)
    if B == 0:
        return out
    blocks = block_table.shape[1]
    if blocks == 0 or n_pages == 0 or page == 0:
        raise ValueError("block_table and caches must hold at least one page")
    with _on(dev):
        nb = lib.nl_paged_attention_workspace_bytes(B, Hq, Hk, d, page, blocks, dt)
        ws = torch.empty(nb, device=dev, dtype=torch.uint8)
        check(lib.nl_paged_attention(q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
                                     dt, page_s, head_s, tok_s, block_table.data_ptr(),
                                     max(block_table.stride(0), blocks), lens.data_ptr(), kn, vn, n_b, n_h, ks, vs,
                                     d ** -0.5 if scale is None else float(scale), out.data_ptr(), out.stride(0),
                                     out.stride(1), lp, ls, ws.data_ptr(), nb, B, Hq, Hk, d, page, blocks, n_pages,
                                     stream_handle()), "nl_paged_attention")
    return out


def paged_kv_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slots: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None) -> None:
    """Write k, v [T, kv_heads, head_dim] (bf16; strided views of a fused qkv
    projection are read in place) into slots[t] (int32 [T]) of the caches.
    Negative slots are padding; no slot may occur twice.  An e4m3 cache holds
    round(x / scale), saturating at 448."""
    _cuda("k", k)
    dev = k.device
    _cuda("v", v, dev)
    _no_grad("paged_kv_write", k, v)
    dt, page_s, head_s, tok_s = _caches(k_cache, v_cache, dev)
    n_pages, Hk, page, d = k_cache.shape
    if k.dim() != 3 or k.shape[1:] != (Hk, d) or v.shape != k.shape:
        raise ValueError(f"k and v must be [tokens, {Hk}, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if d % (16 // k_cache.element_size()):
        raise ValueError(f"head_dim {d}: cache rows must be whole 16-byte pieces")
    T = k.shape[0]
    _ints("slots", slots, (T,), dev)
    k, v = _rows("k", k), _rows("v", v)
    if k.stride() != v.stride():
        k, v = k.contiguous(), v.contiguous()
    ks, vs = _scale("k_scale", k_scale, Hk, k_cache), _scale("v_scale", v_scale, Hk, v_cache)
    if T == 0 or k_cache.numel() == 0:
        return
    with _on(dev):
        check(lib.nl_paged_kv_write(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k_cache.data_ptr(),
                                    v_cache.data_ptr(), dt, page_s, head_s, tok_s, slots.data_ptr(), ks, vs, T, Hk,
                                    d, page, n_pages, stream_handle()), "nl_paged_kv_write")


class BlockPlan(NamedTuple):
    """What one serving step writes and where (all int32, on the device)."""
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
    """One serving step of the block tables, on the device and in one launch.

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
    _cuda("block_table", block_table)
    dev = block_table.device
    _ints("block_table", block_table, (None, None), dev)
    B, blocks = block_table.shape
    for name, t in (("lens", lens), ("new_lens", new_lens), ("done", done), ("lens_out", lens_out)):
        if t is not None:
            _ints(name, t, (B,), dev)
    _ints("free_pages", free_pages, (None,), dev)
    for name, t in (("n_free", n_free), ("n_free_out", n_free_out)):
        if t is not None:
            _ints(name, t, (1,), dev)
    n_pages = free_pages.shape[0]
    if B == 0 or B > MAX_ROWS or blocks == 0 or n_pages == 0:
        raise ValueError(f"block_table must have 1 to {MAX_ROWS} rows and at least one page a row, got "
                         f"{tuple(block_table.shape)} and {n_pages} pages")
    if page_size < 1 or n_tokens < 0 or blocks * page_size > 2**31 - 1 or n_pages * page_size > 2**31 - 1:
        raise ValueError(f"page_size {page_size}, n_tokens {n_tokens}: out of range")
    sizes = [n_tokens, n_tokens, B + 1, B, B, 1]
    slots, positions, cu, status, lo, nf = torch.empty(sum(sizes), device=dev, dtype=torch.int32).split(sizes)
    lens_out = lo if lens_out is None else lens_out
    n_free_out = nf if n_free_out is None else n_free_out
    with _on(dev):
        check(lib.nl_update_block_tables(block_table.data_ptr(), max(block_table.stride(0), blocks), lens.data_ptr(),
                                         new_lens.data_ptr(), 0 if done is None else done.data_ptr(),
                                         free_pages.data_ptr(), n_free.data_ptr(), lens_out.data_ptr(),
                                         n_free_out.data_ptr(), slots.data_ptr(), positions.data_ptr(),
                                         cu.data_ptr(), status.data_ptr(), B, blocks, page_size, n_pages, n_tokens,
                                         stream_handle()), "nl_update_block_tables")
    return BlockPlan(slots, positions, cu, lens_out, n_free_out, status)


__all__ = ["paged_decode_attention", "paged_kv_write", "update_block_tables", "BlockPlan", "ROW_OK", "ROW_NO_PAGES",
           "ROW_TOO_LONG", "ROW_NO_SLOTS", "ROW_INVALID", "MAX_ROWS"]
