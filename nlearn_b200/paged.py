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

from functools import lru_cache
from typing import NamedTuple

import torch

from . import _lib
from ._lib import ARGS, check, lib, raw_stream

_CACHE_DT = {torch.bfloat16: _lib.BF16, torch.float8_e4m3fn: _lib.E4M3}
HEAD_DIMS = (64, 128)

# A call of these operators is a few microseconds of GPU work, so the checks
# below read each property of a tensor once, and the messages are made only
# when one of them fails.


def _refuse_place(name: str, t: torch.Tensor, index: int) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name}: nlearn_b200 paged operators run on CUDA tensors only (no CPU fallback)")
    raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")


def _launch(name: str, index: int, *fields) -> None:
    """Calls a C entry point with its packed arguments on the current stream of
    device `index`, which entry points take to be the current device."""
    args = ARGS[name].pack(*fields)
    if index == torch._C._cuda_getDevice():
        status = getattr(lib, name)(args, raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = getattr(lib, name)(args, raw_stream(index))
    if status:
        check(status, name)


def _ints1(name: str, t: torch.Tensor, n: int, index: int) -> int:
    """Checks a contiguous int32 vector of n elements; -> its address."""
    if t.dtype is torch.int32 and t.dim() == 1 and t.numel() == n and t.is_contiguous() and t.get_device() == index:
        return t.data_ptr()
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.get_device() != index:
        _refuse_place(name, t, index)
    raise ValueError(f"{name} must be a contiguous vector of {n} elements, got shape {tuple(t.shape)} with strides "
                     f"{t.stride()}")


def _ints2(name: str, t: torch.Tensor, rows: int | None, index: int):
    """Checks an int32 matrix with contiguous rows; -> (rows, columns, row pitch)."""
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.get_device() != index:
        _refuse_place(name, t, index)
    if t.dim() != 2:
        raise ValueError(f"{name} must be a matrix, got shape {tuple(t.shape)}")
    n, cols = t.shape
    ld, unit = t.stride()
    if (rows is not None and n != rows) or (cols > 1 and unit != 1) or (n > 1 and ld < cols):
        raise ValueError(f"{name} must have {'' if rows is None else rows} contiguous rows that do not overlap, got "
                         f"shape {(n, cols)} with strides {(ld, unit)}")
    return n, cols, max(ld, cols)


def _no_grad(name: str, *ts) -> None:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no backward: call it under torch.no_grad()")


def _rows(name: str, t: torch.Tensor, shape, index: int):
    """bf16 [n, heads, d] with contiguous 16-byte aligned rows (copied only when needed); -> (tensor, strides)."""
    if t.get_device() != index:
        _refuse_place(name, t, index)
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    st = t.stride()
    if st[2] != 1 or st[0] & 7 or st[1] & 7 or t.data_ptr() & 15:
        t = t.contiguous()
        st = t.stride()
    return t, st


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, index: int):
    """Checks both caches; -> (dtype code, shape, strides)."""
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.get_device() != index:
            _refuse_place(name, t, index)
    dtype = k_cache.dtype
    dt = _CACHE_DT.get(dtype)
    if dt is None or v_cache.dtype is not dtype:
        raise TypeError(f"caches must both be bfloat16 or float8_e4m3fn, got {dtype} and {v_cache.dtype}")
    shape, st = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("caches must be [n_pages, kv_heads, page_size, head_dim], both of one shape, got "
                         f"{tuple(shape)} and {tuple(v_cache.shape)}")
    if v_cache.stride() != st:
        raise ValueError(f"caches must have the same strides, got {st} and {v_cache.stride()}")
    per = 7 if dt == _lib.BF16 else 15
    if st[3] != 1 or (st[0] | st[1] | st[2]) & per or (k_cache.data_ptr() | v_cache.data_ptr()) & 15:
        raise ValueError("cache rows must be contiguous and lie on 16-byte boundaries")
    if shape[0] * shape[2] > 2**31 - 1:
        raise ValueError(f"cache has {shape[0] * shape[2]} slots, over the limit of 2**31 - 1")
    return dt, shape, st


def _scale(name: str, t, heads: int, dt: int, index: int) -> int:
    if t is None:
        return 0
    if dt != _lib.E4M3:
        raise ValueError(f"{name} goes with a float8_e4m3fn cache")
    if t.get_device() != index:
        _refuse_place(name, t, index)
    if t.dtype is not torch.float32 or t.shape != (heads,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape ({heads},)")
    return t.data_ptr()


@lru_cache(maxsize=256)
def _workspace_bytes(index: int, *shape) -> int:
    """nl_paged_attention_workspace_bytes of a shape on device `index`."""
    with torch.cuda.device(index):
        return lib.nl_paged_attention_workspace_bytes(*shape)


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
    index = q.get_device()
    if index < 0:
        _refuse_place("q", q, index)
    _no_grad("paged_decode_attention", q, k_new, v_new)
    if q.dim() != 3:
        raise ValueError(f"q must be [batch, heads, head_dim], got {tuple(q.shape)}")
    dt, (n_pages, Hk, page, dk), (page_s, head_s, tok_s, _) = _caches(k_cache, v_cache, index)
    shape = q.shape
    B, Hq, d = shape
    if d != dk or d not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} and the caches', got {d} and {dk}")
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"{Hq} query heads do not share {Hk} kv heads evenly")
    q, (q_b, q_h, _) = _rows("q", q, shape, index)
    _, blocks, table_ld = _ints2("block_table", block_table, B, index)
    lens_p = _ints1("lens", lens, B, index)
    n_b = n_h = kn = vn = 0
    if k_new is not None or v_new is not None:
        if k_new is None or v_new is None:
            raise ValueError("k_new and v_new come together")
        k_new, kst = _rows("k_new", k_new, (B, Hk, d), index)
        v_new, vst = _rows("v_new", v_new, (B, Hk, d), index)
        if kst != vst:
            k_new, v_new = k_new.contiguous(), v_new.contiguous()
            kst = k_new.stride()
        n_b, n_h, _ = kst
        kn, vn = k_new.data_ptr(), v_new.data_ptr()
    ks = _scale("k_scale", k_scale, Hk, dt, index)
    vs = _scale("v_scale", v_scale, Hk, dt, index)
    if out is None:
        out = q.new_empty(shape)
        o_b, o_h = Hq * d, d
    else:
        if out.get_device() != index:
            _refuse_place("out", out, index)
        o_b, o_h, unit = out.stride() if out.dim() == 3 else (0, 0, 0)
        if out.shape != shape or out.dtype is not torch.bfloat16 or unit != 1:
            raise ValueError(f"out must be bfloat16 {tuple(shape)} with contiguous rows")
    lp = ls = 0
    if lse is not None:
        if lse.get_device() != index:
            _refuse_place("lse", lse, index)
        if lse.shape != (B, Hq) or lse.dtype is not torch.float32 or (Hq > 1 and lse.stride(1) != 1):
            raise ValueError(f"lse must be float32 {(B, Hq)} with contiguous rows")
        lp, ls = lse.data_ptr(), lse.stride(0)
    if B == 0:
        return out
    if blocks == 0 or n_pages == 0 or page == 0:
        raise ValueError("block_table and caches must hold at least one page")
    nb = _workspace_bytes(index, B, Hq, Hk, d, page, blocks, dt)
    ws = torch.empty(nb, device=q.device, dtype=torch.uint8) if nb else None
    _launch("nl_paged_attention", index, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
            lens_p, kn, vn, ks, vs, out.data_ptr(), lp, ws.data_ptr() if nb else 0, q_b, q_h, page_s, head_s, tok_s,
            table_ld, n_b, n_h, o_b, o_h, ls, nb, B, Hq, Hk, d, page, blocks, n_pages, dt,
            d ** -0.5 if scale is None else scale)
    return out


def paged_kv_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slots: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                   v_scale: torch.Tensor | None = None) -> None:
    """Write k, v [T, kv_heads, head_dim] (bf16; strided views of a fused qkv
    projection are read in place) into slots[t] (int32 [T]) of the caches.
    Negative slots are padding; no slot may occur twice.  An e4m3 cache holds
    round(x / scale), saturating at 448."""
    index = k.get_device()
    if index < 0:
        _refuse_place("k", k, index)
    _no_grad("paged_kv_write", k, v)
    dt, (n_pages, Hk, page, d), (page_s, head_s, tok_s, _) = _caches(k_cache, v_cache, index)
    if k.dim() != 3:
        raise ValueError(f"k must be [tokens, {Hk}, {d}], got {tuple(k.shape)}")
    T = k.shape[0]
    if d & (7 if dt == _lib.BF16 else 15):
        raise ValueError(f"head_dim {d}: cache rows must be whole 16-byte pieces")
    k, kst = _rows("k", k, (T, Hk, d), index)
    v, vst = _rows("v", v, (T, Hk, d), index)
    if kst != vst:
        k, v = k.contiguous(), v.contiguous()
        kst = k.stride()
    sp = _ints1("slots", slots, T, index)
    ks = _scale("k_scale", k_scale, Hk, dt, index)
    vs = _scale("v_scale", v_scale, Hk, dt, index)
    if T == 0 or k_cache.numel() == 0:
        return
    _launch("nl_paged_kv_write", index, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), sp, ks, vs,
            kst[0], kst[1], page_s, head_s, tok_s, T, Hk, d, page, n_pages, dt)


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
    index = block_table.get_device()
    if index < 0:
        _refuse_place("block_table", block_table, index)
    B, blocks, table_ld = _ints2("block_table", block_table, None, index)
    if free_pages.dim() != 1:
        raise ValueError(f"free_pages must be a vector, got shape {tuple(free_pages.shape)}")
    n_pages = free_pages.numel()
    if B == 0 or B > MAX_ROWS or blocks == 0 or n_pages == 0:
        raise ValueError(f"block_table must have 1 to {MAX_ROWS} rows and at least one page a row, got "
                         f"{tuple(block_table.shape)} and {n_pages} pages")
    if page_size < 1 or n_tokens < 0 or blocks * page_size > 2**31 - 1 or n_pages * page_size > 2**31 - 1:
        raise ValueError(f"page_size {page_size}, n_tokens {n_tokens}: out of range")
    lens_p, new_p = _ints1("lens", lens, B, index), _ints1("new_lens", new_lens, B, index)
    done_p = 0 if done is None else _ints1("done", done, B, index)
    free_p, nf_p = _ints1("free_pages", free_pages, n_pages, index), _ints1("n_free", n_free, 1, index)
    if lens_out is None:
        lens_out = torch.empty_like(lens)
        lo_p = lens_out.data_ptr()
    else:
        lo_p = _ints1("lens_out", lens_out, B, index)
    if n_free_out is None:
        n_free_out = torch.empty_like(n_free)
        nfo_p = n_free_out.data_ptr()
    else:
        nfo_p = _ints1("n_free_out", n_free_out, 1, index)
    status = torch.empty_like(lens)
    slots, positions, cu = lens.new_empty(n_tokens), lens.new_empty(n_tokens), lens.new_empty(B + 1)
    _launch("nl_update_block_tables", index, block_table.data_ptr(), lens_p, new_p, done_p, free_p, nf_p, lo_p, nfo_p,
            slots.data_ptr(), positions.data_ptr(), cu.data_ptr(), status.data_ptr(), table_ld, B, blocks, page_size,
            n_pages, n_tokens)
    return BlockPlan(slots, positions, cu, lens_out, n_free_out, status)


__all__ = ["paged_decode_attention", "paged_kv_write", "update_block_tables", "BlockPlan", "ROW_OK", "ROW_NO_PAGES",
           "ROW_TOO_LONG", "ROW_NO_SLOTS", "ROW_INVALID", "MAX_ROWS"]
