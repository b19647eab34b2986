"""Plain 64-bit restatements of the paged serving operators (NumPy), from
their definitions: attention over a paged cache, block tables, logits
processing.  No reference counterpart: the definitions are this library's."""
from __future__ import annotations

import math

import numpy as np


def paged_attention(q, k_cache, v_cache, table, lens, scale):
    """q [B, Hq, d]; caches [n_pages, Hk, P, d] as the values they stand for;
    pages outside the cache take no part.  -> o, lse, and a = sum p|v| / sum p
    (what an error of p is weighed with)."""
    B, Hq, d = q.shape
    n_pages, Hk, P, _ = k_cache.shape
    g = Hq // Hk
    o = np.zeros((B, Hq, d))
    a = np.zeros((B, Hq, d))
    lse = np.full((B, Hq), -np.inf)
    for b in range(B):
        rows = [(int(table[b, j // P]), j % P) for j in range(int(lens[b]))]
        rows = [(p, r) for p, r in rows if 0 <= p < n_pages]
        if not rows:
            continue
        pg, rw = np.array(rows).T
        for h in range(Hk):
            k = k_cache[pg, h, rw].astype(np.float64)
            v = v_cache[pg, h, rw].astype(np.float64)
            s = scale * q[b, h * g:(h + 1) * g].astype(np.float64) @ k.T
            m = s.max(1, keepdims=True)
            e = np.exp(s - m)
            z = e.sum(1, keepdims=True)
            o[b, h * g:(h + 1) * g] = e @ v / z
            a[b, h * g:(h + 1) * g] = e @ np.abs(v) / z
            lse[b, h * g:(h + 1) * g] = (m + np.log(z))[:, 0]
    return o, lse, a


def update_tables(table, lens, new, done, free, n_free, P, n_tokens):
    """One step, row after row, on Python lists.  -> dict of the results."""
    B, blocks = len(lens), len(table[0])
    n_pages = len(free)
    table = [list(map(int, r)) for r in table]
    lens, free = list(map(int, lens)), list(map(int, free))
    up = lambda x: -(-x // P)  # noqa: E731
    top = max(0, min(int(n_free), n_pages))
    stack_end = top
    for b in range(B):
        if done[b] and 0 < lens[b] <= blocks * P:
            for i in range(up(lens[b])):
                if stack_end < n_pages:
                    free[stack_end] = table[b][i]
                stack_end += 1
    avail = min(stack_end, n_pages)
    cu, status, out = [0], [], []
    wanted = used = 0
    taken = {}
    for b in range(B):
        n = int(new[b])
        bad = lens[b] < 0 or lens[b] > blocks * P
        len0 = 0 if done[b] and not bad else lens[b]
        first = cu[-1]
        cu.append(first + max(0, n))
        if bad or n < 0:
            st = 4
        elif len0 + n > blocks * P:
            st = 2
        elif n and first + n > n_tokens:
            st = 3
        else:
            st = 0
            need = up(len0 + n) - up(len0)
            if need and wanted + need > avail:
                st = 1
            else:
                taken[b] = (len0, n, first, [free[avail - 1 - wanted - i] for i in range(need)])
                used += need
            wanted += need
        status.append(st)
        out.append(len0 + n if st == 0 else len0)
    slots, pos = [-1] * n_tokens, [-1] * n_tokens
    for b, (len0, n, first, pages) in taken.items():
        for i, pg in enumerate(pages):
            table[b][up(len0) + i] = pg
        for i in range(n):
            p = len0 + i
            pg = table[b][p // P]
            pos[first + i] = p
            slots[first + i] = pg * P + p % P if 0 <= pg < n_pages else -1
    return dict(table=table, free=free, slots=slots, positions=pos, cu=cu, lens=out, n_free=avail - used,
                status=status)


def process_logits(x, tokens=None, lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None,
                   bias_ids=None, bias=None, mask=None, mask_rows=None):
    """x [B, V] -> f64 [B, V]."""
    y = x.astype(np.float64).copy()
    B, V = y.shape
    for b in range(B):
        if tokens is not None:
            n = max(0, min(int(lens[b]), tokens.shape[1]))
            m = max(0, min(int(prompt_lens[b]), n)) if prompt_lens is not None else 0
            row = [int(t) for t in tokens[b, :n]]
            count = {}
            for i, t in enumerate(row):
                if 0 <= t < V:
                    count[t] = count.get(t, 0) + (1 if i >= m else 0)
            for t, c in count.items():
                if repetition is not None:
                    r = float(repetition[b])
                    y[b, t] = y[b, t] / r if y[b, t] > 0 else y[b, t] * r
                if c:
                    if frequency is not None:
                        y[b, t] -= float(frequency[b]) * c
                    if presence is not None:
                        y[b, t] -= float(presence[b])
        if bias is not None:
            for t, v in zip(bias_ids[b], bias[b]):
                if 0 <= t < V:
                    y[b, t] += float(v)
        if mask is not None:
            r = b if mask_rows is None else int(mask_rows[b])
            if 0 <= r < mask.shape[0]:
                for v in range(V):
                    if not (int(mask[r, v // 32]) >> (v % 32)) & 1:
                        y[b, v] = -math.inf
    return y
