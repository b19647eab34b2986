"""Paged attention, key-value writes and block tables on the GPU against the
64-bit restatements of oracle/paged.py.

Tolerance of the attention's output (bf16): half a bf16 step of the value,
2^-8 |o|, and the error of the probabilities weighed with the values,
e * sum p|v| / sum p.  For a bf16 cache p = hi + lo is off by at most 2^-16, a
score (f32 sum of at most 128 products of inputs of size ~1: |terms| sum to
under 2^4 after scaling, 2^-24 each step) by under 2^-13, twice (maximum
and score): e = 2^-11 holds both.  For e4m3 p is f16, half a step 2^-11 more:
e = 2^-10.  An f16 p below 2^-14 has steps of 2^-24: it is off by up to 2^-25,
where the largest p, and so their sum, is at least 2^7 (the running maximum
is kept there): 2^-32 of each |v| more, which shows where the keys that weigh have a
value of 0.  lse (f32): the score error, 2^-12, and 2^-22 of its size."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import paged as OP  # noqa: E402
from nlearn_b200 import _lib  # noqa: E402
from nlearn_b200.paged import (paged_decode_attention, paged_kv_write, update_block_tables)  # noqa: E402

E4M3 = torch.float8_e4m3fn


def make_cache(n_pages, hk, page, d, layout, dtype, gen, dev):
    shape = (n_pages, hk, page, d) if layout == "hnd" else (n_pages, page, hk, d)
    x = torch.randn(shape, generator=gen)
    x = (x * 60).to(E4M3) if dtype == E4M3 else x.to(dtype)
    x = x.to(dev)
    return x if layout == "hnd" else x.transpose(1, 2)


def make_case(dev, lens, hq, hk, d, page, layout="hnd", dtype=torch.bfloat16, seed=0, spare=3, poison=True):
    """Sequences on shuffled pages.  Slots past a sequence's end hold NaN, and
    table entries past its last page hold numbers outside the cache."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    blocks = max(1, max((n + page - 1) // page for n in lens)) + 1
    need = [(n + page - 1) // page for n in lens]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((B, blocks), 10**9, dtype=torch.int32)
    at = 0
    k = make_cache(n_pages, hk, page, d, layout, dtype, g, dev)
    v = make_cache(n_pages, hk, page, d, layout, dtype, g, dev)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
        if poison and lens[b] % page:
            k[order[at - 1], :, lens[b] % page:] = float("nan")
            v[order[at - 1], :, lens[b] % page:] = float("nan")
    q = (torch.randn(B, hq, d, generator=g)).bfloat16().to(dev)
    return q, k, v, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)


def check_out(o, lse, q, k, v, table, lens, scale, ks=None, vs=None, e=2.0**-11):
    f = lambda t: t.double().cpu().numpy()  # noqa: E731
    K, V = f(k.float()), f(v.float())
    if ks is not None:
        K, V = K * f(ks)[:, None, None], V * f(vs)[:, None, None]
    ro, rl, a = OP.paged_attention(f(q.float()), K, V, table.cpu().numpy(), lens.cpu().numpy(), scale)
    err = np.abs(f(o.float()) - ro)
    tol = 2.0**-8 * np.abs(ro) + e * a
    if k.dtype == E4M3:
        tol = tol + 2.0**-32 * lens.cpu().numpy()[:, None, None] * np.nanmax(np.abs(V))
    assert (err <= tol).all(), (err - tol).max()
    if lse is not None:
        L = f(lse)
        assert np.array_equal(np.isneginf(L), np.isneginf(rl))
        fin = np.isfinite(rl)
        assert (np.abs(L[fin] - rl[fin]) <= 2.0**-12 + 2.0**-22 * np.abs(rl[fin])).all()


EDGE = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (6, 2), (8, 1), (14, 2), (16, 1), (17, 1), (40, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_head_layouts(cuda, hq, hk, d):
    c = make_case(cuda, EDGE, hq, hk, d, 16, seed=hq * d)
    lse = torch.empty(len(EDGE), hq, device=cuda)
    o = paged_decode_attention(*c, lse=lse)
    torch.cuda.synchronize()
    check_out(o, lse, *c, d ** -0.5)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 200])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_page_sizes_and_layouts(cuda, page, layout):
    c = make_case(cuda, [5, 0, 211, 64, 1, 499], 8, 2, 64, page, layout, seed=page)
    lse = torch.empty(6, 8, device=cuda)
    o = paged_decode_attention(*c, lse=lse, scale=0.3)
    torch.cuda.synchronize()
    check_out(o, lse, *c, 0.3)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("lens,hq,hk,d", [([20011], 4, 1, 128), ([20011], 16, 1, 64), ([4097, 33], 8, 8, 64),
                                          ([1] * 700, 8, 8, 64), ([0, 0, 9000, 0, 1, 6001, 0], 16, 2, 128),
                                          (list(range(0, 640)), 2, 2, 64)])
def test_split_lengths(cuda, lens, hq, hk, d):
    """Sequences cut over many CTAs, many sequences in one CTA, empty rows between."""
    c = make_case(cuda, lens, hq, hk, d, 16, seed=len(lens))
    lse = torch.empty(len(lens), hq, device=cuda)
    o = paged_decode_attention(*c, lse=lse)
    o2 = paged_decode_attention(*c)
    torch.cuda.synchronize()
    check_out(o, lse, *c, d ** -0.5)
    assert torch.equal(o, o2)            # nothing depends on the order in which CTAs finish
    assert _lib.device_error() == 0


@pytest.mark.parametrize("hq,hk,d,page,layout,dtype", [(8, 8, 64, 16, "nhd", torch.bfloat16),
                                                       (24, 8, 128, 16, "hnd", torch.bfloat16),
                                                       (32, 4, 128, 24, "nhd", E4M3), (8, 4, 64, 48, "hnd", E4M3),
                                                       (6, 3, 64, 16, "hnd", torch.bfloat16)])
def test_many_sequences(cuda, hq, hk, d, page, layout, dtype):
    """Several ends of sequences in every CTA: one head per warp where the heads
    come in fours, and the new token appended in the same call."""
    rng = np.random.default_rng(hq)
    lens = rng.integers(0, 400, 170).tolist() + [1500, 0, 1]
    q, k, v, table, ln = make_case(cuda, lens, hq, hk, d, page, layout, dtype, seed=hq + d)
    B = len(lens)
    kn, vn = (torch.randn(B, hk, d, device=cuda).bfloat16() for _ in range(2))
    lse = torch.empty(B, hq, device=cuda)
    o = paged_decode_attention(q, k, v, table, ln, kn, vn, lse=lse, scale=0.02 if dtype == E4M3 else None)
    o2 = paged_decode_attention(q, k, v, table, ln, scale=0.02 if dtype == E4M3 else None)
    torch.cuda.synchronize()
    check_out(o, lse, q, k, v, table, ln, 0.02 if dtype == E4M3 else d ** -0.5, e=2.0**-10)
    assert torch.equal(o, o2) and _lib.device_error() == 0


@pytest.mark.parametrize("d,page,layout,hq,hk", [(64, 16, "hnd", 8, 8), (128, 16, "nhd", 8, 2), (64, 5, "nhd", 4, 4),
                                                 (128, 64, "hnd", 32, 2)])
def test_e4m3_cache(cuda, d, page, layout, hq, hk):
    lens = EDGE + [1500]
    c = make_case(cuda, lens, hq, hk, d, page, layout, E4M3, seed=page)
    g = torch.Generator().manual_seed(1)
    ks, vs = ((torch.rand(hk, generator=g) + 0.5) / 60 for _ in range(2))
    ks, vs = ks.to(cuda), vs.to(cuda)
    lse = torch.empty(len(lens), hq, device=cuda)
    o = paged_decode_attention(*c, k_scale=ks, v_scale=vs, lse=lse)
    torch.cuda.synchronize()
    check_out(o, lse, *c, d ** -0.5, ks, vs, e=2.0**-10)
    # q of any size: it is scaled into f16's range by powers of two per row
    for mul in (2.0**-60, 2.0**40):
        q = c[0].clone()
        q[:, ::2] *= mul
        sc = d ** -0.5 / mul if mul > 1 else d ** -0.5
        o = paged_decode_attention(q, *c[1:], k_scale=ks, v_scale=vs, scale=sc, lse=lse)
        torch.cuda.synchronize()
        check_out(o, lse, q, *c[1:], sc, ks, vs, e=2.0**-10)
    # no scales: the values themselves
    o = paged_decode_attention(*c, scale=1e-3)
    torch.cuda.synchronize()
    check_out(o, None, *c, 1e-3, e=2.0**-10)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("hq,hk,d,page,layout", [(8, 8, 64, 16, "hnd"), (40, 2, 128, 24, "nhd"), (4, 4, 64, 1, "nhd")])
def test_append(cuda, dtype, hq, hk, d, page, layout):
    """The new key and value take part and land in their slot; every other
    byte of the caches stays."""
    lens = EDGE + [777]
    q, k, v, table, ln = make_case(cuda, lens, hq, hk, d, page, layout, dtype, seed=3)
    B = len(lens)
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(B, (hq + 2 * hk) * d, generator=g).bfloat16().to(cuda)
    kn, vn = qkv[:, hq * d:(hq + hk) * d].view(B, hk, d), qkv[:, (hq + hk) * d:].view(B, hk, d)
    ks = vs = None
    if dtype == E4M3:
        ks, vs = (torch.rand(hk, generator=g).to(cuda) + 0.5) / 60, (torch.rand(hk, generator=g).to(cuda) + 0.5) / 60
    want_k, want_v = k.clone(), v.clone()
    for b, n in enumerate(lens):
        if n:
            pg, r = int(table[b, (n - 1) // page]), (n - 1) % page
            if dtype == E4M3:
                want_k[pg, :, r] = (kn[b].float() / ks[:, None]).clamp(-448, 448).to(E4M3)
                want_v[pg, :, r] = (vn[b].float() / vs[:, None]).clamp(-448, 448).to(E4M3)
            else:
                want_k[pg, :, r], want_v[pg, :, r] = kn[b], vn[b]
    lse = torch.empty(B, hq, device=cuda)
    o = paged_decode_attention(q, k, v, table, ln, kn, vn, k_scale=ks, v_scale=vs, lse=lse)
    torch.cuda.synchronize()
    bits = lambda t: t.view(torch.uint8) if dtype == E4M3 else t.view(torch.int16)  # noqa: E731
    assert torch.equal(bits(k.contiguous()), bits(want_k.contiguous()))
    assert torch.equal(bits(v.contiguous()), bits(want_v.contiguous()))
    check_out(o, lse, q, k, v, table, ln, d ** -0.5, ks, vs, e=2.0**-10)
    again = paged_decode_attention(q, k, v, table, ln, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert torch.equal(o, again)         # the token is in the cache now
    assert _lib.device_error() == 0


def test_bad_pages_and_lengths(cuda):
    """Pages outside the cache take no part and set device error 4; a length
    past the table is clamped and sets 3; a negative one is empty."""
    q, k, v, table, ln = make_case(cuda, [40, 100, 33, 20], 4, 2, 64, 16, seed=5, poison=False)
    table[0, 0] = k.shape[0]
    table[1, 3] = -7
    table[3, :2] = 2**31 - 1             # a row with no page at all
    assert _lib.device_error() == 0
    kn = torch.randn(4, 2, 64, device=cuda).bfloat16()
    before = k.clone()
    lse = torch.empty(4, 4, device=cuda)
    o = paged_decode_attention(q, k, v, table, ln, lse=lse)
    torch.cuda.synchronize()
    assert _lib.device_error() == 4
    check_out(o, lse, q, k, v, table, ln, 64 ** -0.5)
    assert (o[3] == 0).all() and torch.isneginf(lse[3]).all()
    # an append into a page outside the cache is dropped
    ln2 = torch.tensor([0, 64, 0, 20], dtype=torch.int32, device=cuda)
    paged_decode_attention(q, k, v, table, ln2, kn, kn)
    torch.cuda.synchronize()
    assert _lib.device_error() == 4 and torch.equal(k, before)
    cap = table.shape[1] * 16
    table[1] = torch.arange(table.shape[1]) % k.shape[0]
    ln3 = torch.tensor([0, cap + 5, -3, 0], dtype=torch.int32, device=cuda)
    o = paged_decode_attention(q, k, v, table, ln3, kn, kn, lse=lse)
    torch.cuda.synchronize()
    assert _lib.device_error() == 3 and torch.equal(k, before)
    check_out(o, lse, q, k, v, table, torch.tensor([0, cap, 0, 0]), 64 ** -0.5)
    assert _lib.device_error() == 0


def test_infinities_and_nan(cuda):
    """NaN in a key or value that counts reaches exactly its own row and head;
    a key of huge size does not overflow the sum."""
    q, k, v, table, ln = make_case(cuda, [70, 70], 4, 2, 64, 16, seed=8)
    k[int(table[0, 1]), 0, 3] = float("nan")
    v[int(table[1, 2]), 1, 5] = float("nan")
    k[int(table[1, 0]), 0, 0] = q[1, 0] * 1e18
    o = paged_decode_attention(q, k, v, table, ln)
    torch.cuda.synchronize()
    bad = torch.isnan(o).all(-1)
    assert bad.tolist() == [[True, True, False, False], [False, False, True, True]]
    assert not torch.isnan(o[0, 2:]).any() and not torch.isnan(o[1, :2]).any()
    # the huge key takes all of the first head's weight
    assert torch.equal(o[1, 0], v[int(table[1, 0]), 0, 0])


def test_strided_operands_streams_and_graph(cuda):
    q, k, v, table, ln = make_case(cuda, [100, 7, 260], 8, 4, 64, 16, seed=11)
    want = paged_decode_attention(q, k, v, table, ln)
    torch.cuda.synchronize()
    wide = torch.zeros(3, 3, 8, 64, device=cuda, dtype=torch.bfloat16)
    wide[:, 1] = q
    odd = torch.zeros(3, 8, 65, device=cuda, dtype=torch.bfloat16)
    odd[..., :64] = q
    big_table = torch.full((3, 40), -1, device=cuda, dtype=torch.int32)
    big_table[:, :table.shape[1]] = table
    out = torch.zeros(3, 8, 66, device=cuda, dtype=torch.bfloat16)
    lse = torch.zeros(3, 20, device=cuda)
    paged_decode_attention(wide[:, 1], k, v, big_table[:, :table.shape[1]], ln, out=out[..., :64], lse=lse[:, :8])
    torch.cuda.synchronize()
    assert torch.equal(out[..., :64], want) and (out[..., 64:] == 0).all() and (lse[:, 8:] == 0).all()
    assert torch.equal(paged_decode_attention(odd[..., :64], k, v, table, ln), want)
    # two calls at once on two streams
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    res = []
    for _ in range(20):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                res.append(paged_decode_attention(q, k, v, table, ln))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in res)
    # captured: replays read the lengths of the moment
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = paged_decode_attention(q, k, v, table, ln)
    for new in ([100, 7, 260], [1, 0, 33], [64, 3, 200]):
        ln.copy_(torch.tensor(new, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        # (slots past the first lengths hold NaN; these lengths stay before them)
        check_out(o, None, q, k, v, table, ln, 64 ** -0.5)
    assert _lib.device_error() == 0


def test_offsets_past_32_bits(cuda):
    """Pages far into caches of more than 2^32 elements' bytes."""
    n_pages, page, hk, d = 2**31 // (16 * 2 * 64) + 1000, 16, 2, 64
    k = torch.empty(n_pages, hk, page, d, device=cuda, dtype=torch.bfloat16)
    v = torch.empty_like(k)
    pages = torch.tensor([n_pages - 1, 5, n_pages - 500, n_pages // 2 + 1], device=cuda)
    g = torch.Generator().manual_seed(2)
    small_k, small_v = (torch.randn(4, hk, page, d, generator=g).bfloat16().to(cuda) for _ in range(2))
    k[pages], v[pages] = small_k, small_v
    q = torch.randn(1, 4, d, generator=g).bfloat16().to(cuda)
    ln = torch.tensor([60], device=cuda, dtype=torch.int32)
    o = paged_decode_attention(q, k, v, pages.int()[None], ln)
    near = paged_decode_attention(q, small_k, small_v, torch.arange(4, device=cuda, dtype=torch.int32)[None], ln)
    torch.cuda.synchronize()
    assert torch.equal(o, near)
    kn = torch.randn(3, hk, d, generator=g).bfloat16().to(cuda)
    slots = torch.tensor([n_pages * page - 1, -1, (n_pages - 2) * page + 3], device=cuda, dtype=torch.int32)
    paged_kv_write(kn, kn, k, v, slots)
    torch.cuda.synchronize()
    assert torch.equal(k[n_pages - 1, :, page - 1], kn[0]) and torch.equal(v[n_pages - 2, :, 3], kn[2])
    assert _lib.device_error() == 0


# ---------------------------------------------------------------- writes
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("T,hk,d,page,layout", [(1, 1, 64, 16, "hnd"), (333, 8, 64, 16, "nhd"), (100, 3, 48, 7, "hnd"),
                                                (2000, 2, 256, 64, "nhd")])
def test_kv_write(cuda, dtype, T, hk, d, page, layout):
    g = torch.Generator().manual_seed(T)
    n_pages = (T + page - 1) // page + 3
    k, v = (make_cache(n_pages, hk, page, d, layout, dtype, g, cuda) for _ in range(2))
    qkv = (torch.randn(T, 3 * hk * d, generator=g) * 40).bfloat16().to(cuda)
    kn, vn = qkv[:, hk * d:2 * hk * d].view(T, hk, d), qkv[:, 2 * hk * d:].view(T, hk, d)
    slots = torch.randperm(n_pages * page, generator=g)[:T].int()
    slots[::7] = -1 if T > 1 else slots[::7]
    ks = vs = None
    fk, fv = kn, vn
    if dtype == E4M3:
        ks, vs = ((torch.rand(hk, generator=g) + 0.05).to(cuda) for _ in range(2))
        fk, fv = ((x.float() / s[:, None]).clamp(-448, 448).to(E4M3) for x, s in ((kn, ks), (vn, vs)))
    wk, wv = k.clone(), v.clone()
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            wk[s // page, :, s % page], wv[s // page, :, s % page] = fk[t], fv[t]
    paged_kv_write(kn, vn, k, v, slots.to(cuda), k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert torch.equal(k.float(), wk.float()) and torch.equal(v.float(), wv.float())
    assert _lib.device_error() == 0


def test_kv_write_bad_slot_and_odd_rows(cuda):
    k = torch.zeros(4, 2, 16, 64, device=cuda, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    odd = torch.randn(3, 2, 65, device=cuda).bfloat16()[..., :64]
    paged_kv_write(odd, odd, k, v, torch.tensor([5, 64, 2**31 - 1], device=cuda, dtype=torch.int32))
    torch.cuda.synchronize()
    assert _lib.device_error() == 4
    assert torch.equal(k[0, :, 5], odd[0]) and int((k != 0).sum()) == int((odd[0] != 0).sum())
    paged_kv_write(odd[:0], odd[:0], k, v, torch.empty(0, device=cuda, dtype=torch.int32))
    assert _lib.device_error() == 0


# ---------------------------------------------------------------- block tables
def run_tables(dev, B, blocks, page, n_pages, lens, new, done, n_free, n_tokens, seed, inplace, use_done=True):
    rng = np.random.default_rng(seed)
    order = rng.permutation(n_pages).astype(np.int32)
    table = rng.integers(-5, n_pages + 5, (B, blocks)).astype(np.int32)
    at = 0
    for b in range(B):
        n = -(-max(0, min(lens[b], blocks * page)) // page)
        table[b, :n] = order[np.arange(at, at + n) % n_pages]
        at += n
    free = rng.integers(0, n_pages, n_pages).astype(np.int32)
    want = OP.update_tables(table, lens, new, done if use_done else [0] * B, free, n_free, page, n_tokens)
    t = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)  # noqa: E731
    wide = torch.full((B, blocks + 3), -9, dtype=torch.int32, device=dev)
    wide[:, :blocks] = t(table)
    T, L, F, N = wide[:, :blocks], t(lens), t(free), t([n_free])
    plan = update_block_tables(T, L, t(new), F, N, page, n_tokens, done=t(done) if use_done else None,
                               lens_out=L if inplace else None, n_free_out=N if inplace else None)
    torch.cuda.synchronize()
    for name, got in (("slots", plan.slots), ("positions", plan.positions), ("cu", plan.cu), ("lens", plan.lens),
                      ("status", plan.status), ("table", T), ("free", F)):
        assert np.array_equal(got.cpu().numpy(), np.array(want[name]).reshape(got.shape)), name
    assert plan.n_free.item() == want["n_free"]
    assert (wide[:, blocks:] == -9).all()
    if inplace:
        assert plan.lens is L and plan.n_free is N
    else:
        assert L.cpu().tolist() == list(lens) and N.item() == n_free


@pytest.mark.parametrize("B,page,new_max,inplace", [(1, 16, 1, True), (7, 16, 5, False), (33, 1, 40, True),
                                                    (300, 24, 1, True), (1100, 16, 3, False), (64, 16, 700, True),
                                                    (5000, 8, 2, True)])
@pytest.mark.parametrize("short", [False, True])
def test_update_tables(cuda, B, page, new_max, inplace, short):
    rng = np.random.default_rng(B + page)
    blocks = 60
    cap = blocks * page
    lens = rng.integers(0, cap // 2 + 1, B)
    lens[rng.random(B) < 0.2] = 0
    new = rng.integers(0, new_max + 1, B)
    done = (rng.random(B) < 0.15).astype(int)
    pages = int((-(-lens // page)).sum())
    want = int((-(-(lens + new) // page) + lens // page).sum())
    n_pages = max(1, pages + want + 5)
    n_free = max(0, want // 3) if short else min(n_pages - pages, want + 3)
    n_tokens = int(new.sum()) * (2 if short else 3) // 3 + (0 if short else 11 + new_max)
    run_tables(cuda, B, blocks, page, n_pages, lens, new, done, n_free, n_tokens, B, inplace)


def test_update_tables_refusals_and_edges(cuda):
    # invalid counts, lengths past the table, rows that end and start again, a full stack
    run_tables(cuda, 8, 4, 16, 40, [0, -1, 65, 64, 10, 64, 30, 0], [64, 1, 1, 1, -2, 64, 3, 65],
               [0, 1, 1, 0, 0, 1, 1, 1], 20, 300, 1, True)
    run_tables(cuda, 3, 4, 16, 6, [60, 60, 60], [1, 1, 1], [1, 1, 1], 4, 10, 2, True)     # stack overflows: capped
    run_tables(cuda, 3, 4, 16, 6, [0, 0, 0], [1, 1, 1], [0, 0, 0], 900, 10, 3, False)      # n_free past the pages
    run_tables(cuda, 3, 4, 16, 6, [0, 0, 0], [1, 1, 1], [0, 0, 0], -4, 10, 4, False)
    run_tables(cuda, 2, 4, 16, 9, [16, 17], [1, 1], [0, 0], 9, 0, 5, False)                # no slots at all
    run_tables(cuda, 2, 4, 16, 9, [16, 17], [16, 0], [0, 0], 9, 40, 6, True, use_done=False)
    # one row after another finds no pages; a row that needs none is still served
    run_tables(cuda, 5, 4, 16, 9, [0, 5, 0, 7, 0], [40, 3, 1, 4, 1], [0] * 5, 2, 100, 8, True)


def test_update_tables_wide_and_large_counts(cuda):
    """Eight CTAs (a long flat list), more rows than threads, and counts that
    overflow 32 bits together."""
    rng = np.random.default_rng(0)
    B = 2000
    lens, new = rng.integers(0, 200, B), rng.integers(0, 200, B)
    done = (rng.random(B) < 0.3).astype(int)
    run_tables(cuda, B, 30, 16, 60000, lens, new, done, 9000, int(new.sum()) - 5000, 1, True)
    t = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    table, L, N = torch.zeros(4, 4, dtype=torch.int32, device=cuda), t([0, 0, 0, 0]), t([6])
    plan = update_block_tables(table, L, t([2**31 - 1, 2**31 - 1, 5, 0]), t(list(range(6))), N, 16, 40)
    assert plan.status.tolist() == [2, 2, 3, 0] and plan.cu.tolist() == [0, 2**31 - 1, 2**31 - 1, 2**31 - 1,
                                                                          2**31 - 1]
    assert plan.n_free.item() == 6 and (plan.slots == -1).all()


def test_update_tables_longest_flat_list(cuda):
    t = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    n = 2**31 - 1
    table, free = torch.zeros(2, 4, dtype=torch.int32, device=cuda), t(list(range(6)))
    plan = update_block_tables(table, t([0, 3]), t([20, 2]), free, t([6]), 16, n)
    torch.cuda.synchronize()
    assert plan.slots.numel() == n and plan.status.tolist() == [0, 0]
    # row 0 takes pages 5 and 4, row 1 goes on in its page 0
    assert plan.slots[:22].tolist() == list(range(80, 96)) + list(range(64, 68)) + [3, 4]
    assert plan.positions[:22].tolist() == list(range(20)) + [3, 4]
    for part in (plan.slots, plan.positions):
        assert part[22:].max().item() == -1 and part[22:].min().item() == -1


def test_tables_write_attention_together(cuda):
    """Prompts of ragged lengths, then decode steps with rows that end and
    start again, all in one captured step: outputs equal a plain recompute."""
    B, hq, hk, d, page, blocks, n_pages = 5, 8, 4, 64, 8, 12, 40
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().to(cuda)  # noqa: E731
    k = torch.full((n_pages, hk, page, d), float("nan"), device=cuda, dtype=torch.bfloat16)
    v = k.clone()
    i32 = dict(device=cuda, dtype=torch.int32)
    table, lens = torch.full((B, blocks), -1, **i32), torch.zeros(B, **i32)
    free, n_free = torch.arange(n_pages, **i32), torch.tensor([n_pages], **i32)
    new, done = torch.zeros(B, **i32), torch.zeros(B, **i32)
    hist_k, hist_v = [[] for _ in range(B)], [[] for _ in range(B)]

    def admit(rows, sizes):
        new.zero_()
        new[rows] = torch.tensor(sizes, **i32)
        plan = update_block_tables(table, lens, new, free, n_free, page, sum(sizes) + 3, done=done, lens_out=lens,
                                   n_free_out=n_free)
        kx, vx = rnd(sum(sizes) + 3, hk, d), rnd(sum(sizes) + 3, hk, d)
        paged_kv_write(kx, vx, k, v, plan.slots)
        torch.cuda.synchronize()
        assert plan.status.sum().item() == 0
        for b in range(B):
            if done[b]:
                hist_k[b], hist_v[b] = [], []
            for t in range(int(plan.cu[b]), int(plan.cu[b + 1])):
                hist_k[b].append(kx[t])
                hist_v[b].append(vx[t])
        done.zero_()

    admit([0, 1, 3, 4], [17, 1, 30, 8])
    q, kn, vn = rnd(B, hq, d), rnd(B, hk, d), rnd(B, hk, d)
    graph = torch.cuda.CUDAGraph()
    keep = [t.clone() for t in (table, lens, free, n_free, k, v)]
    with torch.cuda.graph(graph):
        update_block_tables(table, lens, new, free, n_free, page, B, lens_out=lens, n_free_out=n_free)
        o = paged_decode_attention(q, k, v, table, lens, kn, vn)
    for a, b in zip((table, lens, free, n_free, k, v), keep):
        a.copy_(b)
    for step in range(14):
        if step == 6:
            done[1] = 1
            done[4] = 1
            admit([1, 2], [9, 3])        # row 4 ends, row 1 starts anew, row 2 joins
        new.copy_((lens > 0).int())
        for t in (q, kn, vn):
            t.copy_(rnd(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            if int(new[b]):
                hist_k[b].append(kn[b].clone())
                hist_v[b].append(vn[b].clone())
        assert lens.tolist() == [len(h) for h in hist_k]
        used = sum(-(-len(h) // page) for h in hist_k)
        assert n_free.item() == n_pages - used
        for b in range(B):
            if not hist_k[b]:
                assert (o[b] == 0).all()
                continue
            K, V = torch.stack(hist_k[b], 1), torch.stack(hist_v[b], 1)
            one = torch.arange(1, **i32)[None]
            check_out(o[b:b + 1], None, q[b:b + 1], K[None], V[None], one, torch.tensor([K.shape[1]]), d ** -0.5)
    assert _lib.device_error() == 0


def test_wrapper_refusals(cuda):
    q, k, v, table, ln = make_case(cuda, [10, 20], 4, 2, 64, 16)
    call = paged_decode_attention
    bad = [
        (ValueError, lambda: call(q[..., :32], k, v, table, ln)),
        (ValueError, lambda: call(q[:, :3], k, v, table, ln)),
        (ValueError, lambda: call(q[0], k, v, table, ln)),
        (TypeError, lambda: call(q.float(), k, v, table, ln)),
        (TypeError, lambda: call(q, k.half(), v.half(), table, ln)),
        (TypeError, lambda: call(q, k, v.to(E4M3), table, ln)),
        (ValueError, lambda: call(q, k, v[:-1], table, ln)),
        (ValueError, lambda: call(q, k, v.transpose(1, 2).contiguous().transpose(1, 2), table, ln)),
        (TypeError, lambda: call(q, k, v, table.long(), ln)),
        (TypeError, lambda: call(q, k, v, table, ln.long())),
        (ValueError, lambda: call(q, k, v, table[:1], ln)),
        (ValueError, lambda: call(q, k, v, table[:, :0], ln)),
        (ValueError, lambda: call(q, k, v, table, ln, q[:, :2])),
        (ValueError, lambda: call(q, k, v, table, ln, q, q)),
        (ValueError, lambda: call(q, k, v, table, ln, k_scale=torch.ones(2, device=cuda))),
        (ValueError, lambda: call(q, k, v, table, ln, out=torch.empty(2, 4, 64, device=cuda))),
        (ValueError, lambda: call(q, k, v, table, ln, lse=torch.empty(2, 3, device=cuda))),
        (ValueError, lambda: call(q.cpu(), k, v, table, ln)),
        (ValueError, lambda: call(q, k, v, table, ln.cpu())),
        (RuntimeError, lambda: call(q.clone().requires_grad_(), k, v, table, ln)),
        (RuntimeError, lambda: call(q, k.clone().requires_grad_(), v, table, ln)),
        (RuntimeError, lambda: call(q, k, v, table, ln, out=torch.empty_like(q).requires_grad_())),
        (RuntimeError, lambda: call(q, k.to(E4M3), v.to(E4M3), table, ln,
                                    k_scale=torch.ones(2, device=cuda, requires_grad=True))),
        (ValueError, lambda: paged_kv_write(q, q, k, v, ln)),
        (TypeError, lambda: paged_kv_write(q[:, :2], q[:, :2], k, v, ln.float())),
        (ValueError, lambda: update_block_tables(table, ln, ln, ln, ln[:1], 0, 5)),
        (ValueError, lambda: update_block_tables(table, ln, ln, ln, ln, 16, 5)),
        (TypeError, lambda: update_block_tables(table, ln, ln.long(), ln, ln[:1], 16, 5)),
    ]
    for i, (err, fn) in enumerate(bad):
        with pytest.raises(err):
            fn()
            raise AssertionError(i)
    assert call(q[:0], k, v, table[:0], ln[:0]).shape == (0, 4, 64)
    assert _lib.device_error() == 0
