"""Cases of the paged serving operators: decode attention over a paged
key-value cache, the write of new keys and values into pages, the block tables
and slot maps of a serving step, and the logits processing before sampling.

Every case can be run in plain torch operations (``own`` false) or through the
public entry points of nlearn_b200 (``own`` true) on the same inputs.

Layouts: a cache is [n_pages, kv_heads, page_size, head_dim] by its logical
axes, stored either that way ("hnd") or with the token axis before the head
axis ("nhd"); a block table row lists the pages of one sequence in order.
"""
import math

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one chat turn of the repository's own model (8 heads of 64, 512 positions): latency
        dict(name="attn-1x512", op="attention", batch=1, heads=8, kv_heads=8, dim=64, page=16, layout="hnd",
             cache="bf16", length=512, ragged=False, append=True, lse=False),
        # the decode benchmark's batch of 32, sequences at all ages, one row not in use
        dict(name="attn-32x512", op="attention", batch=32, heads=8, kv_heads=8, dim=64, page=16, layout="hnd",
             cache="bf16", length=512, ragged=True, append=True, lse=False),
        # long contexts with shared key heads, token-major pages
        dict(name="attn-gqa-48x8192", op="attention", batch=48, heads=32, kv_heads=8, dim=128, page=32, layout="nhd",
             cache="bf16", length=8192, ragged=True, append=False, lse=True),
        # the same kind of batch on an 8-bit cache
        dict(name="attn-e4m3-64x4097", op="attention", batch=64, heads=32, kv_heads=8, dim=128, page=16,
             layout="hnd", cache="e4m3", length=4097, ragged=True, append=False, lse=False),
        # one very long document: all of the card on one sequence
        dict(name="attn-1x131072", op="attention", batch=1, heads=32, kv_heads=8, dim=128, page=16, layout="hnd",
             cache="bf16", length=131072, ragged=False, append=False, lse=True),
        # prefill of a few short prompts: keys and values lie inside the fused q|k|v rows
        dict(name="write-499", op="write", tokens=499, kv_heads=8, dim=64, page=16, layout="hnd"),
        # prefill of a full training-sized batch of tokens
        dict(name="write-16384", op="write", tokens=16384, kv_heads=8, dim=128, page=32, layout="nhd"),
        # one decode step of 256 rows: a page for one row in sixteen, a few rows end
        dict(name="tables-decode-256", op="tables", batch=256, page=16, length=4096, new=1, admit=False),
        # admission of 96 prompts of up to 2048 tokens
        dict(name="tables-admit-96", op="tables", batch=96, page=16, length=4096, new=2048, admit=True),
        # one row of the repository's vocabulary, a short history
        dict(name="logits-1", op="logits", batch=1, vocab=50257, pitch=50304, dtype="f32", history=512, bias=4,
             mask=True),
        # the decode benchmark's batch, every rule at once
        dict(name="logits-32", op="logits", batch=32, vocab=50257, pitch=50304, dtype="f32", history=512, bias=16,
             mask=True),
        # a large batch with long histories, 16-bit logits in rows that are not 16-byte aligned
        dict(name="logits-256-bf16", op="logits", batch=256, vocab=50257, pitch=50257, dtype="bf16", history=4096,
             bias=32, mask=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "write", "tables", "logits"])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
        dim, cache = rng.choice([64, 128]), rng.choice(["bf16", "bf16", "e4m3"])
        batch = _log_int(rng, 1, 200)
        row = 2 * kv_heads * dim * (2 if cache == "bf16" else 1)
        most = min(131072, (400 << 20) // (batch * row))
        return dict(op=op, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([8, 16, 16, 24, 32, 64]), layout=rng.choice(["hnd", "nhd"]), cache=cache,
                    length=_log_int(rng, 1, max(2, most)), ragged=rng.random() < 0.7,
                    append=cache == "bf16" and rng.random() < 0.5, lse=rng.random() < 0.5)
    if op == "write":
        return dict(op=op, tokens=_log_int(rng, 1, 16384), kv_heads=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([64, 128]), page=rng.choice([8, 16, 24, 32, 64]),
                    layout=rng.choice(["hnd", "nhd"]))
    if op == "tables":
        admit = rng.random() < 0.5
        return dict(op=op, batch=_log_int(rng, 1, 96 if admit else 1024), page=rng.choice([8, 16, 24, 32, 64]),
                    length=rng.randint(2048, 4096), new=rng.randint(64, 2048) if admit else 1, admit=admit)
    vocab = rng.choice([1000, 50257, 50257, rng.randint(2, 50257)])
    return dict(op=op, batch=_log_int(rng, 1, 256), vocab=vocab, pitch=vocab + rng.choice([0, 0, 1, 47]),
                dtype=rng.choice(["f32", "bf16"]), history=_log_int(rng, 1, 4096), bias=rng.choice([0, 1, 7, 32]),
                mask=rng.random() < 0.6)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _lengths(case, g):
    """Sequence lengths of the batch; a ragged batch has every age, one of one
    token and, from four rows on, one row that is not in use."""
    b, n = case["batch"], case["length"]
    if not case["ragged"]:
        return torch.full((b,), n, device=DEV, dtype=torch.int32)
    lens = torch.randint(1, n + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
    lens[0] = n
    if b > 2:
        lens[2] = 1
    if b > 3:
        lens[3] = 0
    return lens


def _cache(n_pages, case, g):
    h, p, d = case["kv_heads"], case["page"], case["dim"]
    shape = (n_pages, h, p, d) if case["layout"] == "hnd" else (n_pages, p, h, d)
    x = torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16)
    if case.get("cache") == "e4m3":
        x = (x * 100).float().clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return x if case["layout"] == "hnd" else x.transpose(1, 2)


def _prepare_attention(case, seed):
    g = _gen(seed)
    b, hq, hk, d, p = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case, g)
    blocks = -(-case["length"] // p)
    need = (lens.long() + p - 1) // p
    n_pages = b * blocks + 3
    order = torch.randperm(n_pages, device=DEV, generator=g).int()
    start = (need.cumsum(0) - need)[:, None] + torch.arange(blocks, device=DEV)
    live = torch.arange(blocks, device=DEV) < need[:, None]
    table = torch.where(live, order[start.clamp(max=n_pages - 1)], torch.full_like(start, -1).int())
    # q, k, v of the new token as the fused projection writes them: one row a sequence
    qkv = torch.randn(b, (hq + 2 * hk) * d, device=DEV, generator=g, dtype=torch.bfloat16)
    s = dict(op="attention", q=qkv[:, :hq * d].view(b, hq, d) * 1.5, k=_cache(n_pages, case, g),
             v=_cache(n_pages, case, g), table=table, lens=lens, page=p, k_new=None, v_new=None, k_scale=None,
             v_scale=None, lse=None)
    if case["append"]:
        s["q"] = qkv[:, :hq * d].view(b, hq, d)
        s["k_new"] = qkv[:, hq * d:(hq + hk) * d].view(b, hk, d)
        s["v_new"] = qkv[:, (hq + hk) * d:].view(b, hk, d)
    if case["cache"] == "e4m3":
        s["k_scale"] = (0.5 + torch.rand(hk, device=DEV, generator=g)) / 100
        s["v_scale"] = (0.5 + torch.rand(hk, device=DEV, generator=g)) / 100
    if case["lse"]:
        s["lse"] = torch.empty(b, hq, device=DEV)
    return s


def _prepare_write(case, seed):
    g = _gen(seed)
    t, h, d, p = case["tokens"], case["kv_heads"], case["dim"], case["page"]
    n_pages = -(-t // p) + 5
    qkv = torch.randn(t, 3 * h * d, device=DEV, generator=g, dtype=torch.bfloat16)
    slots = torch.randperm(n_pages * p, device=DEV, generator=g)[:t].view(-1).sort().values
    # whole pages in any order, rows in order inside a page; one row in 61 is padding
    pages = torch.randperm(n_pages, device=DEV, generator=g)
    slots = (pages[slots // p] * p + slots % p).int()
    slots[::61] = -1
    return dict(op="write", k=qkv[:, h * d:2 * h * d].view(t, h, d), v=qkv[:, 2 * h * d:].view(t, h, d), slots=slots,
                kc=_cache(n_pages, case, g), vc=_cache(n_pages, case, g))


def _tokens(case):
    return case["batch"] * case["new"] * 5 // 9 + 7 if case["admit"] else case["batch"] + 7


def _prepare_tables(case, seed):
    g = _gen(seed)
    b, p, n = case["batch"], case["page"], case["length"]
    blocks = -(-n // p)
    if case["admit"]:
        lens = torch.zeros(b, device=DEV, dtype=torch.int32)
        new = torch.randint(1, case["new"] + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
        done = torch.zeros(b, device=DEV, dtype=torch.int32)
    else:
        lens = torch.randint(1, n, (b,), device=DEV, generator=g, dtype=torch.int32)
        new = (torch.rand(b, device=DEV, generator=g) < 0.97).int()
        done = (torch.rand(b, device=DEV, generator=g) < 0.03).int()
        new = new * (1 - done)
    have = (lens.long() + p - 1) // p
    used = have.sum()
    n_pages = b * blocks
    order = torch.randperm(n_pages, device=DEV, generator=g).int()
    at = (have.cumsum(0) - have)[:, None] + torch.arange(blocks, device=DEV)
    live = torch.arange(blocks, device=DEV) < have[:, None]
    table = torch.where(live, order[at.clamp(max=n_pages - 1)], torch.full_like(at, -1).int())
    # other batches hold most of the rest: some steps run out of free pages
    n_free = torch.randint(1, b * (-(-case["new"] // p) + 1) // 2 + 4, (1,), device=DEV, generator=g)
    n_free = torch.minimum(n_free, n_pages - used).int()
    i = torch.arange(n_pages, device=DEV)
    free = torch.where(i < n_free, order[(used + i).clamp(max=n_pages - 1)], torch.full_like(order, -1))
    # rows of the flat token list: the last prompts may not fit, or rows at the end are padding
    tokens = _tokens(case)
    return dict(op="tables", table=table, lens=lens, new=new, done=done, free=free, n_free=n_free, page=p,
                tokens=tokens)


def _prepare_logits(case, seed):
    g = _gen(seed)
    b, v, n = case["batch"], case["vocab"], case["history"]
    logits = torch.randn(b, case["pitch"], device=DEV, generator=g) * 3
    logits = logits.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)[:, :v]
    # histories repeat themselves: tokens from a skewed distribution
    u = torch.rand(b, n, device=DEV, generator=g)
    tokens = (u.pow(4) * v).int().clamp_(max=v - 1)
    lens = torch.randint(1, n + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
    lens[0] = n
    prompt = (lens.float() * torch.rand(b, device=DEV, generator=g)).int()
    s = dict(op="logits", logits=logits, tokens=tokens, lens=lens, prompt_lens=prompt,
             repetition=1 + 0.3 * torch.rand(b, device=DEV, generator=g),
             frequency=0.5 * torch.rand(b, device=DEV, generator=g),
             presence=0.5 * torch.rand(b, device=DEV, generator=g), bias_ids=None, bias=None, mask=None)
    if case["bias"]:
        k = min(case["bias"], v)
        s["bias_ids"] = torch.rand(b, v, device=DEV, generator=g).topk(k, dim=1).indices.int()
        s["bias"] = torch.randn(b, k, device=DEV, generator=g) * 2
    if case["mask"]:
        words = (v + 31) // 32
        s["mask"] = torch.randint(-2**31, 2**31, (b, words), device=DEV, generator=g).int()
    return s


def prepare(case, seed):
    return {"attention": _prepare_attention, "write": _prepare_write, "tables": _prepare_tables,
            "logits": _prepare_logits}[case["op"]](case, seed)


# ---------------------------------------------------------------- plain forms
def _put(cache, page, off, rows):
    """cache[page, :, off] = rows for the rows whose page is not negative."""
    n = cache.shape[0]
    live = (page >= 0) & (page < n)
    pg, of = torch.where(live, page, 0).long(), torch.where(live, off, 0).long()
    old = cache[pg, :, of]
    keep = cache[0, :, 0].clone()          # dead rows all aim at this place: it keeps its value
    cache[pg, :, of] = torch.where(live[:, None, None], rows.to(cache.dtype), old)
    hit = (live & (pg == 0) & (of == 0)).float()
    put = (hit[:, None, None] * rows.float()).sum(0).to(cache.dtype)
    cache[0, :, 0] = torch.where(hit.sum() > 0, put, keep)


def _plain_attention(s):
    q, table, lens, p = s["q"], s["table"], s["lens"], s["page"]
    b, hq, d = q.shape
    hk = s["k"].shape[1]
    if s["k_new"] is not None:
        at = (lens - 1).clamp(min=0)
        page = table.gather(1, (at // p).long()[:, None])[:, 0]
        page = torch.where(lens > 0, page, torch.full_like(page, -1))
        _put(s["k"], page, at % p, s["k_new"])
        _put(s["v"], page, at % p, s["v_new"])
    n = table.shape[1] * p
    idx = table.clamp(min=0).long()
    k = s["k"][idx].float().transpose(1, 2).reshape(b, hk, n, d)       # [b, blocks, hk, p, d] -> [b, hk, n, d]
    v = s["v"][idx].float().transpose(1, 2).reshape(b, hk, n, d)
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][:, None, None], v * s["v_scale"][:, None, None]
    live = (torch.arange(n, device=q.device) < lens[:, None])[:, None, None]
    v = torch.where(live[:, :, 0, :, None], v, torch.zeros((), device=q.device))
    sc = torch.matmul(q.float().view(b, hk, hq // hk, d), k.transpose(2, 3)) / math.sqrt(d)
    sc = torch.where(live, sc, torch.full((), -math.inf, device=q.device))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(sc - m)
    z = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(z > 0, z, torch.ones_like(z))
    out = [o.reshape(b, hq, d).to(q.dtype)]
    if s["lse"] is not None:
        out.append((m + torch.log(z)).reshape(b, hq))
    if s["k_new"] is not None:
        out += [s["k"], s["v"]]
    return out


def _plain_write(s):
    p = s["kc"].shape[2]
    page = torch.where(s["slots"] >= 0, s["slots"] // p, torch.full_like(s["slots"], -1))
    off = s["slots"].clamp(min=0) % p
    _put(s["kc"], page, off, s["k"])
    _put(s["vc"], page, off, s["v"])
    return [s["kc"], s["vc"]]


def _plain_tables(s):
    table, lens, p = s["table"], s["lens"].long(), s["page"]
    new, done, free, t = s["new"].long(), s["done"].bool(), s["free"], s["tokens"]
    dev = table.device
    n_pages, blocks = free.numel(), table.shape[1]
    up = lambda x: (x + p - 1) // p  # noqa: E731
    # pages of the rows that ended go on top of the free pages, row after row
    back = torch.where(done, up(lens), torch.zeros_like(lens))
    at = s["n_free"].long() + (back.cumsum(0) - back)[:, None] + torch.arange(blocks, device=dev)
    hit = torch.arange(blocks, device=dev) < back[:, None]
    room = torch.cat([free, free.new_zeros(1)])
    room.scatter_(0, torch.where(hit, at, torch.full_like(at, n_pages)).view(-1), table.view(-1))
    free.copy_(room[:n_pages])
    avail = s["n_free"].long() + back.sum()
    len0 = torch.where(done, torch.zeros_like(lens), lens)
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    status = torch.zeros_like(lens)
    status = torch.where(cu[:-1] + new > t, torch.full_like(status, 3), status)
    status = torch.where(len0 + new > blocks * p, torch.full_like(status, 2), status)
    take = torch.where(status == 0, up(len0 + new) - up(len0), torch.zeros_like(lens))
    off = take.cumsum(0) - take
    status = torch.where((take > 0) & (off + take > avail), torch.ones_like(status), status)
    ok = status == 0
    take = torch.where(ok, take, torch.zeros_like(take))
    col = torch.arange(blocks, device=dev)[None, :] - up(len0)[:, None]
    fresh = (col >= 0) & (col < take[:, None])
    src = (avail - 1 - off[:, None] - col).clamp(0, n_pages - 1)
    table.copy_(torch.where(fresh, free[src], table))
    i = torch.arange(t, device=dev)
    row = torch.searchsorted(cu[1:].contiguous(), i, right=True).clamp(max=lens.numel() - 1)
    live = (i < cu[-1]) & ok[row]
    pos = len0[row] + i - cu[row]
    page = table[row, (pos // p).clamp(0, blocks - 1)].long()
    slot = torch.where(live, page * p + pos % p, torch.full_like(pos, -1))
    pos = torch.where(live, pos, torch.full_like(pos, -1))
    return [slot.int(), pos.int(), cu.int(), (len0 + torch.where(ok, new, torch.zeros_like(new))).int(),
            (avail - take.sum()).int().view(1), status.int(), table, free]


def _plain_logits(s):
    x = s["logits"].float()
    b, v = x.shape
    i = torch.arange(s["tokens"].shape[1], device=x.device)
    tok = s["tokens"].long()
    seen = (i < s["lens"][:, None]).float()
    made = seen * (i >= s["prompt_lens"][:, None]).float()
    every = torch.zeros(b, v, device=x.device).scatter_add_(1, tok, seen)
    count = torch.zeros(b, v, device=x.device).scatter_add_(1, tok, made)
    r = s["repetition"][:, None]
    x = torch.where(every > 0, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(count > 0, x - s["frequency"][:, None] * count - s["presence"][:, None], x)
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias"])
    if s["mask"] is not None:
        c = torch.arange(v, device=x.device)
        bit = (s["mask"][:, c // 32] >> (c % 32).int()) & 1
        x = torch.where(bit != 0, x, torch.full((), -math.inf, device=x.device))
    return [x.to(s["logits"].dtype)]


# ---------------------------------------------------------------- one pass
def run(state):
    s = state
    if not own:
        return {"attention": _plain_attention, "write": _plain_write, "tables": _plain_tables,
                "logits": _plain_logits}[s["op"]](s)
    if s["op"] == "attention":
        from nlearn_b200.paged import paged_decode_attention
        out = [paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["k_new"], s["v_new"],
                                      k_scale=s["k_scale"], v_scale=s["v_scale"], lse=s["lse"])]
        if s["lse"] is not None:
            out.append(s["lse"])
        if s["k_new"] is not None:
            out += [s["k"], s["v"]]
        return out
    if s["op"] == "write":
        from nlearn_b200.paged import paged_kv_write
        paged_kv_write(s["k"], s["v"], s["kc"], s["vc"], s["slots"])
        return [s["kc"], s["vc"]]
    if s["op"] == "tables":
        from nlearn_b200.paged import update_block_tables
        plan = update_block_tables(s["table"], s["lens"], s["new"], s["free"], s["n_free"], s["page"], s["tokens"],
                                   done=s["done"])
        return [plan.slots, plan.positions, plan.cu, plan.lens, plan.n_free, plan.status, s["table"], s["free"]]
    from nlearn_b200.kernels.logits import process_logits
    return [process_logits(s["logits"], tokens=s["tokens"], lens=s["lens"], prompt_lens=s["prompt_lens"],
                           repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                           bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"])]


# ---------------------------------------------------------------- the floor
def work(case):
    op = case["op"]
    if op == "attention":
        b, hq, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        keys = b * case["length"] * (0.5 if case["ragged"] else 1.0)
        el = 1 if case["cache"] == "e4m3" else 2
        bytes_ = keys * hk * d * 2 * el + b * hq * d * 4 + keys / case["page"] * 4 + b * 4
        if case["append"]:
            bytes_ += 2 * b * hk * d * 4
        if case["lse"]:
            bytes_ += b * hq * 4
        return {"bytes": bytes_, "flops": 4.0 * keys * hq * d}
    if op == "write":
        return {"bytes": case["tokens"] * (8.0 * case["kv_heads"] * case["dim"] + 4), "flops": 0}
    if op == "tables":
        b = case["batch"]
        pages = b * (case["new"] / 2 if case["admit"] else 1) / case["page"]
        return {"bytes": 28.0 * b + _tokens(case) * 8.0 + pages * 8, "flops": 0}
    el = 2 if case["dtype"] == "bf16" else 4
    bytes_ = case["batch"] * (2.0 * case["vocab"] * el + 2.0 * case["history"] + 8.0 * case["bias"] + 20)
    if case["mask"]:
        bytes_ += case["batch"] * case["vocab"] / 8
    return {"bytes": bytes_, "flops": 0}


# ---------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    """From the definitions, in 64 bits, one sequence after the other.  Copies
    and whole numbers have no computed value: None."""
    if case["op"] == "attention":
        s = _prepare_attention(case, seed)
        b, hq, hk, d, p = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "page"))
        out = torch.zeros(b, hq, d, device=DEV, dtype=torch.float64)
        lse = torch.full((b, hq), -math.inf, device=DEV, dtype=torch.float64)
        for i, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            pages = s["table"][i, :(n + p - 1) // p].long()
            k, v = (s[x][pages].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :n].clone() for x in ("k", "v"))
            if s["k_new"] is not None:
                k[:, n - 1], v[:, n - 1] = s["k_new"][i].double(), s["v_new"][i].double()
            if s["k_scale"] is not None:
                k *= s["k_scale"].double()[:, None, None]
                v *= s["v_scale"].double()[:, None, None]
            sc = torch.einsum("hgd,hnd->hgn", s["q"][i].double().view(hk, hq // hk, d), k) * d ** -0.5
            lse[i] = torch.logsumexp(sc, -1).view(hq)
            out[i] = torch.einsum("hgn,hnd->hgd", torch.softmax(sc, -1), v).reshape(hq, d)
        return [out] + ([lse] if case["lse"] else []) + ([None, None] if case["append"] else [])
    if case["op"] == "logits":
        s = _prepare_logits(case, seed)
        y = s["logits"].double()
        v = case["vocab"]
        for i in range(case["batch"]):
            n, m = int(s["lens"][i]), int(s["prompt_lens"][i])
            seen = torch.bincount(s["tokens"][i, :n], minlength=v) > 0
            made = torch.bincount(s["tokens"][i, m:n], minlength=v).double()
            r, f, a = (s[x][i].double() for x in ("repetition", "frequency", "presence"))
            row = y[i]
            row[seen] = torch.where(row[seen] > 0, row[seen] / r, row[seen] * r)
            row -= f * made + a * (made > 0)
            if s["bias_ids"] is not None:
                row.index_add_(0, s["bias_ids"][i].long(), s["bias"][i].double())
            if s["mask"] is not None:
                words = s["mask"][i].long() & 0xFFFFFFFF
                allowed = (words[:, None] >> torch.arange(32, device=DEV) & 1).flatten()[:v].bool()
                row[~allowed] = -math.inf
        return [y]
    return None
