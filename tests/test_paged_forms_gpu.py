"""Forms of the paged operators beside those of test_paged_gpu.py: short
sequences in wide tables, scores and values that are infinite, and the decoder
over an e4m3 cache against a recompute over the same rounded keys and values."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle.model import OracleGPT, causal_attention, gelu_tanh, layer_norm  # noqa: E402
from nlearn_b200 import _lib  # noqa: E402
from nlearn_b200.generate import PagedDecoder  # noqa: E402
from nlearn_b200.paged import paged_decode_attention  # noqa: E402

from test_paged_decode_gpu import CFG, oracle, params, prompts  # noqa: E402,F401
from test_paged_gpu import E4M3, check_out, make_case  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("lens,hq,hk,d,page", [([512], 8, 8, 64, 16), ([1, 0, 17, 512] * 8, 8, 8, 64, 16),
                                               ([40, 3, 700, 0, 1], 32, 8, 128, 32), ([5, 90], 40, 1, 128, 24)])
def test_short_sequences_in_wide_tables(cuda, dtype, lens, hq, hk, d, page):
    """A table for 131072 tokens a row: pages past a sequence's end are never looked at."""
    q, k, v, table, ln = make_case(cuda, lens, hq, hk, d, page, dtype=dtype, seed=d)
    wide = torch.full((len(lens), 131072 // page), 10**9, dtype=torch.int32, device=cuda)
    wide[:, :table.shape[1]] = table
    new = torch.randn(len(lens), 2, hk, d, device=cuda).bfloat16()
    lse = torch.empty(len(lens), hq, device=cuda)
    o = paged_decode_attention(q, k, v, wide, ln, new[:, 0], new[:, 1], lse=lse, scale=0.02)
    torch.cuda.synchronize()
    check_out(o, lse, q, k, v, wide, ln, 0.02)
    assert _lib.device_error() == 0


def test_infinite_keys_and_values(cuda):
    """Keys whose score is -inf have no weight, a row of them is like a row with no
    key; an infinite value leaves its column only."""
    q, k, v, table, ln = make_case(cuda, [70, 70, 3000], 4, 2, 64, 16, seed=8, poison=False)
    q[..., 0] = 1.0
    page = lambda b, j: (int(table[b, j // 16]), slice(None), j % 16, 0)  # noqa: E731
    for b, gone in ((0, range(0, 70)), (1, range(10, 60)), (2, range(0, 2990))):
        for j in gone:
            k[page(b, j)] = -float("inf")
    lse = torch.empty(3, 4, device=cuda)
    o = paged_decode_attention(q, k, v, table, ln, lse=lse)
    torch.cuda.synchronize()
    assert (o[0] == 0).all() and torch.isneginf(lse[0]).all()
    for b, left in ((1, [*range(10), *range(60, 70)]), (2, range(2990, 3000))):
        K, V = (torch.stack([x[int(table[b, j // 16]), :, j % 16] for j in left], 1)[None] for x in (k, v))
        n = torch.tensor([len(left)], dtype=torch.int32)
        check_out(o[b:b + 1], lse[b:b + 1], q[b:b + 1], K, V, torch.zeros(1, 1, dtype=torch.int32), n, 0.125)
    want = o.clone()
    v[int(table[1, 0]), 1, 5, 7] = float("inf")
    o = paged_decode_attention(q, k, v, table, ln)
    torch.cuda.synchronize()
    hit = ~torch.isfinite(o)
    assert hit[1, 2:, 7].all() and int(hit.sum()) == 2 and torch.equal(o[~hit], want[~hit])
    assert _lib.device_error() == 0


def logits_over_rounded_cache(model: OracleGPT, toks, n_prompt):
    """The oracle's forward with the positions after the prompt attending over keys and
    values rounded to e4m3, as the cache holds them (the prompt's own attention runs before
    they are rounded)."""
    p, H, S = model.p, model.H, len(toks)
    D = p["wte"].shape[1]
    x = p["wte"][torch.from_numpy(toks).long()][None] + p["wpe"][:S][None]
    for layer in range(model.L):
        w = f"blocks.{layer}."
        h = layer_norm(x, p[w + "ln1.g"], p[w + "ln1.b"], model.eps)
        qkv = (h @ p[w + "wqkv"]).view(1, S, 3, H, D // H)
        Q, K, V = (qkv[:, :, i].transpose(1, 2) for i in range(3))
        Kr, Vr = (t.bfloat16().float().clamp(-448, 448).to(E4M3).float() for t in (K, V))
        o = torch.cat((causal_attention(Q, K, V)[:, :, :n_prompt], causal_attention(Q, Kr, Vr)[:, :, n_prompt:]), 2)
        x = x + o.transpose(1, 2).reshape(1, S, D) @ p[w + "wo"]
        h = layer_norm(x, p[w + "ln2.g"], p[w + "ln2.b"], model.eps)
        x = x + gelu_tanh(h @ p[w + "w1"] + p[w + "b1"]) @ p[w + "w2"] + p[w + "b2"]
    x = layer_norm(x, p["lnf.g"], p["lnf.b"], model.eps)
    return (x @ p["head.w"][:, :model.V])[0].numpy()


def test_decoder_over_an_e4m3_cache(cuda, params):  # noqa: F811
    """Logits within twice the bf16 decoder's bar (2e-2 of the largest): a key or value that
    bf16 puts on the other side of an e4m3 border, some 2^-8 / 2^-3 = 3 % of them, is off by
    an eighth, 2 % of their norm."""
    ps = prompts([37, 1, 64, 16], 3)
    dec = PagedDecoder(params, CFG, max_batch=4, seed=7, cache_dtype=E4M3)
    rows = dec.add(ps)
    steps = [dec.logits[:, :CFG.vocab].cpu().numpy()]
    for _ in range(9):
        dec.step(1)
        steps.append(dec.logits[:, :CFG.vocab].cpu().numpy())
    model = oracle(params)
    for row, p in zip(rows, ps):
        toks = dec.tokens(row)
        with torch.no_grad():
            full = logits_over_rounded_cache(model, toks[:-1], p.size)
        for i, got in enumerate(steps):
            ref = full[p.size - 1 + i]
            assert np.abs(got[row] - ref).max() / np.abs(ref).max() < 4e-2, (row, i)
    assert _lib.device_error() == 0
