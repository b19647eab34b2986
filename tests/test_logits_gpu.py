"""Logits processing on the GPU against the 64-bit restatement.

Tolerance: f32 logits of size up to ~2^5 go through at most five f32 operations
(divide or multiply, two for the counted penalties, one bias sum per listed
entry, the add): 8 half steps of the largest value on the way, bounded by
2^-24 * 8 * (|x| max(r, 1/r) + f c + a + sum |bias|).  A bf16 result adds half a
bf16 step of the value, 2^-8 |y|."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import paged as OP  # noqa: E402
from nlearn_b200 import _lib  # noqa: E402
from nlearn_b200.kernels.logits import process_logits  # noqa: E402


def make(dev, B, V, pitch, dtype, L, n_bias, seed):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy((rng.standard_normal((B, pitch)) * 4).astype(np.float32)).to(dtype)
    tok = rng.integers(0, max(1, min(V, 60)), (B, L)).astype(np.int32)
    tok[rng.random((B, L)) < 0.2] = V - 1
    tok[rng.random((B, L)) < 0.1] = -1          # ignored
    tok[rng.random((B, L)) < 0.1] = V           # ignored
    lens = rng.integers(0, L + 1, B).astype(np.int32)
    lens[0] = L
    prompt = (lens * rng.random(B)).astype(np.int32)
    kw = dict(tokens=tok, lens=lens, prompt_lens=prompt, repetition=(0.5 + rng.random(B)).astype(np.float32),
              frequency=rng.standard_normal(B).astype(np.float32), presence=rng.standard_normal(B).astype(np.float32))
    if n_bias:
        ids = rng.integers(-1, V + 1, (B, n_bias)).astype(np.int32)
        ids[:, n_bias // 2] = ids[:, 0]         # an id listed again
        kw.update(bias_ids=ids, bias=(rng.standard_normal((B, n_bias)) * 3).astype(np.float32))
    words = (V + 31) // 32 + 1
    kw.update(mask=rng.integers(-2**31, 2**31, (B, words)).astype(np.int32))
    return x.to(dev)[:, :V], kw


def call(x, kw, **more):
    return process_logits(x, **{k: torch.from_numpy(v).to(x.device) for k, v in kw.items()}, **more)


def check(y, x, kw):
    X = x.double().cpu().numpy()
    ref = OP.process_logits(X, **kw)
    got = y.double().cpu().numpy()
    assert np.array_equal(np.isfinite(ref), np.isfinite(got)) and np.array_equal(np.isneginf(ref), np.isneginf(got))
    r = kw.get("repetition")
    size = np.abs(X) * (np.maximum(r, 1 / r)[:, None] if r is not None else 1)
    for k in ("frequency", "presence"):
        if k in kw:
            size = size + np.abs(kw[k])[:, None] * (kw["tokens"].shape[1] if k == "frequency" else 1)
    if "bias" in kw:
        size = size + np.abs(kw["bias"]).sum(1)[:, None]
    fin = np.isfinite(ref)
    tol = 2.0**-21 * size + (2.0**-8 * np.abs(np.where(fin, ref, 0)) if y.dtype == torch.bfloat16 else 0)
    assert (np.abs(got - ref)[fin] <= tol[fin]).all()


@pytest.mark.parametrize("B,V,pitch", [(1, 1, 1), (3, 31, 40), (2, 1000, 1000), (2, 4097, 4099), (5, 8192, 8192),
                                       (2, 50257, 50304), (1, 50257, 50257)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_rules(cuda, B, V, pitch, dtype):
    x, kw = make(cuda, B, V, pitch, dtype, 300, 9, B + V)
    keep = x.clone()
    y = call(x, kw)
    torch.cuda.synchronize()
    check(y, x, kw)
    assert torch.equal(x, keep)
    z = x.clone()
    assert call(z, kw, out=z) is z               # in place: the same values
    torch.cuda.synchronize()
    assert torch.equal(z, y)


@pytest.mark.parametrize("parts", [(), ("tokens",), ("bias",), ("mask",), ("tokens", "repetition"),
                                   ("tokens", "frequency", "presence"), ("tokens", "prompt_lens", "presence", "mask")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parts(cuda, parts, dtype):
    """Each rule alone, out of place and in place inside a wider row whose
    other columns stay as they are."""
    x, kw = make(cuda, 4, 5001, 5010, dtype, 77, 5, 3)
    use = {k: v for k, v in kw.items() if k in parts or (k == "lens" and "tokens" in parts) or
           (k == "bias_ids" and "bias" in parts)}
    check(call(x, use), x, use)
    wide = torch.full((4, 5016), 7.0, device=cuda, dtype=dtype)
    wide[:, 3:5004] = x
    call(wide[:, 3:5004], use, out=wide[:, 3:5004])
    torch.cuda.synchronize()
    check(wide[:, 3:5004], x, use)
    assert (wide[:, :3] == 7).all() and (wide[:, 5004:] == 7).all()


@pytest.mark.parametrize("V", [1, 7, 1000, 4099])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place_rows_with_few_and_many_tokens(cuda, V, dtype):
    """Rows of one call that are worked on where they lie and through a copy, at every
    place in a 16-byte unit; what lies between the rows stays."""
    x, kw = make(cuda, 9, V, V, dtype, 700, 3, V)
    kw.pop("mask")
    kw["lens"][:] = [700, 0, 1, 3, 700, 20, 699, 512, 40]
    kw["prompt_lens"] = kw["lens"] // 2
    for off in (0, 1, 3):
        buf = torch.full((9 * (V + 3) + off,), 77.0, device=cuda).to(dtype)
        z = buf[off:].view(9, V + 3)[:, :V]
        z.copy_(x)
        assert call(z, kw, out=z) is z
        torch.cuda.synchronize()
        check(z, x, kw)
        assert (buf[off:].view(9, V + 3)[:, V:] == 77).all() and (buf[:off] == 77).all()


@pytest.mark.parametrize("rules", [("mask",), ("mask", "tokens", "lens", "repetition"), ("bias_ids", "bias"), ()])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_at_different_places_of_a_unit(cuda, rules, dtype):
    """Input and output rows that begin at different bytes of a 16-byte unit, rows of a
    few columns among them."""
    for V in (1, 5, 9, 33, 2051, 9001):
        x, kw = make(cuda, 5, V, V, dtype, 30, 3, V)
        kw = {k: kw[k] for k in rules}
        for a, b in ((0, 1), (1, 0), (3, 6), (2, 2), (5, 5)):
            src = torch.full((5 * (V + a) + 8,), 77.0, device=cuda).to(dtype)
            dst = torch.full((5 * (V + b) + 8,), 77.0, device=cuda).to(dtype)
            xi, yi = src[a:a + 5 * (V + a)].view(5, V + a)[:, :V], dst[b:b + 5 * (V + b)].view(5, V + b)[:, :V]
            xi.copy_(x)
            call(xi, kw, out=yi)
            torch.cuda.synchronize()
            check(yi, x, kw)
            left = dst.clone()
            left[b:b + 5 * (V + b)].view(5, V + b)[:, :V] = 77.0
            assert (left == 77).all()


@pytest.mark.parametrize("n_bias", [1, 3, 4, 5, 127, 128, 129, 600])
def test_lists_of_biases(cuda, n_bias):
    x, kw = make(cuda, 3, 500, 500, torch.float32, 40, n_bias, n_bias)
    y = call(x, kw)
    torch.cuda.synchronize()
    check(y, x, kw)


def test_mask_rows_and_nothing_left(cuda):
    x = torch.randn(4, 100, device=cuda)
    mask = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    mask[1, 0] = 0b1010
    rows = torch.tensor([1, -1, 0, 2], dtype=torch.int32, device=cuda)
    y = process_logits(x, mask=mask, mask_rows=rows)
    torch.cuda.synchronize()
    assert torch.equal(y[1], x[1]) and torch.equal(y[3], x[3])       # no mask, and one past the last
    assert torch.isneginf(y[2]).all()                                # nothing allowed
    assert torch.equal(y[0, [1, 3]], x[0, [1, 3]]) and torch.isneginf(y[0]).sum() == 98
    # masks of no rows at all: with mask_rows nothing is masked
    assert torch.equal(process_logits(x, mask=mask[:0], mask_rows=rows), x)


def test_infinite_logits_and_parameters(cuda):
    """-inf stays -inf under every rule; parameters of a row touch only the
    columns they name, infinite ones too; the lowest values do not wrap."""
    low = torch.finfo(torch.float32).min
    x = torch.tensor([[1.0, -float("inf"), low, float("inf"), float("nan"), 0.0]], device=cuda)
    tok = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=cuda)
    n = torch.tensor([4], dtype=torch.int32, device=cuda)
    one = lambda v: torch.tensor([v], device=cuda)  # noqa: E731
    y = process_logits(x, tokens=tok, lens=n, repetition=one(2.0))
    assert y[0, :4].tolist() == [0.5, -float("inf"), -float("inf"), float("inf")] and torch.isnan(y[0, 4])
    assert y[0, 5] == 0
    y = process_logits(x, tokens=tok[:, :1], lens=n, frequency=one(float("inf")))
    assert y[0, 0] == -float("inf") and y[0, 3] == float("inf") and y[0, 5] == 0
    ban = process_logits(x, bias_ids=torch.tensor([[3, 0]], dtype=torch.int32, device=cuda),
                         bias=torch.tensor([[0.0, -float("inf")]], device=cuda))
    assert ban[0, 0] == -float("inf") and ban[0, 3] == float("inf")


def test_lengths_past_the_history(cuda):
    x = torch.randn(3, 64, device=cuda)
    tok = torch.zeros(3, 5, dtype=torch.int32, device=cuda)
    one = torch.ones(3, device=cuda)
    y = process_logits(x, tokens=tok, lens=torch.tensor([9, -2, 3], dtype=torch.int32, device=cuda),
                       prompt_lens=torch.tensor([1, 1, 77], dtype=torch.int32, device=cuda), frequency=one,
                       presence=one)
    torch.cuda.synchronize()
    want = x.clone()
    want[0, 0] = want[0, 0] - 4 - 1
    assert torch.allclose(y, want, rtol=0, atol=2.0**-19)
    empty = process_logits(x, tokens=tok[:, :0], lens=torch.zeros(3, dtype=torch.int32, device=cuda), presence=one)
    assert torch.equal(empty, x)


def test_graph_and_refusals(cuda):
    x, kw = make(cuda, 3, 3000, 3000, torch.float32, 50, 4, 1)
    t = {k: torch.from_numpy(v).to(cuda) for k, v in kw.items()}
    y = process_logits(x, **t)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = process_logits(x, **t)
    t["lens"].copy_(torch.tensor([0, 20, 50], dtype=torch.int32))
    kw["lens"] = np.array([0, 20, 50], np.int32)
    g.replay()
    torch.cuda.synchronize()
    check(z, x, kw)
    assert not torch.equal(y, z)
    i = t["tokens"]
    one = torch.ones(3, device=cuda)
    bad = [(TypeError, dict(), x.double()), (ValueError, dict(), x[0]), (ValueError, dict(), x.t()),
           (ValueError, dict(tokens=i), x), (ValueError, dict(repetition=one), x), (ValueError, dict(lens=t["lens"]), x),
           (TypeError, dict(tokens=i.long(), lens=t["lens"]), x), (ValueError, dict(bias=t["bias"]), x),
           (ValueError, dict(bias=t["bias"][:, :1], bias_ids=t["bias_ids"]), x),
           (ValueError, dict(mask=t["mask"][:, :5]), x), (ValueError, dict(mask=t["mask"][:2]), x),
           (RuntimeError, dict(tokens=i, lens=t["lens"], presence=one.clone().requires_grad_()), x),
           (RuntimeError, dict(), x.clone().requires_grad_()),
           (ValueError, dict(mask_rows=t["lens"]), x), (ValueError, dict(out=x[:, :10]), x),
           (ValueError, dict(tokens=i, lens=t["lens"], frequency=one.double()), x),
           (ValueError, dict(out=torch.empty(4, 3000, device=cuda).flatten()[100:9100].view(3, 3000)), x.cpu())]
    for n, (err, kws, arg) in enumerate(bad):
        with pytest.raises(err):
            process_logits(arg, **kws)
            raise AssertionError(n)
    both = torch.randn(9, 1000, device=cuda)
    with pytest.raises(ValueError):
        process_logits(both[:8], out=both[1:])
    assert _lib.device_error() == 0
