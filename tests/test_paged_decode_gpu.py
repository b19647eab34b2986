"""Generation over the paged cache against the oracle's full recompute
(oracle/model.py), as tests/test_decode_gpu.py does for the one-position
decoder: logits within max|err|/max|ref| 2e-2 at every step of every row, the
drawn token the oracle's choice up to that tolerance, rules applied as
oracle/paged.py restates them; rows and pages that come free are used again;
captured steps give the tokens of eager ones."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import decode as OD  # noqa: E402
from oracle import paged as OP  # noqa: E402
from oracle.model import OracleGPT  # noqa: E402
from nlearn_b200 import _lib  # noqa: E402
from nlearn_b200.generate import PagedDecoder, generate  # noqa: E402
from nlearn_b200.model import FlatParams, GPTConfig  # noqa: E402

CFG = GPTConfig(vocab=1003, d_model=256, n_heads=4, n_layers=2, d_ff=512, max_seq=128)


@pytest.fixture(scope="module")
def params(cuda):
    P = FlatParams(CFG, cuda, seed=3)
    for name, shape, _ in P.specs:      # wider logits than the initial weights give: choices are clear
        if name == "head.w":
            P.f(name).mul_(8.0)
    P.refresh_shadow()
    return P


def oracle(P):
    params = {}
    for name, shape, _ in P.specs:
        w = P.f(name).detach().float().cpu()
        params[name] = w.bfloat16().float() if len(shape) == 2 else w
    return OracleGPT(params, n_layers=CFG.n_layers, n_heads=CFG.n_heads, vocab=CFG.vocab, eps=CFG.ln_eps)


def prompts(sizes, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, CFG.vocab, n).astype(np.int32) for n in sizes]


def check_row(model, toks, n_prompt, row, seed, T, **rules):
    """Every drawn token is the oracle's choice up to the logits' tolerance."""
    with torch.no_grad():
        full = model.logits(torch.from_numpy(toks[None, :-1].astype(np.int64))).numpy()[0]
    for i in range(n_prompt, len(toks)):
        raw = full[i - 1:i]
        ref = OP.process_logits(raw, tokens=toks[None, :i], lens=[i], prompt_lens=[n_prompt], **rules)[0]
        # a logit off by e moves by e * max(r, 1 / r) under the penalties
        r = max(float(rules.get("repetition", [1.0])[0]), 1.0)
        tol = 2 * 2e-2 * np.abs(raw).max() * r / (T or 1.0) + 1e-3
        if T > 0:
            u = OD.uniforms(seed, i - 1, row, CFG.vocab).astype(np.float64)
            ref = ref / T - np.log(-np.log(u))
        assert ref[toks[i]] >= ref.max() - tol, (row, i)


@pytest.mark.parametrize("page,dtype", [(16, torch.bfloat16), (5, torch.bfloat16), (16, torch.float8_e4m3fn)])
def test_logits_match_full_recompute(cuda, params, page, dtype):
    sizes = [37, 1, 64, 16]
    ps = prompts(sizes)
    dec = PagedDecoder(params, CFG, max_batch=5, page_size=page, seed=7, cache_dtype=dtype)
    rows = dec.add(ps)
    steps = [dec.logits[:, :CFG.vocab].cpu().numpy()]
    for _ in range(9):
        dec.step(1, use_graph=False)
        steps.append(dec.logits[:, :CFG.vocab].cpu().numpy())
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    model = oracle(params)
    for row, p in zip(rows, ps):
        toks = dec.tokens(row)
        assert len(toks) == p.size + 10 and np.array_equal(toks[:p.size], p)
        with torch.no_grad():
            full = model.logits(torch.from_numpy(toks[None, :-1].astype(np.int64))).numpy()[0]
        # (half a step of e4m3 is 2^-4, sixteen times bf16's 2^-8)
        bar = 2e-2 if dtype == torch.bfloat16 else 16 * 2e-2
        for i, got in enumerate(steps):
            ref = full[p.size - 1 + i]
            assert np.abs(got[row] - ref).max() / np.abs(ref).max() < bar, (row, i)
        if dtype == torch.bfloat16:
            check_row(model, toks, p.size, row, 7, 1.0)


def test_graph_gives_the_eager_tokens(cuda, params):
    ps = prompts([9, 30, 3], 1)
    out = [PagedDecoder(params, CFG, max_batch=3, seed=5).generate(ps, [12, 20, 7], use_graph=g) for g in (True, False)]
    for a, b in zip(*out):
        np.testing.assert_array_equal(a, b)
    assert [len(a) for a in out[0]] == [21, 50, 10]


def test_rows_and_pages_are_used_again(cuda, params):
    """Ten prompts through three rows and fewer pages than they need together:
    greedy tokens are the oracle's for each prompt, whoever ran beside it."""
    sizes = [5, 60, 17, 1, 33, 40, 2, 90, 16, 31]
    ps, counts = prompts(sizes, 2), [6, 9, 1, 14, 3, 20, 30, 8, 0, 5]
    dec = PagedDecoder(params, CFG, max_batch=3, n_pages=12, page_size=16, temperature=0.0)
    out = dec.generate(ps, counts)
    assert _lib.device_error() == 0
    assert dec.n_free.item() == 12 and sorted(dec.free_pages.tolist()) == list(range(12))
    model = oracle(params)
    for p, n, toks in zip(ps, counts, out):
        assert len(toks) == p.size + n and np.array_equal(toks[:p.size], p)
        check_row(model, toks, p.size, 0, 0, 0.0)
    again = dec.generate(ps[:4], 5)
    for p, toks in zip(ps[:4], again):
        assert np.array_equal(toks[:p.size], p) and len(toks) == p.size + 5


def test_rules(cuda, params):
    """Penalties, biases and a mask that changes between steps, each row its own."""
    ps = prompts([20, 20, 20, 20], 3)
    dec = PagedDecoder(params, CFG, max_batch=4, temperature=0.0)
    a, = dec.add(ps[:1], repetition=1.8, frequency=0.7, presence=0.4)
    b, = dec.add(ps[1:2], bias={7: 60.0, 11: -50.0})
    allowed = list(range(100, 140))
    c, = dec.add(ps[2:3], allowed=allowed)
    d, = dec.add(ps[3:])
    dec.step(6)
    dec.set_allowed(c, [999])
    dec.step(5)
    dec.set_allowed(c, None)
    dec.step(2)
    toks = {r: dec.tokens(r) for r in (a, b, c, d)}
    assert _lib.device_error() == 0
    model = oracle(params)
    one = lambda v: np.array([v])  # noqa: E731
    check_row(model, toks[a], 20, a, 0, 0.0, repetition=one(1.8), frequency=one(0.7), presence=one(0.4))
    check_row(model, toks[b], 20, b, 0, 0.0, bias_ids=np.array([[7, 11]]), bias=np.array([[60.0, -50.0]]))
    check_row(model, toks[d], 20, d, 0, 0.0)
    t = toks[c][20:]
    assert all(x in allowed for x in t[:7]) and (t[7:12] == 999).all()
    # with penalties of nothing the tokens are those of no rules
    dec.release([a, b, c, d])
    e, = dec.add(ps[3:])
    dec.step(13)
    np.testing.assert_array_equal(dec.tokens(e), toks[d])


def test_entry_point(cuda, params):
    ps = prompts([12, 40], 4)
    out = generate(params, ps, [5, 3], temperature=0.0)
    assert [len(t) for t in out] == [17, 43]
    one = generate(params, ps[0], 5, temperature=0.0, repetition=1.3)
    assert one.shape == (17,)
    both = generate(params, [p[:10] for p in ps], 4, temperature=0.0)      # equal lengths: the one-position decoder
    assert both.shape == (2, 14)
    long = generate(params, [np.arange(300) % CFG.vocab, ps[0]], 8, temperature=0.0)
    assert len(long[0]) == CFG.max_seq and np.array_equal(long[0][:CFG.max_seq - 8],
                                                          (np.arange(300) % CFG.vocab)[-(CFG.max_seq - 8):])
    assert _lib.device_error() == 0


def test_allowed_of_several_rows(cuda, params):
    """Any iterable of ids holds for every row of the call."""
    dec = PagedDecoder(params, CFG, max_batch=3)
    rows = dec.add(prompts([4, 9, 5]), allowed=(i for i in range(50, 53)))
    dec.step(4)
    for r, n in zip(rows, (4, 9, 5)):
        assert all(50 <= t < 53 for t in dec.tokens(r)[n:])


def test_refusals(cuda, params):
    dec = PagedDecoder(params, CFG, max_batch=2, n_pages=3, page_size=16, max_len=48)
    with pytest.raises(RuntimeError):
        dec.add(prompts([3, 3, 3]))
    with pytest.raises(ValueError):
        dec.add([np.zeros(48, np.int32)])
    with pytest.raises(ValueError):
        dec.add([np.zeros(0, np.int32)])
    with pytest.raises(RuntimeError):
        dec.add(prompts([30, 30]))
    with pytest.raises(ValueError):
        dec.add(prompts([3]), bias={i: 1.0 for i in range(33)})
    with pytest.raises(ValueError):
        dec.add(prompts([3]), allowed=[CFG.vocab])
    with pytest.raises(ValueError):
        dec.add(prompts([3]), allowed=[])
    with pytest.raises(ValueError):
        dec.release([0])
    r, s = dec.add(prompts([15, 32]))
    with pytest.raises(RuntimeError):
        dec.generate(prompts([3]), 2)
    with pytest.raises(RuntimeError):     # row s would need a third page for its key 32
        dec.step(3)
    dec.release([s])
    dec.step(32)                          # row r: 48 tokens, its full length
    dec.step()
    with pytest.raises(RuntimeError):
        dec.step()
    assert len(dec.tokens(r)) == 49 and _lib.device_error() == 0
    for kw in (dict(max_len=129), dict(page_size=0), dict(max_batch=0)):
        with pytest.raises(ValueError):
            PagedDecoder(params, CFG, **kw)


def test_rows_at_their_own_positions(cuda):
    """The embedding and the sampler by rows: idle rows, positions and tokens
    outside their tables, and the random bits of the shared-position sampler."""
    lib = _lib.lib
    st = torch.cuda.current_stream().cuda_stream
    wte, wpe = torch.randn(50, 256, device=cuda).bfloat16(), torch.randn(8, 256, device=cuda).bfloat16()
    tok = torch.tensor([3, 49, 7, 50, -1, 2], device=cuda, dtype=torch.int32)
    lens = torch.tensor([1, 8, 0, 2, 3, 9], device=cuda, dtype=torch.int32)
    x = torch.full((6, 256), 9.0, device=cuda).bfloat16()
    assert _lib.device_error() == 0
    assert lib.nl_decode_embed_rows(tok.data_ptr(), lens.data_ptr(), wte.data_ptr(), wpe.data_ptr(), x.data_ptr(), 6,
                                    256, 8, 50, st) == 0
    torch.cuda.synchronize()
    assert _lib.device_error() == 3
    assert torch.equal(x[0], (wte[3].float() + wpe[0].float()).bfloat16())
    assert torch.equal(x[1], (wte[49].float() + wpe[7].float()).bfloat16()) and (x[2:] == 0).all()
    V = 1000
    lg = (torch.randn(4, V, device=cuda) * 2)
    lens = torch.tensor([5, 0, 9, 1], device=cuda, dtype=torch.int32)
    tok = torch.full((4,), -3, device=cuda, dtype=torch.int32)
    out = torch.full((4, 10), -4, device=cuda, dtype=torch.int32)
    for T in (0.0, 0.8):
        assert lib.nl_sample_tokens_rows(lg.data_ptr(), V, V, T, 11, lens.data_ptr(), tok.data_ptr(), out.data_ptr(),
                                         10, 4, st) == 0
        torch.cuda.synchronize()
        for b, n in enumerate(lens.tolist()):
            if n == 0:
                assert tok[b] == -3 and (out[b] == -4).all()
                continue
            want = OD.sample(lg.cpu().numpy(), 11, n - 1, T)[b]
            assert tok[b] == want and out[b, n] == want
    assert _lib.device_error() == 0
