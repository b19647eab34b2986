"""PagedDecoder when rows are used again: random bits, iterators, errors on the way."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import decode as OD  # noqa: E402
from nlearn_b200 import _lib  # noqa: E402
from nlearn_b200.generate import Decoder, PagedDecoder, generate  # noqa: E402
from nlearn_b200.model import FlatParams  # noqa: E402

from test_paged_decode_gpu import CFG, check_row, oracle, prompts  # noqa: E402


@pytest.fixture(scope="module")
def params(cuda):
    return FlatParams(CFG, cuda, seed=3)     # (flat logits: draws are all but uniform)


def test_prompts_of_one_row_draw_independently(cuda, params):
    """One prompt many times through fewer rows: every completion its own, each the
    oracle's choice under the random bits of its number."""
    p = prompts([7])[0]
    out = PagedDecoder(params, CFG, max_batch=1, seed=4).generate([p] * 5, 12)
    assert len({tuple(t[7:]) for t in out}) == 5
    model = oracle(params)
    for number, toks in enumerate(out):
        check_row(model, toks, 7, number, 4, 1.0)
    # another number of rows: the same draws (the logits' rounding may move a close one)
    for number, toks in enumerate(PagedDecoder(params, CFG, max_batch=3, seed=4).generate([p] * 5, 12)):
        check_row(model, toks, 7, number, 4, 1.0)
    # many more prompts than rows through the entry point
    many = generate(params, [p] * 35 + [p[:3]], 12, seed=4)
    assert len({tuple(t[-12:]) for t in many}) == 36


def test_a_second_run_draws_anew_and_a_new_decoder_repeats(cuda, params):
    p = prompts([5, 9], 1)
    dec = PagedDecoder(params, CFG, max_batch=2, seed=1)
    first, second = dec.generate(p, 10), dec.generate(p, 10)
    assert dec.next_request == 4
    assert all(not np.array_equal(a, b) for a, b in zip(first, second))
    dec.next_request = 0                      # the numbers decide, not the history
    for got in (dec.generate(p, 10), PagedDecoder(params, CFG, max_batch=2, seed=1).generate(p, 10)):
        for a, b in zip(first, got):
            np.testing.assert_array_equal(a, b)


def test_numbers_past_31_bits(cuda, params):
    p = prompts([4])[0]
    dec = PagedDecoder(params, CFG, max_batch=1, seed=2)
    dec.next_request = 2**32 - 1
    a, b = dec.generate([p, p], 6)            # numbers 2^32 - 1 and (wrapped) 0
    model = oracle(params)
    check_row(model, a, 4, 2**32 - 1, 2, 1.0)
    check_row(model, b, 4, 0, 2, 1.0)


def test_sampler_by_requests(cuda):
    V, lib = 1000, _lib.lib
    st = torch.cuda.current_stream().cuda_stream
    i32 = dict(device=cuda, dtype=torch.int32)
    lg = torch.randn(4, V, device=cuda) * 2
    lens, req = torch.tensor([5, 0, 9, 1], **i32), torch.tensor([70000, 3, -1, 0], **i32)
    tok, out = torch.full((4,), -3, **i32), torch.full((4, 10), -4, **i32)
    assert lib.nl_sample_tokens_requests(lg.data_ptr(), V, V, 0.8, 11, lens.data_ptr(), req.data_ptr(), tok.data_ptr(),
                                         out.data_ptr(), 10, 4, st) == 0
    torch.cuda.synchronize()
    for b, (n, r) in enumerate(zip(lens.tolist(), req.tolist())):
        if n == 0:
            assert tok[b] == -3 and (out[b] == -4).all()
            continue
        g = -np.log(-np.log(OD.uniforms(11, n - 1, r & 0xFFFFFFFF, V).astype(np.float64)))
        want = int(np.argmax(lg[b].cpu().numpy().astype(np.float64) / 0.8 + g))
        assert tok[b] == want and out[b, n] == want
    assert _lib.device_error() == 0


def test_release_takes_any_iterable(cuda, params):
    dec = PagedDecoder(params, CFG, max_batch=3, temperature=0.0)
    rows = dec.add(prompts([20, 3, 40]))
    dec.step(2)
    dec.release(r for r in rows[:2])
    assert dec.free_rows() == rows[:2] and dec.new.tolist() == [0, 0, 1]
    assert dec.free_page_count() == dec.n_free.item() == dec.n_pages - 3
    again = dec.add(prompts([5], 1))
    dec.step(3)
    alone = PagedDecoder(params, CFG, max_batch=3, temperature=0.0)
    alone.add(prompts([5], 1))
    alone.step(3)
    np.testing.assert_array_equal(dec.tokens(again[0]), alone.tokens(0))
    assert dec.tokens(rows[1]).size == 0 and _lib.device_error() == 0


def test_allowed_holds_for_every_admission(cuda, params):
    """An iterator of ids, and more prompts than rows."""
    ps = prompts([3, 30, 8, 1, 12], 2)
    out = PagedDecoder(params, CFG, max_batch=2).generate(ps, 5, allowed=(i for i in range(50, 53)))
    assert all(50 <= t < 53 for p, toks in zip(ps, out) for t in toks[p.size:])
    many = generate(params, [ps[0]] * 33 + [ps[1]], 2, allowed=iter([9]))
    assert all((t[-2:] == 9).all() for t in many)


def fail_at(monkeypatch, call):
    """The call-th product of the decoder's layers raises on the host."""
    from nlearn_b200 import generate as G
    count, real = [0], G.gemm_ex

    def gemm(*args, **kw):
        count[0] += 1
        if count[0] == call:
            raise MemoryError("planted")
        return real(*args, **kw)
    monkeypatch.setattr(G, "gemm_ex", gemm)


def fail():
    raise MemoryError("planted")


def same_books(dec):
    """The host's count of rows and pages is the device's."""
    torch.cuda.synchronize()
    assert dec.lens.tolist() == [max(0, n - 1) for n in dec._len]
    assert dec.new.tolist() == [int(n > 0) for n in dec._len]
    assert dec.n_free.item() == dec.free_page_count()
    held = [p for r, n in enumerate(dec.lens.tolist()) for p in dec.block_table[r, :dec._pages(n)].tolist()]
    assert sorted(held + dec.free_pages[:dec.n_free.item()].tolist()) == list(range(dec.n_pages))


@pytest.mark.parametrize("call", [1, 3, 6])
def test_an_admission_that_fails_leaves_no_rows(cuda, params, monkeypatch, call):
    ps = prompts([20, 3, 40], 5)
    dec = PagedDecoder(params, CFG, max_batch=3, n_pages=12, seed=8)
    kept, = dec.add(ps[:1])
    with monkeypatch.context() as m:
        fail_at(m, call)
        with pytest.raises(MemoryError):
            dec.add(ps[1:])
    assert dec.free_rows() == [1, 2] and dec.next_request == 1
    same_books(dec)
    dec.add(ps[1:])
    dec.step(3)
    want = PagedDecoder(params, CFG, max_batch=3, n_pages=12, seed=8)
    want.add(ps[:1])
    want.add(ps[1:])
    want.step(3)
    for r in range(3):
        np.testing.assert_array_equal(dec.tokens(r), want.tokens(r))
    same_books(dec)
    assert _lib.device_error() == 0


def test_a_capture_that_fails_is_made_again(cuda, params, monkeypatch):
    ps = prompts([20, 3], 6)
    dec = PagedDecoder(params, CFG, max_batch=2, seed=8)
    dec.add(ps)
    dec.step()
    with monkeypatch.context() as m:
        fail_at(m, 2)
        with pytest.raises(MemoryError):
            dec.step()
    same_books(dec)
    dec.step(3)
    want = PagedDecoder(params, CFG, max_batch=2, seed=8)
    want.add(ps)
    want.step(4, use_graph=False)
    for r in range(2):
        np.testing.assert_array_equal(dec.tokens(r), want.tokens(r))
    same_books(dec)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("call", [1, 4, "drawn"])
@pytest.mark.parametrize("use_graph", [True, False])
def test_a_step_that_fails_is_taken_back(cuda, params, monkeypatch, call, use_graph):
    """Rows on the edge of a page among them: the page is taken once."""
    ps = prompts([16, 3, 15, 32], 7)
    dec = PagedDecoder(params, CFG, max_batch=4, seed=8)
    dec.add(ps)
    for _ in range(2):
        with monkeypatch.context() as m:
            if call == "drawn":               # (stopped by hand when the step is already on its way)
                real = dec._step
                m.setattr(dec, "_step", lambda rules: (real(rules), fail()))
            else:
                fail_at(m, call)
            with pytest.raises(MemoryError):
                dec.step(use_graph=use_graph)
        same_books(dec)
    dec.step(4, use_graph=use_graph)
    want = PagedDecoder(params, CFG, max_batch=4, seed=8)
    want.add(ps)
    want.step(4, use_graph=False)
    for r in range(4):
        np.testing.assert_array_equal(dec.tokens(r), want.tokens(r))
    same_books(dec)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("call", [2, 20, 60])
def test_a_generation_that_fails_leaves_no_rows(cuda, params, monkeypatch, call):
    ps = prompts([20, 3, 40, 7], 9)
    dec = PagedDecoder(params, CFG, max_batch=2, temperature=0.0)
    with monkeypatch.context() as m:
        fail_at(m, call)
        with pytest.raises(MemoryError):
            dec.generate(ps, 8, use_graph=False)
    assert dec.free_rows() == [0, 1] and dec.n_free.item() == dec.n_pages
    same_books(dec)
    for a, b in zip(dec.generate(ps, 8), PagedDecoder(params, CFG, max_batch=2, temperature=0.0).generate(ps, 8)):
        np.testing.assert_array_equal(a, b)
    assert _lib.device_error() == 0


def test_graphs_of_many_seeds(cuda, params):
    """A graph for each (rules, seed, temperature), the last ones kept; seeds in
    turn use theirs again."""
    ps = prompts([5, 9], 10)
    dec = PagedDecoder(params, CFG, max_batch=2)
    for seed in range(dec.MAX_GRAPHS + 5):
        dec.seed = seed
        dec.generate(ps, 5)
        assert len(dec._graphs) <= dec.MAX_GRAPHS
    assert [k[1] for k in dec._graphs] == list(range(5, dec.MAX_GRAPHS + 5))
    kept = dict(dec._graphs)
    for seed in (10, 11, 10):
        dec.seed, dec.next_request = seed, 0
        out = dec.generate(ps, 5)
        want = PagedDecoder(params, CFG, max_batch=2, seed=seed).generate(ps, 5, use_graph=False)
        assert all(np.array_equal(a, b) for a, b in zip(out, want))
    assert all(dec._graphs[k] is g for k, g in kept.items())
    assert _lib.device_error() == 0


def test_entry_point_keeps_the_shape_of_its_prompts(cuda, params):
    ps = np.stack(prompts([9, 9, 9], 11))
    plain = generate(params, ps, 4, temperature=0.0)
    ruled = generate(params, ps, 4, temperature=0.0, repetition=1.0)     # a rule that changes nothing
    assert isinstance(plain, np.ndarray) and isinstance(ruled, np.ndarray)
    assert plain.shape == ruled.shape == (3, 13) and ruled.dtype == plain.dtype
    np.testing.assert_array_equal(ruled[:, :9], ps)
    by_list = generate(params, list(ps), 4, temperature=0.0, presence=0.5)
    assert isinstance(by_list, list) and [t.shape for t in by_list] == [(13,)] * 3
    each = generate(params, ps, [4, 1, 0], temperature=0.0)
    assert [t.shape for t in each] == [(13,), (10,), (9,)]
    assert generate(params, ps[0], 4, temperature=0.0, presence=0.5).shape == (13,)


@pytest.mark.parametrize("n", [1, 33, 300])
def test_entry_point_takes_any_number_of_biases(cuda, params, n):
    ids = np.random.default_rng(n).permutation(CFG.vocab)[:n]
    toks = generate(params, prompts([6])[0], 5, temperature=0.0, bias={int(i): 500.0 for i in ids})
    assert toks.shape == (11,) and np.isin(toks[6:], ids).all()


@pytest.mark.parametrize("row", [-1, -3, 1, 3])
def test_allowed_of_a_row_that_is_not_in_use(cuda, params, row):
    """A row counted from the end, a free one, one past the last: refused, and nothing changed."""
    dec = PagedDecoder(params, CFG, max_batch=3, temperature=0.0)
    used = dec.add(prompts([4, 5, 6], 3))
    dec.release(used[1:2])
    if row < 0:
        dec.add(prompts([5], 4))                    # (all rows in use: -1 would name the last)
    before, rules = dec.mask_rows.tolist(), list(dec._rules)
    with pytest.raises(ValueError):
        dec.set_allowed(row, [5])
    with pytest.raises(ValueError):
        dec.set_allowed(row, None)
    assert dec.mask_rows.tolist() == before and dec._rules == rules
    dec.set_allowed(0, [5])
    dec.step(2)
    assert (dec.tokens(0)[-2:] == 5).all()


def test_prompt_ids_outside_the_vocabulary(cuda, params):
    """Refused before anything is launched; 64-bit ids do not wrap."""
    dec, one = PagedDecoder(params, CFG, max_batch=2, temperature=0.0), Decoder(params, CFG, batch=1)
    for bad in (np.array([3, CFG.vocab]), np.array([-1, 3]), np.array([2**32 + 5]), [CFG.vocab]):
        with pytest.raises(ValueError):
            dec.add([np.array([1, 2]), bad])
        with pytest.raises(ValueError):
            dec.generate([np.array([1, 2]), bad], 3)
        with pytest.raises(ValueError):
            one.generate(bad, 3)
        with pytest.raises(ValueError):
            generate(params, bad, 3)
        with pytest.raises(ValueError):
            generate(params, [[1, 2, 3], bad], 3)
    assert dec.free_rows() == [0, 1] and dec.n_free.item() == dec.n_pages
    edge = [0, CFG.vocab - 1]
    a = generate(params, edge, 4, temperature=0.0)
    b, = dec.generate([torch.tensor(edge)], 4)
    assert a.dtype == b.dtype == np.int32 and a[:2].tolist() == b[:2].tolist() == edge
    assert generate(params, edge, 0).tolist() == edge and _lib.device_error() == 0


@pytest.mark.parametrize("n", [0, -3])
def test_a_cache_of_no_pages(cuda, params, n):
    with pytest.raises(ValueError):
        PagedDecoder(params, CFG, n_pages=n)
    assert PagedDecoder(params, CFG, max_batch=2, n_pages=1).n_pages == 1


def test_an_admission_without_block_tables(cuda, params, monkeypatch):
    """It fails before the device has given the rows any page."""
    from nlearn_b200 import generate as G
    dec = PagedDecoder(params, CFG, max_batch=3, n_pages=12, seed=8)
    kept, = dec.add(prompts([20], 5))
    real, calls = G.update_block_tables, []

    def tables(*args, **kw):
        calls.append(1)
        return fail() if len(calls) == 1 else real(*args, **kw)
    with monkeypatch.context() as m:
        m.setattr(G, "update_block_tables", tables)
        with pytest.raises(MemoryError):
            dec.add(prompts([3, 40], 6))
    assert dec.free_rows() == [1, 2] and len(calls) == 2
    same_books(dec)
    dec.add(prompts([3, 40], 6))
    dec.step(3)
    same_books(dec)
    assert _lib.device_error() == 0
