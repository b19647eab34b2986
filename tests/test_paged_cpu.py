"""Refusals of the paged serving entry points, before anything is launched:
the C entries' status codes on arguments they must not take (no GPU needed;
the pointers are never read), CPU tensors at the Python entries, and the
NumPy restatements against hand-made cases."""
import struct

import numpy as np
import pytest
import torch

from nlearn_b200._lib import STATUS, lib
from oracle import paged as OP

# the argument structs of include/nl_ops.h (P pointer, q long long, N size_t, i int, f float)
ARGS = {"nl_paged_attention": struct.Struct("@12P11qN8if4x"), "nl_paged_kv_write": struct.Struct("@7P5q6i"),
        "nl_update_block_tables": struct.Struct("@12Pq5i4x"), "nl_process_logits": struct.Struct("@12P5q6i")}
P = 1 << 20  # an aligned non-null address that no refused call reads


def call(name, defaults, kw):
    """The status of a C entry point whose argument struct holds `defaults` changed by `kw`."""
    assert set(kw) <= set(defaults)
    return STATUS[getattr(lib, name)(ARGS[name].pack(*{**defaults, **kw}.values()), None)]


def attention(**kw):
    return call("nl_paged_attention",
                dict(q=P, k=P, v=P, table=P, lens=P, kn=0, vn=0, ks=0, vs=0, o=P, lse=0, ws=P, q_b=512, q_h=64,
                     page_s=1024, head_s=8192, tok_s=64, table_ld=4, n_b=0, n_h=0, o_b=512, o_h=64, lse_b=0, nb=0,
                     B=2, Hq=8, Hk=8, d=64, page=16, blocks=4, n_pages=10, dt=1, scale=1.0), kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(Hq=7), dict(Hk=0), dict(d=80), dict(page=0), dict(blocks=0),
                                dict(n_pages=0), dict(table_ld=3), dict(q=0), dict(lens=0), dict(o=0), dict(kn=P),
                                dict(vn=P), dict(page_s=0), dict(tok_s=-64), dict(blocks=2**27),
                                dict(B=2**24, blocks=2**20)])
def test_attention_shapes(kw):
    assert attention(**kw) == "NL_ERR_SHAPE"


@pytest.mark.parametrize("kw,code", [(dict(dt=0), "NL_ERR_DTYPE"), (dict(dt=7), "NL_ERR_DTYPE"),
                                     (dict(q=P + 8), "NL_ERR_ALIGN"), (dict(tok_s=68), "NL_ERR_ALIGN"),
                                     (dict(dt=2, tok_s=72), "NL_ERR_ALIGN"), (dict(q_h=60), "NL_ERR_ALIGN"),
                                     (dict(kn=P + 2, vn=P), "NL_ERR_ALIGN"), (dict(ws=P + 16), "NL_ERR_ALIGN"),
                                     (dict(page_s=2**33), "NL_ERR_TOO_LARGE"),
                                     (dict(n_pages=2**27, page_s=1024), "NL_ERR_TOO_LARGE")])
def test_attention_types_alignment_size(kw, code):
    assert attention(**kw) == code


def test_attention_workspace_of_refused_shapes():
    for args in ((0, 8, 8, 64, 16, 4, 1), (1, 8, 3, 64, 16, 4, 1), (1, 8, 8, 96, 16, 4, 1), (1, 8, 8, 64, 0, 4, 1)):
        assert lib.nl_paged_attention_workspace_bytes(*args) == 0


def write(**kw):
    return call("nl_paged_kv_write",
                dict(k=P, v=P, kc=P, vc=P, slots=P, ks=0, vs=0, n_t=512, n_h=64, page_s=1024, head_s=8192, tok_s=64,
                     T=3, Hk=8, d=64, page=16, n_pages=10, dt=1), kw)


@pytest.mark.parametrize("kw,code", [(dict(T=0), "NL_ERR_SHAPE"), (dict(d=60), "NL_ERR_SHAPE"),
                                     (dict(dt=2, d=72), "NL_ERR_SHAPE"), (dict(slots=0), "NL_ERR_SHAPE"),
                                     (dict(dt=0), "NL_ERR_DTYPE"), (dict(k=P + 4), "NL_ERR_ALIGN"),
                                     (dict(n_t=500), "NL_ERR_ALIGN"), (dict(page_s=1020), "NL_ERR_ALIGN")])
def test_write_refusals(kw, code):
    assert write(**kw) == code


def tables(**kw):
    return call("nl_update_block_tables",
                dict(table=P, lens=P, new=P, done=0, free=P, n_free=P, lens_out=P, n_free_out=P, slots=P, pos=P,
                     cu=P, status=P, ld=4, B=2, blocks=4, page=16, n_pages=10, n_tokens=5), kw)


@pytest.mark.parametrize("kw", [dict(B=0), dict(B=8193), dict(blocks=0), dict(page=0), dict(n_pages=0),
                                dict(n_tokens=-1), dict(ld=3), dict(blocks=2**30, ld=2**30), dict(n_pages=2**28),
                                dict(lens=0), dict(cu=0), dict(slots=0)])
def test_table_refusals(kw):
    assert tables(**kw) == "NL_ERR_SHAPE"


def logits(**kw):
    return call("nl_process_logits",
                dict(x=P, y=P, tok=0, lens=0, pl=0, rep=0, fr=0, pr=0, ids=0, bias=0, mask=0, mrows=0, ldx=100,
                     ldy=100, ldt=0, ldb=0, ldm=0, dt=0, L=0, n_bias=0, n_masks=0, B=2, V=100), kw)


@pytest.mark.parametrize("kw,code", [(dict(B=0), "NL_ERR_SHAPE"), (dict(B=65536), "NL_ERR_SHAPE"),
                                     (dict(ldx=99), "NL_ERR_SHAPE"), (dict(ldy=99), "NL_ERR_SHAPE"),
                                     (dict(V=2**30, ldx=2**31, ldy=2**31), "NL_ERR_TOO_LARGE"),
                                     (dict(tok=P, lens=P, ldt=2**31, L=2**30), "NL_ERR_TOO_LARGE"),
                                     (dict(ids=P, bias=P, ldb=2**31, n_bias=2**30), "NL_ERR_TOO_LARGE"),
                                     (dict(dt=2), "NL_ERR_DTYPE"), (dict(tok=P, ldt=5, L=5), "NL_ERR_SHAPE"),
                                     (dict(tok=P, lens=P, ldt=4, L=5), "NL_ERR_SHAPE"),
                                     (dict(n_bias=3), "NL_ERR_SHAPE"), (dict(n_bias=-1), "NL_ERR_SHAPE"),
                                     (dict(mask=P, ldm=3, n_masks=2), "NL_ERR_SHAPE"),
                                     (dict(mask=P, ldm=4, n_masks=1), "NL_ERR_SHAPE")])
def test_logits_refusals(kw, code):
    assert logits(**kw) == code


@pytest.mark.parametrize("name", sorted(ARGS))
def test_no_arguments(name):
    assert STATUS[getattr(lib, name)(None, None)] == "NL_ERR_SHAPE"


def test_cpu_tensors_raise():
    from nlearn_b200.kernels.logits import process_logits
    from nlearn_b200.paged import paged_decode_attention, paged_kv_write, update_block_tables
    i = torch.zeros(2, dtype=torch.int32)
    q, c = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 4, 16, 64, dtype=torch.bfloat16)
    for fn, args in ((paged_decode_attention, (q, c, c, i[:, None], i)), (paged_kv_write, (q, q, c, c, i)),
                     (update_block_tables, (i[:, None], i, i, i, i[:1], 16, 2)), (process_logits, (torch.zeros(2, 5),))):
        with pytest.raises(ValueError):
            fn(*args)


def test_restated_tables_by_hand():
    # page size 4, three rows: row 0 grows into a second page, row 1 ends and starts again, row 2 has room
    r = OP.update_tables([[7, -1], [3, 5], [2, -1]], [4, 6, 1], [1, 2, 1], [0, 1, 0], [9, 8, 0, 0, 0, 0, 0, 0, 0, 0],
                         2, 4, 6)
    assert r["free"][:4] == [9, 8, 3, 5]                     # row 1's pages on top
    assert r["table"] == [[7, 5], [3, 5], [2, -1]]           # row 0 takes 5, row 1 then 3
    assert r["lens"] == [5, 2, 2] and r["n_free"] == 2 and r["status"] == [0, 0, 0]
    assert r["cu"] == [0, 1, 3, 4]
    assert r["slots"] == [20, 12, 13, 9, -1, -1] and r["positions"] == [4, 0, 1, 1, -1, -1]
    # too few pages: row 0 is served, row 1 and the later rows that need pages are not
    r = OP.update_tables([[-1, -1]] * 4, [0, 0, 0, 0], [3, 5, 1, 0], [0] * 4, [6, 4], 2, 4, 20)
    assert r["status"] == [0, 1, 1, 0] and r["lens"] == [3, 0, 0, 0] and r["n_free"] == 1


def test_restated_logits_by_hand():
    x = np.array([[2.0, -2.0, 1.0, 0.5]])
    y = OP.process_logits(x, tokens=np.array([[0, 1, 1, 9]]), lens=[4], prompt_lens=[1], repetition=[2.0],
                          frequency=[0.25], presence=[1.0], bias_ids=np.array([[2, 2, -1]]),
                          bias=np.array([[1.0, 0.5, 9.0]]), mask=np.array([[0b0111]]))
    assert y.tolist() == [[1.0, -5.5, 2.5, -np.inf]]


def test_restated_attention_by_hand():
    k = np.zeros((2, 1, 2, 2))
    v = np.arange(8.0).reshape(2, 1, 2, 2)
    o, lse, _ = OP.paged_attention(np.ones((1, 1, 2)), k, v, np.array([[1, 0]]), [3], 1.0)
    assert np.allclose(o[0, 0], (v[1, 0, 0] + v[1, 0, 1] + v[0, 0, 0]) / 3) and np.isclose(lse[0, 0], np.log(3))
