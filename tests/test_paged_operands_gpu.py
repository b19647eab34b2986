"""Operands of the paged operators that share memory: what is written is
refused where its elements coincide, what is only read is taken as it is, and
`out` may be `q` itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from nlearn_b200 import _lib  # noqa: E402
from nlearn_b200.paged import paged_decode_attention, paged_kv_write  # noqa: E402

from test_paged_gpu import E4M3, make_case  # noqa: E402


def test_written_rows_that_overlap(cuda):
    q, k, v, table, ln = make_case(cuda, [10, 20, 33], 4, 2, 64, 16)
    want, lse = torch.empty_like(q), torch.empty(3, 4, device=cuda)
    paged_decode_attention(q, k, v, table, ln, out=want, lse=lse)
    flat = torch.zeros(4096, device=cuda, dtype=torch.bfloat16)
    for strides in ((0, 64, 1), (256, 0, 1), (256, 32, 1), (64, 128, 1)):
        with pytest.raises(ValueError):
            paged_decode_attention(q, k, v, table, ln, out=flat.as_strided((3, 4, 64), strides))
    for strides in ((0, 1), (3, 1)):
        with pytest.raises(ValueError):
            paged_decode_attention(q, k, v, table, ln, lse=torch.zeros(99, device=cuda).as_strided((3, 4), strides))
    assert int(torch.count_nonzero(flat)) == 0
    # rows in any order, with room between them
    for strides in ((256, 64, 1), (64, 192, 1), (300, 65, 1), (70, 211, 1)):
        out, l2 = flat.as_strided((3, 4, 64), strides), torch.zeros(99, device=cuda).as_strided((3, 4), (7, 1))
        paged_decode_attention(q, k, v, table, ln, out=out, lse=l2)
        assert torch.equal(out, want) and torch.equal(l2, lse)
    one = paged_decode_attention(q[:1], k, v, table[:1], ln[:1], out=flat.as_strided((1, 4, 64), (0, 64, 1)))
    assert torch.equal(one, want[:1]) and _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_caches_that_share_slots(cuda, dtype):
    """Heads or pages that are one memory, keys and values that are one array: read, not written."""
    q, k, v, table, ln = make_case(cuda, [10, 20, 33], 4, 1, 64, 16, dtype=dtype, poison=False)
    new = torch.randn(3, 1, 64, device=cuda).bfloat16()
    slots = torch.tensor([1, 2, 3], device=cuda, dtype=torch.int32)
    K, V = (x.expand(-1, 2, -1, -1) for x in (k, v))
    assert torch.equal(paged_decode_attention(q, K, V, table, ln), paged_decode_attention(q, k, v, table, ln))
    paged_decode_attention(q, k, k, table, ln)
    before = k.clone()
    two = new.expand(3, 2, 64)
    for kk, vv, x in ((K, V, two), (k, k, new), (K, K, two)):
        with pytest.raises(ValueError):
            paged_decode_attention(q, kk, vv, table, ln, x, x)
        with pytest.raises(ValueError):
            paged_kv_write(x, x, kk, vv, slots)
    torch.cuda.synchronize()
    assert torch.equal(k.view(torch.uint8), before.view(torch.uint8))
    # halves of one array
    both = torch.stack((k.float(), v.float()), 1).to(dtype)
    assert torch.equal(paged_decode_attention(q, both[:, 0], both[:, 1], table, ln, new, new),
                       paged_decode_attention(q, k, v, table, ln, new, new))
    paged_kv_write(new, new, both[:, 0], both[:, 1], slots)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("hq,hk,d,lens", [(8, 8, 64, [100, 0, 7, 512]), (32, 2, 128, [1, 90, 3000]),
                                          (40, 1, 128, [5000, 33]), (8, 8, 64, [9000, 1, 0, 260]),
                                          (24, 8, 128, list(range(0, 400)))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_out_may_be_q(cuda, hq, hk, d, lens, dtype):
    """Clustered, by keys, by heads and split over CTAs, with the new token beside q in one projection."""
    q, k, v, table, ln = make_case(cuda, lens, hq, hk, d, 16, dtype=dtype, seed=d, poison=False)
    B = len(lens)
    qkv = torch.randn(B, (hq + 2 * hk) * d, device=cuda).bfloat16()
    kn, vn = qkv[:, hq * d:(hq + hk) * d].view(B, hk, d), qkv[:, (hq + hk) * d:].view(B, hk, d)
    q = qkv[:, :hq * d].view(B, hq, d)
    want = paged_decode_attention(q, k, v, table, ln, kn, vn, scale=0.02)
    keep = qkv[:, hq * d:].clone()
    assert paged_decode_attention(q, k, v, table, ln, kn, vn, scale=0.02, out=q) is q
    torch.cuda.synchronize()
    assert torch.equal(q, want) and torch.equal(qkv[:, hq * d:], keep) and _lib.device_error() == 0
