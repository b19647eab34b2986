"""The samplers on the GPU where the restatement's random bits are extreme."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import decode as OD  # noqa: E402
from nlearn_b200 import _lib  # noqa: E402

from test_sampler_cpu import ONES, V, ZEROS  # noqa: E402


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("pos,row,col", ONES + ZEROS)
def test_extreme_bits(cuda, pos, row, col):
    """All ones: a column of probability e^-60 is not drawn; the drawn token is
    the restatement's in both samplers."""
    B = row + 1
    lg = torch.zeros(B, V, device=cuda)
    lg[:, col] = -60.0 if (pos, row, col) in ONES else 60.0
    want = OD.sample(lg.cpu().numpy(), 0, pos, 1.0)
    assert (want[row] == col) == ((pos, row, col) in ZEROS)
    i32 = dict(device=cuda, dtype=torch.int32)
    tok, at, lens = torch.full((B,), -1, **i32), torch.tensor([pos], **i32), torch.full((B,), pos + 1, **i32)
    assert _lib.lib.nl_sample_tokens(lg.data_ptr(), V, V, 1.0, 0, at.data_ptr(), tok.data_ptr(), None, 0, B,
                                     stream()) == 0
    assert tok.tolist() == want.tolist()
    tok.fill_(-1)
    assert _lib.lib.nl_sample_tokens_rows(lg.data_ptr(), V, V, 1.0, 0, lens.data_ptr(), tok.data_ptr(), None, 0, B,
                                          stream()) == 0
    assert tok.tolist() == want.tolist()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("T", [0.0, 0.7])
def test_rows_of_nan(cuda, T):
    """A row of NaN draws a token of the vocabulary and is reported; -inf and NaN
    beside numbers are not drawn; a row of -inf draws its first column."""
    V, nan, inf = 700, float("nan"), float("inf")
    lg = torch.randn(5, V, device=cuda)
    lg[1] = nan
    lg[2, :650], lg[2, 660:] = nan, -inf
    lg[3] = -inf
    i32 = dict(device=cuda, dtype=torch.int32)
    pos, lens = torch.tensor([4], **i32), torch.full((5,), 5, **i32)
    assert _lib.device_error() == 0
    for rows in (False, True):
        tok, out = torch.full((5,), -1, **i32), torch.full((5, 9), -1, **i32)
        fn = _lib.lib.nl_sample_tokens_rows if rows else _lib.lib.nl_sample_tokens
        assert fn(lg.data_ptr(), V, V, T, 3, (lens if rows else pos).data_ptr(), tok.data_ptr(), out.data_ptr(), 9, 5,
                  stream()) == 0
        t = tok.tolist()
        assert t[1] == 0 and 650 <= t[2] < 660 and t[3] == 0 and out[:, 5].tolist() == t
        want = OD.sample(lg.cpu().numpy(), 3, 4, T)
        assert (t[0], t[4]) == (want[0], want[4])
        assert _lib.device_error() == 5
    lg[1] = 0.0
    assert _lib.lib.nl_sample_tokens(lg.data_ptr(), V, V, T, 3, pos.data_ptr(), tok.data_ptr(), None, 0, 5, stream()) == 0
    assert _lib.device_error() == 0
