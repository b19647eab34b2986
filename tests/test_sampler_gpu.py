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
