"""Decode attention at the accuracy of f32 probabilities, where nothing else is
rounded: small scores that are exact in f32, and values of both signs whose
weighted sum nearly cancels, so that an error of a probability is not hidden by
the rounding of the bf16 output.

Tolerance: half a bf16 step of the value, 2^-8 |o|, and e sum p|v| / sum p with
e the errors of p and of the sums.  A score q.k is a sum of two products that f32 holds
exactly; times scale * log2(e) (two half steps, |y| <= 4) it is off by
2^-21, exp2 by 2^-22, a p of two bf16 terms by 2^-16 (of two f16 terms by less),
and the sums over up to 320 keys take at most 32 additions a thread and 8 over
the warps, each off by half an f32 step: 2^-18.  e = 2^-15 holds their sum."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import paged as OP  # noqa: E402
from nlearn_b200 import _lib  # noqa: E402
from nlearn_b200.paged import paged_decode_attention  # noqa: E402

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("hq,hk,d", [(8, 8, 64), (8, 2, 128), (16, 1, 64), (4, 4, 128)])
def test_probabilities_keep_their_bits(cuda, dtype, hq, hk, d):
    """Keys in pairs whose scores differ in the tenth bit, values +c and -c:
    o = sum of c (p - p') / sum p is a thousandth of the values."""
    rng = np.random.default_rng(d + hq)
    lens, page = [2, 16, 64, 130, 320], 16
    blocks = 20
    B = len(lens)
    n = blocks * page
    k = torch.zeros(B, blocks, hk, page, d)
    a = torch.from_numpy(rng.integers(-16, 17, (B, hk, n // 2)) / 8.0).float().repeat_interleave(2, -1)
    b = torch.from_numpy(rng.integers(-8, 9, (B, hk, n)) / 4.0).float()
    c = torch.from_numpy(rng.choice([-1.0, -0.5, 0.5, 1.0], (B, hk, n // 2, d))).float()
    v = torch.stack((c, -c), 3).reshape(B, hk, n, d)
    to_pages = lambda x: x.view(B, hk, blocks, page, -1).transpose(1, 2)  # noqa: E731
    k[..., :1], k[..., 1:2] = to_pages(a), to_pages(b)
    k = k.view(B * blocks, hk, page, d).to(dtype).to(cuda)
    v = to_pages(v).reshape(B * blocks, hk, page, d).to(dtype).to(cuda)
    q = torch.zeros(B, hq, d)
    q[..., 0] = torch.from_numpy(rng.choice([-1.0, 0.5, 0.75, 1.0], (B, hq)))
    q[..., 1] = 2.0**-10
    q = q.bfloat16().to(cuda)
    table = torch.arange(B * blocks, dtype=torch.int32, device=cuda).view(B, blocks)
    ln = torch.tensor(lens, dtype=torch.int32, device=cuda)
    o = paged_decode_attention(q, k, v, table, ln, scale=1.0)
    torch.cuda.synchronize()
    f = lambda t: t.float().double().cpu().numpy()  # noqa: E731
    ref, _, w = OP.paged_attention(f(q), f(k), f(v), table.cpu().numpy(), lens, 1.0)
    err = np.abs(f(o) - ref)
    tol = 2.0**-8 * np.abs(ref) + 2.0**-15 * w
    assert (err <= tol).all(), (err / tol).max()
    assert _lib.device_error() == 0
