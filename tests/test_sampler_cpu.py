"""The sampler's random bits at their extremes (oracle/decode.py)."""
import numpy as np
import pytest

from oracle import decode as OD

# (pos, row, column) of seed 0 whose 24 random bits are all ones / all zeros, at the repository's vocabulary
ONES = [(91, 0, 41690), (19, 1, 27536), (21, 1, 26731), (240, 1, 29904)]
ZEROS = [(245, 0, 12334), (268, 0, 4045), (109, 1, 22758), (260, 2, 30395)]
V = 50257


@pytest.mark.parametrize("pos,row,col", ONES + ZEROS)
def test_extreme_bits_give_finite_noise(pos, row, col):
    u = OD.uniforms(0, pos, row, V)
    assert u[col] == (u.max() if (pos, row, col) in ONES else u.min())
    assert 0 < u.min() and u.max() < 1 and u.dtype == np.float32
    assert np.isfinite(-np.log(-np.log(u))).all()


@pytest.mark.parametrize("pos,row,col", ONES)
def test_an_unlikely_token_is_not_drawn(pos, row, col):
    lg = np.zeros((row + 1, V), np.float32)
    lg[:, col] = -60.0
    assert OD.sample(lg, 0, pos, 1.0)[row] != col
