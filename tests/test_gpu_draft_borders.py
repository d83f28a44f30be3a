"""Sampled verification at the borders of its decisions: random numbers a few 1e-13 to each side of one, at logits far apart,
against the float64 walk (oracle/draft.py)."""
import numpy as np
import pytest
import torch

from oracle import draft as O
from tests.test_gpu_draft import D, run   # noqa: F401

pytestmark = pytest.mark.gpu


def borders(temperature, factor, count):
    """(x, u): float32 logits x and random numbers u whose u is within 3e-13 .. 1e-11 of factor * e / (1 + e), e = exp(x / temperature)."""
    x = -np.arange(8.0, 22.0, 2.0 ** -17).astype(np.float32)[np.random.default_rng(1).permutation(14 * 2 ** 17)]
    e = np.exp(x.astype(np.float64) / temperature)
    p = factor * e / (1 + e)
    u = p.astype(np.float32)
    off = np.abs(u.astype(np.float64) / p - 1)
    at = np.nonzero((off > 3e-13) & (off < 1e-11))[0][:count]
    assert len(at) == count
    return [(x[i], u[i], bool(u[i] < p[i])) for i in at]


@pytest.mark.parametrize("temperature", [0.8, 0.37, 1.0])
@pytest.mark.parametrize("drawn", [False, True])
def test_random_numbers_beside_a_border_of_unlike_logits(D, temperature, drawn):   # noqa: F811
    """float64 arithmetic decides to some 1e-14: exponentials of numbers up to 60 to 1e-14, sums and products to 1e-16."""
    q = np.full((2, 4), 0.25, np.float32) if drawn else None
    below = 0
    for x, u, accept in borders(temperature, 4.0 if drawn else 1.0, 24):
        logits = np.full((2, 4), -np.inf, np.float32)
        logits[:, 0], logits[:, 2] = 0.0, x
        got = run(D, logits, [0, 2], [-1, 0], torch.float32, temperature, [0.0, u], q, 1)
        assert got == O.verify(logits, [0, 2], [-1, 0], temperature, [0.0, u], q, 1)
        assert (len(got[0]) == 2) == accept, (x, u)
        below += accept
    assert 0 < below < 24
