"""Sampled verification at the borders of its decisions: random numbers a few 1e-13 to each side of one, at logits far apart, and what is
left after refusals that took nearly all probability; against the float64 walk (oracle/draft.py)."""
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


@pytest.mark.parametrize("chunked", [False, True])
def test_what_is_left_after_refusals_of_nearly_everything(D, chunked):   # noqa: F811
    """Two refused tokens leave 2^-46 of the probability, half of it on a third: that one is decided by the rest's own sum, and so
    is the token after it.  (A random number of 1 - 2^-24 refuses what leaves more than 2^-24.)"""
    V = 9000
    most = 0.99999994
    for seed in range(16):
        rng = np.random.default_rng(seed)
        at = rng.choice(V, 400, replace=False) if chunked else rng.choice(4000, 400, replace=False)
        logits = np.full((5, V), -np.inf, np.float32)
        small = np.exp(0.5 * rng.normal(size=397))
        row = np.concatenate([np.log(2) * np.array([0.0, -22.5, -45.0]), np.log(small / small.sum()) - 45 * np.log(2)]).astype(np.float32)
        logits[0, at] = row
        logits[1:, 5] = 0.0
        e = np.exp(row.astype(np.float64))
        border = e[2] / e[2:].sum()
        tokens, parents = [0, at[0], at[1], at[0], at[2]], [-1, 0, 0, 0, 0]   # (one of them a second time)
        for side in (-1e-6, 1e-6):
            u = [float(rng.random()), most, most, most, np.float32(border * (1 + side))]
            want = O.verify(logits, tokens, parents, 1.0, u)
            assert want[0] == ([0, 4] if side < 0 else [0])
            assert run(D, logits, tokens, parents, torch.float32, 1.0, u) == want, (seed, side)


@pytest.mark.parametrize("V", [40, 4096, 9000])
def test_rows_without_a_finite_logit_and_drafted_tokens(D, V):   # noqa: F811
    """Rows all -inf or NaN (every token counts alike) and rows with infinities, with children on some of their tokens."""
    rng = np.random.default_rng(V)
    for fill in (-np.inf, np.nan, 0.0):
        for k in range(8):
            logits = np.full((5, V), fill, np.float32)
            if fill == 0.0:
                logits[:, rng.choice(V, 7, replace=False)] = np.inf
            kids = rng.choice(V, 4, replace=False) if fill != 0.0 else rng.choice(np.nonzero(np.isinf(logits[0]))[0], 4, replace=False)
            u = rng.random(5).astype(np.float32)
            if k % 2:
                u[1:] = 0.99999994
            tokens, parents = [0, *kids], [-1, 0, 0, 0, 0]
            assert run(D, logits, tokens, parents, torch.float32, 0.7, u) == O.verify(logits, tokens, parents, 0.7, u)


@pytest.mark.parametrize("drawn", [False, True])
def test_random_numbers_beside_a_second_sibling_s_border(D, drawn):   # noqa: F811
    """After a refusal: the residual's share of the second child, where it holds 1.1 times the draft's at least (a digit of cancellation)."""
    V, temperature, rng, found = 24, 0.7, np.random.default_rng(3), 0
    logits = (3 * rng.normal(size=(300000, V))).astype(np.float32)
    q = np.maximum(rng.dirichlet(np.ones(V), 300000), 1e-9).astype(np.float32)
    p = logits.astype(np.float64) / temperature
    p = np.exp(p - p.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    if drawn:
        r = np.maximum(p - q, 0)
        r /= r.sum(1, keepdims=True)
        border = r[:, 1] / q[:, 1]
        fits = (q[:, 0] * 0.99 > p[:, 0]) & (p[:, 1] > 1.1 * q[:, 1]) & (border < 0.99)
    else:
        border = p[:, 1] / p[:, 1:].sum(1)
        fits = (p[:, 0] < 0.99) & (border < 0.99)
    u = border.astype(np.float32)
    off = np.abs(u / np.maximum(border, 1e-300) - 1)
    for i in np.nonzero(fits & (off > 3e-13) & (off < (1e-10 if drawn else 2e-11)))[0][:12]:
        rows, us, qs = np.repeat(logits[i:i + 1], 3, 0), [0.3, 0.99999994, u[i]], np.repeat(q[i:i + 1], 3, 0) if drawn else None
        got = run(D, rows, [0, 0, 1], [-1, 0, 0], torch.float32, temperature, us, qs, 2)
        assert (got[0] == [0, 2]) == (u[i] < border[i])
        assert got == O.verify(rows, [0, 0, 1], [-1, 0, 0], temperature, us, qs, 2)
        found += 1
    assert found >= 4
