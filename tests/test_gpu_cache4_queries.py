"""Queries that the append to a 4-bit cache returns: float64 rounded once to bf16 (oracle/draft.py)."""
import numpy as np
import pytest
import torch

from oracle import draft as O
from tests.test_gpu_cache4 import BF, C, f64, gen, make_cache   # noqa: F401

pytestmark = pytest.mark.gpu


def nearest_bf16(v):
    """float64 to the nearest bf16 number, ties to even, and how far each is from a tie of two (of its size)."""
    m, e = np.frexp(v)
    m = m * 2.0 ** 8
    return np.ldexp(np.rint(m), e - 8), np.abs(np.abs(m - np.floor(m)) - 0.5) * 2.0 ** -8


def test_queries_are_rounded_once(C):   # noqa: F811
    """Millions of queries, of which some dozens lie so near the middle of two bf16 numbers that float32 is on it."""
    L, hq, hk, d, eps = 4096, 16, 1, 128, 2.0 ** -20
    rnd = gen(8)
    y = rnd(L, (hq + 2 * hk) * d).to(BF)
    qn = (1 + 0.1 * rnd(d)).to(BF)
    inv = 1.0 / (1e6 ** (torch.arange(d // 2, device="cuda", dtype=torch.float32) / (d // 2)))
    c = make_cache(rnd, hk, L, d)
    q = C.cache_write(y, qn, qn, eps, L, hq, hk, d, c[0], c[1], 0, inv, c[2], c[3])
    ref, _, _, mag = O.normed_rows(f64(y), f64(qn), f64(qn), eps, hq, hk, d, np.arange(L), f64(inv))
    want, off = nearest_bf16(ref)
    # angles of 4096 in float64: 2^-41; an element that far from a tie may go either way
    sure = off * np.abs(ref) > 2.0 ** -40 * mag[:, :hq]
    assert sure.mean() > 0.9999 and ((off < 2.0 ** -25) & sure).sum() > 20
    assert (f64(q).transpose(1, 0, 2) == want)[sure].all()


def test_queries_of_every_size(C):   # noqa: F811
    """Zeros, subnormal and overflowing queries, NaN: as one rounding of float64 gives them."""
    d, sizes = 64, [0.0, 1e-44, 3e-41, 1e-39, 1e-38, 1.0, 3e38]
    y = torch.ones(1, 3 * d, device="cuda", dtype=BF)
    y[0, 1:d:2] = -1.0
    qn = torch.ones(d, dtype=BF)
    qn[:len(sizes)] = torch.tensor(sizes).to(BF)
    one, inv = torch.ones(d, device="cuda", dtype=BF), torch.zeros(d // 2, device="cuda")
    c = make_cache(gen(1), 1, 4, d)
    for scale in (1.0, 1.0078125, 0.00390625):
        gain = (qn.double() * scale).to(BF).cuda()
        q = C.cache_write(y, gain, one, 0.0, 1, 1, 1, d, c[0], c[1], 0, inv, c[2], c[3])
        assert np.array_equal(f64(q)[0, 0], f64(y)[0, :d] * f64(gain))
    q = C.cache_write(y * 3, one, one, 6.0, 1, 1, 1, d, c[0], c[1], 0, inv, c[2], c[3])
    assert np.array_equal(f64(q)[0, 0], f64(y)[0, :d] * nearest_bf16(np.array(3 / 15 ** 0.5))[0])
    y[0, 5] = float("nan")
    assert torch.isnan(C.cache_write(y, one, one, 0.0, 1, 1, 1, d, c[0], c[1], 0, inv, c[2], c[3])).all()
