"""Attention over an 8-bit cache whose value rows are zeros, tiny, or far apart in size: what a row without values does to the others, and
rows that hold nearly all probability, against the float64 restatement with a tolerance relative to the result."""
import numpy as np
import pytest
import torch

from oracle import draft as O
from tests.test_gpu_cache import bits, f64, gen, make_cache, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def C():
    from mxfp4_int8_m5_amd import sc_cache
    return sc_cache


def check_relative(out, q, c, masks, pos, scale):
    """As tests.test_gpu_cache.check_attention, without its term of the largest value: a weight (probability times scale) is a
    half-precision number with the largest between 2^8 and 2^14, so that one of less than 2^-14 is off by up to 2^-25, which is 2^-33 of
    the largest; a code is up to 127."""
    hk, _, d = c[0].shape
    T, hq = q.shape[1], q.shape[0]
    k, v, qs, vs = values(c[0], c[2]), values(c[1], c[3]), f64(q), f64(c[3])
    ref, mag = O.attention(qs.transpose(1, 0, 2), k, v, masks, pos, scale)
    got = f64(out).reshape(T, hq, d)
    low = np.zeros((T, hq, 1))
    for i in range(T):
        rows = np.array(list(range(pos)) + [pos + j for j in range(T) if masks[i] >> j & 1], int)
        for h in range(hq):
            g = h // (hq // hk)
            s = k[g, rows] @ qs[h, i] * scale
            p = np.exp(s - s.max())
            low[i, h] = 2.0 ** -33 * 127 * len(rows) * (p / p.sum() * vs[g, rows]).max()
    tol = 1.05 * (2.0 ** -11 * mag + 2.0 ** -8 * np.abs(ref)) + low
    assert (np.abs(got - ref) <= tol).all(), np.max(np.abs(got - ref) / np.maximum(tol, 1e-300))


def cache_of(rnd, hk, rows, d, size, lift, empty):
    """Values of about `size`; the rows of `empty` hold zeros, with scores `lift` powers of two above the others' for queries of ones."""
    c = make_cache(rnd, True, hk, rows, d)
    c[0][:] = 100
    score = torch.rand(hk, rows, device="cuda")
    score[:, empty] += lift * float(np.log(2))
    c[2][:] = score / (100 * d ** 0.5)
    c[3][:] = size / 127 * torch.exp2(torch.rand(hk, rows, device="cuda"))
    c[1][:, empty], c[3][:, empty] = 0, 0
    return c


@pytest.mark.parametrize("d,pos,splits", [(128, 31, 1), (64, 0, 1), (256, 90, 1), (128, 700, 3)])
@pytest.mark.parametrize("size", [1.0, 1e-6, 1e-7, 1e-9, 1e-12])
@pytest.mark.parametrize("lift", [0, 12, 22, 24])
def test_rows_of_zeros_count_in_the_denominator_alone(C, d, pos, splits, size, lift):
    T, hq, hk = 5, 4, 2
    rnd = gen(pos + d)
    q = torch.ones(T, hq, d, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    masks = O.line_masks([-1, 0, 0, 1, 3])
    for empty in ([pos], [0], [pos // 2, pos + 3], list(range(0, pos + T, 2))):
        c = cache_of(rnd, hk, pos + T, d, size, lift, empty)
        check_relative(C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=splits), q, c, masks, pos, d ** -0.5)


@pytest.mark.parametrize("size", [2.0 ** -98, 2.0 ** -60, 1e-12, 2.0 ** 30, 2.0 ** 100])
@pytest.mark.parametrize("pos,splits", [(200, 1), (30000, 1), (30000, 8)])
def test_values_of_any_size(C, size, pos, splits):
    """The denominator holds as many rows of as small values as the append writes."""
    T, hq, hk, d = 2, 4, 2, 128
    rnd = gen(pos)
    q = torch.ones(T, hq, d, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    c = cache_of(rnd, hk, pos + T, d, size, 0, [])
    for grow in (0.0, 12.0):   # scores that rise along the rows
        c[2][:] += grow * float(np.log(2)) * torch.linspace(0, 1, pos + T, device="cuda") / (100 * d ** 0.5)
        check_relative(C.attn_tree(q, *c[:2], pos, None, *c[2:], splits=splits), q, c, [1, 3], pos, d ** -0.5)


def test_a_long_context_of_zeros(C):
    """All rows but one hold zeros, their scores rising: the one's share of them."""
    T, hq, hk, d, pos = 1, 2, 1, 64, 70000
    q = torch.ones(T, hq, d, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    for splits in (1, 64):
        c = cache_of(gen(3), hk, pos + T, d, 1.0, 0, list(range(0, pos)))
        c[2][:] += 14 * float(np.log(2)) * torch.linspace(0, 1, pos + T, device="cuda") / (100 * d ** 0.5)
        check_relative(C.attn_tree(q, *c[:2], pos, None, *c[2:], splits=splits), q, c, [1], pos, d ** -0.5)


def test_appended_zeros_beside_small_values(C):
    """The rows as the append makes them."""
    T, hq, hk, d = 33, 4, 2, 128
    rnd = gen(5)
    y = rnd(T, (hq + 2 * hk) * d)
    y[:, (hq + hk) * d:] *= 1e-8
    y[::3, (hq + hk) * d:] = 0
    n, inv = torch.ones(d, device="cuda", dtype=torch.bfloat16), torch.zeros(d // 2, device="cuda")
    c = make_cache(rnd, True, hk, T, d)
    q = C.cache_write(y.to(torch.bfloat16), n, n, 1e-6, T, hq, hk, d, c[0], c[1], 0, inv, c[2], c[3])
    masks = [(1 << (i + 1)) - 1 for i in range(T)]
    check_relative(C.attn_tree(q, *c[:2], 0, None, *c[2:]), q, c, masks, 0, d ** -0.5)
