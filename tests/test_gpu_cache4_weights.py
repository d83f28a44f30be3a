"""Attention over a 4-bit cache where rounded probabilities would show: values that cancel, against float64 (oracle/draft.py), at the shapes of
test_gpu_cache4.py."""
import numpy as np
import pytest
import torch

from oracle import draft as O
from tests.test_gpu_cache4 import ATTEND, BF, C, bits, f64, gen, make_cache, tree, values   # noqa: F401

pytestmark = pytest.mark.gpu


def check_close(out, q, cache, masks, pos, scale):
    """As check_attention, with weights of 16 bits."""
    d = 2 * cache[0].shape[2]
    T, hq = q.shape[1], q.shape[0]
    ref, mag = O.attention(f64(q).transpose(1, 0, 2), values(cache[0], cache[2]), values(cache[1], cache[3]), masks, pos, scale)
    got = f64(out).reshape(T, hq, d)
    # the result's rounding (2^-8).  A weight is held in two bf16 parts: 2^-8 of 2^-8, in numerator and denominator, 2^-15 in all.  Scores of
    # up to 32: the queries' parts 2^-23 of a block's largest value, float32 sums and differences some 2^-18 of a weight, both ways; float32
    # sums of 32 keys a step, a hundred steps in a row, 2^-17.  All below 2^-14 of sum p |v|.
    tol = 1.01 * 2.0 ** -8 * np.abs(ref) + 2.0 ** -14 * mag + 1e-30
    assert got.shape == ref.shape and (np.abs(got - ref) <= tol).all(), np.max(np.abs(got - ref) / tol)


@pytest.mark.parametrize("T,hq,hk,d,pos,splits", ATTEND)
def test_values_that_cancel(C, T, hq, hk, d, pos, splits):   # noqa: F811
    """Rows in pairs of the same key and opposite values, but for the keys' scale: results far below what is added up."""
    rnd = gen(T * 100 + pos + d)
    c = make_cache(rnd, hk, pos + T, d)
    n = (pos + T) // 2 * 2
    for t in c[:2]:
        t[:, 1:n:2] = t[:, :n:2]
    c[1][:, 1:n:2] ^= 0x88          # the signs of both codes of a byte
    c[3][:, 1:n:2] = c[3][:, :n:2]
    c[2][:, 1:n:2] = c[2][:, :n:2] - (rnd(hk, n // 2, 1) > 1).to(torch.uint8)
    q = (1.5 * rnd(T, hq, d)).to(BF).transpose(0, 1)
    masks = O.line_masks(tree(T, pos))
    check_close(C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=splits), q, c, masks, pos, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_mean_of_many_values(C, d):   # noqa: F811
    """Weights that are equal, or differ in their last bits: a mean whose summands are a thousand times larger."""
    T, hq, hk, pos = 3, 4, 2, 2045
    rnd = gen(d)
    c = make_cache(rnd, hk, pos + T, d, 0.0)
    q = (2.0 ** -6 * rnd(T, hq, d)).to(BF).transpose(0, 1)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    for splits in (1, 5, None):
        check_close(C.attn_tree(q, *c[:2], pos, None, *c[2:], splits=splits), q, c, chain, pos, d ** -0.5)
