"""MXFP4 rows and products at the sizes that the largest tile takes, with more rows than a launch has groups, and long prompts' norms, each
against the float64 restatement (oracle/mx.py)."""
import numpy as np
import pytest
import torch

from oracle import mx as O
from tests.test_gpu_mx import BF, X, check_product, f64, gen, host, operands, same   # noqa: F401

pytestmark = pytest.mark.gpu

# the 256 x 256 tile: rows and columns that end inside it, stages of 256 that K ends inside, bytes of four stages that it ends inside
LARGE = [(4090, 4096, 1152), (2040, 8192, 1152), (2500, 5136, 2176), (1800, 2064, 8320), (3900, 2064, 4224)]


@pytest.mark.parametrize("M,N,K", LARGE)
def test_products_of_the_largest_tile(X, M, N, K):   # noqa: F811
    rnd = gen(M + N + K)
    x, w = operands(X, rnd, M, N, K)
    xq = X.quantize(x)
    rows = np.unique(np.concatenate([np.arange(0, M, M // 30), np.arange(M - 20, M)]))
    at = torch.from_numpy(rows).cuda()
    xv, wv = O.values(*host(*(t[at] for t in xq))), O.values(*host(*w))
    for epi in (1, 2, 3):
        res = rnd(M, N).to(BF) if epi == 2 else None
        out = X.mm(*xq, *w, epi, res)
        check_product(out[at], xv, wv, epi, None if res is None else f64(res[at]))
        assert torch.equal(X.linear(x, *w, epi, res), out)
        again = X.mm(xq[0][at], xq[1][at], *w, epi, None if res is None else res[at])   # a smaller tile: the same sums in another order
        # of float32 sums 2^-20 of the magnitudes apart at most, a bf16 step (2^-7) for those beside a border
        check_product(again, xv, wv, epi, None if res is None else f64(res[at]))


def test_a_nan_in_the_largest_tile(X):   # noqa: F811
    """A block's NaN reaches its row or column and no other, blocks behind the end of K among them."""
    M, N, K = 4090, 4096, 1152
    rnd = gen(1)
    x, w = operands(X, rnd, M, N, K)
    (xc, xs), (wc, ws) = X.quantize(x), w
    clean = X.mm(xc, xs, wc, ws)
    xs, ws = xs.clone(), ws.clone()
    for i, j in ((0, 0), (300, 35), (M - 1, 17)):
        xs[i, j] = 255
    for i, j in ((5, 35), (257, 0), (N - 1, 8)):
        ws[i, j] = 255
    out = X.mm(xc, xs, wc, ws)
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[[0, 300, M - 1]] = True
    bad[:, [5, 257, N - 1]] = True
    assert torch.equal(torch.isnan(out), bad) and torch.equal(out[~bad], clean[~bad])


def test_the_largest_tile_in_a_graph(X):   # noqa: F811
    M, N, K = 4090, 4096, 1152
    rnd = gen(2)
    x, w = operands(X, rnd, M, N, K)
    X.linear(x, *w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = X.linear(x, *w)
    for i in range(3):
        x.copy_((rnd(M, K) * 2 ** i).to(BF))
        want = X.linear(x, *w)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_more_rows_than_groups_of_a_launch(X):   # noqa: F811
    """Rows of one block times three columns: less than four bytes of weights' scales, and over 65535 groups of 16 rows."""
    M, N, K = 1100003, 3, 32
    rnd = gen(3)
    x, w = operands(X, rnd, M, N, K)
    xq = X.quantize(x)
    check_product(X.mm(*xq, *w), O.values(*host(*xq)), O.values(*host(*w)), 1, None)


@pytest.mark.parametrize("M,K", [(4096, 2048), (3000, 4096), (500, 8192), (300, 16384)])
def test_long_prompts_norms_take_float64s_codes(X, M, K):   # noqa: F811
    """Millions of values, of which some are next to a border: all codes are float64's.  Rows of very different sizes."""
    rnd = gen(M)
    x = (rnd(M, K) * torch.exp(3 * rnd(M, 1))).to(BF)
    w = (1 + 0.3 * rnd(K)).to(BF)
    assert same(X.quantize(x, w, 1e-6), O.quantize(O.rmsnorm(f64(x), f64(w), 1e-6), 10, 252))


def test_norms_on_the_borders(X):   # noqa: F811
    """Rows of ones and minus ones, whose norm is one, so that the values are the gains: every border between two codes, at many exponents,
    exactly, and (eps) a little below."""
    K = 64 * 32
    base = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 4, 1, 3])
    w = np.ones(K)
    for b in range(64):
        w[32 * b:32 * b + 12] = base * 2.0 ** (2 * b - 70)
        w[32 * b + 12:32 * b + 32] = 4 * 2.0 ** (2 * b - 70) if b % 2 else 7.96875 * 2.0 ** (2 * b - 70)
    w = torch.from_numpy(w).to(BF).cuda()
    x = torch.where(gen(4)(1040, K) < 0, -1.0, 1.0).to(BF)
    x[5] *= 2.0 ** 60
    x[6] *= 2.0 ** -60
    for rows in (x, x[:7]):   # a wave a row, four waves a row
        for eps in (0.0, 2.0 ** -30, 2.0 ** -24, 2.0 ** -20, 2.0 ** -10):
            assert same(X.quantize(rows, w, eps), O.quantize(O.rmsnorm(f64(rows), f64(w), eps), 10, 252)), eps


@pytest.mark.parametrize("M,N,K", [(3, 600, 256), (40, 130, 512), (300, 1500, 384), (2040, 8192, 1152)])
@pytest.mark.parametrize("at", [1, 2, 3])
def test_scales_at_any_address(X, M, N, K, at):   # noqa: F811
    """Bytes that start off a word, of rows of whole words: the results of aligned ones, which take other tiles and sums of another order."""
    rnd = gen(M + at)
    x, w = operands(X, rnd, M, N, K)
    xq = X.quantize(x)

    def moved(t):
        out = torch.empty(t.numel() + at, dtype=torch.uint8, device="cuda")[at:].view(t.shape)
        return out.copy_(t)

    rows = np.arange(0, M, max(1, M // 40))
    pick = torch.from_numpy(rows).cuda()
    xv, wv = O.values(*host(xq[0][pick], xq[1][pick])), O.values(*host(*w))
    for s, ws in ((moved(xq[1]), w[1]), (xq[1], moved(w[1])), (moved(xq[1]), moved(w[1]))):
        check_product(X.mm(xq[0], s, w[0], ws)[pick], xv, wv, 1, None)
        assert np.array_equal(f64(X.dequantize(w[0], ws)), O.values(*host(*w)))
    check_product(X.linear(x, w[0], moved(w[1]))[pick], xv, wv, 1, None)


def test_rows_beyond_a_launchs_threads(X):   # noqa: F811
    """2^25 rows of one block: more threads than a launch has in one dimension; there and back."""
    M = (1 << 25) + 3
    x = torch.arange(M * 32, device="cuda", dtype=torch.int32).remainder(251).sub(125).to(BF).view(M, 32)
    codes, scales = X.quantize(x)
    few = torch.cat([torch.arange(0, M, 1000003, device="cuda"), torch.arange(M - 20, M, device="cuda")])
    assert same((codes[few], scales[few]), O.quantize(f64(x[few])))
    back = X.dequantize(codes, scales)
    assert np.array_equal(f64(back[few]), O.values(*host(codes[few], scales[few])))
    del back
    gain = torch.ones(32, device="cuda", dtype=BF)
    codes, scales = X.quantize(x, gain, 1e-6)
    assert same((codes[few], scales[few]), O.quantize(O.rmsnorm(f64(x[few]), np.ones(32), 1e-6), 10, 252))
