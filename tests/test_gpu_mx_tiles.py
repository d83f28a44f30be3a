"""Products of MXFP4 operands by every tile, whole words of scales a row and not, whose workgroups take several tiles in turn: results whole,
against float64 of the values (include/scmx_mx.h).  test_mx_tile_choice.py holds that these sizes take the tiles they are listed under."""
import pytest
import torch

from tests.test_gpu_mx import BF, X, gen, operands   # noqa: F401

# rows and columns of a tile; whole words of scales a row; sizes M, N, K with more tiles than a launch has workgroups, rows that end inside
# a tile behind whole ones, columns that are 0, 4, 12 and an odd number behind the last 16, and one, some and an odd and even number
# of stages of 256 of K
TILES = [
    (32, 128, True, [(8346, 144, 128), (131, 17396, 512), (134, 16391, 640), (196, 16428, 1280), (195, 17456, 2048)]),
    (32, 128, False, [(8310, 144, 32), (8237, 132, 96), (193, 16769, 288), (196, 16812, 544)]),
    (64, 128, True, [(389, 16592, 128), (386, 16532, 256), (392, 16579, 384), (387, 16460, 1152), (391, 16608, 640), (392, 16519, 2048)]),
    (64, 128, False, [(386, 16468, 96), (394, 16512, 288), (387, 16503, 544), (392, 16668, 1184), (392, 16544, 2912)]),
    (128, 128, True, [(385, 18864, 128), (388, 18756, 384), (392, 19036, 640), (387, 19235, 1152), (776, 12864, 1536), (390, 18740, 1536)]),
    (128, 128, False, [(388, 18752, 32), (390, 18892, 288), (516, 14516, 544), (387, 19203, 1184), (388, 18864, 2912)]),
    (256, 256, True, [(1539, 17904, 1152), (8860, 3232, 1536), (1538, 17552, 2048), (2454, 9776, 4096)]),
]


def product(x, w, epi, res):
    """float64 x w^T with the epilogue, and how far float32 sums may be off it."""
    y, mag = x @ w.t(), x.abs() @ w.abs().t()
    if epi == 1:
        return y, 2.0 ** -20 * mag
    if epi == 2:
        return y + res, 2.0 ** -20 * mag
    (g, u), (mg, mu) = (t.unflatten(1, (-1, 2, 2)).unbind(2) for t in (y, mag))
    g, u, mg, mu = (t.flatten(1) for t in (g, u, mg, mu))
    silu = g * torch.sigmoid(g)
    # (as in test_gpu_mx.check_product: silu' is at most 1.1, an exponential's and a quotient's last bits)
    return silu * u, 2.0 ** -20 * (1.1 * mg * u.abs() + mu * silu.abs() + (silu * u).abs() * (1 + g.abs()))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [s for *_, sizes in TILES for s in sizes])
def test_every_tile_in_turn(X, M, N, K):   # noqa: F811
    rnd = gen(M + N + K)
    x, w = operands(X, rnd, M, N, K)
    xq = X.quantize(x)
    xv, wv = (X.dequantize(*t, torch.float32).double() for t in (xq, w))
    for epi in (1, 2, 3):
        if epi == 3 and N % 4:
            continue
        res = rnd(M, N).to(BF) if epi == 2 else None
        ref, err = product(xv, wv, epi, None if res is None else res.double())
        out = X.mm(*xq, *w, epi, res)
        off = (out.double() - ref).abs() - (2.0 ** -8 * ref.abs() + 1.02 * err + 1e-38)
        assert out.shape == ref.shape and (off <= 0).all(), (epi, [t.item() for t in (off <= 0).logical_not().nonzero()[0]])
        del ref, err, off
        assert torch.equal(X.mm(*xq, *w, epi, res), out)   # the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [sizes[-1] for *_, sizes in TILES])
def test_every_tile_in_turn_in_a_graph(X, M, N, K):   # noqa: F811
    """Captured with the rows' quantisation, replayed over other rows."""
    rnd = gen(M)
    x, w = operands(X, rnd, M, N, K)
    X.linear(x, *w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = X.linear(x, *w)
    for i in range(3):
        x.copy_((rnd(M, K) * 2.0 ** i).to(BF))
        want = X.linear(x, *w)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [sizes[i] for *_, sizes in TILES for i in (1, -1)])
def test_a_nan_in_every_tile_in_turn(X, M, N, K):   # noqa: F811
    """A block's NaN reaches its row or its column and no other, in first and later tiles of a workgroup."""
    rnd = gen(N)
    x, w = operands(X, rnd, M, N, K)
    (xc, xs), (wc, ws) = X.quantize(x), w
    clean = X.mm(xc, xs, wc, ws)
    xs, ws = xs.clone(), ws.clone()
    rows, cols = [0, 77, M // 2, M - 1], [3, N // 2 + 1, N - 1]
    for i, r in enumerate(rows):
        xs[r, -1 - i if i < K // 32 else 0] = 255
    for i, c in enumerate(cols):
        ws[c, i if i < K // 32 else 0] = 255
    out = X.mm(xc, xs, wc, ws)
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[rows] = True
    bad[:, cols] = True
    assert torch.equal(torch.isnan(out), bad) and torch.equal(out[~bad], clean[~bad])
