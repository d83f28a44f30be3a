"""Rows to MXFP4 and back and products of MXFP4 operands on the GPU (include/scmx_mx.h), against a float64 restatement (oracle/mx.py) at the
sizes, strides and values where they can go wrong; what they refuse."""
import numpy as np
import pytest
import torch

from oracle import mx as O

BF = torch.bfloat16


@pytest.fixture(scope="module")
def X():
    from mxfp4_int8_m5_amd import sc_mx
    return sc_mx


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731


def f64(t):
    return t.double().cpu().numpy()


def host(*ts):
    return tuple(t.cpu().numpy() for t in ts)


def same(got, want):
    """The same codes and scales."""
    (gc, gs), (wc, ws) = host(*got), want
    return gc.shape == wc.shape and gs.shape == ws.shape and (gs == ws).all() and (gc == wc).all()


# ---- quantisation --------------------------------------------------------------------------------------------------------

# a block, rows that end inside a wave's piece and behind several, many rows, more values than a wave takes of a row at once
ROWS = [(1, 32), (1, 2048), (3, 96), (7, 544), (5, 2080), (130, 160), (1, 16384), (2, 20000 // 32 * 32), (1030, 1024), (257, 4128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", ROWS)
def test_quantize(X, M, K, dtype):
    rnd = gen(M + K)
    wide = (rnd(M + 1, K + 64) * torch.exp(2 * rnd(M + 1, K + 64))).to(dtype)
    x = wide[:M, :K]
    want = O.quantize(f64(x))
    assert same(X.quantize(x.contiguous()), want)
    assert same(X.quantize(x), want)                                   # rows of a wider tensor
    assert same(X.quantize(wide.reshape(-1)[3:3 + M * K].view(M, K)), O.quantize(f64(wide.reshape(-1)[3:3 + M * K].view(M, K))))   # off 16 bytes
    odd = wide[:, 1:K + 1][:M]
    assert same(X.quantize(odd), O.quantize(f64(odd)))
    if M < 200:
        turned = x.t().contiguous().t()                                # K is not the fast axis
        assert same(X.quantize(turned), want)
    codes, scales = X.quantize(x)
    v = O.values(*host(codes, scales))
    assert np.array_equal(f64(X.dequantize(codes, scales)), v) and np.array_equal(f64(X.dequantize(codes, scales, torch.float32)), v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
def test_quantize_borders_and_extremes(X, dtype):
    """Every border between two codes and the values beside it, at every exponent of the type; zeros, subnormals, the largest values, NaN
    and infinities."""
    info = torch.finfo(dtype)
    base = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7])
    near = np.concatenate([base, base * (1 + info.eps), base * (1 - info.eps), [0, -0.0, 4]])
    rows = []
    lo, hi = int(np.floor(np.log2(info.tiny))) - 12, int(np.floor(np.log2(info.max)))
    for e in range(lo, hi - 1):
        rows.append(np.ldexp(np.concatenate([near, [4, 4]]), e))
        rows.append(-np.ldexp(np.concatenate([near, [4, 7.5]]), e))
    v = torch.from_numpy(np.array(rows)).to(dtype)
    v = v.masked_fill(~torch.isfinite(v), 0)
    v = torch.cat([v, torch.full((1, 32), info.max, dtype=dtype), torch.zeros(1, 32, dtype=dtype), torch.full((1, 32), info.smallest_normal, dtype=dtype)])
    odd = torch.ones(4, 32, dtype=dtype)
    odd[0, 7], odd[1, 31], odd[2, 0] = float("nan"), float("inf"), -float("inf")
    v = torch.cat([v, odd])
    want = O.quantize(f64(v))
    got = X.quantize(v.cuda())
    assert same(got, want)
    back, ref = f64(X.dequantize(*got, torch.float32)), O.values(*want)
    assert np.array_equal(back, ref, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", ROWS)
def test_quantize_of_the_norm(X, M, K):
    if K > 16384:
        with pytest.raises(ValueError):
            X.quantize(torch.zeros(M, K, device="cuda", dtype=BF), torch.ones(K, device="cuda", dtype=BF), 1e-6)
        return
    rnd = gen(M * 3 + K)
    wide = (rnd(M, K + 8) * torch.exp(rnd(K + 8))).to(BF)
    x, w = wide[:, :K], (1 + 0.2 * rnd(K)).to(BF)
    eps = 2.0 ** -20   # (the same number in float32)
    want = O.quantize(O.rmsnorm(f64(x), f64(w), eps), 10, 252)
    assert same(X.quantize(x, w, eps), want)       # float64 to the code: equal, borders and all
    assert same(X.quantize(x.contiguous(), w, torch.tensor([eps])), want)
    odd = torch.cat([w[:1], w])[1:]                # a weight off 16 bytes
    x = wide.reshape(-1)[:M * K].view(M, K)
    assert odd.data_ptr() % 16 and same(X.quantize(x, odd, eps), O.quantize(O.rmsnorm(f64(x), f64(w), eps), 10, 252))


@pytest.mark.gpu
def test_norms_of_rows_that_are_not_ordinary(X):
    """Zeros, a NaN, an infinity, tiny and huge rows and weights."""
    K = 256
    x = gen(5)(8, K).to(BF)
    x[0], x[1, 5], x[2, 200], x[3], x[4] = 0, float("nan"), float("inf"), 1e-30, 1e30
    w = gen(6)(K).to(BF)
    w[:32], w[32:64], w[64:96] = 1e-38, 3e38, 0
    with np.errstate(invalid="ignore"):
        want = O.quantize(O.rmsnorm(f64(x), f64(w), 1e-6), 10, 252)
    got = X.quantize(x, w, 1e-6)
    assert (got[1].cpu().numpy() == want[1]).all()
    a, b = O.values(*host(*got)), O.values(*want)
    assert np.array_equal(a, b, equal_nan=True)


@pytest.mark.gpu
def test_values_of_every_byte(X):
    """Every scale byte with every code, in both types: float32 whole, bf16 whole where its range reaches."""
    row = torch.arange(16, dtype=torch.uint8).repeat(2)
    codes = (row[0::2] | row[1::2] << 4).repeat(256, 1).cuda()
    scales = torch.arange(256, dtype=torch.uint8)[:, None].cuda()
    with np.errstate(over="ignore"):
        ref = O.values(*host(codes, scales)).astype(np.float32)
    assert np.array_equal(X.dequantize(codes, scales, torch.float32).cpu().numpy(), ref, equal_nan=True)
    assert np.array_equal(X.dequantize(codes, scales).float().cpu().numpy()[:253], ref[:253])


# ---- products ------------------------------------------------------------------------------------------------------------

def operands(X, rnd, M, N, K):
    x = (rnd(M, K) * torch.exp(rnd(K))).to(BF)
    w = X.quantize(rnd(N, K) * K ** -0.5 * torch.exp(rnd(N, 1)))
    return x, w


def check_product(out, x, w, epi, res):
    ref, mag = O.product(x, w, epi, res)
    # float32 sums of K exact products: 2^-24 of the magnitudes' sum a step, of which few add up (2^-20); then one rounding to bf16
    # (2^-8); the gate's exponential and quotient are a few 2^-23 of a result whose gate is off by f: silu' is at most 1.1
    if epi == 3:
        mg, mu, g, u = mag
        silu = np.abs(g / (1 + np.exp(-np.clip(g, -700, None))))
        err = 2.0 ** -20 * (1.1 * mg * np.abs(u) + mu * silu + np.abs(ref) * (1 + np.abs(g)))
    else:
        err = 2.0 ** -20 * mag
    got = f64(out)
    assert got.shape == ref.shape
    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 1.02 * err + 1e-38).all(), np.nanmax(np.abs(got - ref) / (2.0 ** -8 * np.abs(ref) + err + 1e-38))


# one block of K, K that ends inside a step, rows and columns of every tile that end inside it, single ones, more than one tile of each kind
SIZES = [(1, 4, 32), (1, 1, 64), (1, 2048, 2048), (2, 100, 96), (3, 36, 4000), (5, 2048, 6144), (8, 60, 128), (16, 257, 160), (17, 64, 32), (17, 64, 256), (33, 1, 32),
         (40, 130, 544), (64, 512, 2912), (100, 61, 224), (128, 4096, 512), (130, 1500, 320), (333, 5004, 2912), (500, 7, 4096), (700, 2052, 96), (2048, 4096, 288),
         (2000, 8000, 192), (4100, 4164, 64), (3, 70000, 64), (70000, 3, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SIZES)
def test_products(X, M, N, K):
    rnd = gen(M + N + K)
    x, w = operands(X, rnd, M, N, K)
    xq = X.quantize(x)
    xv, wv = O.values(*host(*xq)), O.values(*host(*w))
    few = slice(0, None) if M * N < 4e6 else np.unique(np.concatenate([np.arange(0, M, max(1, M // 40)), [M - 1]]))   # rows that are checked
    for epi in (1, 2, 3):
        if epi == 3 and N % 4:
            continue
        res = rnd(M, N).to(BF) if epi == 2 else None
        out = X.mm(*xq, *w, epi, res)
        rows = few if not isinstance(few, slice) else np.arange(M)
        check_product(out[torch.from_numpy(rows).cuda()], xv[rows], wv, epi, None if res is None else f64(res)[rows])
        whole = X.linear(x, *w, epi, res)
        assert torch.equal(whole, out) if M > 16 else np.allclose(f64(whole), f64(out), rtol=2.0 ** -7, atol=1e-2 * np.abs(f64(out)).max())
        if M <= 16:
            check_product(whole, xv, wv, epi, None if res is None else f64(res))


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(1, 2048), (4, 96), (9, 4096), (40, 544), (300, 1024)])
def test_linear_of_the_norm_and_of_strided_rows(X, M, K):
    rnd, N = gen(M), 132
    wide = (rnd(M, K + 40) * torch.exp(rnd(K + 40))).to(BF)
    x, nw = wide[:, :K], (1 + 0.1 * rnd(K)).to(BF)
    w = X.quantize(rnd(N, K))
    for xs in (x, wide[:, 7:K + 7], wide.t().contiguous().t()[:, :K]):
        xv = O.values(*O.quantize(O.rmsnorm(f64(xs), f64(nw), 1e-5), 10, 252))
        check_product(X.linear(xs, *w, 1, None, nw, 1e-5), xv, O.values(*host(*w)), 1, None)
        check_product(X.linear(xs, *w), O.values(*O.quantize(f64(xs))), O.values(*host(*w)), 1, None)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 64), (16, 64), (50, 200), (300, 400)])
def test_products_of_blocks_that_are_not_numbers(X, M, N):
    """A NaN block reaches its row's results (its column's, of a weight) and no other; exponents far apart."""
    rnd, K = gen(M), 416
    x, w = operands(X, rnd, M, N, K)
    (xc, xs), (wc, ws) = X.quantize(x), w
    clean = X.mm(xc, xs, wc, ws)
    xs2, ws2 = xs.clone(), ws.clone()
    xs2[M - 1, 12], ws2[N - 1, 3] = 255, 255
    out = X.mm(xc, xs2, wc, ws2)
    assert torch.isnan(out[M - 1]).all() and torch.isnan(out[:, N - 1]).all()
    assert torch.equal(out[:M - 1, :N - 1], clean[:M - 1, :N - 1])
    xs[:, ::2], ws[:, ::2] = 20, 230
    xs[:, 1::2], ws[:, 1::2] = 120, 100
    check_product(X.mm(xc, xs, wc, ws), O.values(*host(xc, xs)), O.values(*host(wc, ws)), 1, None)


@pytest.mark.gpu
def test_no_rows(X):
    e = torch.empty(0, 64, device="cuda", dtype=BF)
    w = X.quantize(torch.ones(8, 64, device="cuda"))
    codes, scales = X.quantize(e)
    assert codes.shape == (0, 32) and scales.shape == (0, 2) and X.dequantize(codes, scales).shape == (0, 64)
    assert X.linear(e, *w).shape == X.mm(codes, scales, *w).shape == (0, 8) and X.linear(e, *w, 3).shape == (0, 4)


@pytest.mark.gpu
def test_packed_weights_as_mxfp4(X):
    """The code words of a packed weight in the published format are a standard MXFP4 tensor's."""
    from mxfp4_int8_m5_amd import sc_format as F, sc_kernels as S, sc_weights as W
    w = gen(1)(96, 256) * 0.05
    codes, bc, ws, q = F.quantize(w)
    pw = W.PackedWeight([(codes.cpu().numpy().view(np.uint32), bc.cpu().numpy(), ws.cpu().numpy())])
    c, s = X.from_packed(pw)
    assert np.array_equal(O.values(*host(c, s)), f64(q) * f64(ws)[:, None])
    x = gen(2)(33, 256).to(BF)
    check_product(X.linear(x, c, s, 1), O.values(*O.quantize(f64(x))), O.values(*host(c, s)), 1, None)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 6, 40, 600])
def test_captured_and_on_other_streams(X, M):
    """A captured quantisation and product, replayed over new inputs between eager calls; two streams at once."""
    rnd, N, K = gen(M), 512, 1024
    x, w = operands(X, rnd, M, N, K)
    nw = torch.ones(K, device="cuda", dtype=BF)
    step = lambda t: X.linear(X.linear(t, *w, 1, None, nw, 1e-6), *v, 2, t)   # noqa: E731
    v = X.quantize(rnd(K, N))
    static = x.clone()
    step(static)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(static)
    for i in range(4):
        new = (rnd(M, K) * (i + 1)).to(BF)
        static.copy_(new)
        want = step(new)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s, t in zip(streams, (x, -x)):
        with torch.cuda.stream(s):
            outs.append([step(t) for _ in range(8)])
    torch.cuda.synchronize()
    for t, os in zip((x, -x), outs):
        assert all(torch.equal(o, step(t)) for o in os)


@pytest.mark.gpu
def test_refusals(X):
    z = lambda *s, t=BF: torch.zeros(*s, dtype=t, device="cuda")   # noqa: E731
    u8 = lambda *s: z(*s, t=torch.uint8)   # noqa: E731
    w = (u8(8, 32), u8(8, 2))
    bad = [lambda: X.quantize(z(2, 48)), lambda: X.quantize(z(2, 0)), lambda: X.quantize(z(64)), lambda: X.quantize(z(2, 64, t=torch.int32)),
           lambda: X.quantize(z(2, 64, t=torch.float32), z(64), 1e-6), lambda: X.quantize(z(2, 64), z(32), 1e-6), lambda: X.quantize(z(2, 64), z(64, t=torch.float32), 1e-6),
           lambda: X.quantize(z(2, 64).cpu()), lambda: X.dequantize(u8(2, 32), u8(2, 3)), lambda: X.dequantize(u8(2, 32), u8(3, 2)),
           lambda: X.dequantize(u8(2, 32), u8(2, 2), torch.float16), lambda: X.dequantize(z(2, 32, t=torch.int8), u8(2, 2)), lambda: X.dequantize(u8(2, 32).cpu(), u8(2, 2)),
           lambda: X.dequantize(u8(32, 2).t(), u8(2, 2)), lambda: X.mm(u8(2, 16), u8(2, 1), *w), lambda: X.mm(u8(2, 32), u8(2, 2), *w, 2), lambda: X.mm(u8(2, 32), u8(2, 2), *w, 4),
           lambda: X.mm(u8(2, 32), u8(2, 2), u8(6, 32), u8(6, 2), 3), lambda: X.mm(u8(2, 32), u8(2, 2), *w, 2, z(2, 7)), lambda: X.mm(u8(2, 32), u8(2, 2), *w, 2, z(2, 8, t=torch.float32)),
           lambda: X.linear(z(2, 32), *w), lambda: X.linear(z(2, 64, t=torch.float32), *w), lambda: X.linear(z(64), *w), lambda: X.linear(z(2, 64), *w, 0), lambda: X.linear(z(2, 64), *w, 2),
           lambda: X.linear(z(2, 64), u8(0, 32), u8(0, 2)), lambda: X.linear(z(2, 64), *w, 1, None, z(63), 1e-6), lambda: X.linear(z(2, 64), w[0].cpu(), w[1])]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
