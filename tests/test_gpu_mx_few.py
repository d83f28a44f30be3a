"""Linear layers of few MXFP4 rows, whose rows become codes in the product's own launch: long rows, every kind of workgroup, and each value
beside a border of two codes (include/scmx_mx.h; oracle/mx.py)."""
import numpy as np
import pytest
import torch

from oracle import mx as O
from tests.test_gpu_mx import BF, X, check_product, f64, gen, host, operands   # noqa: F401

pytestmark = pytest.mark.gpu

# columns of a workgroup: 8 where that leaves no CU two workgroups (N to 2048 for up to 16 rows), else 16; blocks of K at a time: 256, or 128
# for 16 columns and K to 4096.  K of one and several rounds that ends inside one and at its end, columns and rows that end inside a workgroup
FEW = [(1, 4100, 8224), (3, 64, 16416), (16, 2100, 6176), (1, 16384, 8192), (5, 2052, 4128), (16, 2049, 8192), (2, 5000, 20000), (16, 2300, 4096), (7, 2047, 8224),
       (16, 100, 32768), (9, 3001, 4064), (1, 1, 8224), (4, 8, 65536), (33, 20, 16416), (64, 130, 12320)]


@pytest.mark.parametrize("M,N,K", FEW)
def test_long_rows(X, M, N, K):   # noqa: F811
    from mxfp4_int8_m5_amd import _lib
    assert _lib.load().scmx_mx_linear_workspace(M, N, K, 0) == 0   # one launch: no place for codes
    rnd = gen(M + N + K)
    wide = (rnd(M, K + 24) * torch.exp(rnd(K + 24))).to(BF)
    w = X.quantize(rnd(N, K) * K ** -0.5 * torch.exp(rnd(N, 1)))
    wv = O.values(*host(*w))
    for x in (wide[:, :K], wide[:, 5:K + 5]):   # rows of a wider tensor, and off 16 bytes
        xq = X.quantize(x)
        xv = O.values(*host(*xq))
        for epi in (1, 2, 3):
            if epi == 3 and N % 4:
                continue
            res = rnd(M, N).to(BF) if epi == 2 else None
            out = X.linear(x, *w, epi, res)
            check_product(out, xv, wv, epi, None if res is None else f64(res))
            if M <= 16:   # the same kernel and sums as of codes
                assert torch.equal(out, X.mm(*xq, *w, epi, res))


def extremes():
    """bf16 [.., 32]: every border of two codes, the values beside it, at every exponent; zeros, subnormals, the largest values."""
    info = torch.finfo(BF)
    base = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7])
    near = np.concatenate([base, base * (1 + info.eps), base * (1 - info.eps), [0, -0.0, 4]])
    rows = []
    for e in range(-138, 127):
        rows.append(np.ldexp(np.concatenate([near, [4, 4]]), e))
        rows.append(-np.ldexp(np.concatenate([near, [4, 7.5]]), e))
    v = torch.from_numpy(np.array(rows)).to(BF)
    v = v.masked_fill(~torch.isfinite(v), 0)
    return torch.cat([v, torch.full((1, 32), info.max, dtype=BF), torch.zeros(1, 32, dtype=BF), torch.full((1, 32), info.smallest_normal, dtype=BF)])


@pytest.mark.parametrize("N", [32, 2080])
def test_codes_of_every_border_and_exponent(X, N):   # noqa: F811
    """Weights with a one a row return the values that the codes stand for; workgroups of 8 and of 16 columns."""
    v = extremes().cuda()
    codes = torch.zeros(N, 16, dtype=torch.uint8, device="cuda")
    n = torch.arange(N, device="cuda")
    codes[n, n % 32 // 2] = torch.where(n % 2 == 0, 0x02, 0x20).to(torch.uint8)
    scales = torch.full((N, 1), 127, dtype=torch.uint8, device="cuda")
    want = O.values(*O.quantize(f64(v)))[:, np.arange(N) % 32]
    for i in range(0, len(v), 16):
        x = v[i:i + 16]
        out, ref = X.linear(x, codes, scales), want[i:i + 16]
        assert torch.equal(out, X.mm(*X.quantize(x), codes, scales))
        normal = (np.abs(ref) >= 2.0 ** -126) | (ref == 0)   # (what is below float32's normal numbers may be 0 in the matrix instructions)
        got = f64(out)
        assert (got == ref)[normal].all() and (np.abs(got) <= np.abs(ref))[~normal].all()


@pytest.mark.parametrize("N", [32, 2080])
def test_blocks_that_are_not_numbers(X, N):   # noqa: F811
    """A NaN or an infinity anywhere in a block makes its row's results NaN and no other row's."""
    K = 8224
    rnd = gen(N)
    x, w = operands(X, rnd, 12, N, K)
    clean = X.linear(x, *w)
    bad = x.clone()
    bad[1, 0], bad[4, 4096 + 31], bad[6, K - 1], bad[11, 8200] = float("nan"), float("inf"), -float("inf"), float("nan")
    out, hit = X.linear(bad, *w), [1, 4, 6, 11]
    ok = [i for i in range(12) if i not in hit]
    assert torch.isnan(out[hit]).all() and torch.equal(out[ok], clean[ok])
