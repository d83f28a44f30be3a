"""4-bit caches at more tokens and rows than a launch has threads in one dimension (include/scmx_mx.h)."""
import pytest
import torch

from tests.test_gpu_cache4 import BF, C, gen   # noqa: F401

pytestmark = pytest.mark.gpu


def room(need):
    """Skips where the card has not so many bytes left."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < need:
        pytest.skip("needs more of the card's memory than is free")


def test_more_tokens_than_a_launch_has_workgroups(C):   # noqa: F811
    """2^24 tokens and some: each what it gives alone."""
    L, hq, hk, d = (1 << 24) + 5, 1, 1, 64
    room(24 << 30)
    few = torch.cat([torch.arange(0, L, 1000003, device="cuda"), torch.arange((1 << 22) - 2, (1 << 22) + 3, device="cuda"), torch.arange(L - 9, L, device="cuda")])
    pattern = gen(1)(1021, (hq + 2 * hk) * d).to(BF)
    y = pattern.repeat(-(-L // 1021), 1)[:L]
    n, inv = (1 + 0.1 * gen(2)(d)).to(BF), torch.zeros(d // 2, device="cuda")
    big = tuple(torch.zeros((hk, L, w), dtype=torch.uint8, device="cuda") for w in (d // 2, d // 2, d // 32, d // 32))
    q = C.cache_write(y, n, n, 1e-6, L, hq, hk, d, big[0], big[1], 0, inv, big[2], big[3])
    small = tuple(torch.zeros((hk, len(few), w), dtype=torch.uint8, device="cuda") for w in (d // 2, d // 2, d // 32, d // 32))
    ref = C.cache_write(y[few], n, n, 1e-6, len(few), hq, hk, d, small[0], small[1], 0, inv, small[2], small[3])
    assert torch.equal(q[:, few], ref) and all(torch.equal(b[:, few], s) for b, s in zip(big, small))


def test_more_rows_than_a_launch_has_threads(C):   # noqa: F811
    """2^29 rows of 64 and some read back: 2^32 words of codes."""
    n, hk, d = (1 << 29) + 3, 1, 64
    room(190 << 30)
    big = tuple(torch.zeros((hk, n, w), dtype=torch.uint8, device="cuda") for w in (d // 2, d // 2, d // 32, d // 32))
    few = torch.cat([torch.arange(0, n, 50000017, device="cuda"), torch.arange((1 << 27) - 3, (1 << 27) + 3, device="cuda"), torch.arange(n - 9, n, device="cuda")])
    small = tuple(torch.randint(0, 250, (hk, len(few), t.shape[2]), device="cuda", dtype=torch.uint8) for t in big)
    for b, s in zip(big, small):
        b[:, few] = s
    k, v = C.cache_read(*big, n)
    for got, ref in zip((k, v), C.cache_read(*small, len(few))):
        assert torch.equal(got[:, few], ref)
        got[:, few] = 0
        assert not any(part.any() for part in got[0].split(1 << 26))   # all the others are zeros
    del k, v, got, big
    torch.cuda.empty_cache()
