"""bf16 and 8-bit caches at more tokens than a launch has workgroups in one dimension (include/scmx_cache.h)."""
import pytest
import torch

from tests.test_gpu_cache4 import BF, C, gen   # noqa: F401
from tests.test_gpu_cache4_large import room

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True])
def test_more_tokens_than_a_launch_has_workgroups(C, eight):   # noqa: F811
    """2^24 tokens and some: each what it gives alone."""
    L, hq, hk, d = (1 << 24) + 5, 1, 1, 64
    room(24 << 30)
    few = torch.cat([torch.arange(0, L, 1000003, device="cuda"), torch.arange((1 << 22) - 2, (1 << 22) + 3, device="cuda"), torch.arange(L - 9, L, device="cuda")])
    y = gen(1)(1021, (hq + 2 * hk) * d).to(BF).repeat(-(-L // 1021), 1)[:L]
    n, inv = (1 + 0.1 * gen(2)(d)).to(BF), torch.zeros(d // 2, device="cuda")

    def append(rows):
        kv = [torch.zeros((hk, len(rows), d), dtype=torch.int8 if eight else BF, device="cuda") for _ in range(2)]
        scales = [torch.zeros((hk, len(rows)), device="cuda") if eight else None for _ in range(2)]
        q = C.cache_write(rows, n, n, 1e-6, len(rows), hq, hk, d, *kv, 0, inv, *scales)
        return [q, *kv, *(scales if eight else [])]

    for big, small in zip(append(y), append(y[few])):
        assert torch.equal(big[:, few], small)
