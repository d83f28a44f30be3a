"""Captured steps of the Qwen3 drivers against eager ones: over the store's evictions."""
import gc
import weakref

import numpy as np
import pytest
import torch

from tests.test_gpu_draft_model import ids_of
from tests.test_gpu_model import default_format_afterwards, make_tiny   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny():
    return make_tiny(4, 2, 64)


def test_evicted_steps_are_captured_again(tiny):
    """Fresh caches, trees of several sizes, more temperatures than are kept: the eager steps' bits, and only the latest cache is held."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    m = Q.FusedQwen3(args, state, packed)
    eager, graph = Q.DraftQwen3(m), Q.DraftQwen3(m, graphs=True)
    rng, refs = np.random.default_rng(1), []
    for prompt in range(3):
        caches = [m.make_cache(150, bits=8) for _ in range(2)]
        refs.append(weakref.ref(caches[1][0]))
        for c in caches:
            m.hidden(ids_of(args, 9 + prompt, prompt), c)
        for i, t in enumerate((0.0, 0.5, 0.6, 0.7, 0.8, 0.9, 0.5, 0.0)):
            T = 3 + (i + prompt) % 3
            tree = DraftTree([-1] + [int(rng.integers(0, k)) for k in range(1, T)])
            tokens = torch.tensor(rng.integers(args.vocab_size, size=T), device="cuda")
            u = torch.tensor(rng.random(T), dtype=torch.float32, device="cuda")
            a, b = eager.step(tokens, tree, caches[0], t, u), graph.step(tokens, tree, caches[1], t, u)
            assert all(torch.equal(x, y) for x, y in zip(a, b)), (prompt, t)
        assert len({k[3] for k in graph.graphs}) <= 5
        del caches, c
    gc.collect()
    assert [r() is None for r in refs] == [True, True, False]
