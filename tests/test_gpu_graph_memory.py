"""Captured steps of the Qwen3 drivers after a cache's layers, or their tensors, were replaced in place: the new memory is used, and
nothing is written to the old."""
import pytest
import torch

from tests.test_gpu_draft_model import ids_of
from tests.test_gpu_model import default_format_afterwards, make_tiny   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("kind", [True, "step", "drafted"])
def test_layers_replaced_in_place(kind, bits):
    Q, args, state, packed = make_tiny(4, 2, 64)
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    m = Q.FusedQwen3(args, state, packed)
    tree = DraftTree([-1, 0, 0, 1])

    def run(graphs, replace):
        cache = m.make_cache(100, bits=bits)
        dec = Q.DraftQwen3(m, graphs=bool(graphs)) if kind == "drafted" else Q.DecodeQwen3(m, graphs=graphs)
        outs, old = [], []
        for prompt in range(3):
            if prompt == 1 and replace:     # other layers in the same list
                old += [(t, t.clone()) for c in cache for t in (c.k, c.v)]
                cache[:] = m.make_cache(100, bits=bits)
            elif prompt == 2 and replace:   # other tensors in the same layers
                old += [(t, t.clone()) for c in cache for t in (c.k, c.v)]
                for c, n in zip(cache, m.make_cache(100, bits=bits)):
                    c.__dict__.update(n.__dict__)
            elif prompt:
                cache = m.make_cache(100, bits=bits)
            m.hidden(ids_of(args, 10 + prompt, prompt), cache)
            for step in range(3):
                ids = ids_of(args, 4, 10 * prompt + step)
                outs += [t.clone() for t in dec.step(ids, tree, cache)] if kind == "drafted" else [dec.step(ids[:1], cache).clone()]
        assert all(torch.equal(t, before) for t, before in old)
        return outs

    want = run(False, False)
    assert all(torch.equal(a, b) for a, b in zip(want, run(kind if kind != "drafted" else True, True)))
