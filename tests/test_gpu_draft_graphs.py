"""Captured steps of the Qwen3 drivers against eager ones: over the store's evictions, and over caches long enough that the attention's
ranges go by the cache in a graph and by the position outside."""
import gc
import weakref

import numpy as np
import pytest
import torch

from tests.test_gpu_draft_model import ids_of
from tests.test_gpu_model import default_format_afterwards, make_tiny, rel   # noqa: F401

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


@pytest.mark.parametrize("kw", [{"graphs": True}, {"graphs": "step"}, {"graphs": "step", "fuse_attn": False}])
@pytest.mark.parametrize("rows,same", [(150, True), (2000, False)])
@pytest.mark.parametrize("bits", [8, 16])
def test_captured_decode_steps_are_the_eager_ones(tiny, kw, rows, same, bits):
    """One range: the same bits.  More: sums of the same weights in another order, so that a bf16 value now and then rounds to its
    neighbour (2^-8 of it) and an INT8 activation with it; all of them rounded afresh, a prefill against a decoder, make 2e-2."""
    Q, args, state, packed = tiny
    m = Q.FusedQwen3(args, state, packed)
    for n in (20, rows - 30):
        out = []
        for k in (kw | {"graphs": False}, kw):
            cache = m.make_cache(rows, bits=bits)
            m.hidden(ids_of(args, n, 2), cache)
            dec, ids = Q.DecodeQwen3(m, **k), ids_of(args, 6, 3)
            out.append(torch.cat([dec.step(ids[j:j + 1], cache) for j in range(6)]))
        if same:
            assert torch.equal(*out)
        else:
            assert rel(out[1], out[0]) < 1e-2, rel(out[1], out[0])


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n", [20, 700, 1950])
def test_captured_drafted_steps_over_a_long_cache(tiny, bits, n):
    """A cache of 2000 rows: its ranges at a position that fills one of them, a few, all."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    m = Q.FusedQwen3(args, state, packed)
    tree = DraftTree([-1, 0, 0, 1, 1, 2, 3, 3, 0])
    tokens = ids_of(args, 9, 5)
    out = []
    for graphs in (False, True):
        cache = m.make_cache(2000, bits=bits)
        m.hidden(ids_of(args, n, 4), cache)
        dec = Q.DraftQwen3(m, graphs=graphs)
        for _ in range(2):   # the step again over the same rows: captured, replayed
            logits = dec.step(tokens, tree, cache)[3]
            for c in cache:
                c.offset = n
        out.append(logits)
    assert rel(out[1], out[0]) < 1e-2, rel(out[1], out[0])
    # node 6's line is a prefill's
    line = [0, 1, 3, 6]
    cache = m.make_cache(2000, bits=bits)
    m.hidden(ids_of(args, n, 4), cache)
    ref = m(tokens[line], cache)
    assert rel(out[1][line], ref) < 3e-2, rel(out[1][line], ref)


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_places_without_a_draft(tiny, graphs, temperature):
    """Tokens outside the vocabulary are never taken and change nothing for the nodes beside them."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    from oracle import draft as O
    m = Q.FusedQwen3(args, state, packed)
    tree, V = DraftTree([-1, 0, 0, 0, 1, 2, 2]), args.vocab_size
    dec, u = Q.DraftQwen3(m, graphs=graphs), torch.rand(7, generator=torch.Generator().manual_seed(1)).cuda()
    out = []
    for none in ((-1, V, 2 ** 40, -2 ** 40), (3, 4, 5, 6)):
        cache = m.make_cache(100, bits=8)
        m.hidden(ids_of(args, 12, 6), cache)
        tokens = torch.tensor([7, none[0], 9, none[1], 11, none[2], none[3]], device="cuda")
        path, count, token, logits = dec.step(tokens, tree, cache, temperature, u)
        out.append(logits)
        want = O.verify(logits.float().cpu().numpy(), tokens.tolist(), tree.parent_list, temperature, u.cpu().numpy())
        assert (path[:int(count)].tolist(), int(token)) == want
        assert none[0] >= 0 or not set(path.tolist()) & {1, 3, 5, 6}
    assert torch.equal(out[0][[0, 2]], out[1][[0, 2]])
