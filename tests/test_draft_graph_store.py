"""Host logic of the drafted steps' graph store (no GPU): the latest cache's graphs, of a bounded number of temperatures, whatever
trees, drafts and caches come by."""
import gc
import types
import weakref

import pytest
import torch


class Layer:
    def __init__(self):
        self.k, self.offset = torch.zeros(1, 4096, 64), 0


class Graph:
    def replay(self):
        pass


@pytest.fixture
def dec(monkeypatch):
    """A DraftQwen3 whose steps are captured as nothing: the store is the real one."""
    from mxfp4_int8_m5_amd import fused_qwen3 as Q
    monkeypatch.setattr(Q.S, "set_format", lambda fmt: None)
    fused = types.SimpleNamespace(epilogue="gemm", args=None, device="cpu", fmt=None, lm_head=torch.zeros(10, 4), embed=torch.zeros(10, 4))
    dec = Q.DraftQwen3(fused, graphs=True)
    dec.captured = 0

    def capture(key, fn, inputs, owner=None):
        if dec._lookup(key, owner) is None:
            dec.captured += 1
            T = inputs[0].numel()
            out = torch.full((T,), -1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64), torch.zeros(T, 10)
            dec.graphs[key] = (Graph(), [t.clone() for t in inputs], out, owner)
        return dec.graphs[key]

    monkeypatch.setattr(dec, "_capture", capture)
    return dec


def step(dec, cache, parents, temperature=0.0, drawn=False):
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    T = len(parents)
    dec.step(torch.zeros(T, dtype=torch.int64), DraftTree(parents, device="cpu"), cache, temperature, torch.zeros(T) if temperature else None,
             torch.zeros(T, 10) if drawn else None)


def test_fresh_caches_and_trees_of_several_sizes_leave_the_latest_cache(dec):
    refs = []
    for prompt in range(30):
        cache = [Layer(), Layer()]
        refs += [weakref.ref(c) for c in cache]
        for _ in range(2):
            step(dec, cache, list(range(-1, prompt % 7)))
            step(dec, cache, [-1, 0], 0.5 + prompt % 3, drawn=prompt % 2 == 1)
        assert all(e[3] is cache for e in dec.graphs.values()) and dec.captured == 2 * (prompt + 1)
        del cache
    gc.collect()
    assert sum(r() is not None for r in refs) == 2


def test_the_latest_temperatures_stay(dec):
    cache = [Layer()]
    step(dec, cache, [-1, 0])
    for t in (0.5, 0.6, 0.7, 0.8, 0.6, 0.9):
        step(dec, cache, [-1, 0], t)
        step(dec, cache, [-1, 0, 0], t)
    assert {k[3] for k in dec.graphs} == {0.0, 0.7, 0.8, 0.6, 0.9} and len(dec.graphs) == 9 and dec.captured == 11
    for t in (0.0, 0.7, 0.8, 0.6, 0.9):
        step(dec, cache, [-1, 0], t)
    assert dec.captured == 11
    for i in range(100):
        step(dec, cache, [-1, 0], 1.0 + i / 100)
    assert len(dec.graphs) == 5


def test_children_beyond_those_tried_do_not_capture_anew(dec):
    cache = [Layer()]
    for kids in (16, 17, 40, 63):
        step(dec, cache, [-1] + [0] * kids + [1] * (63 - kids), 0.5, drawn=True)
    assert dec.captured == 1
    step(dec, cache, [-1], 0.5, drawn=True)
    step(dec, cache, list(range(-1, 63)), 0.5, drawn=True)
    assert dec.captured == 3
