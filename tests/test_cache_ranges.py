"""Ranges that the rows of a cache are cut into, by the cache's kind (no GPU)."""
import os

import pytest


@pytest.fixture(scope="module")
def C():
    import mxfp4_int8_m5_amd as p
    if not os.path.exists(p._lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return p.sc_cache


def test_a_kind_by_either_name(C):
    """The names of make_cache, and 4, ask the kernel of that cache."""
    from mxfp4_int8_m5_amd import _lib
    sizes = [(T, n, hq, hk, d) for T in (1, 5, 64) for n in (40, 3000, 40000) for hq, hk in ((16, 8), (32, 8), (14, 2)) for d in (64, 128, 256)]
    four, more = [_lib.load().scmx_attn_tree4_splits(*s) for s in sizes], [_lib.load().scmx_attn_tree_splits(*s) for s in sizes]
    assert four != more
    for bits, want in (("mxfp4", four), (4, four), (16, more), (8, more)):
        assert [C.attn_tree_splits(*s, bits=bits) for s in sizes] == want
    assert [C.attn_tree_splits(*s) for s in sizes] == more


@pytest.mark.parametrize("bits", ["mxfp8", 2, 32, None, "4"])
def test_other_kinds_are_refused(C, bits):
    with pytest.raises(ValueError):
        C.attn_tree_splits(1, 1000, 16, 8, 128, bits=bits)
