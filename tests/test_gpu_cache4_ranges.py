"""Attention over 4-bit caches whose values are beside float32's largest, against float64 (oracle/draft.py)."""
import pytest
import torch

from oracle import draft as O
from oracle import mx as M
from tests.test_gpu_cache4 import BF, C, bits, check_attention, f64, gen, make_cache, tree   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("T,hq,hk,pos,splits", [(1, 1, 1, 63, 1), (1, 4, 2, 900, None), (5, 4, 2, 70, 2), (40, 8, 2, 333, 1), (17, 2, 1, 3000, 7)])
def test_values_beside_the_largest(C, T, hq, hk, pos, splits, d):   # noqa: F811
    """V's bytes up to 252: sums of weights times such values pass float32, the result, their mean, does not."""
    rnd = gen(d + pos)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    q = rnd(T, hq, d).to(BF).transpose(0, 1)
    for case in range(7):
        c = make_cache(rnd, hk, pos + T, d)
        if case == 0:      # all rows the same: 6 * 2^125
            c[0][:], c[1][:], c[3][:] = 0x00, 0x77, 252
        elif case == 1:    # random codes
            c[3][:] = 252
        elif case == 2:    # a block of them beside ordinary ones
            c[3][..., -1] = 252
        elif case == 3:    # in the last rows only: tiles before have their sums already
            c[3][:, pos // 2 + 11:] = 252
        elif case == 4:    # one row, behind scores that fall
            c[3][:, pos // 3] = 252
        elif case == 5:    # about where sums of all rows there can be begin to pass float32
            c[3][:] = torch.where(rnd(hk, pos + T, d // 32) > 0, 211, 212).to(torch.uint8)
        else:              # rows of the tree, which some nodes do not see
            c[3][:, pos:] = 252
        masks = chain if case < 6 else O.line_masks(tree(T, pos))
        out = C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=splits)
        assert torch.isfinite(out).all(), case
        check_attention(out, q, c, masks, pos, d ** -0.5)


def test_large_values_behind_scores_that_grow_and_fall(C):   # noqa: F811
    """The reference moves before and after the largest values come."""
    T, hq, hk, d, pos = 2, 2, 1, 128, 1200
    rnd = gen(3)
    q = torch.ones(T, hq, d, device="cuda", dtype=BF).transpose(0, 1)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    ramp = torch.linspace(-70, 70, pos + T)
    for shape in (ramp, ramp.flip(0), ramp.abs(), -ramp.abs()):
        for rows in (slice(0, 40), slice(580, 620), slice(1150, None), slice(0, None)):
            c = make_cache(rnd, hk, pos + T, d)
            codes, scales = M.quantize((shape / d ** 0.5)[:, None].expand(-1, d).double().numpy())
            c[0][:], c[2][:] = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
            c[3][:, rows] = 251
            for splits in (1, 4):
                out = C.attn_tree(q, *c[:2], pos, None, *c[2:], splits=splits)
                assert torch.isfinite(out).all()
                check_attention(out, q, c, chain, pos, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_values_of_rows_that_a_node_does_not_see(C, d):   # noqa: F811
    """The nodes that do not see them give the bits they give without."""
    T, hq, hk, pos = 37, 6, 2, 290
    rnd = gen(d)
    c = make_cache(rnd, hk, pos + T, d)
    q = rnd(T, hq, d).to(BF).transpose(0, 1)
    masks = O.line_masks(tree(T, 3))
    for splits in (1, 3):
        clean = C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=splits)
        large = [t.clone() for t in c]
        large[3][:, pos + 4], large[3][:, pos + 11] = 252, 250
        out = C.attn_tree(q, *large[:2], pos, bits(masks), *large[2:], splits=splits)
        check_attention(out, q, large, masks, pos, d ** -0.5)
        unseen = [i for i in range(T) if not (masks[i] >> 4 & 1 or masks[i] >> 11 & 1)]
        assert unseen and torch.equal(out[unseen], clean[unseen])
