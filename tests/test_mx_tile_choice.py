"""The tile that products of MXFP4 operands take on 256 CUs, recomputed from the constants of the source: the sizes of test_gpu_mx_tiles.py
take the tiles that they are listed under, several a workgroup, and every form of each tile is among them."""
import os
import re

import pytest

from tests.test_gpu_mx_tiles import TILES

CUS = 256
with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mxfp4-int8-m5_amd", "csrc", "mx_gemm.hip")) as f:
    SOURCE = f.read()
RULE = SOURCE[SOURCE.index("static int tile_of("):SOURCE.index('extern "C" int scmx_mx_mm(')]
FEW = int(re.search(r"constexpr int FEW = (\d+);", SOURCE).group(1))


def numbers(name):
    return [float(x) for x in re.search(name + r"\[4\] = \{([^}]*)\}", RULE).group(1).split(",")]


BM, BN, ALONE, ALONE_ENDS, FULL, FULL_ENDS = (numbers(n) for n in (r"\bBM", r"\bBN", r"\bALONE", "ALONE_ENDS", r"\bFULL", "FULL_ENDS"))
FEW_STAGE, FEW_ENDS = (float(x) for x in re.search(r"\(([\d.]+) \* stages \+ ([\d.]+)\);", RULE).groups())
ODD_ALONE, ODD_FULL = (float(x) for x in re.findall(r"words \? 0 : ([\d.]+)", RULE))


def tile(m, n, k, words):
    """(rows, columns) of the tile, or None for the kernel of few rows."""
    if m <= FEW or k // 32 * min(m, n) < 16:
        return None
    up = lambda a, b: -(-a // b)   # noqa: E731
    stages, best = up(k, 256), None
    least = max(up(m, 16) * up(n, 16) / CUS, 1) * (FEW_STAGE * stages + FEW_ENDS)
    for i in range(3 if n % 16 or not words else 4):
        tiles = up(m, int(BM[i])) * up(n, int(BN[i]))
        load = tiles / CUS if tiles < CUS else up(tiles, CUS)
        us = max((ALONE[i] + (0 if words else ODD_ALONE)) * stages + ALONE_ENDS[i], ((FULL[i] + (0 if words else ODD_FULL)) * stages + FULL_ENDS[i]) * load)
        if us < least:
            least, best = us, (int(BM[i]), int(BN[i]))
    return best


@pytest.mark.parametrize("bm,bn,words,m,n,k", [(bm, bn, words, *s) for bm, bn, words, sizes in TILES for s in sizes])
def test_the_sizes_take_their_tiles(bm, bn, words, m, n, k):
    assert tile(m, n, k, k % 128 == 0) == (bm, bn) and (k % 128 == 0) == words
    held = 2 if bm + bn <= 256 else 1   # workgroups a CU
    assert -(-m // bm) * -(-n // bn) > CUS * held and m % bm and m > bm


@pytest.mark.parametrize("bm,bn,words,sizes", TILES)
def test_every_form_is_reached(bm, bn, words, sizes):
    stages = {-(-k // 256) for _, _, k in sizes}
    assert {s % 2 for s in stages} == {0, 1} or bm + bn == 512 and {5, 6, 8} <= stages
    assert any(k % 256 for _, _, k in sizes) and (bm + bn == 512 or 1 in stages)
    rest = {n % 16 if n % 4 == 0 else "odd" for _, n, _ in sizes}
    assert rest == {0} if bm + bn == 512 else {0, "odd"} <= rest and rest & {4, 12}
