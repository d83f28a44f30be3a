"""KV caches in 4 bits on the GPU (include/scmx_mx.h): the append (norm, rotation, codes), the read-back, the accepted rows moved together, and
the attention of drafted tokens, each against a float64 restatement (oracle/draft.py, oracle/mx.py) at the sizes, masks and values where
it can go wrong; what each refuses."""
import numpy as np
import pytest
import torch

from oracle import draft as O
from oracle import mx as M

BF = torch.bfloat16


@pytest.fixture(scope="module")
def C():
    from mxfp4_int8_m5_amd import sc_cache
    return sc_cache


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731


def f64(t):
    return t.double().cpu().numpy()


def make_cache(rnd, hk, rows, d, spread=1.0):
    """(k, v, kscale, vscale): random codes, the blocks' scales up to `spread` powers of two apart."""
    codes = [(rnd(hk, rows, d // 2) * 1000).int().remainder(256).to(torch.uint8) for _ in range(2)]
    scales = [(125 + spread * rnd(hk, rows, d // 32)).round().to(torch.uint8) for _ in range(2)]
    return (*codes, *scales)


def values(c, s):
    return M.values(c.cpu().numpy(), s.cpu().numpy())


# ---- append and read-back ------------------------------------------------------------------------------------------------

WRITES = [(1, 1, 1, 64, 0, 1), (1, 16, 8, 128, 300, 400), (7, 14, 2, 64, 0, 7), (5, 3, 3, 256, 100000, 100005), (300, 4, 2, 128, 17, 500), (33, 16, 4, 256, 5, 38),
          (2, 40, 1, 64, 262143, 262145), (1000, 2, 5, 64, 3, 1003)]


@pytest.mark.gpu
@pytest.mark.parametrize("L,hq,hk,d,pos,rows", WRITES)
def test_cache_write(C, L, hq, hk, d, pos, rows):
    rnd, eps = gen(L + d), 2.0 ** -20
    y = (rnd(L + 1, (hq + 2 * hk) * d) * torch.exp(rnd((hq + 2 * hk) * d))).to(BF)   # one row more than tokens
    y[0, (hq + hk) * d:(hq + hk + 1) * d] = 0   # a value row of zeros
    qn, kn = (1 + 0.1 * rnd(d)).to(BF), (1 + 0.1 * rnd(d)).to(BF)
    inv = 1.0 / (1e6 ** (torch.arange(d // 2, device="cuda", dtype=torch.float32) / (d // 2)))
    depth = torch.randint(0, 5, (L,), device="cuda", dtype=torch.int32) if L < 64 else None
    c = make_cache(rnd, hk, rows, d)
    before = [t.clone() for t in c]
    q = C.cache_write(y, qn, kn, eps, L, hq, hk, d, c[0], c[1], pos, inv, c[2], c[3], depth)
    at = pos + (depth.cpu().numpy() if depth is not None else np.arange(L))
    rq, rk, rv, mag = O.normed_rows(f64(y), f64(qn), f64(kn), eps, hq, hk, d, at, f64(inv))
    assert q.shape == (hq, L, d) and q.transpose(0, 1).is_contiguous()
    # float64 rounded through float32 (2^-24) to bf16 (2^-8); angles of 1e5 in turns off by 2^-37
    assert (np.abs(f64(q).transpose(1, 0, 2) - rq) <= (2.0 ** -8 + 2.0 ** -23) * np.abs(rq) + 2.0 ** -33 * mag[:, :hq]).all()
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[pos:pos + L] = False
    for i, (ref, least, most) in enumerate(((rk, 10, 252), (rv, 0, 254))):
        codes, scales = M.quantize(ref.transpose(1, 0, 2), least, most)
        got, bytes_ = (t[:, pos:pos + L].cpu().numpy() for t in (c[i], c[2 + i]))
        assert (bytes_ == scales).all() and (got == codes).all()   # the definition's codes, borders and all
        for t, o in ((c[i], before[i]), (c[2 + i], before[2 + i])):
            assert torch.equal(t[:, keep], o[:, keep])             # the other rows: as they were
    n = min(rows, pos + L + 1)
    kb, vb = C.cache_read(*c, n - pos, pos)
    for b, i in ((kb, 0), (vb, 1)):
        assert b.shape == (hk, n - pos, d) and np.array_equal(f64(b), values(c[i], c[2 + i])[:, pos:n])


@pytest.mark.gpu
def test_cache_write_from_accumulators(C):
    """acc with its scales gives what the bf16 rows made of them give."""
    rnd, hq, hk, d, L = gen(3), 4, 2, 128, 9
    acc = (rnd(L, (hq + 2 * hk) * d) * 20000).to(torch.int32)
    xs, ws = torch.rand(L, device="cuda") * 1e-2, torch.rand((hq + 2 * hk) * d, device="cuda") * 1e-2
    y = (acc.float() * xs[:, None] * ws).to(BF)
    n = torch.ones(d, device="cuda", dtype=BF)
    inv = torch.rand(d // 2, device="cuda")
    outs = []
    for kw in ({"y": y}, {"y": None, "acc": acc, "xscale": xs, "wscale": ws}):
        k, v, ks, vs = make_cache(gen(4), hk, 20, d)
        q = C.cache_write(kw.pop("y"), n, n, 1e-6, L, hq, hk, d, k, v, 3, inv, ks, vs, **kw)
        outs.append((q, k, v, ks, vs))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.gpu
def test_rows_that_are_not_finite_and_tiny_ones(C):
    """A block of a value row with an infinity or NaN is NaN, the other blocks are themselves; a key row with one is NaN; tiny and huge
    values stand."""
    d, L = 64, 5
    y = torch.ones(L, 3 * d, device="cuda", dtype=BF)
    y[0, 2 * d + 5] = float("inf")
    y[1, 2 * d + 63] = float("nan")
    y[2, 2 * d:] = 2.0 ** -120
    y[3, 2 * d:] = 3.0e38
    y[1, d] = float("nan")
    n, inv = torch.ones(d, device="cuda", dtype=BF), torch.zeros(d // 2, device="cuda")
    k, v, ks, vs = make_cache(gen(1), 1, L, d)
    C.cache_write(y, n, n, 1e-6, L, 1, 1, d, k, v, 0, inv, ks, vs)
    kb, vb = C.cache_read(k, v, ks, vs, L)
    assert torch.isnan(vb[0, 0, :32]).all() and (vb[0, 0, 32:] == 1).all() and torch.isnan(vb[0, 1, 32:]).all() and (vb[0, 1, :32] == 1).all()
    assert torch.isnan(kb[0, 1]).all() and torch.isfinite(kb[0, [0, 2, 3, 4]]).all()
    assert (vb[0, 2] == 2.0 ** -120).all() and (vb[0, 3] == 6 * 2.0 ** 125).all() and (vb[0, 4] == 1).all()


@pytest.mark.gpu
def test_a_device_position_outside_the_cache_appends_and_moves_nothing(C):
    hq, hk, d, rows = 2, 1, 64, 12
    y = gen(2)(4, 4 * d).to(BF)
    n, inv = torch.ones(d, device="cuda", dtype=BF), torch.ones(d // 2, device="cuda")
    for bad in (-1, rows - 3, 2 ** 40):
        c = make_cache(gen(5), hk, rows, d)
        old = [t.clone() for t in c]
        pos = torch.tensor([bad], device="cuda")
        q = C.cache_write(y, n, n, 1e-6, 4, hq, hk, d, c[0], c[1], pos, inv, c[2], c[3])
        C.cache_keep([c], torch.tensor([1, 2, 3, 0], device="cuda", dtype=torch.int32), torch.tensor([4], device="cuda", dtype=torch.int32), pos)
        assert not C.attn_tree(q, c[0], c[1], pos, None, c[2], c[3], splits=2).any()
        assert all(torch.equal(a, b) for a, b in zip(c, old))


@pytest.mark.gpu
@pytest.mark.parametrize("path,count", [([0, 2, 5, -1, -1, -1], 3), ([3, 3, 0, 1, 9, -7], 6), ([5, 4, 3, 2, 1, 0], 99), ([1, 2, 3, 4, 5, 0], -4), ([0], 1), (list(range(1, 64)) + [0], 64)])
def test_cache_keep(C, path, count):
    for layers, hk, d, pos in ((1, 2, 64, 0), (3, 1, 256, 4), (35, 2, 128, 7)):
        T = len(path)
        rows = pos + T + 3
        rnd = gen(T + layers)
        cs = [make_cache(rnd, hk, rows, d) for _ in range(layers)]
        old = [[t.clone() for t in c] for c in cs]
        C.cache_keep(cs, torch.tensor(path, device="cuda", dtype=torch.int32), torch.tensor([count], device="cuda", dtype=torch.int32), pos)
        src = [pos + p if j < count and 0 <= p < T else pos + j for j, p in enumerate(path)]
        src = list(range(pos)) + src + list(range(pos + T, rows))
        for c, o in zip(cs, old):
            for a, b in zip(c, o):
                assert torch.equal(a, b[:, src])


# ---- attention -----------------------------------------------------------------------------------------------------------

def tree(T, seed):
    rng = np.random.default_rng(seed)
    return [-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, T)]


def bits(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device="cuda")


def check_attention(out, q, cache, masks, pos, scale):
    d = 2 * cache[0].shape[2]
    T, hq = q.shape[1], q.shape[0]
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    ref, mag = O.attention(f64(q).transpose(1, 0, 2), k, v, masks, pos, scale)
    got = f64(out).reshape(T, hq, d)
    # the weights' rounding to bf16 (2^-8 in numerator and denominator) and the result's (2^-8); the queries' two parts (2^-23 of a block's
    # largest value), scores in float32 and the exponential's last bits are some 2^-16 of a weight, far below the five per cent
    tol = 1.05 * (2.0 ** -8 * mag + 2.0 ** -7 * np.abs(ref)) + 1e-30
    assert got.shape == ref.shape and (np.abs(got - ref) <= tol).all(), np.max(np.abs(got - ref) / tol)


# T, hq, hk, d, pos, splits: one row in all, ends inside and at the borders of tiles of 32 keys, trees across two and three tiles,
# one and several blocks of query rows, rows past the last query, a range per tile group and empty ranges
ATTEND = [(1, 1, 1, 64, 0, 1), (1, 16, 8, 128, 300, None), (1, 14, 2, 64, 31, 1), (2, 2, 1, 128, 30, 2), (7, 14, 2, 64, 901, None), (16, 16, 8, 128, 1000, 3),
          (17, 2, 2, 128, 31, 1), (33, 4, 4, 128, 64, 1), (64, 8, 2, 128, 500, None), (64, 32, 2, 64, 95, 2), (5, 16, 4, 256, 256, None), (64, 4, 2, 256, 33, 2),
          (64, 3, 3, 128, 0, 1), (40, 8, 1, 128, 1, 64), (3, 8, 8, 256, 2500, 9), (12, 5, 1, 64, 2047, 7), (1, 32, 8, 128, 5000, 20),
          (9, 4, 2, 128, 700, 64), (2, 6, 2, 256, 1200, 40), (1, 4, 2, 128, 20000, None)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,hq,hk,d,pos,splits", ATTEND)
def test_attn_tree(C, T, hq, hk, d, pos, splits):
    rnd = gen(T * 1000 + pos)
    c = make_cache(rnd, hk, pos + T + 5, d)
    q = (1.5 * rnd(T, hq, d)).to(BF).transpose(0, 1)
    for s in c[2:]:
        s[:, pos + T:] = 255   # rows behind the tree hold anything
    masks = O.line_masks(tree(T, pos))
    check_attention(C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=splits), q, c, masks, pos, d ** -0.5)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    out = C.attn_tree(q.contiguous(), *c[:2], pos, None, *c[2:], scale=0.11, splits=splits)   # another layout of q, the default mask
    check_attention(out, q, c, chain, pos, 0.11)
    dev = C.attn_tree(q, *c[:2], torch.tensor([pos], device="cuda"), None, *c[2:], scale=0.11, splits=splits)
    if splits is not None:
        assert torch.equal(dev, out)   # the same ranges: the same bits
    else:
        check_attention(dev, q, c, chain, pos, 0.11)


@pytest.mark.gpu
@pytest.mark.parametrize("pos,splits", [(0, 1), (3, 1), (700, 3)])
def test_any_mask_and_nodes_that_see_nothing(C, pos, splits):
    """Masks that are no tree: empty ones (without rows below them: zeros), ones without the node itself, all ones."""
    T, hq, hk, d = 20, 4, 2, 128
    rnd = gen(pos)
    c = make_cache(rnd, hk, pos + T, d)
    q = rnd(T, hq, d).to(BF).transpose(0, 1)
    rng = np.random.default_rng(1)
    masks = [0, (1 << T) - 1, 1 << 19, 0] + [int(rng.integers(0, 1 << T)) for _ in range(T - 4)]
    masks[6] |= ((1 << 44) - 1) << T   # bits beyond the tree say nothing
    out = C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=splits)
    check_attention(out, q, c, [m & (1 << T) - 1 for m in masks], pos, d ** -0.5)
    assert pos or not out[[0, 3]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("pos", [0, 29, 290])
def test_what_a_node_does_not_see_does_not_reach_it(C, pos, d):
    """NaN blocks in rows of the tree: the nodes that do not see them give the bits they give without; those that do, NaN: everywhere of a
    key's, in the block's dimensions of a value's."""
    T, hq, hk = 37, 6, 2
    rnd = gen(7)
    c = make_cache(rnd, hk, pos + T, d)
    q = rnd(T, hq, d).to(BF).transpose(0, 1)
    masks = O.line_masks(tree(T, 3))
    clean = C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=2).view(T, hk, hq // hk, d // 32, 32)
    last = d // 32 - 1
    c[2][0, pos + 4, 1], c[3][0, pos + 11, last], c[3][1, pos + 36, 0] = 255, 255, 255
    out = C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=2).view(T, hk, hq // hk, d // 32, 32)
    for i in range(T):
        sees = [masks[i] >> b & 1 for b in (4, 11, 36)]
        for h in range(hk):
            for blk in range(d // 32):
                nan = (h == 0 and sees[0]) or (h == 0 and sees[1] and blk == last) or (h == 1 and sees[2] and blk == 0)
                assert torch.isnan(out[i, h, :, blk]).all() if nan else torch.equal(out[i, h, :, blk], clean[i, h, :, blk])


@pytest.mark.gpu
def test_scores_that_grow_and_fall_along_the_rows(C):
    """The reference moves many times, or never after the first tile; one row holds nearly all weight; scales far apart."""
    T, hq, hk, d, pos = 4, 4, 2, 64, 1500
    rnd = gen(9)
    q = torch.ones(T, hq, d, device="cuda", dtype=BF).transpose(0, 1)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    ramp = torch.linspace(-60, 60, pos + T, device="cuda")
    for shape in (ramp, ramp.flip(0), ramp.abs() * 3, torch.where(torch.arange(pos + T, device="cuda") == 777, 90.0, 0.0)):
        c = make_cache(rnd, hk, pos + T, d, 6.0)
        rows = (shape / d ** 0.5)[:, None].expand(-1, d).cpu().double().numpy()
        codes, scales = M.quantize(rows)
        c[0][:], c[2][:] = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
        c[3][:, 40:60] = 60
        check_attention(C.attn_tree(q, *c[:2], pos, None, *c[2:], splits=4), q, c, chain, pos, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -30, 1.0, 2.0 ** 20, 2.0 ** 60])
def test_queries_of_any_size(C, size, d):
    """Queries far from one, small blocks beside large ones, values of all eight bits, and one of infinities beside finite ones."""
    T, hq, hk, pos = 6, 4, 2, 200
    rnd = gen(21)
    c = make_cache(rnd, hk, pos + T, d)
    q = rnd(T, hq, d)
    q[1] *= 2.0 ** -12
    q[2, :, 32:] *= 2.0 ** -9
    q[3] = q[3].sign() * (1 + 127 / 128)
    q = (q * size).to(BF).transpose(0, 1)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    check_attention(C.attn_tree(q, *c[:2], pos, None, *c[2:], scale=0.09 / size), q, c, chain, pos, 0.09 / size)
    if size == 2.0 ** 20:
        q = rnd(T, hq, d).to(BF).transpose(0, 1)
        bad = q.clone()
        bad[:, 2, 5], bad[:, 4, d - 1] = float("inf"), float("nan")
        a, b = (C.attn_tree(x, *c[:2], pos, None, *c[2:]) for x in (q, bad))
        assert torch.isnan(b[2]).all() and torch.isnan(b[4]).all()
        b[2], b[4] = a[2], a[4]
        check_attention(b, q, c, chain, pos, d ** -0.5)


@pytest.mark.gpu
def test_a_score_keeps_the_bits_of_its_query(C):
    """Scores of two keys that differ in the last bits of a query: the weights' ratio tells them from queries of four bits."""
    d = 128
    q = torch.zeros(1, 1, d, device="cuda")
    q[0, 0, :32] = torch.linspace(1.0, 1.9921875, 32, device="cuda")   # eight bits
    q[0, 0, 32:] = q[0, 0, :32].repeat(3) * 2.0 ** -7
    q = q.to(BF)
    k = np.zeros((1, 2, d))
    k[0, 0], k[0, 1, ::2], k[0, 1, 1::2] = 1.0, 3.0, -1.0
    v = np.zeros((1, 2, d))
    v[0, 0] = 1.0
    parts = [torch.from_numpy(t).cuda() for x in (k, v) for t in M.quantize(x)]
    c = (parts[0], parts[2], parts[1], parts[3])
    f = f64(q)[0, 0]
    diff = (k[0, 0] @ f - k[0, 1] @ f) * 0.05
    out = C.attn_tree(q.transpose(0, 1), c[0], c[1], 1, None, c[2], c[3], scale=0.05)
    want = 1 / (1 + np.exp(-diff))
    # both weights and the result round to bf16: 2^-8 each; a query of four bits would be off by 2^-5 of sum |q k| * 0.05 = 0.15 and more
    assert np.abs(f64(out) - want).max() <= 1.02 * 3 * 2.0 ** -8 * want


@pytest.mark.gpu
def test_a_cache_longer_than_32_bits_of_bytes(C):
    """The last KV head's rows lie beyond 2^32 bytes; reading, writing and moving there."""
    hk, d = 3, 256
    rows = (2 ** 32 // (d // 2)) * 5 // 8   # two heads end beyond 2^32 bytes
    T, hq, pos = 3, 3, rows - 40
    c = tuple(torch.zeros((hk, rows, n), dtype=torch.uint8, device="cuda") for n in (d // 2, d // 2, d // 32, d // 32))
    small = make_cache(gen(11), hk, 40, d)
    for s in c[2:]:
        s[:] = 127
    for big, s in zip(c, small):
        big[:, rows - 40:] = s
    q = (2 * gen(12)(T, hq, d)).to(BF).transpose(0, 1)
    out = f64(C.attn_tree(q, *c[:2], pos, None, *c[2:])).reshape(T, hq, d)
    k, v = values(small[0], small[2]), values(small[1], small[3])
    for i in range(T):
        for h in range(hq):
            s = k[h, :i + 1] @ f64(q)[h, i] * d ** -0.5   # rows before the tree are zeros: score 0, value 0
            top = max(s.max(), 0)
            p = np.exp(s - top)
            den = p.sum() + pos * np.exp(-top)
            ref, mag = p @ v[h, :i + 1] / den, p @ np.abs(v[h, :i + 1]) / den
            # rounded weights of 1 in a float32 denominator of millions: sums of ones are exact to 2^24 a lane
            assert (np.abs(out[i, h] - ref) <= 1.05 * (2.0 ** -8 * mag + 2.0 ** -7 * np.abs(ref)) + 1e-30).all()
    kb, vb = C.cache_read(*c, 40, rows - 40)
    assert np.array_equal(f64(kb), k) and np.array_equal(f64(vb), v)
    C.cache_keep([c], torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda"), torch.tensor([2], dtype=torch.int32, device="cuda"), pos)
    assert all(torch.equal(b[:, pos:], s[:, [2, 0, 2] + list(range(3, 40))]) for b, s in zip(c, small))
    y = gen(13)(T, (hq + 2 * hk) * d).to(BF)
    one = torch.ones(d, device="cuda", dtype=BF)
    C.cache_write(y, one, one, 1e-6, T, hq, hk, d, c[0], c[1], pos, torch.zeros(d // 2, device="cuda"), c[2], c[3])
    kb, vb = C.cache_read(*c, T, pos)
    assert np.array_equal(f64(vb), M.values(*M.quantize(f64(y).reshape(T, -1, d)[:, hq + hk:].transpose(1, 0, 2))))


@pytest.mark.gpu
def test_refusals(C):
    z = lambda *s, t=torch.uint8: torch.zeros(*s, dtype=t, device="cuda")   # noqa: E731
    k, v, ks, vs = z(2, 8, 32), z(2, 8, 32), z(2, 8, 2), z(2, 8, 2)
    q = z(2, 1, 64, t=BF)
    n, inv, y = z(64, t=BF), z(32, t=torch.float32), z(1, 384, t=BF)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    write = lambda k, v, ks, vs, pos=0: C.cache_write(y, n, n, 1e-6, 1, 2, 2, 64, k, v, pos, inv, ks, vs)   # noqa: E731
    f32 = z(2, 8, t=torch.float32)
    bad = [lambda: C.attn_tree(q, k, v, 0, None, ks, z(2, 8, 1)), lambda: C.attn_tree(q, k, v, 0, None, ks, None), lambda: C.attn_tree(q, k, v, 8, None, ks, vs),
           lambda: C.attn_tree(q, k, v, 0, None, ks, f32), lambda: C.attn_tree(q, k, v, 0, None, f32, f32), lambda: C.attn_tree(q, k, v, 0), lambda: C.attn_tree(q, z(2, 8, 24), z(2, 8, 24), 0, None, ks, vs),
           lambda: C.attn_tree(z(2, 65, 64, t=BF), z(2, 80, 32), z(2, 80, 32), 0, None, z(2, 80, 2), z(2, 80, 2)), lambda: C.attn_tree(z(2, 1, 96, t=BF), z(2, 8, 48), z(2, 8, 48), 0, None, z(2, 8, 3), z(2, 8, 3)),
           lambda: C.attn_tree(q, k, v, 0, None, ks, vs, splits=65), lambda: C.attn_tree(q, k, v, 0, None, ks, vs, scale=float("nan")), lambda: C.attn_tree(q, k.cpu(), v, 0, None, ks, vs),
           lambda: C.cache_read(k, v, ks, vs, 9), lambda: C.cache_read(k, v, ks, vs, 2, 7), lambda: C.cache_read(k, v, ks, vs, 1, -1), lambda: C.cache_read(k, v, z(2, 8, 4), vs, 1),
           lambda: write(k, k, ks, vs), lambda: write(k, v, ks, ks), lambda: write(k, v, ks, vs, 8), lambda: write(k, v, ks, vs, -1), lambda: write(z(1, 8, 32), v, ks, vs), lambda: write(k, v, f32, f32),
           lambda: C.cache_keep([(k, v, ks, vs), (z(2, 8, 64, t=torch.int8), z(2, 8, 64, t=torch.int8), f32, f32.clone())], i32(0), i32(1), 0), lambda: C.cache_keep([(k, v, ks, vs)] * 2, i32(0), i32(1), 0),
           lambda: C.cache_keep([(k, v, ks, ks)], i32(0), i32(1), 0), lambda: C.cache_keep([(k, v, ks, vs)], i32(*range(9)), i32(1), 0)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")


@pytest.mark.gpu
def test_captured_steps_over_two_caches(C):
    """Append and attention of a tree captured with the position on the device, replayed along a growing cache between eager steps over
    another one: each replay gives the eager bits."""
    T, hq, hk, d, rows = 5, 8, 2, 128, 900
    rnd = gen(31)
    n, inv = torch.ones(d, device="cuda", dtype=BF), torch.rand(d // 2, device="cuda")
    a, b = (make_cache(gen(32), hk, rows, d) for _ in range(2))
    y, pos = torch.zeros(T, (hq + 2 * hk) * d, device="cuda", dtype=BF), torch.zeros(1, dtype=torch.int64, device="cuda")
    mask = bits(O.line_masks(tree(T, 1)))

    def step(c, at):
        q = C.cache_write(y, n, n, 1e-6, T, hq, hk, d, c[0], c[1], at, inv, c[2], c[3])
        return C.attn_tree(q, *c[:2], at, mask, *c[2:], splits=6)

    step(a, pos)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(a, pos)
    for i, at in enumerate((0, 5, 400, 700, 895)):
        y.copy_(rnd(T, (hq + 2 * hk) * d))
        pos.fill_(at)
        g.replay()
        want = step(b, at)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(s[:, at:at + T], t[:, at:at + T]) for s, t in zip(a, b))
