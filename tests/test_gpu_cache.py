"""KV caches in bf16 and 8 bits on the GPU: the append (norm, rotation, quantisation), the read-back, the accepted rows moved together,
and the attention of drafted tokens, each against a float64 restatement (oracle/draft.py) at the sizes, masks and values where it can go
wrong; what each refuses."""
import numpy as np
import pytest
import torch

from oracle import draft as O

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


def make_cache(rnd, eight, hk, rows, d, spread=0.0):
    """(k, v, kscale, vscale) of random rows, in 8 bits with scales up to `spread` powers of two apart."""
    if not eight:
        return rnd(hk, rows, d).to(BF), rnd(hk, rows, d).to(BF), None, None
    codes = [(rnd(hk, rows, d) * 42).round().clamp(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [torch.exp2(spread * rnd(hk, rows)) / 40 for _ in range(2)]
    return (*codes, *scales)


def values(c, s):
    return f64(c) if s is None else f64(c) * f64(s)[..., None]


# ---- append and read-back ------------------------------------------------------------------------------------------------

WRITES = [(1, 1, 1, 64, 0, 1), (1, 16, 8, 128, 300, 400), (7, 14, 2, 64, 0, 7), (5, 3, 3, 256, 100000, 100005), (300, 4, 2, 128, 17, 500), (33, 16, 4, 256, 5, 38),
          (2, 40, 1, 64, 262143, 262145)]


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("L,hq,hk,d,pos,rows", WRITES)
def test_cache_write(C, L, hq, hk, d, pos, rows, eight):
    rnd = gen(L + d)
    y = (rnd(L + 1, (hq + 2 * hk) * d) * torch.exp(rnd((hq + 2 * hk) * d))).to(BF)   # one row more than tokens
    y[0, (hq + hk) * d:(hq + hk + 1) * d] = 0   # a value row of zeros
    qn, kn = (1 + 0.1 * rnd(d)).to(BF), (1 + 0.1 * rnd(d)).to(BF)
    inv = 1.0 / (1e6 ** (torch.arange(d // 2, device="cuda", dtype=torch.float32) / (d // 2)))
    depth = torch.randint(0, 5, (L,), device="cuda", dtype=torch.int32) if L < 64 else None
    k, v, ks, vs = make_cache(rnd, eight, hk, rows, d)
    before = [None if t is None else t.clone() for t in (k, v, ks, vs)]
    q = C.cache_write(y, qn, kn, 1e-6, L, hq, hk, d, k, v, pos, inv, ks, vs, depth)
    at = pos + (depth.cpu().numpy() if depth is not None else np.arange(L))
    rq, rk, rv, mag = O.normed_rows(f64(y), f64(qn), f64(kn), 1e-6, hq, hk, d, at, f64(inv))
    # float32: the norm's sum, square root, quotient and products are a few 2^-24 of each operand of the rotation, sine and cosine
    # 2^-23 of it beside; 2^-20 of what went in covers them.  Then one rounding: bf16 2^-8, a code half a scale.
    f32 = 2.0 ** -20 * mag
    assert q.shape == (hq, L, d) and q.transpose(0, 1).is_contiguous()
    assert (np.abs(f64(q).transpose(1, 0, 2) - rq) <= 2.0 ** -8 * np.abs(rq) + 1.01 * f32[:, :hq] + 1e-30).all()
    for new, scales, ref, err, old, olds in ((k, ks, rk, f32[:, hq:], before[0], before[2]), (v, vs, rv, 0 * rv, before[1], before[3])):
        ref, err = ref.transpose(1, 0, 2), err.transpose(1, 0, 2)
        got = values(new, scales)[:, pos:pos + L]
        if eight:
            _, s = O.quantize_rows(ref)
            assert np.allclose(f64(scales)[:, pos:pos + L], s, rtol=2.0 ** -22 + 2.0 ** -18, atol=0)
            # half a step of the scale, the scale's and the quotient's float32 roundings on 127 steps
            assert (np.abs(got - ref) <= s[..., None] * (0.5 + 127 * 2.0 ** -17) + 1.01 * err).all()
            keep = torch.ones(rows, dtype=torch.bool, device="cuda")
            keep[pos:pos + L] = False
            assert torch.equal(scales[:, keep], olds[:, keep])
        else:
            assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 1.01 * err + 1e-30).all()
        assert torch.equal(new[:, :pos], old[:, :pos]) and torch.equal(new[:, pos + L:], old[:, pos + L:])   # the other rows: as they were
    if not eight:
        assert torch.equal(v[:, pos:pos + L], y[:L].view(L, hq + 2 * hk, d)[:, hq + hk:].transpose(0, 1))   # values pass unchanged
    else:
        n = min(rows, pos + L + 1)
        kb, vb = C.cache_read(k, v, ks, vs, n - pos, pos)
        for b, c, s in ((kb, k, ks), (vb, v, vs)):
            ref = values(c, s)[:, pos:n]
            assert b.shape == (hk, n - pos, d) and (np.abs(f64(b) - ref) <= 2.0 ** -8 * np.abs(ref) * (1 + 2.0 ** -15)).all()


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
        k, v, ks, vs = make_cache(gen(4), True, hk, 20, d)
        q = C.cache_write(kw.pop("y"), n, n, 1e-6, L, hq, hk, d, k, v, 3, inv, ks, vs, **kw)
        outs.append((q, k, v, ks, vs))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.gpu
def test_rows_that_are_not_finite_and_tiny_ones(C):
    """8 bits: a row with an infinity or NaN has the scale NaN and reads back as NaN; one below 2^-100 is zeros; the row beside it is
    untouched by either.  bf16: as they are."""
    hq = hk = 1
    d, L = 64, 5
    y = torch.ones(L, 3 * d, device="cuda", dtype=BF)
    y[0, 2 * d + 5] = float("inf")
    y[1, 2 * d + 63] = float("nan")
    y[2, 2 * d:] = 2.0 ** -110
    y[3, 2 * d:] = 3.0e38
    y[1, d] = float("nan")
    n, inv = torch.ones(d, device="cuda", dtype=BF), torch.zeros(d // 2, device="cuda")
    k, v, ks, vs = make_cache(gen(1), True, hk, L, d)
    C.cache_write(y, n, n, 1e-6, L, hq, hk, d, k, v, 0, inv, ks, vs)
    kb, vb = C.cache_read(k, v, ks, vs, L)
    assert torch.isnan(vb[0, :2]).all() and torch.isnan(kb[0, 1]).all() and torch.isfinite(kb[0, [0, 2, 3, 4]]).all()
    assert not vb[0, 2].any() and vs[0, 2] == 0 and torch.equal(vb[0, 3], y[3, 2 * d:]) and (vb[0, 4] == 1).all()
    k, v, _, _ = make_cache(gen(1), False, hk, L, d)
    C.cache_write(y, n, n, 1e-6, L, hq, hk, d, k, v, 0, inv)
    assert torch.equal(v[0].nan_to_num(7), y[:, 2 * d:].nan_to_num(7))


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_a_device_position_outside_the_cache_appends_and_moves_nothing(C, eight):
    hq, hk, d, rows = 2, 1, 64, 12
    y = gen(2)(4, 4 * d).to(BF)
    n, inv = torch.ones(d, device="cuda", dtype=BF), torch.ones(d // 2, device="cuda")
    for bad in (-1, rows - 3, 2 ** 40):
        c = make_cache(gen(5), eight, hk, rows, d)
        old = [None if t is None else t.clone() for t in c]
        pos = torch.tensor([bad], device="cuda")
        q = C.cache_write(y, n, n, 1e-6, 4, hq, hk, d, c[0], c[1], pos, inv, c[2], c[3])
        C.cache_keep([c], torch.tensor([1, 2, 3, 0], device="cuda", dtype=torch.int32), torch.tensor([4], device="cuda", dtype=torch.int32), pos)
        assert not C.attn_tree(q, c[0], c[1], pos, None, c[2], c[3], splits=2).any()
        assert all(a is None or torch.equal(a, b) for a, b in zip(c, old))


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("path,count", [([0, 2, 5, -1, -1, -1], 3), ([3, 3, 0, 1, 9, -7], 6), ([5, 4, 3, 2, 1, 0], 99), ([1, 2, 3, 4, 5, 0], -4), ([0], 1), (list(range(1, 64)) + [0], 64)])
def test_cache_keep(C, path, count, eight):
    for layers, hk, d, pos in ((1, 2, 64, 0), (3, 1, 256, 4), (35, 2, 128, 7)):
        T = len(path)
        rows = pos + T + 3
        rnd = gen(T + layers)
        cs = [make_cache(rnd, eight, hk, rows, d) for _ in range(layers)]
        old = [[None if t is None else t.clone() for t in c] for c in cs]
        C.cache_keep(cs, torch.tensor(path, device="cuda", dtype=torch.int32), torch.tensor([count], device="cuda", dtype=torch.int32), pos)
        src = [pos + p if j < count and 0 <= p < T else pos + j for j, p in enumerate(path)]
        src = list(range(pos)) + src + list(range(pos + T, rows))
        for c, o in zip(cs, old):
            for a, b in zip(c, o):
                assert a is None or torch.equal(a, b[:, src])


# ---- attention -----------------------------------------------------------------------------------------------------------

def tree(T, seed):
    rng = np.random.default_rng(seed)
    return [-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, T)]


def bits(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device="cuda")


def check_attention(out, q, cache, masks, pos, scale, eight):
    hk, _, d = cache[0].shape
    T, hq = q.shape[1], q.shape[0]
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    ref, mag = O.attention(f64(q).transpose(1, 0, 2), k, v, masks, pos, scale)
    got = f64(out).reshape(T, hq, d)
    # the weights' rounding (bf16 2^-8 in numerator and denominator, half precision 2^-11 in the numerator; below its normal
    # range 2^-25 of weights whose largest is 2^8 or more) and the result's (2^-8); scores in float32 and the exponential's last
    # bits are some 2^-16 of a weight, far below the five per cent
    w = 2.0 ** -11 if eight else 2.0 ** -8
    tol = 1.05 * (w * mag + (2.0 ** -8 + (0 if eight else 2.0 ** -8)) * np.abs(ref)) + (2.0 ** -33 * (pos + T) * np.abs(v[:, :pos + T]).max() if eight else 0) + 1e-30
    assert got.shape == ref.shape and (np.abs(got - ref) <= tol).all(), np.max(np.abs(got - ref) / tol)


# T, hq, hk, d, pos, splits: one row in all, ends inside and at the borders of tiles of 32 keys, trees across two and three tiles,
# one and several blocks of query rows, rows past the last query, a range per tile group and empty ranges
ATTEND = [(1, 1, 1, 64, 0, 1), (1, 16, 8, 128, 300, None), (1, 14, 2, 64, 31, 1), (2, 2, 1, 128, 30, 2), (7, 14, 2, 64, 901, None), (16, 16, 8, 128, 1000, 3),
          (17, 2, 2, 128, 31, 1), (33, 4, 4, 128, 64, 1), (64, 8, 2, 128, 500, None), (64, 32, 2, 64, 95, 2), (5, 16, 4, 256, 256, None), (64, 4, 2, 256, 33, 2),
          (64, 3, 3, 128, 0, 1), (40, 8, 1, 128, 1, 64), (3, 8, 8, 256, 2500, 9), (12, 5, 1, 64, 2047, 7), (1, 32, 8, 128, 5000, 20),
          (9, 4, 2, 128, 700, 64), (2, 6, 2, 256, 1200, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("T,hq,hk,d,pos,splits", ATTEND)
def test_attn_tree(C, T, hq, hk, d, pos, splits, eight):
    rnd = gen(T * 1000 + pos)
    rows = pos + T + 5
    c = make_cache(rnd, eight, hk, rows, d, 1.0)
    q = (1.5 * rnd(T, hq, d)).to(BF).transpose(0, 1)
    # rows behind the tree hold anything
    if eight:
        c[2][:, pos + T:], c[3][:, pos + T:] = float("nan"), float("inf")
    else:
        c[0][:, pos + T:], c[1][:, pos + T:] = float("nan"), float("inf")
    masks = O.line_masks(tree(T, pos))
    check_attention(C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=splits), q, c, masks, pos, d ** -0.5, eight)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    out = C.attn_tree(q.contiguous(), *c[:2], pos, None, *c[2:], scale=0.11, splits=splits)   # another layout of q, the default mask
    check_attention(out, q, c, chain, pos, 0.11, eight)
    dev = C.attn_tree(q, *c[:2], torch.tensor([pos], device="cuda"), None, *c[2:], scale=0.11, splits=splits)
    if splits is not None:
        assert torch.equal(dev, out)   # the same ranges: the same bits
    else:
        check_attention(dev, q, c, chain, pos, 0.11, eight)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("pos,splits", [(0, 1), (3, 1), (700, 3)])
def test_any_mask_and_nodes_that_see_nothing(C, eight, pos, splits):
    """Masks that are no tree: empty ones (without rows below them: zeros), ones without the node itself, all ones."""
    T, hq, hk, d = 20, 4, 2, 128
    rnd = gen(pos)
    c = make_cache(rnd, eight, hk, pos + T, d)
    q = rnd(T, hq, d).to(BF).transpose(0, 1)
    rng = np.random.default_rng(1)
    masks = [0, (1 << T) - 1, 1 << 19, 0] + [int(rng.integers(0, 1 << T)) for _ in range(T - 4)]
    masks[6] |= ((1 << 44) - 1) << T   # bits beyond the tree say nothing
    out = C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=splits)
    check_attention(out, q, c, [m & (1 << T) - 1 for m in masks], pos, d ** -0.5, eight)
    assert pos or not out[[0, 3]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("pos", [0, 29, 290])
def test_what_a_node_does_not_see_does_not_reach_it(C, eight, pos):
    """Infinities and NaN in rows of the tree: the nodes that do not see them give the bits they give without; those that do, NaN or an
    infinity."""
    T, hq, hk, d = 37, 6, 2, 128
    rnd = gen(7)
    c = make_cache(rnd, eight, hk, pos + T, d)
    q = rnd(T, hq, d).to(BF).transpose(0, 1)
    masks = O.line_masks(tree(T, 3))
    clean = C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=2)
    bad = [4, 11, 36]
    if eight:
        c[2][0, pos + 4], c[3][0, pos + 11], c[3][1, pos + 36] = float("nan"), float("inf"), float("nan")
    else:
        c[0][0, pos + 4, 5], c[1][0, pos + 11, 127], c[1][1, pos + 36, 0] = float("nan"), float("inf"), float("nan")
    out = C.attn_tree(q, *c[:2], pos, bits(masks), *c[2:], splits=2).view(T, hk, -1)
    clean = clean.view(T, hk, -1)
    for i in range(T):
        for h in range(hk):
            sees = any(masks[i] >> b & 1 and h == (1 if b == 36 else 0) for b in bad)
            if sees:
                assert not torch.isfinite(out[i, h]).all()
            else:
                assert torch.equal(out[i, h], clean[i, h])


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_scores_that_grow_and_fall_along_the_rows(C, eight):
    """The reference moves many times, or never after the first tile; one row holds nearly all weight; rows of zeros; scales far apart."""
    T, hq, hk, d, pos = 4, 4, 2, 64, 1500
    rnd = gen(9)
    q = torch.ones(T, hq, d, device="cuda", dtype=BF).transpose(0, 1)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    ramp = torch.linspace(-60, 60, pos + T, device="cuda")
    for shape in (ramp, ramp.flip(0), ramp.abs() * 3, torch.where(torch.arange(pos + T, device="cuda") == 777, 90.0, 0.0)):
        if eight:
            c = make_cache(rnd, True, hk, pos + T, d, 3.0)
            c[0][:] = 100
            c[2][:] = shape.abs().clamp(min=1e-3) / (100 * d ** 0.5)
            c[0][:, shape < 0] = -100
            c[1][:, 40:60], c[3][:, 40:60] = 0, 0
        else:
            c = make_cache(rnd, False, hk, pos + T, d)
            c[0][:] = (shape / d ** 0.5)[:, None].to(BF)
        check_attention(C.attn_tree(q, *c[:2], pos, None, *c[2:], splits=4), q, c, chain, pos, d ** -0.5, eight)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -30, 2.0 ** 20, 2.0 ** 60])
def test_queries_of_any_size(C, eight, size):
    """Queries far outside half precision's range, small ones beside large ones, and one of infinities beside finite ones."""
    T, hq, hk, d, pos = 6, 4, 2, 128, 200
    rnd = gen(21)
    c = make_cache(rnd, eight, hk, pos + T, d)
    q = rnd(T, hq, d)
    q[1] *= 2.0 ** -12
    q = (q * size).to(BF).transpose(0, 1)
    chain = [(1 << (i + 1)) - 1 for i in range(T)]
    check_attention(C.attn_tree(q, *c[:2], pos, None, *c[2:], scale=0.09 / size), q, c, chain, pos, 0.09 / size, eight)
    if size == 2.0 ** 20:
        q = rnd(T, hq, d).to(BF).transpose(0, 1)
        bad = q.clone()
        bad[:, 2, 5] = float("inf")
        a, b = (C.attn_tree(x, *c[:2], pos, None, *c[2:]) for x in (q, bad))
        assert torch.isnan(b[2]).any()
        b[2] = a[2]
        check_attention(b, q, c, chain, pos, d ** -0.5, eight)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_a_cache_longer_than_32_bits_of_bytes(C, eight):
    """The last KV head's rows lie beyond 2^32 bytes (and elements, in 8 bits); reading, writing and moving there."""
    hk, d = 3, 256
    rows = (2 ** 32 // (d * (1 if eight else 2))) * 5 // 8   # two heads end beyond 2^32 bytes
    T, hq, pos = 3, 3, rows - 40
    shape = (hk, rows, d)
    c = [torch.zeros(shape, dtype=torch.int8 if eight else BF, device="cuda") for _ in range(2)] + [torch.zeros(shape[:2], device="cuda") if eight else None] * 1
    c = (c[0], c[1], c[2], torch.zeros(shape[:2], device="cuda") if eight else None)
    rnd = gen(11)
    small = make_cache(rnd, eight, hk, 40, d)
    for big, s in zip(c, small):
        if big is not None:
            big[:, rows - 40:] = s
    # the rows before are zeros: scores 0, values 0; 3 + 37 of them at the end count
    q = (2 * rnd(T, hq, d)).to(BF).transpose(0, 1)
    out = f64(C.attn_tree(q, *c[:2], pos, None, *c[2:])).reshape(T, hq, d)
    k, v = values(small[0], small[2]), values(small[1], small[3])
    for i in range(T):
        for h in range(hq):
            s = k[h, :i + 1] @ f64(q)[h, i] * d ** -0.5
            top = max(s.max(), 0.0)
            e = np.exp(s - top)
            ref = e @ v[h, :i + 1] / (e.sum() + pos * np.exp(-top))
            assert np.abs(out[i, h] - ref).max() <= 2.0 ** -6 * np.abs(ref).max() + 1e-6
    y = rnd(T, 9 * d).to(BF)
    n, inv = torch.ones(d, device="cuda", dtype=BF), torch.zeros(d // 2, device="cuda")
    C.cache_write(y, n, n, 1e-6, T, hq, hk, d, c[0], c[1], pos + 20, inv, c[2], c[3])
    C.cache_keep([c], torch.tensor([2, 0, 1], device="cuda", dtype=torch.int32), torch.tensor([3], device="cuda", dtype=torch.int32), pos + 20)
    _, _, rv, _ = O.normed_rows(f64(y), np.ones(d), np.ones(d), 1e-6, hq, hk, d, [0] * T, np.zeros(d // 2))
    got = values(c[1][:, pos + 20:pos + 23], None if c[3] is None else c[3][:, pos + 20:pos + 23])
    assert np.abs(got - rv.transpose(1, 0, 2)[:, [2, 0, 1]]).max() <= (np.abs(rv).max() / 250 if eight else 0)
    if eight:
        b = C.cache_read(*c, 3, pos + 20)[1]
        assert np.abs(f64(b) - got).max() <= 2.0 ** -8 * np.abs(got).max()


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_other_streams_and_two_calls_at_once(C, eight):
    """Calls on two streams, each with its own workspace, give what they give alone."""
    T, hq, hk, d, pos = 8, 16, 8, 128, 3000
    rnd = gen(13)
    c = make_cache(rnd, eight, hk, pos + T, d)
    qs = [rnd(T, hq, d).to(BF).transpose(0, 1) for _ in range(2)]
    alone = [C.attn_tree(q, *c[:2], pos, None, *c[2:]) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(C.attn_tree(qs[i], *c[:2], pos, None, *c[2:]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, a) for outs, a in zip(got, alone) for o in outs)


@pytest.mark.gpu
def test_caches_that_are_one_or_empty_are_refused(C):
    b = lambda *s, t=BF: torch.zeros(*s, dtype=t, device="cuda")   # noqa: E731
    one, none = b(2, 16, 64), b(0, 16, 64)
    with pytest.raises(ValueError, match="one cache"):
        C.cache_write(b(4, 8 * 64), b(64), b(64), 1e-6, 4, 4, 2, 64, one, one, 0, b(32, t=torch.float32))
    with pytest.raises(ValueError):
        C.attn_tree(b(4, 1, 64), none, none, 0)
    eight = b(2, 16, 64, t=torch.int8), b(2, 16, 64, t=torch.int8), b(2, 16, t=torch.float32), b(2, 16, t=torch.float32)
    for n, row0 in ((2 ** 40, 0), (4, 13), (0, 17), (1, -1), (-1, 3)):   # before anything is allocated
        with pytest.raises(ValueError):
            C.cache_read(*eight, n, row0)


@pytest.mark.gpu
def test_what_is_refused(C):
    hq, hk, d, rows = 4, 2, 64, 16
    b = lambda *s, t=BF: torch.zeros(*s, dtype=t, device="cuda")   # noqa: E731
    k, v, ks, vs = b(hk, rows, d, t=torch.int8), b(hk, rows, d, t=torch.int8), b(hk, rows, t=torch.float32), b(hk, rows, t=torch.float32)
    n, inv, y, q = b(d), b(d // 2, t=torch.float32), b(4, 8 * d), b(hq, 4, d)
    write = lambda **o: C.cache_write(**({"y": y, "qn": n, "kn": n, "eps": 1e-6, "L": 4, "hq": hq, "hk": hk, "d": d, "kcache": k, "vcache": v, "pos": 0,   # noqa: E731
                                          "inv_freq": inv, "kscale": ks, "vscale": vs} | o))
    write()
    assert write(y=y[:0], L=0, pos=rows).shape == (hq, 0, d)
    for o in ({"pos": 13}, {"pos": -1}, {"L": 5}, {"kscale": None}, {"kscale": None, "vscale": None}, {"kcache": k[:, :8]}, {"y": y.float()}, {"qn": n[:32]},
              {"inv_freq": inv.double()}, {"depth": b(4, t=torch.int64)}, {"depth": b(3, t=torch.int32)}, {"y": None}, {"y": None, "acc": y.int()},
              {"pos": b(1, t=torch.int32)}, {"kscale": ks[:, :8], "vscale": vs[:, :8]}, {"y": y.cpu()}, {"kcache": k.cpu(), "vcache": v.cpu()},
              {"kcache": k.transpose(1, 2).contiguous().transpose(1, 2)}, {"hk": 3}):
        with pytest.raises(ValueError):
            write(**o)
    with pytest.raises(ValueError, match="head dim"):
        C.attn_tree(b(4, 1, 32), b(2, 8, 32), b(2, 8, 32), 0)
    attend = lambda **o: C.attn_tree(**({"q": q, "kcache": k, "vcache": v, "pos": 0, "kscale": ks, "vscale": vs} | o))   # noqa: E731
    attend()
    for o in ({"pos": 13}, {"pos": -1}, {"q": q.float()}, {"q": b(3, 4, d)}, {"q": b(hq, 65, d)}, {"q": b(hq, 0, d)}, {"mask": b(3, t=torch.int64)}, {"mask": b(4, t=torch.int32)},
              {"kscale": None}, {"splits": 0}, {"splits": 65}, {"scale": float("nan")}, {"kcache": k.float(), "vcache": v.float()}, {"q": q.cpu()}):
        with pytest.raises(ValueError):
            attend(**o)
    for o in ((k, v, ks, vs, 17), (k, v, ks, vs, 4, 13), (k, v, ks, vs, -1), (k, v, None, None, 4), (b(hk, rows, d), b(hk, rows, d), ks, vs, 4)):
        with pytest.raises(ValueError):
            C.cache_read(*o)
    assert [t.shape for t in C.cache_read(k, v, ks, vs, 0)] == [(hk, 0, d)] * 2
    p, one = torch.arange(4, device="cuda", dtype=torch.int32), torch.ones(1, device="cuda", dtype=torch.int32)
    C.cache_keep([], p, one, 0)
    for o in (([(k, v, ks, vs)], p, one, 13), ([(k, v, ks, vs)], p.long(), one, 0), ([(k, v, None, None)], p, one, 0), ([(k, v, ks, vs), (b(hk, rows, d), b(hk, rows, d), None, None)], p, one, 0),
              ([(k[:, ::2], v[:, ::2], ks[:, ::2], vs[:, ::2])], p, one, 0), ([(k, v, ks, vs)], torch.arange(65, device="cuda", dtype=torch.int32), one, 0), ([(k, v, ks, vs)] * 2, p, one, 0),
              ([(k, k, ks, vs)], p, one, 0)):
        with pytest.raises(ValueError):
            C.cache_keep(*o)


def test_ranges_stay_in_bounds(C):
    for T in (1, 7, 64):
        for n in (1, 300, 40000, 2 ** 31 - 1):
            for hq, hk, d in ((1, 1, 64), (16, 8, 128), (64, 1, 256), (65535, 65535, 64)):
                assert 1 <= C.attn_tree_splits(T, n, hq, hk, d) <= 64
