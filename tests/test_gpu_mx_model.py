"""4-bit values where they are used: the Qwen3 drivers over an MXFP4 cache, and a block of MXFP4 linear layers around such a cache."""
import numpy as np
import pytest
import torch

from oracle import draft as D
from oracle import mx as O
from tests.test_gpu_cache4 import check_attention
from tests.test_gpu_draft_model import greedy, ids_of
from tests.test_gpu_model import default_format_afterwards, float_model, make_tiny, rel   # noqa: F401
from tests.test_gpu_mx import BF, check_product, f64, gen, host, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=[(4, 2, 64), (4, 2, 128)])
def tiny(request):
    return make_tiny(*request.param)


def reads_back(monkeypatch, C):
    """The drivers' attention over a 4-bit cache by what the cache reads back as, in float32."""
    def attend(q, k, v, pos, mask=None, ks=None, vs=None):
        hq, T, d = q.shape
        end = int(pos) + T
        rk, rv = (t.float().repeat_interleave(hq // k.shape[0], 0) for t in C.cache_read(k, v, ks, vs, end))
        see = torch.arange(end, device="cuda")[None] <= torch.arange(end - T, end, device="cuda")[:, None]
        p = torch.softmax(((q.float() @ rk.transpose(1, 2).contiguous()) * d ** -0.5).masked_fill(~see, float("-inf")), -1)
        return (p @ rv).transpose(0, 1).reshape(T, -1).to(BF)
    monkeypatch.setattr(C, "attn_tree", attend)


@pytest.mark.parametrize("epilogue", ["gemm", "row"])
def test_prefill_with_a_4_bit_cache(tiny, epilogue, monkeypatch):
    """Long and short prompts, fresh and behind others.  A 4-bit value is off by an eighth of itself at most, in the rms a tenth of a row, and
    so are the scores and their averages: two blocks' attention, beside a residual stream of several times its size, makes less than
    0.15.  Against the same driver whose attention is float32's on the rows that the cache reads back as: the kernels' rounding (2^-8), and
    where a value of the next block's keys lies beside a border its code (a quarter of it, once in some hundred values): 2e-2."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd import sc_cache as C
    ids = ids_of(args, 140, 1)
    m = Q.FusedQwen3(args, state, packed, epilogue=epilogue)
    ref = float_model(Q, args, state, packed, ids.cpu())

    def run():
        cache = m.make_cache(160, bits="mxfp4")
        assert all(isinstance(c, C.Q4Cache) for c in cache)
        out = torch.cat([m.hidden(ids[a:b], cache) for a, b in ((0, 70), (70, 73), (73, 74), (74, 140))])
        assert cache[0].offset == 140
        return out

    got = run()
    assert rel(got, ref) < 0.15, rel(got, ref)
    with monkeypatch.context() as mp:
        reads_back(mp, C)
        want = run()
    assert rel(got, want) < 2e-2, rel(got, want)
    assert m.make_cache(100, bits="mxfp4")[0].k.nbytes * 4 == m.make_cache(100)[0].k.nbytes


@pytest.mark.parametrize("kw", [{}, {"fuse_prologue": True}, {"fuse_attn": False}, {"graphs": True}, {"graphs": "step"}, {"graphs": "step", "fuse_attn": False}])
@pytest.mark.parametrize("rows", [150, 2000])
def test_decode_with_a_4_bit_cache(tiny, kw, rows, monkeypatch):
    """Every form of the decoder continues a prefill.  Against the plain eager form whose attention is float32's on the rows read back (as
    above); captured steps are the eager ones of the same form: their bits where the cache is one range, else sums in another order."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd import sc_cache as C
    m = Q.FusedQwen3(args, state, packed)
    ids, n = ids_of(args, 90, 2), rows - 20

    def run(kw):
        cache = m.make_cache(rows, bits="mxfp4")
        m.hidden(ids_of(args, n, 3), cache)
        dec = Q.DecodeQwen3(m, head=False, **kw)
        out = torch.cat([dec.step(ids[j:j + 1], cache).clone() for j in range(8)])
        assert cache[0].offset == n + 8
        return out

    got = run(kw)
    if "graphs" in kw:
        eager = run(kw | {"graphs": False})
        assert torch.equal(got, eager) if rows == 150 else rel(got, eager) < 1e-2, rel(got, eager)
    with monkeypatch.context() as mp:
        reads_back(mp, C)
        want = run({k: v for k, v in kw.items() if k != "graphs"})
    assert rel(got, want) < 2e-2, rel(got, want)


@pytest.mark.parametrize("graphs", [False, True])
def test_drafted_steps_with_a_4_bit_cache(tiny, graphs):
    """Greedy drafted decoding: every token the largest logit, the accepted line's logits a prefill's of the accepted text, whose keys and
    values are a few thousandths off before they are coded (INT8 activations): codes beside a border differ, so that rows are up to
    sqrt(0.01 * 0.25) = 0.05 apart in the rms, and with what they average to 0.06 of the logits."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd import sc_cache as C
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    m = Q.FusedQwen3(args, state, packed)
    prompt = ids_of(args, 20, 3)
    want = greedy(Q, m, prompt, 40, "mxfp4")
    cache = m.make_cache(200, bits="mxfp4")
    h = m.hidden(prompt, cache)
    text = prompt.tolist() + [int(m.logits(h[-1:]).argmax())]
    dec = Q.DraftQwen3(m, graphs=graphs)
    rng = np.random.default_rng(0)
    trees = [DraftTree.chain(5), DraftTree([-1, 0, 0, 1, 1, 2, 3]), DraftTree.chain(1), DraftTree([-1, 0, 0, 0, 1, 2, 3, 4, 5, 6, 7, 8])]
    counts = []
    for step in range(8):
        tree = trees[step % 4]
        done, off = len(text) - len(prompt), cache[0].offset
        assert off == len(text) - 1
        tokens = [text[-1]] + [want[done + depth - 1] if done + depth - 1 < len(want) and rng.random() < 0.8 else int(rng.integers(args.vocab_size))
                               for depth in tree.depth_list[1:tree.T]]
        path, count, nxt, logits = dec.step(torch.tensor(tokens, device="cuda"), tree, cache)
        n = int(count)
        line = path[:n].tolist()
        assert line[0] == 0 and all(tree.parent_list[b] == a for a, b in zip(line, line[1:])) and cache[0].offset == off + n
        best = logits.argmax(-1)
        assert [tokens[i] for i in line[1:]] + [int(nxt)] == [int(best[i]) for i in line]
        text += [tokens[i] for i in line[1:]] + [int(nxt)]
        counts.append(n)
        fresh = m.make_cache(200, bits="mxfp4")
        ref = m(torch.tensor(text[:-1], device="cuda"), fresh)[off:]
        assert rel(logits[line], ref) < 6e-2, (step, rel(logits[line], ref))
        for c, r in zip(cache, fresh):
            a, b = (C.cache_read(x.k, x.v, x.kscale, x.vscale, off + n) for x in (c, r))
            assert rel(a[0], b[0]) < 0.1 and rel(a[1], b[1]) < 0.1
    assert max(counts) > 1


def test_another_heads_size_is_refused():
    Q, args, state, packed = make_tiny(4, 2, 64)
    from mxfp4_int8_m5_amd import sc_cache as C
    args.head_dim = 96
    with pytest.raises(ValueError):
        C.Q4Cache(args, 16, "cuda")


class Block:
    """A transformer block of MXFP4 linear layers around a 4-bit cache, as a user of the operators writes it."""

    def __init__(self, seed, hidden, wide, hq, hk, d, rows):
        from mxfp4_int8_m5_amd import sc_cache, sc_kernels, sc_mx
        self.X, self.C = sc_mx, sc_cache
        rnd = gen(seed)
        self.hq, self.hk, self.d, self.wide = hq, hk, d, wide
        linear = lambda n, k: sc_mx.quantize(rnd(n, k) * k ** -0.5)   # noqa: E731
        order = torch.as_tensor(sc_kernels.interleave_gate_up(wide), device="cuda")
        self.w = {"qkv": linear((hq + 2 * hk) * d, hidden), "o": linear(hidden, hq * d), "down": linear(hidden, wide),
                  "gu": tuple(t[order] for t in linear(2 * wide, hidden))}
        self.n1, self.n2 = ((1 + 0.1 * rnd(hidden)).to(BF) for _ in range(2))
        self.qn, self.kn = ((1 + 0.1 * rnd(d)).to(BF) for _ in range(2))
        self.inv = 1.0 / (1e4 ** (torch.arange(d // 2, device="cuda", dtype=torch.float32) / (d // 2)))
        zeros = lambda n: torch.zeros(hk, rows, n, dtype=torch.uint8, device="cuda")   # noqa: E731
        self.cache = (zeros(d // 2), zeros(d // 2), zeros(d // 32), zeros(d // 32))

    def __call__(self, x, pos, keep=None):
        X, C, c, L = self.X, self.C, self.cache, x.shape[0]
        y = X.linear(x, *self.w["qkv"], 1, None, self.n1, 1e-6)
        q = C.cache_write(y, self.qn, self.kn, 1e-6, L, self.hq, self.hk, self.d, c[0], c[1], pos, self.inv, c[2], c[3])
        o = torch.cat([C.attn_tree(q[:, i:i + 64].contiguous(), c[0], c[1], pos + i, None, c[2], c[3]) for i in range(0, L, 64)])
        h = X.linear(o, *self.w["o"], 2, x)
        act = X.linear(h, *self.w["gu"], 3, None, self.n2, 1e-6)
        out = X.linear(act, *self.w["down"], 2, h)
        if keep is not None:
            keep.update(y=y, q=q, o=o, h=h, act=act)
        return out


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (8, 2, 128), (4, 1, 256)])
def test_a_block_of_them(hq, hk, d):
    """A prompt of 130, one of 20 behind it and single tokens: every stage against float64 on its own inputs."""
    hidden, wide = 416, 544
    b, rnd = Block(d, hidden, wide, hq, hk, d, 400), gen(9)
    pos = 0
    for L in (130, 20, 1, 1):
        x, s = rnd(L, hidden).to(BF), {}
        out = b(x, pos, s)
        v = {k: O.values(*host(*w)) for k, w in b.w.items()}
        normed = lambda t, n: O.values(*O.quantize(O.rmsnorm(f64(t), f64(n), 1e-6), 10, 252))   # noqa: E731
        coded = lambda t: O.values(*O.quantize(f64(t)))   # noqa: E731
        check_product(s["y"], normed(x, b.n1), v["qkv"], 1, None)
        _, rk, rv, _ = D.normed_rows(f64(s["y"]), f64(b.qn), f64(b.kn), 1e-6, hq, hk, d, pos + np.arange(L), f64(b.inv))
        assert same((b.cache[0][:, pos:pos + L], b.cache[2][:, pos:pos + L]), O.quantize(rk.transpose(1, 0, 2), 10, 252))
        assert same((b.cache[1][:, pos:pos + L], b.cache[3][:, pos:pos + L]), O.quantize(rv.transpose(1, 0, 2)))
        for i in range(0, L, 64):
            n = min(64, L - i)
            seen = tuple(t[:, :pos + i + n] for t in b.cache)
            check_attention(s["o"][i:i + n], s["q"][:, i:i + n], seen, [(1 << (j + 1)) - 1 for j in range(n)], pos + i, d ** -0.5)
        check_product(s["h"], coded(s["o"]), v["o"], 2, f64(x))
        check_product(s["act"], normed(s["h"], b.n2), v["gu"], 3, None)
        check_product(out, coded(s["act"]), v["down"], 2, f64(s["h"]))
        pos += L


def test_a_captured_block(hq=8, hk=2, d=128):
    """A decode step with its position on the device, replayed token after token with eager work between, over two blocks' own caches: the
    eager block's bits."""
    a, b = (Block(1, 512, 1024, hq, hk, d, 300) for _ in range(2))
    rnd = gen(5)
    prompt = rnd(100, 512).to(BF)
    assert torch.equal(a(prompt, 0), b(prompt, 0))
    x, pos = rnd(1, 512).to(BF), torch.tensor([100], device="cuda")
    a(x, pos)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = a(x, pos)
    for i in range(5):
        x.copy_(rnd(1, 512).to(BF))
        pos.fill_(100 + i)
        want = b(x, torch.tensor([100 + i], device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(s, t) for s, t in zip(a.cache, b.cache))
