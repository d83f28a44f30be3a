"""Verification of drafted tokens on the GPU against a float64 walk (oracle/draft.py): node and token numbers are equal.  Then a run of all
operators on drafted tokens together, eager and captured."""
import numpy as np
import pytest
import torch

from oracle import draft as O

BF = torch.bfloat16


@pytest.fixture(scope="module")
def D():
    from mxfp4_int8_m5_amd import sc_draft
    return sc_draft


def tree(T, rng, wide):
    return [-1] + [int(rng.integers(max(0, i - wide), i)) for i in range(1, T)]


def problem(T, V, seed, wide, drawn, dtype=BF):
    """Logits with a few likely tokens; children likely tokens of their parent's (drawn: from a draft near the target); some twice."""
    rng = np.random.default_rng(seed)
    logits = rng.normal(size=(T, V)) * 2
    for t in range(T):
        logits[t, rng.integers(0, V, 4)] += 8
    parents = tree(T, rng, wide)
    logits = torch.tensor(logits, dtype=torch.float32).to(dtype).float().numpy()
    draft = np.stack([O.softmax64(logits[t] + 0.8 * rng.normal(size=V), 0.8) for t in range(T)]).astype(np.float32) if drawn else None
    tokens = np.zeros(T, np.int64)
    for i in range(1, T):
        p = parents[i]
        tokens[i] = rng.choice(V, p=draft[p].astype(np.float64) / draft[p].astype(np.float64).sum()) if drawn else np.argsort(-logits[p])[rng.integers(0, min(3, V))]
    return logits, tokens, parents, draft, rng.random(T).astype(np.float32)


def run(D, logits, tokens, parents, dtype=BF, temperature=0.0, u=None, draft=None, siblings=None):
    dev = lambda a, t: None if a is None else torch.tensor(np.asarray(a), dtype=t, device="cuda")   # noqa: E731
    path, count, nxt = D.verify_drafts(dev(logits, dtype), dev(tokens, torch.int64), dev(parents, torch.int32), temperature, dev(u, torch.float32), dev(draft, torch.float32),
                                       siblings)
    n = int(count)
    path = path.tolist()
    assert path[n:] == [-1] * (len(path) - n)
    return path[:n], int(nxt)


# chunks of the vocabulary are 4096 tokens: one, borders, odd ends, an unaligned row
VOCABS = [1, 2, 50, 4095, 4096, 4097, 8193, 32000, 50304]


@pytest.mark.gpu
@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("mode", ["greedy", "given", "drawn"])
def test_verify(D, V, mode):
    lengths = []
    for seed, (T, wide, temperature) in enumerate([(1, 1, 1.0), (2, 1, 0.7), (8, 1, 1.3), (13, 4, 0.8), (64, 6, 0.6), (40, 64, 1.0)]):
        dtype = BF if seed % 2 else torch.float32
        if V > 30000 and T > 13:
            T = 13
        logits, tokens, parents, draft, u = problem(T, V, 100 * seed + V, wide, mode == "drawn", dtype)
        kids = max(parents.count(i) for i in range(T))
        t = 0.0 if mode == "greedy" else temperature
        for k in range(4):
            us = np.random.default_rng(k).random(T).astype(np.float32) * (1.0 if k else 0.2)
            got = run(D, logits, tokens, parents, dtype, t, us, draft, min(max(kids, 1), 16))
            assert got == O.verify(logits, tokens, parents, t, us, draft), (seed, k)
            lengths.append(len(got[0]))
    assert mode == "greedy" or V < 50 or max(lengths) > 1   # some drafts are taken (greedy: next test)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 17, 64])
@pytest.mark.parametrize("stop", [0.0, 0.1, 1.0])
def test_long_accepted_lines(D, T, stop):
    """A chain of the target's own tokens, broken now and then; and the same nodes hanging on the root's line with wrong siblings before."""
    V = 6000
    rng = np.random.default_rng(T)
    logits = rng.normal(size=(T, V)).astype(np.float32)
    best = logits.argmax(1)
    for parents in (list(range(-1, T - 1)), [-1] + [(i - 1) // 2 * 2 for i in range(1, T)]):
        tokens = [0] + [int(best[p]) if (i % 2 == 0 or parents[1:] == list(range(T - 1))) and rng.random() >= stop else 17 for i, p in enumerate(parents[1:], 1)]
        got = run(D, logits, tokens, parents, torch.float32)
        assert got == O.verify(logits, tokens, parents)
        if stop == 0:
            assert len(got[0]) == (T if parents[1:] == list(range(T - 1)) else (T + 1) // 2)
        sharp = 40 * logits   # nearly all mass on one token
        u = rng.random(T).astype(np.float32)
        assert run(D, sharp, tokens, parents, torch.float32, 0.9, u) == O.verify(sharp, tokens, parents, 0.9, u)


@pytest.mark.gpu
def test_siblings_twice_unknown_tokens_and_certain_ones(D):
    V = 5000
    logits = np.full((4, V), -np.inf, np.float32)
    logits[:, 7] = 0.0   # all probability on one token
    for draft in (None, np.eye(V, dtype=np.float32)[[9, 9, 9, 9]]):
        for tokens in ([0, 7, 7, 7], [0, 3, 7, 7], [0, -1, V, 7], [0, 2 ** 40, 3, 3]):
            for u in (0.0, 0.5, 0.99999994):
                us = np.full(4, u, np.float32)
                parents = [-1, 0, 0, 0]
                d = draft
                assert run(D, logits, tokens, parents, torch.float32, 1.0, us, d, 3) == O.verify(logits, tokens, parents, 1.0, us, d, 3)
    # a draft that is the target: always taken; the same token twice, refused once, is not taken the second time
    p = np.zeros((3, 4), np.float32)
    assert run(D, p, [0, 2, 1], [-1, 0, 1], torch.float32, 1.0, [0.6, 0.99, 0.99], np.full((3, 4), 0.25, np.float32), 1) == ([0, 1, 2], 2)
    assert run(D, p, [0, 2, 2], [-1, 0, 0], torch.float32, 1.0, [0.99, 0.5, 0.0], None) == O.verify(p, [0, 2, 2], [-1, 0, 0], 1.0, [0.99, 0.5, 0.0]) == ([0], 3)
    # only the first `siblings` children are tried against a draft
    q = np.full((4, 4), 0.25, np.float32)
    logits = np.array([[0, 0, 0, 9.0]] * 4, np.float32)
    for siblings in (1, 2, 3):
        us = [0.5, 0.9, 0.9, 0.9]
        assert run(D, logits, [0, 0, 1, 3], [-1, 0, 0, 0], torch.float32, 1.0, us, q, siblings) == O.verify(logits, [0, 0, 1, 3], [-1, 0, 0, 0], 1.0, us, q, siblings)


@pytest.mark.gpu
def test_equal_infinite_and_nan_logits(D):
    V = 4100
    x = np.zeros((6, V), np.float32)
    x[1, 4099] = x[1, 5] = np.inf
    x[2] = -np.inf
    x[3] = np.nan
    x[4, 4097] = x[4, 4098] = 3.0
    x[5, :] = np.nan
    x[5, 4099] = -5.0
    for dtype in (torch.float32, BF):
        for t in range(6):
            row = x[[t]]
            assert run(D, row, [0], [-1], dtype)[1] == O.verify(row, [0], [-1])[1] == [0, 5, 0, 0, 4097, 4099][t]
            for u in (0.0, 0.3, 0.5, 0.7, 0.99999994):
                assert run(D, row, [0], [-1], dtype, 0.5, [u])[1] == O.verify(row, [0], [-1], 0.5, [u])[1]


@pytest.mark.gpu
def test_random_numbers_near_a_border_and_far_tails(D):
    """Flat rows: the border of token i is i / V; u just below and above it.  A long tail of tokens of 1e-12 each."""
    V = 2 ** 15
    x = np.zeros((1, V), np.float32)
    for i in (1, 4095, 4096, 4097, V - 1):
        for u in (np.float32(i / V), np.nextafter(np.float32(i / V), np.float32(0)), np.nextafter(np.float32(i / V), np.float32(1))):
            assert run(D, x, [0], [-1], torch.float32, 1.0, [u])[1] == int(np.floor(float(u) * V))
    x[0, 1:] = -27.6
    for u in (0.0, 0.99999, 0.99999994):
        assert run(D, x, [0], [-1], torch.float32, 1.0, [u])[1] == O.verify(x, [0], [-1], 1.0, [u])[1]


@pytest.mark.gpu
@pytest.mark.parametrize("there,u", [(2 * 4096 + 5, 0.0), (2 * 4096 + 5, 0.99999994), (3, 0.0), (3, 0.99999994), (4096 + 77, 0.0), (4096 + 77, 0.99999994)])
def test_a_chunk_whose_likely_tokens_were_all_refused(D, there, u):
    """What is left of its sum is rounding, and no token of it is ever the next one."""
    V, T = 3 * 4096, 17
    for seed in range(12):
        rng = np.random.default_rng(seed)
        logits = np.full((T, V), -np.inf, np.float32)
        tokens = np.concatenate([[0], 4096 + rng.choice(4096, 16, replace=False)])
        tokens = tokens[tokens != there]
        parents = [-1] + [0] * (len(tokens) - 1)
        logits = logits[:len(tokens)]
        logits[0, tokens[1:]] = 3 * rng.normal(size=len(tokens) - 1)
        logits[0, there] = 0.0
        us = np.full(len(tokens), 0.99999994, np.float32)
        us[0] = u
        assert O.verify(logits, tokens, parents, 1.0, us) == ([0], there)
        assert run(D, logits, tokens, parents, torch.float32, 1.0, us) == ([0], there), seed


@pytest.mark.gpu
@pytest.mark.parametrize("V", [262144, 262145, 300001, 4194304])
def test_vocabularies_of_more_chunks_than_a_wave_has_lanes(D, V):
    T = 3 if V < 400000 else 2
    rng = np.random.default_rng(V)
    logits = rng.normal(size=(T, V)).astype(np.float32)
    logits[:, -3:] += 6   # the last chunk counts
    best = logits.argmax(1)
    q = np.exp(logits + 0.5 * rng.normal(size=(T, V)).astype(np.float32))
    q = (q / q.sum(1, keepdims=True)).astype(np.float32)
    parents = [-1, 0, 0][:T]
    for tokens in ([0, int(best[0]), 5][:T], [0, 7, V - 1][:T]):
        assert run(D, logits, tokens, parents, torch.float32) == O.verify(logits, tokens, parents)
        for k in range(3):
            u = rng.random(T).astype(np.float32) * (1.0 if k else 0.01)
            for draft in (None, q):
                assert run(D, logits, tokens, parents, torch.float32, 1.1, u, draft, 2) == O.verify(logits, tokens, parents, 1.1, u, draft, 2)


@pytest.mark.gpu
def test_parents_that_are_none(D):
    """Numbers that name no earlier node are nobody's children; nothing is read outside."""
    V = 100
    logits, tokens, _, _, u = problem(6, V, 1, 1, False, torch.float32)
    for parents in ([-1, 70, -5, 3, 2 ** 31 - 1, 5], [0, 0, 2, 2, 4, 4], [-2 ** 31, 1, 1, 9, 4, 0]):
        for t in (0.0, 1.0):
            path, nxt = run(D, logits, tokens, parents, torch.float32, t, u)
            assert path[0] == 0 and all(parents[b] == a for a, b in zip(path, path[1:])) and 0 <= nxt < V
        run(D, logits, tokens, parents, torch.float32, 1.0, u, np.full((6, V), 1 / V, np.float32), 4)


@pytest.mark.gpu
def test_verify_refuses(D):
    b = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")   # noqa: E731
    ok = {"logits": b(4, 10), "tokens": b(4, t=torch.int64), "parents": b(4, t=torch.int32), "temperature": 1.0, "uniforms": b(4), "draft": b(4, 10), "siblings": 1}
    D.verify_drafts(**ok)
    for o in ({"logits": b(4, 10, t=torch.float16)}, {"logits": b(65, 10), "tokens": b(65, t=torch.int64), "parents": b(65, t=torch.int32), "uniforms": b(65), "draft": None},
              {"logits": b(0, 10), "tokens": b(0, t=torch.int64), "parents": b(0, t=torch.int32), "uniforms": b(0), "draft": None}, {"logits": b(4, 0), "draft": None},
              {"tokens": b(4, t=torch.int32)}, {"parents": b(4, t=torch.int64)}, {"tokens": b(3, t=torch.int64)}, {"temperature": -1.0}, {"temperature": float("nan")},
              {"temperature": 1e-9}, {"uniforms": None}, {"uniforms": b(3)}, {"uniforms": b(4, t=torch.float64)}, {"draft": b(4, 9)}, {"draft": b(4, 10, t=BF)}, {"siblings": None},
              {"logits": b(4, 10).cpu()}, {"logits": b(10, 4).T}, {"draft": b(10, 4).T}):
        with pytest.raises(ValueError):
            D.verify_drafts(**(ok | o))
    D.verify_drafts(**(ok | {"temperature": 0.0, "uniforms": None, "draft": None, "siblings": None}))


def test_draft_tree():
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    t = DraftTree([-1, 0, 0, 1, 3, 0], device="cpu")
    assert (t.T, t.siblings, t.depth_list) == (6, 3, [0, 1, 1, 2, 3, 1])
    assert t.mask.tolist() == [1, 3, 5, 11, 27, 33] and t.parents.tolist() == [-1, 0, 0, 1, 3, 0] and t.depth.tolist() == t.depth_list
    c = DraftTree.chain(64, device="cpu")
    assert c.siblings == 1 and c.depth.tolist() == list(range(64)) and c.mask[63] == -1 and c.mask[62] == 2 ** 63 - 1
    assert DraftTree([-1], device="cpu").siblings == 0
    for bad in ([], [0], [-1, 1], [-1, -1], [-1] + [0] * 64):
        with pytest.raises(ValueError):
            DraftTree(bad, device="cpu")


# ---- all of it together --------------------------------------------------------------------------------------------------

class Steps:
    """Drafted steps on two blocks' caches: append, attend, verify, keep, the position moved on by what was accepted; everything that
    changes lives on the device, so that one captured step serves every position."""

    def __init__(self, eight, T, d=64, hq=4, hk=2, V=300, rows=200):
        from mxfp4_int8_m5_amd import sc_cache, sc_draft
        from tests.test_gpu_cache import gen, make_cache
        self.C, self.D, rnd = sc_cache, sc_draft, gen(17)
        self.shape = (hq, hk, d)
        self.caches = [make_cache(rnd, eight, hk, rows, d) for _ in range(2)]
        self.tree = sc_draft.DraftTree(tree(T, np.random.default_rng(2), 4))
        self.gain, self.inv = (1 + 0.1 * rnd(d)).to(BF), 1.0 / (1e4 ** (torch.arange(d // 2, device="cuda", dtype=torch.float32) / (d // 2)))
        self.embed, self.head = rnd(V, (hq + 2 * hk) * d).to(BF), (0.2 * rnd(hq * d, V)).to(BF)
        self.pos = torch.tensor([5], device="cuda")
        self.tokens, self.u = torch.zeros(T, dtype=torch.int64, device="cuda"), torch.zeros(T, device="cuda")

    def __call__(self):
        C, t, (hq, hk, d) = self.C, self.tree, self.shape
        o = 0
        for k, v, ks, vs in self.caches:
            q = C.cache_write(self.embed[self.tokens], self.gain, self.gain, 1e-6, t.T, hq, hk, d, k, v, self.pos, self.inv, ks, vs, t.depth)
            o = o + C.attn_tree(q, k, v, self.pos, t.mask, ks, vs)
        logits = (o.float() @ self.head.float()).to(BF)
        path, count, nxt = self.D.verify_drafts(logits, self.tokens, t.parents, 0.9, self.u)
        C.cache_keep(self.caches, path, count, self.pos)
        self.pos += count
        return logits, path, count, nxt

    def state(self):
        return [t for c in self.caches for t in c if t is not None] + [self.pos]


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("T", [1, 9])
def test_a_captured_drafted_step_equals_the_eager_one(eight, T):
    """One captured step replayed over growing positions, with eager work between, against the eager step on its own caches: bit for bit."""
    import mxfp4_int8_m5_amd as scmx
    scmx._lib.native()
    eager, graph = Steps(eight, T), Steps(eight, T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    keep = [t.clone() for t in graph.state()]
    with torch.cuda.stream(side):
        graph()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = graph()
    for t, old in zip(graph.state(), keep):
        t.copy_(old)
    rng = np.random.default_rng(3)
    taken = []
    for step in range(6):
        tokens, u = torch.tensor(rng.integers(0, 300, T)), torch.tensor(rng.random(T), dtype=torch.float32)
        for s in (eager, graph):
            s.tokens.copy_(tokens)
            s.u.copy_(u)
        want = eager()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), step
        assert all(torch.equal(a.nan_to_num(9) if a.is_floating_point() else a, b.nan_to_num(9) if b.is_floating_point() else b) for a, b in zip(eager.state(), graph.state()))
        taken.append(int(want[2]))
    assert int(eager.pos) == 5 + sum(taken)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [False, True])
def test_an_accepted_line_is_what_a_chain_of_it_would_have_been(eight):
    """The rows kept of a tree are, bit for bit, those that the accepted tokens leave when appended alone, one after the other."""
    s = Steps(eight, 12)
    hq, hk, d = s.shape
    s.tokens.copy_(torch.arange(12) * 7)
    k, v, ks, vs = s.caches[0]
    start = [None if t is None else t.clone() for t in s.caches[0]]
    y = s.embed[s.tokens]
    q = s.C.cache_write(y, s.gain, s.gain, 1e-6, 12, hq, hk, d, k, v, 5, s.inv, ks, vs, s.tree.depth)
    node, line = 11, []
    while node >= 0:
        line.insert(0, node)
        node = s.tree.parent_list[node]
    path = torch.tensor(line + [-1] * (12 - len(line)), dtype=torch.int32, device="cuda")
    s.C.cache_keep(s.caches[:1], path, torch.tensor([len(line)], dtype=torch.int32, device="cuda"), 5)
    for i, n in enumerate(line):
        q1 = s.C.cache_write(y[n:n + 1], s.gain, s.gain, 1e-6, 1, hq, hk, d, start[0], start[1], 5 + i, s.inv, start[2], start[3])
        assert torch.equal(q1[:, 0], q[:, n])
    n = 5 + len(line)
    for a, b in zip((k, v, ks, vs), start):
        assert a is None or torch.equal(a[:, :n], b[:, :n])
