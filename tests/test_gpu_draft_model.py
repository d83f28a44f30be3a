"""8-bit caches and drafted steps in the Qwen3 drivers, on small random models: against the float32 model, the bf16 cache, the plain
decoder, and the model's own prefill of what was accepted."""
import numpy as np
import pytest
import torch

from tests.test_gpu_model import default_format_afterwards, float_model, make_tiny, rel   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=[(4, 2, 64), (4, 2, 128)])
def tiny(request):
    return make_tiny(*request.param)


def ids_of(args, n, seed):
    return torch.randint(0, args.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("epilogue", ["gemm", "row"])
def test_prefill_with_an_8_bit_cache(tiny, epilogue):
    """Long and short prompts, fresh and behind others, against the float32 model: INT8 activations and 4-bit weights as without (3e-2),
    8-bit keys and values add a step of 1/127 of a row's largest value, some 0.5 per cent of a row a block."""
    Q, args, state, packed = tiny
    ids = ids_of(args, 140, 1)
    m = Q.FusedQwen3(args, state, packed, epilogue=epilogue)
    ref = float_model(Q, args, state, packed, ids.cpu())
    cache = m.make_cache(160, bits=8)
    assert all(c.k.dtype == torch.int8 for c in cache)
    got = torch.cat([m.hidden(ids[a:b], cache) for a, b in ((0, 70), (70, 73), (73, 74), (74, 140))])
    assert cache[0].offset == 140 and rel(got, ref) < 4e-2, rel(got, ref)
    plain = m.hidden(ids, m.make_cache(160))
    assert rel(got, plain) < 2.5e-2, rel(got, plain)


@pytest.mark.parametrize("kw", [{}, {"fuse_prologue": True}, {"fuse_attn": False}, {"graphs": True}, {"graphs": "step"}, {"graphs": "step", "fuse_attn": False}])
def test_decode_with_an_8_bit_cache(tiny, kw):
    """Every form of the decoder continues a prefill over an 8-bit cache as one prefill over all of it would; the graphs' steps are
    the eager ones' bits at the same positions."""
    Q, args, state, packed = tiny
    ids = ids_of(args, 90, 2)
    m = Q.FusedQwen3(args, state, packed)
    full = m.hidden(ids, m.make_cache(100, bits=8))
    cache = m.make_cache(100, bits=8)
    m.hidden(ids[:80], cache)
    dec = Q.DecodeQwen3(m, head=False, **kw)
    rows = torch.cat([dec.step(ids[80 + j:81 + j], cache).clone() for j in range(10)])
    assert cache[0].offset == 90 and rel(rows, full[80:]) < 2e-2, rel(rows, full[80:])


def greedy(Q, m, prompt, n, bits):
    cache = m.make_cache(200, bits=bits)
    h = m.hidden(prompt, cache)
    out, dec = [int(m.logits(h[-1:]).argmax())], Q.DecodeQwen3(m)
    while len(out) < n:
        out.append(int(dec.step(torch.tensor([out[-1]], device="cuda"), cache).argmax()))
    return out


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("graphs", [False, True])
def test_drafted_steps_follow_the_model(tiny, bits, graphs):
    """Greedy drafted decoding with drafts that are right, wrong and mixed.  Every step's logits of the accepted nodes are those of a prefill
    of the accepted text (the cache holds its rows, whatever was refused), and every token the largest logit."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    m = Q.FusedQwen3(args, state, packed)
    prompt = ids_of(args, 20, 3)
    want = greedy(Q, m, prompt, 40, bits)
    cache = m.make_cache(200, bits=bits)
    h = m.hidden(prompt, cache)
    text = prompt.tolist() + [int(m.logits(h[-1:]).argmax())]
    dec = Q.DraftQwen3(m, graphs=graphs)
    rng = np.random.default_rng(0)
    trees = [DraftTree.chain(5), DraftTree([-1, 0, 0, 1, 1, 2, 3]), DraftTree.chain(1), DraftTree([-1, 0, 0, 0, 1, 2, 3, 4, 5, 6, 7, 8])]
    counts = []
    for step in range(10):
        tree = trees[step % 4]
        done = len(text) - len(prompt)
        tokens = [text[-1]] + [want[done + tree.depth_list[i] - 1] if done + tree.depth_list[i] - 1 < len(want) and rng.random() < 0.8 else int(rng.integers(args.vocab_size))
                               for i in range(1, tree.T)]
        off = cache[0].offset
        assert off == len(text) - 1
        path, count, nxt, logits = dec.step(torch.tensor(tokens, device="cuda"), tree, cache)
        n = int(count)
        line = path[:n].tolist()
        assert line[0] == 0 and all(tree.parent_list[b] == a for a, b in zip(line, line[1:])) and cache[0].offset == off + n
        best = logits.argmax(-1)
        assert [tokens[i] for i in line[1:]] + [int(nxt)] == [int(best[i]) for i in line]
        text += [tokens[i] for i in line[1:]] + [int(nxt)]
        counts.append(n)
        fresh = m.make_cache(200, bits=bits)
        ref = m(torch.tensor(text[:-1], device="cuda"), fresh)[off:]
        assert rel(logits[line], ref) < 3e-2, (step, rel(logits[line], ref))
        from mxfp4_int8_m5_amd import sc_cache
        for c, r in zip(cache, fresh):
            end = off + n
            a, b = ([sc_cache.cache_read(x.k, x.v, x.kscale, x.vscale, end) for x in (c, r)] if bits == 8 else [(x.k[:, :end], x.v[:, :end]) for x in (c, r)])
            assert rel(a[0], b[0]) < 2.5e-2 and rel(a[1], b[1]) < 2.5e-2
    assert max(counts) > 1 and min(counts) == 1


@pytest.mark.parametrize("graphs", [False, True])
def test_sampled_drafted_steps(tiny, graphs):
    """With random numbers: the walk is the float64 one on the step's own logits, with and without a draft's probabilities."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    from oracle import draft as O
    m = Q.FusedQwen3(args, state, packed)
    cache = m.make_cache(120, bits=8)
    m.hidden(ids_of(args, 12, 4), cache)
    dec, tree = Q.DraftQwen3(m, graphs=graphs), DraftTree([-1, 0, 1, 0, 3, 3])
    g = torch.Generator(device="cuda").manual_seed(1)
    for step in range(6):
        draft = torch.softmax(2 * torch.randn(6, args.vocab_size, device="cuda", generator=g), -1) if step % 2 else None
        tokens = torch.randint(0, args.vocab_size, (6,), device="cuda", generator=g)
        if draft is not None:
            tokens[1:] = torch.multinomial(draft[tree.parents[1:].long()], 1, generator=g)[:, 0]
        u = torch.rand(6, device="cuda", generator=g)
        path, count, nxt, logits = dec.step(tokens, tree, cache, 0.7, u, draft)
        want = O.verify(logits.float().cpu().numpy(), tokens.tolist(), tree.parent_list, 0.7, u.cpu().numpy(), None if draft is None else draft.cpu().numpy(), tree.siblings)
        assert (path[:int(count)].tolist(), int(nxt)) == want


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_every_step_may_bring_another_tree(tiny, temperature):
    """Trees of one size that live for one step, with other tensors in their place afterwards: captured steps are the eager ones, to the bit."""
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    m = Q.FusedQwen3(args, state, packed)
    runs = []
    for graphs in (False, True):
        rng = np.random.default_rng(5)
        cache = m.make_cache(200, bits=8)
        m.hidden(ids_of(args, 9, 2), cache)
        dec, outs = Q.DraftQwen3(m, graphs=graphs), []
        for step in range(8):
            tree = DraftTree([-1] + [int(rng.integers(0, i)) for i in range(1, 6)])
            u = torch.tensor(rng.random(6), dtype=torch.float32, device="cuda")
            q = torch.tensor(rng.dirichlet(np.ones(args.vocab_size), 6), dtype=torch.float32, device="cuda") if step % 3 == 2 else None
            tokens = torch.tensor(rng.integers(args.vocab_size, size=6), device="cuda")
            outs += [t.cpu() for t in dec.step(tokens, tree, cache, temperature, u, q)]
            del tree, u, q, tokens
            junk = [torch.randint(0, 6, (n,), device="cuda", dtype=torch.int32) for n in (6, 12, 24, 6, 12, 24)]
        runs.append(outs)
        del junk
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_captured_step_refuses_what_an_eager_one_does(tiny):
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    m = Q.FusedQwen3(args, state, packed)
    for graphs in (False, True):
        cache = m.make_cache(40)
        dec, tree, tokens = Q.DraftQwen3(m, graphs=graphs), DraftTree.chain(4), ids_of(args, 4, 1)
        b = lambda *s, t=torch.float32: torch.full(s, 0.25, dtype=t, device="cuda")   # noqa: E731
        V = args.vocab_size
        dec.step(tokens, tree, cache, 0.5, b(4), b(4, V))
        for bad in ((b(1), b(4, V)), (b(4, t=torch.float64), b(4, V)), (b(4), b(V)), (b(4), b(1, V)), (b(4), b(4, V, t=torch.bfloat16)), (None, b(4, V)), (None, None)):
            with pytest.raises(ValueError):
                dec.step(tokens, tree, cache, 0.5, *bad)
        with pytest.raises(ValueError):
            dec.hidden(ids_of(args, 5, 1), tree, cache, 0)


def test_what_the_drivers_refuse(tiny):
    Q, args, state, packed = tiny
    from mxfp4_int8_m5_amd.sc_draft import DraftTree
    m = Q.FusedQwen3(args, state, packed)
    with pytest.raises(ValueError):
        m.make_cache(16, bits=4)
    cache = m.make_cache(8, bits=8)
    with pytest.raises(ValueError, match="full"):
        m.hidden(ids_of(args, 9, 1), cache)
    dec = Q.DraftQwen3(m)
    with pytest.raises(ValueError, match="full"):
        dec.step(ids_of(args, 9, 1), DraftTree.chain(9), cache)
    with pytest.raises(ValueError):
        dec.step(ids_of(args, 3, 1), DraftTree.chain(4), cache)
    with pytest.raises(ValueError):
        dec.step(ids_of(args, 4, 1), DraftTree.chain(4), cache, temperature=0.5)
    m.hidden(ids_of(args, 8, 1), cache)
    with pytest.raises(ValueError, match="full"):
        Q.DecodeQwen3(m).step(ids_of(args, 1, 1), cache)
