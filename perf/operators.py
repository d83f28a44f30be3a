"""What the operators for drafted tokens over a (quantised) KV cache are timed on and compared with: each in its plain form
(elementary torch operations, 32 bits or more) and, with `own`, as a program calls the library's.

    listed()            the cases, by name
    draw(rng)           one more case of the same kinds and ranges, sizes spread over their logarithm
    prepare(case, seed) the inputs a program holds before the call, on the GPU
    run(state)          one pass
    work(case)          bytes and operations that pass cannot do without
    exact(case, seed)   the same outputs from the definitions, in 64 bits

Kinds: "append" (norm, rotary embedding and append of a prompt's q|k|v to an 8-bit cache, the whole cache read back for its
attention), "attend" (a tree of drafted tokens, or one token, against a cache), "verify" (which drafted tokens the target's
probabilities accept, and the token after them), "accept" (the appends of a tree in every block of a model, the accepted rows
moved together in all of them)."""
import math
import random

import torch

own = False
BF = torch.bfloat16
EPS = 1e-6

# query heads, KV heads, head dim: the attention of the dense models of the benchmark and its tests, and of a quarter of and
# twice that width; "wide" heads are those of a hybrid model's few attention blocks
HEADS = {"small": (14, 2, 64), "medium": (16, 8, 128), "large": (32, 8, 128), "wide": (16, 4, 256)}


def listed():
    return [
        # a prompt's next 900 tokens behind a conversation of 1100, into an 8-bit cache
        {"name": "append_900_behind_1100", "kind": "append", "heads": "medium", "tokens": 900, "cached": 1100},
        # a long first prompt of a larger model
        {"name": "append_2501_large", "kind": "append", "heads": "large", "tokens": 2501, "cached": 0},
        # one token of a short conversation, 8-bit cache: what a decode loop calls most
        {"name": "attend_one_300", "kind": "attend", "heads": "medium", "tokens": 1, "cached": 300, "bits": 8, "shape": "chain"},
        # one token behind a long document, 8-bit cache
        {"name": "attend_one_40000", "kind": "attend", "heads": "medium", "tokens": 1, "cached": 40000, "bits": 8, "shape": "chain"},
        # a small model's drafts, heads of 64 that seven query heads share
        {"name": "attend_chain_7_small_901", "kind": "attend", "heads": "small", "tokens": 7, "cached": 901, "bits": 16, "shape": "chain"},
        # an ordinary tree of drafts in an ordinary conversation
        {"name": "attend_tree_16_3000", "kind": "attend", "heads": "medium", "tokens": 16, "cached": 3000, "bits": 16, "shape": "tree"},
        # the widest tree, a larger model, 8-bit cache
        {"name": "attend_tree_64_large_6000", "kind": "attend", "heads": "large", "tokens": 64, "cached": 6000, "bits": 8, "shape": "tree"},
        # greedy decoding with drafts from the text itself
        {"name": "verify_greedy_5", "kind": "verify", "vocab": 50304, "tokens": 5, "mode": "greedy", "shape": "chain", "dtype": "bf16"},
        # drafts drawn from a draft model's probabilities
        {"name": "verify_drawn_8", "kind": "verify", "vocab": 151936, "tokens": 8, "mode": "drawn", "shape": "chain", "dtype": "bf16"},
        # a wide tree of a draft's likeliest tokens, sampled decoding
        {"name": "verify_tree_60", "kind": "verify", "vocab": 151936, "tokens": 60, "mode": "sampled", "shape": "tree", "dtype": "bf16"},
        # the appends of a tree in every block of a model, then the accepted ones moved together
        {"name": "accept_16_28_blocks", "kind": "accept", "heads": "medium", "tokens": 16, "cached": 500, "bits": 16, "blocks": 28, "shape": "tree"},
        # the same with 8-bit caches
        {"name": "accept_48_8bit", "kind": "accept", "heads": "large", "tokens": 48, "cached": 1203, "bits": 8, "blocks": 8, "shape": "tree"},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "verify", "verify", "accept"])
    heads = rng.choice(sorted(HEADS))
    hq, hk, d = HEADS[heads]
    if kind == "append":
        most = 2501 * 48 * 128 // ((hq + 2 * hk) * d)
        cached = rng.choice([0, _spread(rng, 1, 4000)])
        return {"kind": kind, "heads": heads, "tokens": _spread(rng, 1, min(most, 5000)), "cached": min(cached, 2501 * 8 * 128 // (hk * d))}
    if kind == "attend":
        tokens = rng.choice([1, _spread(rng, 2, 64)])
        most = min(40000 * 8 * 128 // (hk * d), 64 * 32 * 128 * 6000 // (tokens * hq * d))
        return {"kind": kind, "heads": heads, "tokens": tokens, "cached": _spread(rng, 1, min(most, 40000)), "bits": rng.choice([8, 16]),
                "shape": rng.choice(["chain", "tree"])}
    if kind == "verify":
        mode = rng.choice(["greedy", "sampled", "drawn"])
        vocab = rng.choice([32000, 50304, 151936, _spread(rng, 100, 151936)])
        return {"kind": kind, "vocab": vocab, "tokens": _spread(rng, 1, 16 if mode == "drawn" else 60), "mode": mode,
                "shape": rng.choice(["chain", "tree"]), "dtype": rng.choice(["bf16", "f32"]) if vocab <= 50304 else "bf16"}
    return {"kind": kind, "heads": heads, "tokens": _spread(rng, 2, 64), "cached": _spread(rng, 1, 1500), "bits": rng.choice([8, 16]),
            "blocks": rng.choice([4, 6, 8]), "shape": rng.choice(["chain", "tree"])}


# ---- trees ---------------------------------------------------------------------------------------------------------------

def _parents(shape, tokens, seed):
    """parents[i] < i of every node, -1 of the root: a chain, or a tree whose nodes hang on one of the six before them."""
    if shape == "chain":
        return list(range(-1, tokens - 1))
    rng = random.Random(seed)
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, tokens)]


def _plan(parents):
    """What a program derives of a tree: depths, each node's line back to the root as bits, its rank among its siblings."""
    depth, mask, rank, kids = [0], [1], [0], [0] * len(parents)
    for i, p in enumerate(parents[1:], 1):
        depth.append(depth[p] + 1)
        mask.append(mask[p] | 1 << i)
        rank.append(kids[p])
        kids[p] += 1
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    bits = torch.tensor([m - (1 << 64) if m >> 63 else m for m in mask], dtype=torch.int64, device="cuda")
    return {"parents": i32(parents), "depth": i32(depth), "mask": bits, "rank": rank, "siblings": max(kids), "deepest": max(depth)}


# ---- inputs --------------------------------------------------------------------------------------------------------------

class _Source:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, device="cuda", generator=self.g)

    def uniform(self, *shape):
        return torch.rand(shape, device="cuda", generator=self.g)

    def gain(self, n):
        return (1.0 + 0.1 * self.normal(n)).to(BF)

    def qkv(self, tokens, heads):
        """What a q|k|v projection gives: channels of unlike scales, one per cent of them large."""
        hq, hk, d = heads
        n = (hq + 2 * hk) * d
        scale = torch.exp(0.4 * self.normal(n)) * torch.where(self.uniform(n) < 0.01, 8.0, 1.0)
        return (self.normal(tokens, n) * scale).to(BF)

    def rows(self, bits, *shape):
        """Cache rows [.., rows, d]: normed and rotated keys, values; in 8 bits with their scales [.., rows]."""
        v = self.normal(*shape).to(BF)
        if bits == 16:
            return v, None
        v = v.float()
        s = v.abs().amax(-1) / 127
        return torch.round(v / s[..., None]).to(torch.int8), s


def prepare(case, seed):
    src, kind = _Source(seed), case["kind"]
    if kind == "verify":
        return _prepare_verify(case, src, seed)
    hq, hk, d = heads = HEADS[case["heads"]]
    tokens, pos, bits = case["tokens"], case["cached"], case.get("bits", 8)
    rows = pos + tokens + 37   # a cache is longer than what is in it
    st = {"kind": kind, "heads": heads, "tokens": tokens, "pos": pos, "bits": bits,
          "inv_freq": 1.0 / (1e6 ** (torch.arange(d // 2, device="cuda", dtype=torch.float32) / (d // 2)))}
    if kind == "attend":
        st["q"] = src.normal(tokens, hq, d).to(BF).transpose(0, 1)   # the [hq, tokens, d] view of what the append writes
        st["k"], st["ks"] = src.rows(bits, hk, rows, d)
        st["v"], st["vs"] = src.rows(bits, hk, rows, d)
        st["mask"] = _plan(_parents(case["shape"], tokens, seed))["mask"]
        return st
    blocks = case.get("blocks", 1)
    st["qn"], st["kn"] = src.gain(d), src.gain(d)
    st["y"] = [src.qkv(tokens, heads) for _ in range(blocks)]
    st["K"], st["KS"] = src.rows(bits, blocks, hk, rows, d)
    st["V"], st["VS"] = src.rows(bits, blocks, hk, rows, d)
    none = [None] * blocks
    st["caches"] = list(zip(*(none if t is None else list(t) for t in (st["K"], st["V"], st["KS"], st["VS"]))))
    if kind == "accept":
        parents = _parents(case["shape"], tokens, seed)
        st["depth"] = _plan(parents)["depth"]
        line, node = [], tokens - 1   # the last node's line back to the root, accepted to its end or to half of it
        while node >= 0:
            line.insert(0, node)
            node = parents[node]
        count = len(line) if seed % 2 else (len(line) + 1) // 2
        st["path"] = torch.tensor(line[:count] + [-1] * (tokens - count), dtype=torch.int32, device="cuda")
        st["count"] = torch.tensor([count], dtype=torch.int32, device="cuda")
    return st


def _prepare_verify(case, src, seed):
    tokens, vocab, mode = case["tokens"], case["vocab"], case["mode"]
    parents = _parents(case["shape"], tokens, seed)
    st = _plan(parents)
    st |= {"kind": "verify", "mode": mode, "temperature": 0.0 if mode == "greedy" else 0.8, "draft": None}
    # a few likely tokens over a long tail
    logits = 2.0 * src.normal(tokens, vocab)
    top = torch.randint(0, vocab, (tokens, 8), device="cuda", generator=src.g)
    logits.scatter_add_(1, top, 9.0 + 2.0 * src.normal(tokens, 8))
    above = st["parents"].clamp(min=0).long()
    if mode == "drawn":   # the draft's probabilities, and children drawn from their parent's
        st["draft"] = torch.softmax(logits / 0.8 + 0.7 * src.normal(tokens, vocab), -1)
        st["tokens"] = torch.multinomial(st["draft"][above], 1, generator=src.g)[:, 0]
    else:   # a node's children are its likeliest tokens in falling order, now and then with one left out
        likely = logits.topk(min(vocab, 16), -1).indices
        at = torch.tensor(st["rank"], device="cuda") + (src.uniform(tokens) < 0.2).long()
        st["tokens"] = likely[above, at.clamp(max=likely.shape[1] - 1)]
    st["logits"] = logits.to(BF) if case["dtype"] == "bf16" else logits
    st["uniforms"] = src.uniform(tokens)
    return st


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(st):
    return {"append": _append, "attend": _attend, "verify": _verify, "accept": _accept}[st["kind"]](st)


def _append(st):
    if own:
        from mxfp4_int8_m5_amd import sc_cache
        hq, hk, d = st["heads"]
        k, v, ks, vs = st["caches"][0]
        q = sc_cache.cache_write(st["y"][0], st["qn"], st["kn"], EPS, st["tokens"], hq, hk, d, k, v, st["pos"], st["inv_freq"], ks, vs)
        return (q, *sc_cache.cache_read(k, v, ks, vs, st["pos"] + st["tokens"]))
    q = _write_plain(st, 0)
    return (q, *_read_plain(st, 0, 0, st["pos"] + st["tokens"]))


def _attend(st):
    if own:
        from mxfp4_int8_m5_amd import sc_cache
        return sc_cache.attn_tree(st["q"], st["k"], st["v"], st["pos"], st["mask"], st["ks"], st["vs"])
    hq, hk, d = st["heads"]
    n = st["pos"] + st["tokens"]
    value = lambda t, s: t[:, :n].float() if s is None else t[:, :n].float() * s[:, :n, None]   # noqa: E731
    k, v = value(st["k"], st["ks"]), value(st["v"], st["vs"])
    q = st["q"].float().reshape(hk, -1, d)   # the query heads of a KV head and their tokens
    s = torch.matmul(q, k.transpose(1, 2)) * d ** -0.5
    s = s.reshape(hq, st["tokens"], n).masked_fill(~_seen(st), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(hk, -1, n)
    o = torch.matmul(p, v).reshape(hq, st["tokens"], d)
    return o.transpose(0, 1).reshape(st["tokens"], hq * d).to(BF)


def _seen(st):
    """Which of the rows each token sees: [tokens, rows]."""
    at = torch.arange(st["tokens"], device="cuda")
    return torch.cat([torch.ones(st["tokens"], st["pos"], dtype=torch.bool, device="cuda"), (st["mask"][:, None] >> at & 1).bool()], 1)


def _verify(st):
    if own:
        from mxfp4_int8_m5_amd import sc_draft
        return sc_draft.verify_drafts(st["logits"], st["tokens"], st["parents"], st["temperature"], st["uniforms"], st["draft"], st["siblings"])
    logits, tokens, parents, u = st["logits"], st["tokens"], st["parents"].long(), st["uniforms"].double()
    count, vocab = logits.shape
    nodes = torch.arange(count, device="cuda")
    x = logits.double()
    x = x.masked_fill(torch.isnan(x), -math.inf)
    top = x.amax(-1, keepdim=True)
    taken = torch.zeros(count, dtype=torch.bool, device="cuda")
    if st["mode"] == "greedy":
        best = torch.where(x == top, torch.arange(vocab, device="cuda"), vocab).amin(-1)   # the lowest of equal ones
        taken = tokens == best[parents]
    else:
        r = torch.where(x == top, 1.0, torch.exp((x - top) / st["temperature"]))
        r = r / r.sum(-1, keepdim=True)
        rank = torch.tensor(st["rank"], device="cuda")
        for k in range(st["siblings"]):   # the k-th children of all nodes
            child = nodes[1:][rank[1:] == k]
            above, token = parents[child], tokens[child]
            drawn = r[above]
            if st["draft"] is None:
                taken[child] = u[child] < drawn.gather(1, token[:, None])[:, 0]
                rest = drawn.scatter(1, token[:, None], 0.0)
            else:
                q = st["draft"][above].double()
                taken[child] = u[child] * q.gather(1, token[:, None])[:, 0] < drawn.gather(1, token[:, None])[:, 0]
                rest = (drawn - q).clamp(min=0)
            mass = rest.sum(-1, keepdim=True)
            r[above] = torch.where(mass > 0, rest / mass, drawn)
    first = torch.full((count,), count, device="cuda").scatter_reduce(0, parents[1:], torch.where(taken, nodes, count)[1:], "amin")
    at, path = nodes[:1], nodes[:1]
    for _ in range(st["deepest"]):   # from the root down: each node's first accepted child
        at = torch.where(at < count, first[at.clamp(max=count - 1)], at)
        path = torch.cat([path, at])
    length = (path < count).sum().reshape(1)
    last = path[length - 1]
    if st["mode"] == "greedy":
        token = best[last]
    else:
        cum = r[last].cumsum(-1)
        token = torch.searchsorted(cum, u[0] * cum[:, -1:], right=True)[:, 0].clamp(max=vocab - 1)
    full = torch.full((count,), -1, dtype=torch.int32, device="cuda")
    full[:path.shape[0]] = torch.where(path < count, path, -1).int()
    return full, length.int(), token


def _accept(st):
    t, pos, blocks = st["tokens"], st["pos"], range(len(st["y"]))
    if own:
        from mxfp4_int8_m5_amd import sc_cache
        hq, hk, d = st["heads"]
        q = [sc_cache.cache_write(y, st["qn"], st["kn"], EPS, t, hq, hk, d, k, v, pos, st["inv_freq"], ks, vs, depth=st["depth"])
             for y, (k, v, ks, vs) in zip(st["y"], st["caches"])]
        sc_cache.cache_keep(st["caches"], st["path"], st["count"], pos)
        if st["bits"] == 16:
            return q, st["K"], st["V"]
        return q, [sc_cache.cache_read(k, v, ks, vs, t, pos) for k, v, ks, vs in st["caches"]]
    q = [_write_plain(st, i) for i in blocks]
    j = torch.arange(t, device="cuda")
    src = torch.where(j < st["count"], st["path"].long(), j)
    for c in (st["K"], st["V"], st["KS"], st["VS"]):
        if c is not None:
            c[:, :, pos:pos + t] = c[:, :, pos:pos + t][:, :, src]
    if st["bits"] == 16:
        return q, st["K"], st["V"]
    return q, [_read_plain(st, i, pos, t) for i in blocks]


def _write_plain(st, block):
    hq, hk, d = st["heads"]
    t, pos = st["tokens"], st["pos"]
    x = st["y"][block].float().reshape(t, hq + 2 * hk, d)
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    n = torch.cat([n[:, :hq] * st["qn"].float(), n[:, hq:hq + hk] * st["kn"].float()], 1)
    at = pos + (st["depth"] if "depth" in st else torch.arange(t, device="cuda"))
    angle = at.double()[:, None, None] * st["inv_freq"].double()   # 32 bits lose the angles of far positions
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = n[..., :d // 2], n[..., d // 2:]
    n = torch.cat([a * c - b * s, b * c + a * s], -1).transpose(0, 1)
    for rows, scales, new in ((st["K"], st["KS"], n[hq:]), (st["V"], st["VS"], x[:, hq + hk:].transpose(0, 1))):
        if st["bits"] == 16:
            rows[block, :, pos:pos + t] = new.to(BF)
        else:
            scale = new.abs().amax(-1) / 127
            scales[block, :, pos:pos + t] = scale
            rows[block, :, pos:pos + t] = torch.round(torch.where(scale > 0, 1 / scale, 0.0)[..., None] * new).to(torch.int8)
    return n[:hq].to(BF)


def _read_plain(st, block, row, n):
    return tuple((c[block, :, row:row + n].float() * s[block, :, row:row + n, None]).to(BF) for c, s in ((st["K"], st["KS"]), (st["V"], st["VS"])))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    t, kind = case["tokens"], case["kind"]
    if kind == "verify":
        each = (2 if case["dtype"] == "bf16" else 4) + (4 if case["mode"] == "drawn" else 0)
        return {"bytes": each * t * case["vocab"] + 20 * t, "flops": t * case["vocab"] * (1 if case["mode"] == "greedy" else 4)}
    hq, hk, d = HEADS[case["heads"]]
    row = hk * (2 * d + 8 if case.get("bits", 8) == 8 else 4 * d)   # bytes of a token's keys and values
    n = case["cached"] + t
    if kind == "attend":
        return {"bytes": 4 * t * hq * d + row * n + 8 * t, "flops": 4 * t * hq * d * n}
    write = 2 * t * (2 * hq + 2 * hk) * d + row * t
    if kind == "append":   # the rows already there are read; all come back in 16 bits
        return {"bytes": write + row * case["cached"] + 4 * hk * d * n, "flops": 8 * t * (hq + hk) * d}
    back = 4 * hk * d * t if case["bits"] == 8 else 0
    return {"bytes": case["blocks"] * (write + back), "flops": 8 * case["blocks"] * t * (hq + hk) * d}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "verify":
        return None   # node and token numbers
    st = prepare(case, seed)
    hq, hk, d = st["heads"]
    t, pos = st["tokens"], st["pos"]
    if case["kind"] == "attend":
        held = lambda c, s: c[:pos + t].double() * (1.0 if s is None else s[:pos + t, None].double())   # noqa: E731
        out = torch.empty(t, hq, d, dtype=torch.float64, device="cuda")
        lines = [int(m) for m in st["mask"]]
        hidden = torch.tensor([[j >= pos and not lines[i] >> (j - pos) & 1 for j in range(pos, pos + t)] for i in range(t)], device="cuda")
        for h in range(hq):
            g = h // (hq // hk)
            score = (st["q"][h].double() / math.sqrt(d)) @ held(st["k"][g], st["ks"] if st["ks"] is None else st["ks"][g]).T
            score[:, pos:][hidden] = -math.inf
            out[:, h] = torch.softmax(score, -1) @ held(st["v"][g], st["vs"] if st["vs"] is None else st["vs"][g])
        return out.reshape(t, hq * d)
    eight, depth = st["bits"] == 8, st["depth"].double() if "depth" in st else torch.arange(t, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones(t, d // 2, dtype=torch.float64, device="cuda"), torch.outer(depth + pos, st["inv_freq"].double()))
    queries, keys, values = [], [], []
    for block, y in enumerate(st["y"]):
        heads = y.double().reshape(t, hq + 2 * hk, d).permute(1, 0, 2)
        gain = torch.cat([st["qn"].double().expand(hq, d), st["kn"].double().expand(hk, d)])[:, None]
        normed = heads[:hq + hk] / ((heads[:hq + hk] ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * gain
        turned = torch.complex(normed[..., :d // 2], normed[..., d // 2:]) * turn
        turned = torch.cat([turned.real, turned.imag], -1)
        queries.append(turned[:hq])
        for new, rows, scales, into in ((turned[hq:], st["K"], st["KS"], keys), (heads[hq + hk:], st["V"], st["VS"], values)):
            whole = rows[block].double()
            if eight:
                whole = whole * scales[block].double()[..., None]
                step = new.abs().amax(-1, keepdim=True) / 127
                new = torch.round(new / step) * step
            whole[:, pos:pos + t] = new
            if "path" in st:
                kept = whole[:, pos + st["path"][:int(st["count"])].long()]
                whole[:, pos:pos + kept.shape[1]] = kept
            into.append(whole)
    if case["kind"] == "append":
        return queries[0], keys[0][:, :pos + t], values[0][:, :pos + t]
    if eight:
        return queries, [(k[:, pos:pos + t], v[:, pos:pos + t]) for k, v in zip(keys, values)]
    return queries, torch.stack(keys), torch.stack(values)
