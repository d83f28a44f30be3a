"""What the operators on microscaled 4-bit values (MXFP4: E2M1 codes, a power of two a block of 32) are timed on and compared with: each in
its plain form (elementary torch operations, 32 bits or more) and, with `own`, as a program calls the library's.

    listed()            the cases, by name
    draw(rng)           one more case of the same kinds and ranges, sizes spread over their logarithm
    prepare(case, seed) the inputs a program holds before the call, on the GPU
    run(state)          one pass
    work(case)          bytes and operations that pass cannot do without
    exact(case, seed)   the same outputs from the definitions, in 64 bits

Kinds: "quantize" (activations, with or without their RMSNorm, or float weights; returned as the values that the codes stand for), "linear"
(rows of bf16 activations, quantised, times an MXFP4 weight), "append" (norm, rotary embedding and append of q|k|v to a 4-bit cache, rows read
back), "attend" (one token, or a tree of drafted tokens, against a 4-bit cache)."""
import math
import random

import torch

own = False
BF = torch.bfloat16
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# query heads, KV heads, head dim: the attention of the dense models of the benchmark and its tests, and of a quarter of and
# twice that width; "wide" heads are those of a hybrid model's few attention blocks
HEADS = {"small": (14, 2, 64), "medium": (16, 8, 128), "large": (32, 8, 128), "wide": (16, 4, 256)}


def listed():
    return [
        # the norm in front of a single token's projections
        {"name": "quantize_norm_1x2048", "kind": "quantize", "rows": 1, "width": 2048, "dtype": "bf16", "norm": True, "wider": 0},
        # the same of a long prompt
        {"name": "quantize_norm_8192x2048", "kind": "quantize", "rows": 8192, "width": 2048, "dtype": "bf16", "norm": True, "wider": 0},
        # gate and up projection of a single token, with the activation
        {"name": "linear_1_gate_up", "kind": "linear", "rows": 1, "out": 12288, "width": 2048, "epilogue": 3},
        # down projection of a few drafted tokens, onto the residual
        {"name": "linear_5_down", "kind": "linear", "rows": 5, "out": 2048, "width": 6144, "epilogue": 2},
        # a short prompt through a layer of odd sizes
        {"name": "linear_333_ragged", "kind": "linear", "rows": 333, "out": 5004, "width": 2912, "epilogue": 1},
        # the joined q|k|v projection of an ordinary prompt
        {"name": "linear_2048_qkv", "kind": "linear", "rows": 2048, "out": 4096, "width": 2048, "epilogue": 1},
        # gate and up projection of a long prompt, with the activation
        {"name": "linear_8192_gate_up", "kind": "linear", "rows": 8192, "out": 12288, "width": 2048, "epilogue": 3},
        # one token's keys and values, behind a long conversation: what a decode loop calls in every block
        {"name": "append_1_behind_5000", "kind": "append", "heads": "medium", "tokens": 1, "cached": 5000, "read": "new"},
        # a prompt's next 900 tokens behind a conversation of 1100, read back for its attention
        {"name": "append_900_behind_1100", "kind": "append", "heads": "medium", "tokens": 900, "cached": 1100, "read": "all"},
        # one token of a short conversation
        {"name": "attend_one_300", "kind": "attend", "heads": "medium", "tokens": 1, "cached": 300, "shape": "chain"},
        # one token behind a long document
        {"name": "attend_one_40000", "kind": "attend", "heads": "medium", "tokens": 1, "cached": 40000, "shape": "chain"},
        # the widest tree of drafts, a larger model
        {"name": "attend_tree_64_large_6000", "kind": "attend", "heads": "large", "tokens": 64, "cached": 6000, "shape": "tree"},
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "append", "attend", "attend"])
    if kind == "quantize":
        norm = rng.random() < 0.5
        dtype = "bf16" if norm else rng.choice(sorted(TYPES))
        width = 32 * _spread(rng, 2, 512)
        most = 8192 * 2048 // width // (2 if dtype == "f32" else 1)
        return {"kind": kind, "rows": _spread(rng, 1, min(most, 16384)), "width": width, "dtype": dtype, "norm": norm,
                "wider": rng.choice([0, 0, 32 * _spread(rng, 1, 64)])}
    if kind == "linear":
        epilogue = rng.choice([1, 2, 3])
        rows = rng.choice([1, _spread(rng, 2, 16), _spread(rng, 17, 8192), _spread(rng, 17, 8192)])
        width, out = 32 * _spread(rng, 4, 256), 4 * _spread(rng, 16, 4096)
        while rows * width * out > 8192 * 12288 * 2048 // 2:
            rows = rows // 2 + 1
        return {"kind": kind, "rows": rows, "out": out, "width": width, "epilogue": epilogue}
    heads = rng.choice(sorted(HEADS))
    hq, hk, d = HEADS[heads]
    if kind == "append":
        cached = rng.choice([0, _spread(rng, 1, 4000)])
        return {"kind": kind, "heads": heads, "tokens": rng.choice([1, _spread(rng, 2, 1000 * 4096 // ((hq + 2 * hk) * d))]),
                "cached": cached, "read": rng.choice(["new", "all"])}
    tokens = rng.choice([1, _spread(rng, 2, 64)])
    most = min(40000 * 8 * 128 // (hk * d), 64 * 32 * 128 * 6000 // (tokens * hq * d))
    return {"kind": kind, "heads": heads, "tokens": tokens, "cached": _spread(rng, 1, min(most, 40000)), "shape": rng.choice(["chain", "tree"])}


# ---- the format ----------------------------------------------------------------------------------------------------------

def _power(e):
    """2^e, exactly: the exponent field of a float32."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _round(v):
    """(codes' values, exponents) of v [.., K], blocks of 32: a power of two two below the largest value's, E2M1 to nearest even."""
    b = v.unflatten(-1, (-1, 32))
    e = (torch.frexp(b.abs().amax(-1, keepdim=True)).exponent - 3).clamp(-126, 126)
    a = (b * _power(-e)).clamp(-6, 6)
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return torch.round(a / step) * step, e


def _rounded(v):
    """v [.., K] as the values that its codes stand for."""
    a, e = _round(v)
    return (a * _power(e)).flatten(-2)


def _packed(v):
    """(codes uint8 [.., K / 2], scales uint8 [.., K / 32]) of v [.., K]: what a program holds."""
    a, e = _round(v)
    m = a.abs()
    c = torch.where(m < 2, 2 * m, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8) | ((a < 0).to(torch.uint8) << 3)
    c = c.flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), (e[..., 0] + 127).to(torch.uint8)


def _values(codes, scales):
    """The float32 values of codes [.., K / 2] and scales [.., K / 32]."""
    level = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = level[(c & 7).long()] * (1.0 - 2.0 * (c >> 3).float())
    return (v.unflatten(-1, (-1, 32)) * _power(scales[..., None].int() - 127)).flatten(-2)


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

    def activations(self, rows, n):
        """Channels of unlike scales, one per cent of them large."""
        return self.normal(rows, n) * torch.exp(0.4 * self.normal(n)) * torch.where(self.uniform(n) < 0.01, 8.0, 1.0)


def _parents(shape, tokens, seed):
    """parents[i] < i of every node, -1 of the root: a chain, or a tree whose nodes hang on one of the six before them."""
    if shape == "chain":
        return list(range(-1, tokens - 1))
    rng = random.Random(seed)
    return [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, tokens)]


def prepare(case, seed):
    src, kind = _Source(seed), case["kind"]
    st = {"kind": kind}
    if kind == "quantize":   # rows of a wider tensor now and then (a part of a joined projection)
        rows, width = case["rows"], case["width"]
        x = src.activations(rows, width + case["wider"]) * (1.0 if case["norm"] or case["dtype"] != "f32" else 0.02)
        st["x"] = x.to(TYPES[case["dtype"]])[:, :width]
        st["gain"] = src.gain(width) if case["norm"] else None
        return st
    if kind == "linear":
        rows, out, width = case["rows"], case["out"], case["width"]
        st["epilogue"] = case["epilogue"]
        st["x"] = src.activations(rows, width).to(BF)
        st["codes"], st["scales"] = _packed(src.normal(out, width) * (0.7 * width ** -0.5) * torch.exp(0.3 * src.normal(out, 1)))
        st["residual"] = src.normal(rows, out).to(BF) if case["epilogue"] == 2 else None
        return st
    hq, hk, d = st["heads"] = HEADS[case["heads"]]
    tokens, pos = st["tokens"], st["pos"] = case["tokens"], case["cached"]
    rows = pos + tokens + 37   # a cache is longer than what is in it
    st["k"], st["ks"] = _packed(src.normal(hk, rows, d))   # normed and rotated keys, values
    st["v"], st["vs"] = _packed(src.normal(hk, rows, d))
    if kind == "attend":
        st["q"] = src.normal(tokens, hq, d).to(BF).transpose(0, 1)   # the [hq, tokens, d] view of what the append writes
        line = [1]   # each node's line back to the root, as bits
        for i, p in enumerate(_parents(case["shape"], tokens, seed)[1:], 1):
            line.append(line[p] | 1 << i)
        st["mask"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in line], dtype=torch.int64, device="cuda")
        return st
    st["inv_freq"] = 1.0 / (1e6 ** (torch.arange(d // 2, device="cuda", dtype=torch.float32) / (d // 2)))
    st["qn"], st["kn"] = src.gain(d), src.gain(d)
    st["y"] = src.activations(tokens, (hq + 2 * hk) * d).to(BF)
    st["first"] = 0 if case["read"] == "all" else pos   # the rows read back: from there on
    return st


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(st):
    return {"quantize": _quantize, "linear": _linear, "append": _append, "attend": _attend}[st["kind"]](st)


def _quantize(st):
    if own:
        from mxfp4_int8_m5_amd import sc_mx
        return sc_mx.dequantize(*sc_mx.quantize(st["x"], st["gain"], EPS))
    x = st["x"]
    if st["gain"] is not None:   # in 64 bits: a value next to the border of two codes takes the right one
        x = x.double()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * st["gain"].double()
        return _rounded(x).to(BF)
    return _rounded(x.float()).to(BF)


def _linear(st):
    if own:
        from mxfp4_int8_m5_amd import sc_mx
        return sc_mx.linear(st["x"], st["codes"], st["scales"], st["epilogue"], st["residual"])
    y = torch.matmul(_rounded(st["x"].float()), _values(st["codes"], st["scales"]).T)
    if st["epilogue"] == 2:
        y = y + st["residual"].float()
    elif st["epilogue"] == 3:   # two gates, their two ups, and so on
        y = y.unflatten(-1, (-1, 2, 2))
        gate, up = y[:, :, 0], y[:, :, 1]
        y = (gate / (1 + torch.exp(-gate)) * up).flatten(-2)
    return y.to(BF)


def _append(st):
    hq, hk, d = st["heads"]
    t, pos, first = st["tokens"], st["pos"], st["first"]
    n = pos + t - first
    if own:
        from mxfp4_int8_m5_amd import sc_cache
        q = sc_cache.cache_write(st["y"], st["qn"], st["kn"], EPS, t, hq, hk, d, st["k"], st["v"], pos, st["inv_freq"], st["ks"], st["vs"])
        return (q, *sc_cache.cache_read(st["k"], st["v"], st["ks"], st["vs"], n, first))
    x = st["y"].double().reshape(t, hq + 2 * hk, d)   # 64 bits: angles of far positions, values next to the border of two codes
    v = x[:, hq + hk:].transpose(0, 1)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    x = torch.cat([x[:, :hq] * st["qn"].double(), x[:, hq:hq + hk] * st["kn"].double()], 1)
    angle = (pos + torch.arange(t, device="cuda")).double()[:, None, None] * st["inv_freq"].double()
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = x[..., :d // 2], x[..., d // 2:]
    x = torch.cat([a * c - b * s, b * c + a * s], -1).transpose(0, 1)
    for new, codes, scales in ((x[hq:], st["k"], st["ks"]), (v, st["v"], st["vs"])):
        codes[:, pos:pos + t], scales[:, pos:pos + t] = _packed(new)
    back = slice(first, first + n)
    return x[:hq].to(BF), _values(st["k"][:, back], st["ks"][:, back]).to(BF), _values(st["v"][:, back], st["vs"][:, back]).to(BF)


def _attend(st):
    if own:
        from mxfp4_int8_m5_amd import sc_cache
        return sc_cache.attn_tree(st["q"], st["k"], st["v"], st["pos"], st["mask"], st["ks"], st["vs"])
    hq, hk, d = st["heads"]
    t, n = st["tokens"], st["pos"] + st["tokens"]
    k, v = _values(st["k"][:, :n], st["ks"][:, :n]), _values(st["v"][:, :n], st["vs"][:, :n])
    q = st["q"].float().reshape(hk, -1, d)   # the query heads of a KV head and their tokens
    s = torch.matmul(q, k.transpose(1, 2)) * d ** -0.5
    seen = torch.cat([torch.ones(t, st["pos"], dtype=torch.bool, device="cuda"),
                      (st["mask"][:, None] >> torch.arange(t, device="cuda") & 1).bool()], 1)
    s = s.reshape(hq, t, n).masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(hk, -1, n)
    o = torch.matmul(p, v).reshape(hq, t, d)
    return o.transpose(0, 1).reshape(t, hq * d).to(BF)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quantize":   # in, and the codes' values out
        n = case["rows"] * case["width"]
        return {"bytes": n * ((4 if case["dtype"] == "f32" else 2) + 2), "flops": n * (5 if case["norm"] else 2)}
    if kind == "linear":
        m, n, k = case["rows"], case["out"], case["width"]
        out = m * (n // 2 if case["epilogue"] == 3 else n * case["epilogue"])
        return {"bytes": 2 * m * k + n * k * 17 // 32 + 2 * out, "flops": 2 * m * n * k}
    hq, hk, d = HEADS[case["heads"]]
    t, n = case["tokens"], case["cached"] + case["tokens"]
    row = hk * d * 17 // 16   # bytes of a token's keys and values
    if kind == "attend":
        return {"bytes": 4 * t * hq * d + row * n + 8 * t, "flops": 4 * t * hq * d * n}
    back = n if case["read"] == "all" else t
    return {"bytes": 2 * t * (2 * hq + 2 * hk) * d + row * back + 4 * hk * d * back, "flops": 8 * t * (hq + hk) * d}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _unit(e):
    return (e + 1023 << 52).view(torch.float64)


def _nearest(v):
    """v [.., K] in 64 bits on the grid of its blocks: of the eight magnitudes the nearest, of two as near the one of even number."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    border = (grid[1:] + grid[:-1]) / 2
    b = v.double().reshape(*v.shape[:-1], -1, 32)
    unit = _unit((b.abs().amax(-1, keepdim=True).view(torch.int64) >> 52) - 1023 - 2)   # by the exponent field
    a = (b / unit).abs()
    low, high = torch.bucketize(a, border), torch.bucketize(a, border, right=True)   # they differ on a border
    return (grid[torch.where(low % 2 == 0, low, high)] * torch.sign(b) * unit).reshape(v.shape)


def _held(codes, scales):
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device="cuda")
    out[..., 0::2], out[..., 1::2] = grid[(codes % 16).long()], grid[(codes // 16).long()]
    return out * _unit(scales.long() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        x = st["x"].double()
        if case["norm"]:
            x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * st["gain"].double()
        return _nearest(x)
    if kind == "linear":
        x, w = _nearest(st["x"]), _held(st["codes"], st["scales"])
        if case["epilogue"] == 3:
            rows = torch.arange(case["out"], device="cuda").reshape(-1, 4)
            gate, up = x @ w[rows[:, :2].flatten()].T, x @ w[rows[:, 2:].flatten()].T
            return gate * torch.sigmoid(gate) * up
        y = x @ w.T
        return y if case["epilogue"] == 1 else y + st["residual"].double()
    hq, hk, d = st["heads"]
    t, pos = st["tokens"], st["pos"]
    if kind == "attend":
        out = torch.empty(t, hq, d, dtype=torch.float64, device="cuda")
        lines = [int(m) for m in st["mask"]]
        hidden = torch.tensor([[not lines[i] >> j & 1 for j in range(t)] for i in range(t)], device="cuda")
        for h in range(hq):
            g = h // (hq // hk)
            score = (st["q"][h].double() / math.sqrt(d)) @ _held(st["k"][g, :pos + t], st["ks"][g, :pos + t]).T
            score[:, pos:][hidden] = -math.inf
            out[:, h] = torch.softmax(score, -1) @ _held(st["v"][g, :pos + t], st["vs"][g, :pos + t])
        return out.reshape(t, hq * d)
    turn = torch.polar(torch.ones(t, d // 2, dtype=torch.float64, device="cuda"),
                       torch.outer(torch.arange(pos, pos + t, device="cuda", dtype=torch.float64), st["inv_freq"].double()))
    heads = st["y"].double().reshape(t, hq + 2 * hk, d).permute(1, 0, 2)
    gain = torch.cat([st["qn"].double().expand(hq, d), st["kn"].double().expand(hk, d)])[:, None]
    normed = heads[:hq + hk] / ((heads[:hq + hk] ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * gain
    turned = torch.complex(normed[..., :d // 2], normed[..., d // 2:]) * turn
    turned = torch.cat([turned.real, turned.imag], -1)
    old = slice(st["first"], pos)
    k = torch.cat([_held(st["k"][:, old], st["ks"][:, old]), _nearest(turned[hq:])], 1)
    v = torch.cat([_held(st["v"][:, old], st["vs"][:, old]), _nearest(heads[hq + hk:])], 1)
    return turned[:hq], k, v
