"""Trees of drafted tokens and their verification against the target's probabilities (include/scmx_cache.h).  The reference decodes a token
at a time (e2e/decode.py:29-99)."""
import torch

from . import _lib
from .sc_cache import BF, MAX_NODES, _check, _on_device

MAX_SIBLINGS = 16   # children of a node that are tried against a draft's probabilities


class DraftTree:
    """The shape of a tree of drafted tokens: parents[i] < i, -1 for node 0, the sequence's newest token.  On the device: `parents` and
    `depth` int32 [T], `mask` int64 [T] (a node sees itself and its line back to the root), views of `packed`.  `siblings`: the most
    children of a node."""

    def __init__(self, parents, device="cuda"):
        parents = [int(p) for p in parents]
        _check(1 <= len(parents) <= MAX_NODES, "a tree has 1..64 nodes")
        _check(parents[0] == -1 and all(0 <= p < i for i, p in enumerate(parents[1:], 1)), "parents[0] is -1, parents[i] one of 0 .. i - 1")
        depth, mask, kids = [0], [1], [0] * len(parents)
        for i, p in enumerate(parents[1:], 1):
            depth.append(depth[p] + 1)
            mask.append(mask[p] | 1 << i)
            kids[p] += 1
        self.T, self.parent_list, self.depth_list, self.siblings = len(parents), parents, depth, max(kids)
        mask = torch.tensor([m - (1 << 64) if m >> 63 else m for m in mask], dtype=torch.int64)
        self.packed = torch.cat([mask.view(torch.int32), torch.tensor(depth + parents, dtype=torch.int32)]).to(device)
        self.mask, self.depth, self.parents = self.unpack(self.packed)

    @staticmethod
    def unpack(packed):
        """(mask, depth, parents): views of int32 [4 T]."""
        T = packed.numel() // 4
        return packed[:2 * T].view(torch.int64), packed[2 * T:3 * T], packed[3 * T:]

    @classmethod
    def chain(cls, T, device="cuda"):
        return cls(range(-1, T - 1), device)


def verify_drafts(logits, tokens, parents, temperature=0.0, uniforms=None, draft=None, siblings=None):
    """Which drafted tokens the target accepts, and the token after them: logits bf16 or float32 [T, V] (the target's after each node),
    tokens int64 [T], parents int32 [T] -> (path int32 [T], count int32 [1], next int64 [1]), all on the device: the accepted nodes from
    node 0 on, -1 behind them, their number, the next token.
    temperature 0: greedy.  Otherwise uniforms float32 [T] in [0, 1) decide (entry 0 draws the next token, entry c tries node c), in
    float64, such that the tokens are distributed as softmax(logits / temperature) whatever the draft was.  draft float32 [T, V]: the
    distributions that a node's children were drawn from, with siblings, the most children of a node (1..16; further ones are not tried).
    Without it the drafts are taken as given (a draft's likeliest tokens, tokens from the text)."""
    _check(logits.dim() == 2 and logits.dtype in (BF, torch.float32), "logits are bfloat16 or float32 [T, V]")
    T, V = logits.shape
    _check(tokens.dtype == torch.int64 and parents.dtype == torch.int32 and tokens.numel() == parents.numel() == T,
           "tokens are int64 [T], parents int32 [T]")
    temperature = float(temperature)
    levels = 0
    if temperature == 0:
        uniforms = draft = None
    else:
        _check(uniforms is not None and uniforms.dtype == torch.float32 and uniforms.numel() == T, "uniforms are float32 [T]")
        if draft is not None:
            _check(draft.dtype == torch.float32 and draft.shape == logits.shape, "draft is float32 [T, V]")
            _check(siblings is not None and 0 <= siblings, "a draft needs siblings, the most children of a node")
            levels = min(max(int(siblings), 1), MAX_SIBLINGS)
    out = _lib.native().verify_drafts(logits, tokens, parents, temperature, uniforms, draft, levels)
    if out is not None:
        return out
    _on_device(logits, tokens, parents, uniforms, draft)
    n = _lib.native()
    path, count, token = n.empty_i32(logits, T), n.empty_i32(logits, 1), n.empty_i64(logits, 1)
    need = n.scmx_verify_workspace(T, V, levels)
    work = n.empty_u8(logits, need)
    n.scmx_verify_drafts(tokens, parents, logits, int(logits.dtype == torch.float32), draft, temperature, uniforms, path, count, token, T,
                         V, levels, work, need)
    return path, count, token
