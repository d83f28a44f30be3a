"""KV caches in bf16, 8 or 4 bits: the append of new tokens, the read-back, attention for one token or a tree of drafted ones, and the
accepted rows of such a tree moved together (include/scmx_cache.h, scmx_mx.h).  The reference's cache holds the model's type and its
decode step takes one token (e2e/decode.py:29-99); these have no counterpart there.

A cache is a pair of tensors kcache, vcache [hk, rows, d]: bf16, or INT8 beside kscale, vscale float32 [hk, rows], one scale a row; in 4 bits
(MXFP4, see sc_mx) codes uint8 [hk, rows, d / 2] beside kscale, vscale uint8 [hk, rows, d / 32].
Tensors are contiguous, on the current device; work goes to the current stream.  A position is an int, or an int64 device tensor (for
graph replay; one whose rows do not fit the cache appends and moves nothing, and its attention is zero)."""
from array import array

import torch

from . import _lib

BF = torch.bfloat16
MAX_NODES = 64   # of a tree: the bits of a mask


class Q8Cache:
    """A block's keys and values in 8 bits, with a write offset: what fused_qwen3.KVCache is in bf16, in half its bytes."""

    def __init__(self, args, max_len, device="cuda"):
        shape = (args.num_key_value_heads, max_len, args.head_dim)
        self.k = torch.zeros(shape, dtype=torch.int8, device=device)
        self.v = torch.zeros(shape, dtype=torch.int8, device=device)
        self.kscale = torch.zeros(shape[:2], dtype=torch.float32, device=device)
        self.vscale = torch.zeros(shape[:2], dtype=torch.float32, device=device)
        self.offset = 0


class Q4Cache:
    """The same in 4 bits (MXFP4): 4.25 bits a value, little more than a quarter of bf16."""

    def __init__(self, args, max_len, device="cuda"):
        hk, d = args.num_key_value_heads, args.head_dim
        _check(d in (64, 128, 256), "a 4-bit cache has heads of 64, 128 or 256")
        zeros = lambda n: torch.zeros((hk, max_len, n), dtype=torch.uint8, device=device)   # noqa: E731
        self.k, self.v, self.kscale, self.vscale = zeros(d // 2), zeros(d // 2), zeros(d // 32), zeros(d // 32)
        self.offset = 0


FEW_BITS = Q8Cache, Q4Cache


def tensors(cache):
    """(k, v, kscale, vscale) of a cache object; the scales are None in bf16."""
    return cache.k, cache.v, getattr(cache, "kscale", None), getattr(cache, "vscale", None)


def _on_device(*ts):
    here = torch.cuda.current_device() if any(t is not None and t.is_cuda for t in ts) else None
    for t in ts:
        if t is not None and (not t.is_cuda or t.get_device() != here):
            raise ValueError("scmx kernels take CUDA (ROCm) tensors on the current device")


def _check(cond, what):
    if not cond:
        raise ValueError(what)


def _check_cache(kcache, vcache, kscale, vscale):
    """(hk, rows, d) of a cache whose tensors belong together."""
    _check(kcache.dim() == 3 and kcache.shape == vcache.shape and kcache.dtype == vcache.dtype,
           "kcache and vcache are [hk, rows, d] of one type")
    _check((kscale is None) == (vscale is None), "an 8-bit cache has both scales, a bf16 one none")
    if kscale is None:
        _check(kcache.dtype == BF, "a cache without scales is bfloat16")
    elif _four(kscale):
        hk, rows, half = kcache.shape
        _check(kcache.dtype == torch.uint8 == vscale.dtype and half % 16 == 0 and tuple(kscale.shape) == tuple(vscale.shape) == (hk, rows, half // 16),
               "a 4-bit cache is uint8 [hk, rows, d / 2] beside uint8 scales [hk, rows, d / 32]")
        return torch.Size((hk, rows, 2 * half))
    else:
        _check(kcache.dtype == torch.int8 and kscale.dtype == vscale.dtype == torch.float32
               and kscale.shape == vscale.shape == kcache.shape[:2], "an 8-bit cache is int8 beside float32 scales [hk, rows]")
    return kcache.shape


def _four(kscale):
    """Whether the cache with these scales is in 4 bits."""
    return kscale is not None and kscale.dtype == torch.uint8


def _position(pos):
    """(device tensor or None, int) of a position."""
    if not torch.is_tensor(pos):
        return None, int(pos)
    _check(pos.dtype == torch.int64 and pos.numel() == 1, "a position on the device is an int64 tensor of one value")
    return pos, 0


def cache_write(y, qn, kn, eps, L, hq, hk, d, kcache, vcache, pos, inv_freq, kscale=None, vscale=None, depth=None, acc=None, xscale=None,
                wscale=None):
    """Per-head RMSNorm of q and k, rotary embedding and the append to rows pos .. pos + L - 1 of a cache in bf16, 8 or 4 bits:
    y bf16 [>= L, (hq + 2 hk) d], or acc int32 with xscale and wscale as in sc_kernels.qkv_headnorm_rope -> q, the [hq, L, d] view of
    [L, hq, d] storage.  depth int32 [L]: token i is rotated as position pos + depth[i] (the depths of a tree's nodes; default i).
    Computed in float32 (4 bits: float64), rounded once."""
    q = _lib.native().cache_write(y, qn, kn, eps, L, hq, hk, d, kcache, vcache, pos, inv_freq, kscale, vscale, depth)
    if q is not None:   # the operands of every step; anything else is converted or refused below
        return q
    src = y if y is not None else acc
    _check(src is not None and src.dim() == 2 and src.shape[0] >= L >= 0 and src.shape[1] == (hq + 2 * hk) * d,
           "y or acc is [>= L, (hq + 2 hk) d]")
    _check(src.dtype == (BF if y is not None else torch.int32), "y is bfloat16, acc int32")
    if y is None:
        _check(xscale is not None and wscale is not None and xscale.dtype == wscale.dtype == torch.float32 and xscale.numel() >= L
               and wscale.numel() == src.shape[1], "acc needs xscale float32 [>= L] and wscale float32 [(hq + 2 hk) d]")
    _check(tuple(_check_cache(kcache, vcache, kscale, vscale)[::2]) == (hk, d), "the cache is [hk, rows, d]")
    _check(qn.dtype == kn.dtype == BF and qn.numel() == kn.numel() == d, "qn and kn are bfloat16 [d]")
    _check(inv_freq.dtype == torch.float32 and inv_freq.numel() == d // 2, "inv_freq is float32 [d / 2]")
    _check(depth is None or (depth.dtype == torch.int32 and depth.numel() == L), "depth is int32 [L]")
    dev_pos, at = _position(pos)
    _on_device(src, qn, kn, kcache, vcache, kscale, vscale, inv_freq, depth, dev_pos, *((xscale, wscale) if y is None else ()))
    q = _lib.native().empty_bf16(src, L, hq, d)
    write = _lib.native().scmx_cache4_write if _four(kscale) else _lib.native().scmx_cache_write
    write(None if y is not None else acc, xscale, wscale, y, qn, kn, float(eps), q, kcache, vcache, kscale, vscale, L, hq, hk, d, inv_freq,
          depth, dev_pos, at, kcache.shape[1])
    return q.transpose(0, 1)


def cache_read(kcache, vcache, kscale, vscale, n, row0=0):
    """Rows row0 .. row0 + n - 1 of an 8-bit or 4-bit cache as bf16: (k, v) [hk, n, d], what a prompt's attention takes."""
    out = _lib.native().cache_read(kcache, vcache, kscale, vscale, n, row0)
    if out is not None:
        return out
    _check(kscale is not None, "rows of an 8-bit cache (a bf16 one is read as it is)")
    hk, rows, d = _check_cache(kcache, vcache, kscale, vscale)
    _check(0 <= n <= rows and 0 <= row0 <= rows - n, f"{n} rows from {row0} on do not fit a cache of {rows} rows")
    _on_device(kcache, vcache, kscale, vscale)
    k, v = (_lib.native().empty_bf16(kcache, hk, n, d) for _ in range(2))
    read = _lib.native().scmx_cache4_read if _four(kscale) else _lib.native().scmx_cache_read
    read(kcache, vcache, kscale, vscale, k, v, hk, d, rows, int(row0), int(n))
    return k, v


def cache_keep(caches, path, count, pos):
    """Row pos + j of every cache takes what row pos + path[j] held, for j < count: the accepted line of a tree moved together, all
    blocks in one launch (up to 32 of them).  caches: (kcache, vcache, kscale, vscale) a block, all of one shape and type; path int32 [T],
    count int32 [1] as verify_drafts returns them.  Rows from pos + count on keep what they hold."""
    if _lib.native().cache_keep(caches, path, count, pos):
        return
    caches = [tuple(c) for c in caches]
    if not caches:
        return
    shape = _check_cache(*caches[0])
    eight, four = caches[0][2] is not None, _four(caches[0][2])
    for c in caches[1:]:
        _check(_check_cache(*c) == shape and (c[2] is not None) == eight and _four(c[2]) == four, "the caches are of one shape and type")
    _check(path.dtype == count.dtype == torch.int32 and count.numel() == 1, "path is int32 [T], count int32 [1]")
    dev_pos, at = _position(pos)
    flat = [t for c in caches for t in c[:4 if eight else 2]]
    _check(all(t.is_contiguous() for t in flat), "scmx kernels take contiguous tensors")
    _on_device(path, count, dev_pos, *flat)
    pointers = array("Q", [t.data_ptr() for t in flat])
    sizes = (shape[0], shape[2], shape[1], path, count, path.numel(), dev_pos, at)
    if four:
        _lib.native().scmx_cache4_keep(pointers.buffer_info()[0], len(caches), *sizes)
    else:
        _lib.native().scmx_cache_keep(pointers.buffer_info()[0], len(caches), int(eight), *sizes)


def attn_tree_splits(T, n, hq, hk, d, bits=16):
    """Ranges that n rows are cut into for T nodes; bits as FusedQwen3.make_cache names them: 16, 8 or "mxfp4" (or 4)."""
    _check(bits in (16, 8, 4, "mxfp4"), 'a cache has 16 or 8 bits, or is in "mxfp4"')
    return (_lib.native().scmx_attn_tree4_splits if bits in (4, "mxfp4") else _lib.native().scmx_attn_tree_splits)(T, n, hq, hk, d)


def attn_tree(q, kcache, vcache, pos, mask=None, kscale=None, vscale=None, scale=None, splits=None):
    """Attention of T drafted tokens (1..64; one: a decode step's) in rows pos .. pos + T - 1 of a cache: q bf16 [hq, T, d], best as the
    view that cache_write returns (any other layout is copied) -> bf16 [T, hq * d].  All see the rows below pos; token i sees row
    pos + j if bit j of mask[i] (int64 [T]; default: a chain) is set; one that sees nothing gets zeros.  splits: ranges the rows are cut
    into (default: by the sizes; by the cache's when the position is on the device)."""
    out = _lib.native().attn_tree(q, kcache, vcache, pos, mask, kscale, vscale, scale, splits)
    if out is not None:
        return out
    q = q.transpose(0, 1).contiguous()   # [T, hq, d]; no copy when q already is a view of it
    T, hq, d = q.shape
    hk, rows, dc = _check_cache(kcache, vcache, kscale, vscale)
    _check(q.dtype == BF and dc == d and hk > 0 and hq % hk == 0, "q is bfloat16 [hq, T, d], hq a multiple of hk")
    _check(1 <= T <= MAX_NODES, "a tree has 1..64 nodes")
    _check(mask is None or (mask.dtype == torch.int64 and mask.numel() == T), "mask is int64 [T]")
    dev_pos, at = _position(pos)
    _on_device(q, kcache, vcache, kscale, vscale, mask, dev_pos)
    out = _lib.native().empty_bf16(q, T, hq * d)
    if splits is None:
        splits = attn_tree_splits(T, rows if dev_pos is not None else at + T, hq, hk, d, 4 if _four(kscale) else 16)
    work = _lib.native().empty_f32(q, splits * T * hq * (d + 2)) if splits > 1 else None
    attend = _lib.native().scmx_attn_tree4 if _four(kscale) else _lib.native().scmx_attn_tree
    attend(q, kcache, vcache, kscale, vscale, mask, dev_pos, at, out, T, hq, hk, d, rows, float(scale if scale is not None else d ** -0.5),
           work, splits)
    return out
