"""Restatement in numpy / float64 of the operators on drafted tokens and 8-bit caches (include/scmx_cache.h), from their
definitions: norm, rotary embedding and 8-bit rows; attention of a tree; verification of drafts, a token at a time.  The reference has no
counterpart to pin them with; tests/test_draft_oracle.py checks them against closed forms."""
import numpy as np

F64 = np.float64


def normed_rows(y, qn, kn, eps, hq, hk, d, positions, inv_freq):
    """float64 q [L, hq, d], k, v [L, hk, d] of the projection's rows y [L, (hq + 2 hk) d], k and q normed and rotated; and the
    absolute values that went into each element of the rotation (how far float32 may be off)."""
    L = len(positions)
    x = np.asarray(y, F64)[:L].reshape(L, hq + 2 * hk, d)
    n = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    n = np.concatenate([n[:, :hq] * np.asarray(qn, F64), n[:, hq:hq + hk] * np.asarray(kn, F64)], 1)
    t = np.asarray(positions, F64)[:, None, None] * np.asarray(inv_freq, F64)
    c, s = np.cos(t), np.sin(t)
    a, b = n[..., :d // 2], n[..., d // 2:]
    r = np.concatenate([a * c - b * s, b * c + a * s], -1)
    mag = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    return r[:, :hq], r[:, hq:], x[:, hq + hk:], mag


def quantize_rows(v):
    """(codes, scale) of rows v [.., d]: scale = max|v| / 127, code = rint(v / scale)."""
    s = np.abs(v).max(-1) / 127
    return np.where(s[..., None] > 0, np.rint(v / np.where(s > 0, s, 1)[..., None]), 0), s


def line_masks(parents):
    """Per node the set of rows of the tree it sees, as a Python integer of bits."""
    m = []
    for i, p in enumerate(parents):
        m.append((m[p] if i else 0) | 1 << i)
    return m


def attention(q, k, v, masks, pos, scale):
    """float64 [T, hq, d]: q [T, hq, d], k, v [hk, >= pos + T, d] (values); and sum p |v|."""
    T, hq, d = q.shape
    hk = k.shape[0]
    out, mag = np.zeros((T, hq, d)), np.zeros((T, hq, d))
    for i in range(T):
        rows = np.array(list(range(pos)) + [pos + j for j in range(T) if masks[i] >> j & 1], int)
        if not len(rows):
            continue
        for h in range(hq):
            kk, vv = k[h // (hq // hk), rows].astype(F64), v[h // (hq // hk), rows].astype(F64)
            s = kk @ q[i, h].astype(F64) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], mag[i, h] = p @ vv, p @ np.abs(vv)
    return out, mag


def softmax64(x, temperature):
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, F64))
    top = x.max()
    with np.errstate(invalid="ignore"):
        e = np.where(x == top, 1.0, np.exp((x - top) / temperature))
    return e / e.sum()


def verify(logits, tokens, parents, temperature=0.0, uniforms=None, draft=None, siblings=16):
    """(path, next): the accepted nodes and the token after them, one test at a time."""
    T, V = logits.shape
    u = None if uniforms is None else [float(x) for x in uniforms]
    cur, path = 0, [0]
    while True:
        kids = [c for c in range(1, T) if parents[c] == cur]
        if temperature == 0:
            best = int(np.argmax(np.where(np.isnan(logits[cur]), -np.inf, logits[cur].astype(F64))))   # the first of equal ones
            taken = next((c for c in kids if tokens[c] == best), None)
        else:
            r = softmax64(logits[cur], temperature)
            taken = None
            for c in kids[:siblings] if draft is not None else kids:
                x = int(tokens[c])
                if draft is None:
                    q = np.zeros(V)
                    if 0 <= x < V:
                        q[x] = 1.0
                else:
                    q = draft[cur].astype(F64)
                if 0 <= x < V and u[c] * q[x] < r[x]:
                    taken = c
                    break
                rest = np.where(q == 1.0, 0.0, r) if draft is None else np.maximum(r - q, 0.0)
                if rest.sum() > 0:
                    r = rest / rest.sum()
        if taken is None:
            if temperature == 0:
                return path, best
            cum = np.cumsum(r)
            over = np.nonzero(cum > u[0] * cum[-1])[0]
            return path, int(over[0]) if len(over) else int(np.nonzero(r)[0][-1])
        cur = taken
        path.append(cur)
