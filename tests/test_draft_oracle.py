"""The float64 restatement of the operators on drafted tokens (oracle/draft.py) against closed forms: what verification gives is distributed
as the target, whatever the draft; the residual's closed form; attention's mask; the 8-bit rows."""
import numpy as np
import pytest

from oracle import draft as O


@pytest.mark.parametrize("drawn", [False, True])
def test_verified_tokens_are_distributed_as_the_target(drawn):
    """The exact distribution of the token at the first place after the root, integrated over the random numbers: for two children
    (drawn from q, or given) it has to be softmax(logits)."""
    rng = np.random.default_rng(5)
    V = 5
    logits, q = rng.normal(size=V) * 2, rng.dirichlet(np.ones(V))
    p = O.softmax64(logits, 0.9)
    got = np.zeros(V)
    pairs = [(a, b, q[a] * q[b]) for a in range(V) for b in range(V)] if drawn else [(1, 3, 1.0)]
    for a, b, weight in pairs:
        r = p.copy()
        left = 1.0
        for x in (a, b):
            qx = q if drawn else np.eye(V)[x]
            take = min(1.0, r[x] / qx[x])
            got[x] += weight * left * take
            left *= 1 - take
            rest = np.maximum(r - qx, 0)
            if rest.sum() > 0:
                r = rest / rest.sum()
        got += weight * left * r
    assert np.allclose(got, p, atol=1e-12)


def test_verify_follows_those_probabilities():
    """verify() takes exactly the decisions above: child c where u_c lies below r / q, and the next token by inversion."""
    rng = np.random.default_rng(6)
    V = 7
    logits = rng.normal(size=(3, V)).astype(np.float32)
    p0 = O.softmax64(logits[0], 1.0)
    for u in (0.0, p0[2] * 0.999, p0[2] * 1.001, 0.9999):
        path, nxt = O.verify(logits, [0, 2, 4], [-1, 0, 0], 1.0, [0.3, u, 0.999999])
        if u < p0[2]:
            assert path == [0, 1] and nxt == np.nonzero(np.cumsum(O.softmax64(logits[1], 1.0)) > 0.3)[0][0]
        else:
            r = np.where(np.isin(np.arange(V), [2, 4]), 0, p0)
            assert path == [0] and nxt == np.nonzero(np.cumsum(r / r.sum()) > 0.3)[0][0]
    assert O.verify(np.array([[1.0, 3.0, 3.0]] * 2), [0, 1], [-1, 0])[1] == 1   # equal logits: the lower token


def test_the_residuals_closed_form():
    """r_k = max(a_k p - b_k q, 0) with a, b from the sums alone equals the step-by-step residual."""
    rng = np.random.default_rng(7)
    p, q = rng.dirichlet(np.ones(50)), rng.dirichlet(np.ones(50))
    r, a, b = p.copy(), 1.0, 0.0
    for _ in range(5):
        s = np.maximum(a * p - (b + 1) * q, 0).sum()
        rest = np.maximum(r - q, 0)
        assert s == pytest.approx(rest.sum(), rel=1e-12)
        r, a, b = rest / rest.sum(), a / s, (b + 1) / s
        assert np.allclose(r, np.maximum(a * p - b * q, 0), atol=1e-14)


def test_attention_and_rows():
    rng = np.random.default_rng(8)
    q, k, v = rng.normal(size=(3, 2, 4)), rng.normal(size=(1, 5, 4)), rng.normal(size=(1, 5, 4))
    o, _ = O.attention(q, k, v, [1, 0, 0b101], 0, 0.5)
    assert np.allclose(o[0], v[0, 0]) and not o[1].any()   # one row seen: its value; none: zeros
    assert O.line_masks([-1, 0, 0, 1]) == [1, 0b11, 0b101, 0b1011]
    c, s = O.quantize_rows(np.array([[1.0, -2.0, 0.5], [0, 0, 0]]))
    assert s[0] == 2 / 127 and list(c[0]) == [64, -127, 32] and not c[1].any() and s[1] == 0
    # rotation keeps the length of each pair; position 0 leaves the norm
    y, g = rng.normal(size=(2, 3 * 8)), np.ones(8)
    qr, kr, vr, _ = O.normed_rows(y, g, g, 0.0, 1, 1, 8, [0, 9], 1.0 / 10 ** np.arange(4))
    assert np.allclose((qr ** 2).sum(-1), 8) and np.allclose(vr, y.reshape(2, 3, 8)[:, 2:])
    assert np.allclose(qr[0, 0], y[0, :8] / np.sqrt((y[0, :8] ** 2).mean()))
