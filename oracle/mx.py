"""Restatement in numpy / float64 of microscaled 4-bit values (include/scmx_mx.h), from their definition: E2M1 codes, an E8M0 exponent for 32
values.  The reference has no counterpart to pin them with; tests/test_mx_oracle.py checks them against closed forms."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize(v, least=0, most=254):
    """(codes uint8 [.., K / 2], scales uint8 [.., K / 32]) of v [.., K]; least, most: of a finite block's byte."""
    v = np.asarray(v, np.float64)
    b = v.reshape(*v.shape[:-1], -1, 32)
    fine = np.isfinite(b).all(-1)
    b = np.where(fine[..., None], b, 0)
    top = np.abs(b).max(-1)
    e = np.frexp(top)[1] - 1 - 2   # floor(log2) less 2
    byte = np.clip(np.where(top == 0, 0, e + 127), least, most).astype(np.int64)
    a = np.minimum(np.ldexp(np.abs(b), 127 - byte[..., None]), 1e9)
    border = (LEVELS[1:] + LEVELS[:-1]) / 2
    code = (a[..., None] > border).sum(-1)
    on = (a[..., None] == border).argmax(-1)   # on border i, between codes i and i + 1: the even one
    code = np.where((a[..., None] == border).any(-1), on + on % 2, code)
    code = code | np.where(np.signbit(b), 8, 0)
    code = np.where(fine[..., None], code, 0).reshape(v.shape).astype(np.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, np.where(fine, byte, 255).astype(np.uint8)


def values(codes, scales):
    """float64 [.., K] of codes and scales."""
    codes, scales = np.asarray(codes), np.asarray(scales).astype(np.int64)
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = LEVELS[c & 7] * np.where(c & 8, -1.0, 1.0)
    v = np.ldexp(v.reshape(*scales.shape, 32), (scales - 127)[..., None])
    return np.where((scales == 255)[..., None], np.nan, v).reshape(c.shape)


def rmsnorm(x, w, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)


def product(x, w, epi=1, res=None):
    """float64 x w^T with the epilogue, and the sum of the products' magnitudes (the gates' and the ups' for SwiGLU)."""
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    if epi == 2:
        return y + res, mag
    if epi == 3:
        y, mag = (t.reshape(len(t), -1, 2, 2) for t in (y, mag))
        g, u = y[:, :, 0].reshape(len(x), -1), y[:, :, 1].reshape(len(x), -1)
        with np.errstate(over="ignore"):
            return g / (1 + np.exp(-g)) * u, (mag[:, :, 0].reshape(g.shape), mag[:, :, 1].reshape(g.shape), g, u)
    return y, mag
