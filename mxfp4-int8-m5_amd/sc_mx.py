"""Microscaled 4-bit values (include/scmx_mx.h): rows to MXFP4 and back, and products of MXFP4 activations with MXFP4 weights on the scaled
matrix instructions.  The reference's activations are INT8 (e2e/sc_kernels.py); these have no counterpart there.

A tensor [rows, K], K a multiple of 32, is a pair: codes uint8 [rows, K / 2] (two E2M1 codes a byte, the even value low) and scales uint8
[rows, K / 32] (E8M0), what a standard MXFP4 checkpoint holds.  Tensors are on the current device; work goes to the current stream."""
import torch

from . import _lib
from . import sc_kernels as S
from .sc_cache import BF, _check, _on_device

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _check_pair(codes, scales, what):
    """(rows, K) of codes and scales that belong together."""
    _check(codes.dim() == scales.dim() == 2 and codes.dtype == scales.dtype == torch.uint8 and codes.shape[0] == scales.shape[0]
           and codes.shape[1] == 16 * scales.shape[1] > 0, f"{what}: codes uint8 [rows, K / 2] and scales uint8 [rows, K / 32]")
    return codes.shape[0], 2 * codes.shape[1]


def _rows(x):
    """x [M, K] whose rows are whole; where they are not, a copy."""
    return x if x.stride(1) == 1 and (x.shape[0] < 2 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _ldx(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def quantize(x, nw=None, eps=0.0):
    """x [M, K] bfloat16, float16 or float32, K a multiple of 32, rows at any stride -> (codes, scales).  nw bfloat16 [K] (x bfloat16, K up to
    16384): of the RMSNorm of x, which is not rounded in between.  A block takes the power of two that its largest magnitude
    has, less two, each value the nearest E2M1 (ties to even, held to 6); a block with a NaN or an infinity becomes NaN."""
    out = _lib.native().mx_quantize(x, nw, eps)
    if out is not None:   # the operands of every step; anything else is converted or refused below
        return out
    _check(x.dim() == 2 and x.dtype in TYPES and x.shape[1] and x.shape[1] % 32 == 0,
           "x is bfloat16, float16 or float32 [M, K], K a multiple of 32")
    _check(nw is None or (x.dtype == nw.dtype == BF and nw.numel() == x.shape[1] <= 16384), "a norm takes x and nw bfloat16, K up to 16384")
    _on_device(x, nw)
    x, (M, K) = _rows(x), x.shape
    codes, scales = _lib.native().empty_u8(x, M, K // 2), _lib.native().empty_u8(x, M, K // 32)
    _lib.native().scmx_mx_quantize(x.data_ptr(), TYPES[x.dtype], _ldx(x), nw, S._eps(eps) if nw is not None else 0.0, codes, scales, M, K)
    return codes, scales


def dequantize(codes, scales, dtype=BF):
    """The values [rows, K] as bfloat16 or float32 (exact but where they pass its range)."""
    out = _lib.native().mx_dequantize(codes, scales, dtype == torch.float32) if dtype in (BF, torch.float32) else None
    if out is not None:
        return out
    M, K = _check_pair(codes, scales, "dequantize")
    _check(dtype in (BF, torch.float32), "values come as bfloat16 or float32")
    _on_device(codes, scales)
    out = (_lib.native().empty_bf16 if dtype == BF else _lib.native().empty_f32)(codes, M, K)
    _lib.native().scmx_mx_dequantize(codes, scales, out, TYPES[dtype], M, K)
    return out


def _check_product(M, K, wcodes, wscales, epi, res, like):
    N, Kw = _check_pair(wcodes, wscales, "weights")
    _check(Kw == K and N > 0, f"weights [N, {Kw}] for rows of {K}")
    _check(epi in (1, 2, 3) and (epi != 3 or N % 4 == 0), "epilogue 1, 2 or 3 (SwiGLU: N a multiple of 4)")
    _check(epi != 2 or (res is not None and res.dtype == BF and tuple(res.shape) == (M, N)), "res is bfloat16 [M, N]")
    return N, _lib.native().empty_bf16(like, M, N // 2 if epi == 3 else N)


def mm(xcodes, xscales, wcodes, wscales, epi=1, res=None):
    """x w^T of MXFP4 rows x [M, K] and weights w [N, K], sums in float32 -> bfloat16: epi 1 [M, N], 2 + res [M, N], 3 SwiGLU of w rows in
    the order of sc_kernels.interleave_gate_up [M, N / 2]."""
    out = _lib.native().mx_mm(xcodes, xscales, wcodes, wscales, epi, res)
    if out is not None:
        return out
    M, K = _check_pair(xcodes, xscales, "rows")
    _on_device(xcodes, xscales, wcodes, wscales, res if epi == 2 else None)
    N, out = _check_product(M, K, wcodes, wscales, epi, res, xcodes)
    _lib.native().scmx_mx_mm(xcodes, xscales, wcodes, wscales, res if epi == 2 else None, out, epi, M, N, K)
    return out


def linear(x, wcodes, wscales, epi=1, res=None, nw=None, eps=0.0):
    """mm of quantize(x, nw, eps): x bfloat16 [M, K], rows at any stride."""
    out = _lib.native().mx_linear(x, wcodes, wscales, epi, res, nw, eps)
    if out is not None:
        return out
    _check(x.dim() == 2 and x.dtype == BF and x.shape[1] and x.shape[1] % 32 == 0, "x is bfloat16 [M, K], K a multiple of 32")
    _check(nw is None or (nw.dtype == BF and nw.numel() == x.shape[1] <= 16384), "nw is bfloat16 [K], K up to 16384")
    res = res if epi == 2 else None
    _on_device(x, nw, wcodes, wscales, res)
    x, (M, K) = _rows(x), x.shape
    N, out = _check_product(M, K, wcodes, wscales, epi, res, x)
    need = _lib.native().scmx_mx_linear_workspace(M, N, K, int(nw is not None))
    _lib.native().scmx_mx_linear(x.data_ptr(), _ldx(x), nw, S._eps(eps) if nw is not None else 0.0, wcodes, wscales, res, out, epi, M, N, K,
                                 _lib.native().empty_u8(x, need) if need else None, need)
    return out


def from_packed(pw):
    """(codes, scales) of a sc_weights.PackedWeight in the 32-block power-of-two format, whose code words are a standard MXFP4
    tensor's: the codes are a view."""
    from .sc_weights import mxfp4_scales
    scales = torch.from_numpy(mxfp4_scales(pw)).to(pw.codes.device)
    return pw.codes.view(torch.uint8).view(pw.N, pw.K // 2), scales
