"""Language-model operators on CUDA torch tensors: the norm with a residual and an 8-bit
output, products of 8-bit operands with block scales (plain and grouped by expert) and
the choice of a token.

Unlike the ops_* on engine Tensors, which copy from and to the host, these work on
device memory: they enqueue on torch's current stream of the tensors' device and
return tensors made there. Inputs keep their strides (rows may be spaced apart, the
last dimension has to be dense). Wrong arguments raise TypeError (not a CUDA tensor, a
wrong dtype) or PdefaError (shapes, strides).
"""
from __future__ import annotations

import math
import sys

from . import _native as N
from .api import PdefaError, _check

BLOCK = 128   # values (of a row, or of both weight dimensions) that share a scale

_T = None


class _Types:
    """torch, and what of it is looked up on every call."""

    def __init__(self):
        import torch
        self.torch = torch
        self.code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self.fp8 = torch.float8_e4m3fn
        self.f32, self.i32 = torch.float32, torch.int32


def _types() -> _Types:
    global _T
    if _T is None:
        if "torch" not in sys.modules:
            raise TypeError("the language-model operators take CUDA torch tensors")
        _T = _Types()
    return _T


def _tensor(t, T, what, device, dtype, ndim):
    if not isinstance(t, T.torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{what}: a CUDA torch.Tensor is needed")
    if t.dtype != dtype:
        raise TypeError(f"{what}: {dtype} is needed, got {t.dtype}")
    if t.dim() != ndim:
        raise PdefaError(f"{what}: {ndim} dimensions are needed, got {tuple(t.shape)}")
    if t.device != device:
        raise PdefaError(f"{what}: is on {t.device}, not on {device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise PdefaError(f"{what}: the last dimension has to be dense (strides {t.stride()})")


def _cuda(t, T, what):
    if not isinstance(t, T.torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{what}: a CUDA torch.Tensor is needed")
    return t.device


def _stream(T, device) -> int:
    return T.torch.cuda.current_stream(device).cuda_stream


def _rows(t):
    """t as [rows, columns]: its leading dimensions as one (a view)."""
    if t.dim() == 2:
        return t
    if t.dim() == 1:
        return t.unsqueeze(0)
    if t.numel() == 0:
        return t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError as e:
        raise PdefaError(f"rows of shape {tuple(t.shape)}, strides {t.stride()} are not evenly spaced") from e


def _norm(what, x, weight, residual, eps, fp8):
    T = _types()
    device = _cuda(x, T, what)
    code = T.code.get(x.dtype)
    if code is None:
        raise TypeError(f"{what}: x must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() == 0:
        raise PdefaError(f"{what}: x needs a dimension")
    shape = x.shape
    x2 = _rows(x)
    rows, cols = x2.shape
    _tensor(x2, T, f"{what}: x", device, x.dtype, 2)
    _tensor(weight, T, f"{what}: weight", device, T.f32 if getattr(weight, "dtype", None) == T.f32 else x.dtype, 1)
    if weight.shape[0] != cols:
        raise PdefaError(f"{what}: weight of {weight.shape[0]} for rows of {cols}")
    empty = T.torch.empty
    r = h = None
    if residual is not None:
        if not isinstance(residual, T.torch.Tensor) or residual.shape != shape:
            raise PdefaError(f"{what}: the residual needs x's shape {tuple(shape)}")
        r = _rows(residual)
        _tensor(r, T, f"{what}: residual", device, x.dtype, 2)
        h = empty(shape, dtype=x.dtype, device=device)
    scales = None
    nb = (cols + BLOCK - 1) // BLOCK
    if fp8:
        y = empty(shape, dtype=T.fp8, device=device)
        scales = empty((*shape[:-1], nb), dtype=T.f32, device=device)
    else:
        y = empty(shape, dtype=x.dtype, device=device)
    rc = N.lib().engine_rms_norm_device(
        x2.data_ptr(), x2.stride(0), None if r is None else r.data_ptr(), 0 if r is None else r.stride(0),
        weight.data_ptr(), None if h is None else h.data_ptr(), cols, y.data_ptr(), cols,
        None if scales is None else scales.data_ptr(), nb, rows, cols, code, T.code[weight.dtype], eps,
        device.index, _stream(T, device))
    if rc:
        _check(rc, what)
    return y, scales, h


def ops_rms_norm(x, weight, residual=None, eps: float = 1e-6):
    """y = h * weight / sqrt(mean(h^2) + eps) over the last dimension, h = x + residual
    (32 bits). x [..., cols] float32, float16 or bfloat16; residual like x; weight [cols]
    of x's type or float32. Returns y, or (y, h) with a residual, both of x's type."""
    y, _, h = _norm("ops_rms_norm", x, weight, residual, eps, False)
    return y if residual is None else (y, h)


def ops_rms_norm_fp8(x, weight, residual=None, eps: float = 1e-6):
    """ops_rms_norm with its result in 8 bits: (q, scales), or (q, scales, h) with a
    residual. q [..., cols] float8_e4m3fn, scales [..., ceil(cols / 128)] float32, y being
    q times the scale of its 128 columns: the operands of ops_matmul_fp8."""
    q, scales, h = _norm("ops_rms_norm_fp8", x, weight, residual, eps, True)
    return (q, scales) if residual is None else (q, scales, h)


def _out_code(T, what, out_dtype):
    if out_dtype is None:
        return T.torch.bfloat16, 2
    code = T.code.get(out_dtype)
    if code is None:
        raise TypeError(f"{what}: out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    return out_dtype, code


def ops_matmul_fp8(a, a_scales, b, b_scales, out_dtype=None):
    """a @ b.T for 8-bit operands with block scales -> [M, N] of out_dtype (bfloat16).
    a [M, K] float8_e4m3fn with a_scales [M, ceil(K / 128)] float32 (as ops_rms_norm_fp8
    makes them); b [N, K] float8_e4m3fn with b_scales [ceil(N / 128), ceil(K / 128)]."""
    what = "ops_matmul_fp8"
    T = _types()
    device = _cuda(a, T, f"{what}: a")
    _tensor(a, T, f"{what}: a", device, T.fp8, 2)
    _tensor(b, T, f"{what}: b", device, T.fp8, 2)
    _tensor(a_scales, T, f"{what}: a_scales", device, T.f32, 2)
    _tensor(b_scales, T, f"{what}: b_scales", device, T.f32, 2)
    m, k = a.shape
    n, kb = b.shape[0], (k + BLOCK - 1) // BLOCK
    if b.shape[1] != k or a_scales.shape != (m, kb) or b_scales.shape != ((n + BLOCK - 1) // BLOCK, kb):
        raise PdefaError(f"{what}: shapes do not fit: a {tuple(a.shape)}, a_scales {tuple(a_scales.shape)}, "
                         f"b {tuple(b.shape)}, b_scales {tuple(b_scales.shape)}")
    out_dtype, code = _out_code(T, what, out_dtype)
    out = T.torch.empty((m, n), dtype=out_dtype, device=device)
    rc = N.lib().engine_matmul_fp8_device(
        a.data_ptr(), a.stride(0), a_scales.data_ptr(), a_scales.stride(0), b.data_ptr(), b.stride(0),
        b_scales.data_ptr(), b_scales.stride(0), out.data_ptr(), n, code, m, n, k, device.index, _stream(T, device))
    if rc:
        _check(rc, what)
    return out


def ops_matmul_grouped_fp8(a, a_scales, b, b_scales, offsets, out_dtype=None):
    """ops_matmul_fp8 with a weight per expert -> [rows, N] of out_dtype (bfloat16).
    a [rows, K] with its rows sorted by expert; b [experts, N, K] with b_scales [experts,
    ceil(N / 128), ceil(K / 128)]; offsets [experts + 1] int32, rising, on the GPU: rows
    offsets[e] .. offsets[e + 1] - 1 meet expert e. Rows of no expert give 0."""
    what = "ops_matmul_grouped_fp8"
    T = _types()
    device = _cuda(a, T, f"{what}: a")
    _tensor(a, T, f"{what}: a", device, T.fp8, 2)
    _tensor(b, T, f"{what}: b", device, T.fp8, 3)
    _tensor(a_scales, T, f"{what}: a_scales", device, T.f32, 2)
    _tensor(b_scales, T, f"{what}: b_scales", device, T.f32, 3)
    _tensor(offsets, T, f"{what}: offsets", device, T.i32, 1)
    rows, k = a.shape
    experts, n = b.shape[0], b.shape[1]
    kb = (k + BLOCK - 1) // BLOCK
    if (b.shape[2] != k or a_scales.shape != (rows, kb) or b_scales.shape != (experts, (n + BLOCK - 1) // BLOCK, kb)
            or offsets.shape[0] != experts + 1):
        raise PdefaError(f"{what}: shapes do not fit: a {tuple(a.shape)}, a_scales {tuple(a_scales.shape)}, "
                         f"b {tuple(b.shape)}, b_scales {tuple(b_scales.shape)}, offsets {tuple(offsets.shape)}")
    out_dtype, code = _out_code(T, what, out_dtype)
    out = T.torch.empty((rows, n), dtype=out_dtype, device=device)
    if experts == 0:
        return out.zero_()
    rc = N.lib().engine_matmul_grouped_fp8_device(
        a.data_ptr(), a.stride(0), a_scales.data_ptr(), a_scales.stride(0), b.data_ptr(), b.stride(1), b.stride(0),
        b_scales.data_ptr(), b_scales.stride(1), b_scales.stride(0), offsets.data_ptr(), experts, out.data_ptr(), n,
        code, rows, n, k, device.index, _stream(T, device))
    if rc:
        _check(rc, what)
    return out


def ops_sample(logits, noise, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits -> (tokens int32 [rows], probs float32 [rows]).

    logits [rows, vocab] float32, float16 or bfloat16 (-inf: ruled out); noise [rows,
    vocab] float32 of independent exponential variates (Tensor.exponential_()).
    temperature, top_p, min_p float32 [rows] and top_k int32 [rows], each optional:
    temperature 0 takes the largest logit, top_k <= 0, top_p >= 1 and min_p <= 0 are off.
    With w = exp((logit - largest) / temperature) a token is kept if fewer than top_k
    tokens are before it (larger, or equal with a lower index), their mass is below
    top_p of the row's, and w >= min_p. probs is the token's share of the row's whole
    mass. A row of -inf alone gives token -1 and probability 0."""
    what = "ops_sample"
    T = _types()
    device = _cuda(logits, T, f"{what}: logits")
    code = T.code.get(logits.dtype)
    if code is None:
        raise TypeError(f"{what}: logits must be float32, float16 or bfloat16, got {logits.dtype}")
    _tensor(logits, T, f"{what}: logits", device, logits.dtype, 2)
    _tensor(noise, T, f"{what}: noise", device, T.f32, 2)
    rows, vocab = logits.shape
    if noise.shape != logits.shape:
        raise PdefaError(f"{what}: noise {tuple(noise.shape)} for logits {tuple(logits.shape)}")
    ptr = [None] * 4
    for i, (t, dtype, name) in enumerate(((temperature, T.f32, "temperature"), (top_k, T.i32, "top_k"),
                                          (top_p, T.f32, "top_p"), (min_p, T.f32, "min_p"))):
        if t is not None:
            _tensor(t, T, f"{what}: {name}", device, dtype, 1)
            if t.shape[0] != rows:
                raise PdefaError(f"{what}: {name} of {t.shape[0]} for {rows} rows")
            ptr[i] = t.data_ptr()
    tokens = T.torch.empty(rows, dtype=T.i32, device=device)
    probs = T.torch.empty(rows, dtype=T.f32, device=device)
    rc = N.lib().engine_sample_device(
        logits.data_ptr(), logits.stride(0), code, noise.data_ptr(), noise.stride(0), ptr[0], ptr[1], ptr[2], ptr[3],
        rows, vocab, tokens.data_ptr(), probs.data_ptr(), device.index, _stream(T, device))
    if rc:
        _check(rc, what)
    return tokens, probs
