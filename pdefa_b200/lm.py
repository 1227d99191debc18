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
    """torch, the library and what of both is looked up on every call."""

    def __init__(self):
        import torch
        self.Tensor, self.empty, self.empty_like = torch.Tensor, torch.empty, torch.empty_like
        self.code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self.fp8, self.f32, self.i32, self.bf16 = torch.float8_e4m3fn, torch.float32, torch.int32, torch.bfloat16
        # torch.cuda.current_stream() without the Stream object around the handle (2 us a call)
        self.stream = torch._C._cuda_getCurrentRawStream
        lib = N.lib()
        self.rms_norm, self.sample = lib.engine_rms_norm_device, lib.engine_sample_device
        self.matmul, self.grouped = lib.engine_matmul_fp8_device, lib.engine_matmul_grouped_fp8_device


def _types() -> _Types:
    global _T
    if _T is None:
        if "torch" not in sys.modules:
            raise TypeError("the language-model operators take CUDA torch tensors")
        _T = _Types()
    return _T


def _tensor(t, T, what, device, dtype, ndim):
    """Refuses what is not a dense-rowed tensor of `dtype` on GPU `device`."""
    if not isinstance(t, T.Tensor) or not t.is_cuda:
        raise TypeError(f"{what}: a CUDA torch.Tensor is needed")
    if t.dtype != dtype:
        raise TypeError(f"{what}: {dtype} is needed, got {t.dtype}")
    if t.dim() != ndim:
        raise PdefaError(f"{what}: {ndim} dimensions are needed, got {tuple(t.shape)}")
    if t.get_device() != device:
        raise PdefaError(f"{what}: is on GPU {t.get_device()}, not on {device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise PdefaError(f"{what}: the last dimension has to be dense (strides {t.stride()})")


def _gpu(t, T, what) -> int:
    if not isinstance(t, T.Tensor) or not t.is_cuda:
        raise TypeError(f"{what}: a CUDA torch.Tensor is needed")
    return t.get_device()


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
    gpu = _gpu(x, T, what)
    dtype = x.dtype
    code = T.code.get(dtype)
    if code is None:
        raise TypeError(f"{what}: x must be float32, float16 or bfloat16, got {dtype}")
    shape = x.shape
    if not shape:
        raise PdefaError(f"{what}: x needs a dimension")
    x2 = _rows(x)
    rows, cols = x2.shape
    _tensor(x2, T, what, gpu, dtype, 2)
    wcode = code
    if getattr(weight, "dtype", None) == T.f32:
        wcode = 0
        _tensor(weight, T, what, gpu, T.f32, 1)
    else:
        _tensor(weight, T, what, gpu, dtype, 1)
    if weight.shape[0] != cols:
        raise PdefaError(f"{what}: weight of {weight.shape[0]} for rows of {cols}")
    # empty_like costs half of empty, but keeps strides that are not those of whole rows
    dense = x.is_contiguous()
    device = x.device
    h, r_ptr, r_stride, h_ptr = None, None, 0, None
    if residual is not None:
        if not isinstance(residual, T.Tensor) or residual.shape != shape:
            raise PdefaError(f"{what}: the residual needs x's shape {tuple(shape)}")
        r = _rows(residual)
        _tensor(r, T, what, gpu, dtype, 2)
        h = T.empty_like(x) if dense else T.empty(shape, dtype=dtype, device=device)
        r_ptr, r_stride, h_ptr = r.data_ptr(), r.stride(0), h.data_ptr()
    nb = (cols + BLOCK - 1) // BLOCK
    if fp8:
        y = T.empty_like(x, dtype=T.fp8) if dense else T.empty(shape, dtype=T.fp8, device=device)
        scales = T.empty((*shape[:-1], nb), dtype=T.f32, device=device)
        s_ptr = scales.data_ptr()
    else:
        y = T.empty_like(x) if dense else T.empty(shape, dtype=dtype, device=device)
        scales, s_ptr = None, None
    rc = T.rms_norm(x2.data_ptr(), x2.stride(0), r_ptr, r_stride, weight.data_ptr(), h_ptr, cols, y.data_ptr(), cols,
                    s_ptr, nb, rows, cols, code, wcode, eps, gpu, T.stream(gpu))
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
    code = T.code.get(out_dtype)
    if code is None:
        raise TypeError(f"{what}: out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    return code


def ops_matmul_fp8(a, a_scales, b, b_scales, out_dtype=None):
    """a @ b.T for 8-bit operands with block scales -> [M, N] of out_dtype (bfloat16).
    a [M, K] float8_e4m3fn with a_scales [M, ceil(K / 128)] float32 (as ops_rms_norm_fp8
    makes them); b [N, K] float8_e4m3fn with b_scales [ceil(N / 128), ceil(K / 128)]."""
    what = "ops_matmul_fp8"
    T = _types()
    gpu = _gpu(a, T, what)
    _tensor(a, T, "ops_matmul_fp8: a", gpu, T.fp8, 2)
    _tensor(b, T, "ops_matmul_fp8: b", gpu, T.fp8, 2)
    _tensor(a_scales, T, "ops_matmul_fp8: a_scales", gpu, T.f32, 2)
    _tensor(b_scales, T, "ops_matmul_fp8: b_scales", gpu, T.f32, 2)
    m, k = a.shape
    n, kb = b.shape[0], (k + BLOCK - 1) // BLOCK
    if b.shape[1] != k or a_scales.shape != (m, kb) or b_scales.shape != ((n + BLOCK - 1) // BLOCK, kb):
        raise PdefaError(f"{what}: shapes do not fit: a {tuple(a.shape)}, a_scales {tuple(a_scales.shape)}, "
                         f"b {tuple(b.shape)}, b_scales {tuple(b_scales.shape)}")
    out_dtype = out_dtype or T.bf16
    code = _out_code(T, what, out_dtype)
    out = T.empty((m, n), dtype=out_dtype, device=a.device)
    rc = T.matmul(a.data_ptr(), a.stride(0), a_scales.data_ptr(), a_scales.stride(0), b.data_ptr(), b.stride(0),
                  b_scales.data_ptr(), b_scales.stride(0), out.data_ptr(), n, code, m, n, k, gpu, T.stream(gpu))
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
    gpu = _gpu(a, T, what)
    _tensor(a, T, "ops_matmul_grouped_fp8: a", gpu, T.fp8, 2)
    _tensor(b, T, "ops_matmul_grouped_fp8: b", gpu, T.fp8, 3)
    _tensor(a_scales, T, "ops_matmul_grouped_fp8: a_scales", gpu, T.f32, 2)
    _tensor(b_scales, T, "ops_matmul_grouped_fp8: b_scales", gpu, T.f32, 3)
    _tensor(offsets, T, "ops_matmul_grouped_fp8: offsets", gpu, T.i32, 1)
    rows, k = a.shape
    experts, n = b.shape[0], b.shape[1]
    kb = (k + BLOCK - 1) // BLOCK
    if (b.shape[2] != k or a_scales.shape != (rows, kb) or b_scales.shape != (experts, (n + BLOCK - 1) // BLOCK, kb)
            or offsets.shape[0] != experts + 1):
        raise PdefaError(f"{what}: shapes do not fit: a {tuple(a.shape)}, a_scales {tuple(a_scales.shape)}, "
                         f"b {tuple(b.shape)}, b_scales {tuple(b_scales.shape)}, offsets {tuple(offsets.shape)}")
    out_dtype = out_dtype or T.bf16
    code = _out_code(T, what, out_dtype)
    out = T.empty((rows, n), dtype=out_dtype, device=a.device)
    if experts == 0:
        return out.zero_()
    b_expert, ldb, _ = b.stride()
    s_expert, lds, _ = b_scales.stride()
    rc = T.grouped(a.data_ptr(), a.stride(0), a_scales.data_ptr(), a_scales.stride(0), b.data_ptr(), ldb, b_expert,
                   b_scales.data_ptr(), lds, s_expert, offsets.data_ptr(), experts, out.data_ptr(), n, code, rows, n, k,
                   gpu, T.stream(gpu))
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
    gpu = _gpu(logits, T, what)
    dtype = logits.dtype
    code = T.code.get(dtype)
    if code is None:
        raise TypeError(f"{what}: logits must be float32, float16 or bfloat16, got {dtype}")
    _tensor(logits, T, "ops_sample: logits", gpu, dtype, 2)
    _tensor(noise, T, "ops_sample: noise", gpu, T.f32, 2)
    rows, vocab = shape = logits.shape
    if noise.shape != shape:
        raise PdefaError(f"{what}: noise {tuple(noise.shape)} for logits {tuple(shape)}")

    def per_row(t, dtype, name):
        if t is None:
            return None
        _tensor(t, T, name, gpu, dtype, 1)
        if t.shape[0] != rows:
            raise PdefaError(f"{name} of {t.shape[0]} for {rows} rows")
        return t.data_ptr()

    t_ptr = per_row(temperature, T.f32, "ops_sample: temperature")
    k_ptr = per_row(top_k, T.i32, "ops_sample: top_k")
    p_ptr = per_row(top_p, T.f32, "ops_sample: top_p")
    m_ptr = per_row(min_p, T.f32, "ops_sample: min_p")
    device = logits.device
    tokens = T.empty(rows, dtype=T.i32, device=device)
    probs = T.empty(rows, dtype=T.f32, device=device)
    rc = T.sample(logits.data_ptr(), logits.stride(0), code, noise.data_ptr(), noise.stride(0), t_ptr, k_ptr, p_ptr,
                  m_ptr, rows, vocab, tokens.data_ptr(), probs.data_ptr(), gpu, T.stream(gpu))
    if rc:
        _check(rc, what)
    return tokens, probs
