"""Language-model operators on CUDA torch tensors: the norm with a residual and an 8-bit
output, products of 8-bit operands with block scales (plain and grouped by expert) and
the choice of a token.

Unlike the ops_* on engine Tensors, which copy from and to the host, these work on
device memory: they enqueue on torch's current stream of the tensors' device and
return tensors made there; nothing waits. Inputs keep their strides (rows may be spaced
apart, the last dimension has to be dense). Wrong arguments raise TypeError (not a CUDA
tensor, a wrong dtype) or PdefaError (shapes, strides). There are no gradients: the engine
only infers. The kernels' device-side waits are bounded; one that runs out is recorded in
the device's error word (engine_device_error).

The argument checks and the calls are in lib/lm_torch-*.so (torch_ext/lm_torch.cpp).
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import os
import sys

from . import _native as N
from .api import PdefaError, _check

BLOCK = 128   # values (of a row, or of both weight dimensions) that share a scale

_B = None


def _binding():
    """The binding of the installed torch, bound to the engine's entry points."""
    global _B
    if _B is None:
        if "torch" not in sys.modules:
            raise TypeError("the language-model operators take CUDA torch tensors")
        from . import build
        lib = N.lib()
        root = build.torch_root()
        if root is None:
            raise TypeError("the language-model operators take CUDA torch tensors: this torch has no CUDA")
        path = build.torch_lib(root)
        if not os.path.isfile(path):
            build.build_torch_binding(False)        # raises RuntimeError with the compiler's output
        loader = importlib.machinery.ExtensionFileLoader("lm_torch", path)
        b = importlib.util.module_from_spec(importlib.util.spec_from_loader("lm_torch", loader))
        loader.exec_module(b)
        address = lambda f: C.cast(f, C.c_void_p).value   # noqa: E731
        b.bind(address(lib.engine_rms_norm_device), address(lib.engine_matmul_fp8_device),
               address(lib.engine_matmul_grouped_fp8_device), address(lib.engine_sample_device), PdefaError, _check)
        _B = b
    return _B


def ops_rms_norm(x, weight, residual=None, eps: float = 1e-6):
    """y = h * weight / sqrt(mean(h^2) + eps) over the last dimension, h = x + residual
    (32 bits). x [..., cols] float32, float16 or bfloat16; residual like x; weight [cols]
    of x's type or float32. Returns y, or (y, h) with a residual, both of x's type."""
    return (_B or _binding()).rms_norm(x, weight, residual, eps, False)


def ops_rms_norm_fp8(x, weight, residual=None, eps: float = 1e-6):
    """ops_rms_norm with its result in 8 bits: (q, scales), or (q, scales, h) with a
    residual. q [..., cols] float8_e4m3fn, scales [..., ceil(cols / 128)] float32, y being
    q times the scale of its 128 columns: the operands of ops_matmul_fp8."""
    return (_B or _binding()).rms_norm(x, weight, residual, eps, True)


def ops_matmul_fp8(a, a_scales, b, b_scales, out_dtype=None):
    """a @ b.T for 8-bit operands with block scales -> [M, N] of out_dtype (bfloat16).
    a [M, K] float8_e4m3fn with a_scales [M, ceil(K / 128)] float32 (as ops_rms_norm_fp8
    makes them); b [N, K] float8_e4m3fn with b_scales [ceil(N / 128), ceil(K / 128)]."""
    return (_B or _binding()).matmul(a, a_scales, b, b_scales, out_dtype)


def ops_matmul_grouped_fp8(a, a_scales, b, b_scales, offsets, out_dtype=None):
    """ops_matmul_fp8 with a weight per expert -> [rows, N] of out_dtype (bfloat16).
    a [rows, K] with its rows sorted by expert; b [experts, N, K] with b_scales [experts,
    ceil(N / 128), ceil(K / 128)]; offsets [experts + 1] int32, rising, on the GPU: rows
    offsets[e] .. offsets[e + 1] - 1 meet expert e. Rows of no expert give 0. 1024 experts
    at most."""
    return (_B or _binding()).grouped(a, a_scales, b, b_scales, offsets, out_dtype)


def ops_sample(logits, noise, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits -> (tokens int32 [rows], probs float32 [rows]).

    logits [rows, vocab] float32, float16 or bfloat16 (-inf: ruled out); noise [rows,
    vocab] float32 of independent exponential variates (Tensor.exponential_()); a token whose
    variate is negative, -0 or NaN is out of the race.
    temperature, top_p, min_p float32 [rows] and top_k int32 [rows], each optional:
    temperature 0 takes the largest logit, top_k <= 0, top_p >= 1 and min_p <= 0 are off.
    With w = exp((logit - largest) / temperature) a token is kept if fewer than top_k
    tokens are before it (larger, or equal with a lower index), their mass is below
    top_p of the row's, and w >= min_p. probs is the token's share of the row's whole
    mass. A row of -inf alone gives token -1 and probability 0."""
    return (_B or _binding()).sample(logits, noise, temperature, top_k, top_p, min_p)
