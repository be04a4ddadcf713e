"""RMS norm with the residual's addition (include/mnb_norm.h).

``rms_norm_fp8`` makes the e4m3 rows that ``MatMulFp8`` multiplies,
``rms_norm`` rows of X's own type, as ``MatMulNBitsMoE`` takes them; with a
residual both return the sum too, which the next residual addition needs.
``MatMulNBits.run_rmsnorm`` and ``MatMulFp8.run_rmsnorm`` take the norm with their
product. There is no CPU fallback, and no gradient: backward() through a result raises.
"""
from __future__ import annotations

import ctypes

from . import _check, _raw_stream, library
from .fp8 import BLOCK, _elsewhere, _without_gradient

PREFIX = "onnx_light_cpu_amd::RmsNorm"
_INF = float("inf")

_lib = None
_types = None  # torch dtype -> MNB_TYPE_* of include/mnb_fp8.h


def _library():
    """libmnb.so with the norm's signature."""
    global _lib, _types
    if _lib is None:
        import torch
        L = library()
        vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
        L.mnb_rms_norm.argtypes = [i64, i64, i32, vp, i64, vp, i64, vp, ctypes.c_float, i32, vp,
                                   vp, vp, vp]
        _types = {torch.float32: 1, torch.float16: 10, torch.bfloat16: 16}
        _lib = L
    return _lib


def _wants_gradient(X, gamma, residual):
    if (X.requires_grad or gamma.requires_grad
            or (residual is not None and residual.requires_grad)):
        import torch
        return torch.is_grad_enabled()
    return False


def _rows(X, K):
    """(X, values between its rows), a copy where its rows are not evenly apart."""
    if X.is_contiguous():
        return X, K
    if X.dim() == 2 and X.stride(1) == 1 and X.stride(0) >= K:
        return X, X.stride(0)
    return X.contiguous(), K


def _run(X, gamma, epsilon, residual, codes, stream):
    # The smallest calls are bound by this function, not by their 3 us of kernel: results
    # come from empty_like and new_empty, which take a third less than empty.
    import torch
    L = _lib or _library()
    dtype, device, shape = X.dtype, X.device, X.shape
    x_type = _types.get(dtype)
    if x_type is None or not X.is_cuda:
        raise ValueError(f"{PREFIX}: X must be a float32, float16 or bfloat16 device tensor")
    if not shape or shape[-1] == 0:
        raise ValueError(f"{PREFIX}: X must be [..., K] with K >= 1")
    K = shape[-1]
    if gamma.shape != (K,) or gamma.dtype != torch.float32 or gamma.device != device:
        raise ValueError(f"{PREFIX}: gamma must be float32 [{K}] on {device}")
    if residual is not None and (residual.shape != shape or residual.dtype != dtype
                                 or residual.device != device):
        raise ValueError(f"{PREFIX}: residual must be of X's shape, type and device")
    if not 0.0 <= epsilon < _INF:
        raise ValueError(f"{PREFIX}: epsilon must be finite and not negative, got {epsilon}")
    if _wants_gradient(X, gamma, residual):
        return _without_gradient(PREFIX, lambda: _run(X, gamma, epsilon, residual, codes, stream),
                                 X, gamma, residual)
    elsewhere = _elsewhere(device, stream)
    if elsewhere is not None:
        with elsewhere:
            return _run(X, gamma, epsilon, residual, codes, None)
    X, ldx = _rows(X, K)  # of rows that are apart, empty_like makes dense ones
    if not gamma.is_contiguous():
        gamma = gamma.contiguous()
    total = from_ = to = scales_to = None
    ldr = 0
    if residual is not None:
        residual, ldr = _rows(residual, K)
        total = torch.empty_like(X)
        from_, to = residual.data_ptr(), total.data_ptr()
    if codes:
        Y = torch.empty_like(X, dtype=torch.float8_e4m3fn)
        scales = gamma.new_empty(shape[:-1] + ((K + BLOCK - 1) // BLOCK,))
        scales_to = scales.data_ptr()
    else:
        Y, scales = torch.empty_like(X), None
    status = L.mnb_rms_norm(X.numel() // K, K, x_type, X.data_ptr(), ldx, from_, ldr,
                            gamma.data_ptr(), epsilon, 17 if codes else x_type, Y.data_ptr(),
                            scales_to, to, _raw_stream(device))
    if status != 0:
        _check(status, "rms_norm")
    return Y, scales, total


def rms_norm(X, gamma, epsilon: float = 1e-5, residual=None, stream=None):
    """Y [..., K] = h / sqrt(mean(h^2) + epsilon) * gamma of X's type, h = X + residual
    rounded to it; X a float32, float16 or bfloat16 device tensor, residual the same
    or None, gamma float32 [K]. With a residual: (Y, h). 2-D inputs may have any row
    stride."""
    Y, _, total = _run(X, gamma, epsilon, residual, False, stream)
    return Y if total is None else (Y, total)


def rms_norm_fp8(X, gamma, epsilon: float = 1e-5, residual=None, stream=None):
    """(codes float8_e4m3fn [..., K], scales float32 [..., ceil(K / 128)]) of the norm that
    rms_norm rounds, in quantize_fp8's format: the codes nearest to 448 times its unrounded
    values over their block's largest; with a residual: (codes, scales, h)."""
    Y, scales, total = _run(X, gamma, epsilon, residual, True, stream)
    return (Y, scales) if total is None else (Y, scales, total)
