"""The 8-bit floating-point product with block scales (include/mnb_fp8.h).

``quantize_fp8`` turns rows into e4m3 codes with one scale for each row's block
of 128 values; ``MatMulFp8`` multiplies such rows, or rows that it quantizes
itself, by an e4m3 weight with a scale for each block of 128 x 128. Both stand
beside ``MatMulNBits``: the same weight layout [N, K], prepared once, the same
errors, and no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import (MatMulNBits, _check, _dev_ptr, _host_ptr, _raw_stream, library)

BLOCK = 128
PREFIX = "onnx_light_cpu_amd::MatMulFp8"
QUANTIZE_PREFIX = "onnx_light_cpu_amd::QuantizeFp8"

_lib = None
_types = None  # torch dtype -> MNB_TYPE_* of include/mnb_fp8.h
# Workspaces by thread and stream, of all objects: their calls there run one after
# another, and a model has hundreds of them (8192 rows of K = 14336: 117 MB a call).
_shared_works = {}


def release_workspaces():
    """Gives the workspaces that MatMulFp8 and MatMulNBitsMoE calls share back to torch's
    allocator; the next calls have new ones."""
    _shared_works.clear()


def _library():
    """libmnb.so with the 8-bit entry points' signatures."""
    global _lib, _types
    if _lib is None:
        import torch
        L = library()
        vp, i64, i32, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t
        L.mnb_fp8_quantize.argtypes = [i64, i64, i32, vp, i64, vp, vp, vp]
        for name in ("mnb_fp8_plan_create", "mnb_fp8_plan_create_device"):
            getattr(L, name).argtypes = [i64, i64, vp, vp, ctypes.POINTER(vp)]
        L.mnb_fp8_plan_destroy.argtypes = [vp]
        L.mnb_fp8_plan_device_bytes.argtypes = [vp, ctypes.POINTER(sz)]
        L.mnb_fp8_workspace_bytes.argtypes = [vp, i64, i32, ctypes.POINTER(sz)]
        L.mnb_fp8_run.argtypes = [vp, i64, i32, vp, vp, i32, vp, vp, sz, vp]
        L.mnb_fp8_kernel_name.argtypes = [vp, i64]
        L.mnb_fp8_kernel_name.restype = ctypes.c_char_p
        _types = {torch.float32: 1, torch.float16: 10, torch.bfloat16: 16,
                  torch.float8_e4m3fn: 17}
        _lib = L
    return _lib


def _elsewhere(device, stream):
    """What has to be made current for a call on `device` and `stream`, so that what
    it allocates, copies and launches is ordered there; None where it is."""
    import torch
    if stream is None:
        return None if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)
    if stream.device != device:
        raise ValueError(f"stream of {stream.device}, tensors on {device}")
    return torch.cuda.stream(stream)


def _laid_out(shape, want):
    """Whether values of `shape` lie in memory as those of `want`: axes of 1 apart, the
    same one, or with neighbouring axes joined into one."""
    want = [n for n in want if n != 1]
    for n in shape:
        joined = 1
        while joined < n and want:
            joined *= want.pop(0)
        if joined != n:
            return False
    return not want


def quantize_fp8(X, stream=None):
    """(codes float8_e4m3fn [..., K], scales float32 [..., ceil(K / 128)]) of the
    rows of X (a float32, float16 or bfloat16 device tensor [..., K]): with amax
    the largest magnitude of a row's block of 128, at least 2^-100, scale =
    amax / 448 and code = 448 x / amax rounded to e4m3. A 2-D X may have any row
    stride."""
    import torch
    L = _lib or _library()
    x_type = _types.get(X.dtype, 17)
    if x_type == 17 or not X.is_cuda:
        raise ValueError(f"{QUANTIZE_PREFIX}: X must be a float32, float16 or bfloat16 device "
                         "tensor")
    shape, device = X.shape, X.device
    if not shape or shape[-1] == 0:
        raise ValueError(f"{QUANTIZE_PREFIX}: X must be [..., K] with K >= 1")
    elsewhere = _elsewhere(device, stream)
    if elsewhere is not None:
        with elsewhere:
            return quantize_fp8(X)
    K = ldx = shape[-1]
    if X.is_contiguous():
        codes = torch.empty_like(X, dtype=torch.float8_e4m3fn)
    else:
        if X.dim() == 2 and X.stride(1) == 1 and X.stride(0) >= K:
            ldx = X.stride(0)
        else:
            X = X.contiguous()
        codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty(shape[:-1] + ((K + BLOCK - 1) // BLOCK,), dtype=torch.float32,
                         device=device)
    status = L.mnb_fp8_quantize(X.numel() // K, K, x_type, X.data_ptr(), ldx, codes.data_ptr(),
                                scales.data_ptr(), _raw_stream(device))
    if status != 0:
        _check(status, "quantize_fp8")
    return codes, scales


class MatMulFp8:
    """One 8-bit projection: Y[..., N] = A[..., K] * W^T with e4m3 weights W
    [N, K], a float32 scale for each of W's blocks of 128 x 128 and one for each
    row's block of 128 of A. Calls of one object on several streams or threads may
    overlap."""

    op_type = "MatMulFp8"

    def __init__(self, K: int, N: int):
        self.K, self.N = int(K), int(N)
        self._plan = ctypes.c_void_p()
        self._device = None
        self._needs = {}  # workspace bytes by (rows, dtype)

    _works = _shared_works
    _stream_workspace = MatMulNBits._stream_workspace

    # -- constants ---------------------------------------------------------
    def _check_sizes(self, W, scales):
        if self.K <= 0 or self.N <= 0:
            return  # the C ABI reports it
        blocks = [-(-self.N // BLOCK), -(-self.K // BLOCK)]
        w, s = math.prod(W.shape), math.prod(scales.shape)
        if w != self.N * self.K:
            raise ValueError(f"{PREFIX}: W has {w} values, expected N*K = {self.N * self.K}")
        if s != blocks[0] * blocks[1]:
            raise ValueError(f"{PREFIX}: scales has {s} elements, expected "
                             f"{blocks[0] * blocks[1]}")
        if not _laid_out(W.shape, [self.N, self.K]):
            raise ValueError(f"{PREFIX}: W must be [N, K] = {[self.N, self.K]}, got "
                             f"{list(W.shape)}")
        if not _laid_out(scales.shape, blocks):
            raise ValueError(f"{PREFIX}: scales must be [ceil(N / 128), ceil(K / 128)] = {blocks}, "
                             f"got {list(scales.shape)}")

    def prepare(self, W, scales):
        """Uploads host (numpy) constants once, to the current device: W uint8
        (e4m3 codes) [N, K], scales float32 [ceil(N / 128), ceil(K / 128)] (axes may be
        joined, as in flat arrays)."""
        import torch
        self.release()
        W = np.ascontiguousarray(W, dtype=np.uint8)
        scales = np.ascontiguousarray(scales, dtype=np.float32)
        self._check_sizes(W, scales)
        _check(_library().mnb_fp8_plan_create(self.K, self.N, _host_ptr(W), _host_ptr(scales),
                                              ctypes.byref(self._plan)), "prepare")
        self._device = torch.device("cuda", torch.cuda.current_device())
        return self

    def prepare_device(self, W, scales):
        """Lays out device (torch) constants once: W float8_e4m3fn or uint8
        [N, K], scales float32 [ceil(N / 128), ceil(K / 128)]. They may be freed
        afterwards."""
        import torch
        self.release()
        if not W.is_cuda or W.dtype not in (torch.float8_e4m3fn, torch.uint8):
            raise ValueError(f"{PREFIX}: W must be a float8_e4m3fn or uint8 device tensor")
        if scales.device != W.device or scales.dtype != torch.float32:
            raise ValueError(f"{PREFIX}: scales must be a float32 tensor on W's device")
        self._check_sizes(W, scales)
        with torch.cuda.device(W.device):
            w, s = W.contiguous(), scales.contiguous()
            _check(_library().mnb_fp8_plan_create_device(self.K, self.N, _dev_ptr(w), _dev_ptr(s),
                                                         ctypes.byref(self._plan)),
                   "prepare_device")
        self._device = W.device
        return self

    def release(self):
        if self._plan:
            _library().mnb_fp8_plan_destroy(self._plan)
            self._plan = ctypes.c_void_p()
        self._needs = {}

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    # -- compute -----------------------------------------------------------
    def __call__(self, A, scales=None, out=None, out_dtype=None, stream=None):
        """Y[..., N] on A's device. A: float8_e4m3fn codes [..., K] with scales
        float32 [..., ceil(K / 128)] (as quantize_fp8 gives them), or a float32,
        float16 or bfloat16 tensor, quantized first. Y's type: out's, out_dtype,
        else A's (float32 for codes). Products are exact for a float32 or float16 Y; a
        bfloat16 Y loses up to 7 2^-13 of the sum of their magnitudes (mnb_fp8.h)."""
        import torch
        if not self._plan:
            raise ValueError(f"{PREFIX}: prepare() was not called")
        a_type = _types.get(A.dtype)
        device = A.device
        if a_type is None or device != self._device:
            raise ValueError(f"{PREFIX}: A must be a float8_e4m3fn, float32, float16 or bfloat16 "
                             f"tensor on {self._device}")
        K, N, shape = self.K, self.N, A.shape
        if not shape or shape[-1] != K:
            raise ValueError(f"{PREFIX}: A must be [..., {K}], got {list(shape)}")
        rows = shape[:-1]
        if a_type == 17:
            want = rows + ((K + BLOCK - 1) // BLOCK,)
            if (scales is None or scales.shape != want or scales.dtype != torch.float32
                    or scales.device != device):
                raise ValueError(f"{PREFIX}: codes need float32 scales {list(want)} on {device}")
        elif scales is not None:
            raise ValueError(f"{PREFIX}: scales belong to float8_e4m3fn codes")
        dtype = out.dtype if out is not None else out_dtype or (
            torch.float32 if a_type == 17 else A.dtype)
        if out_dtype not in (None, dtype):
            raise ValueError(f"{PREFIX}: out is {dtype}, out_dtype {out_dtype}")
        y_type = _types.get(dtype, 17)
        if y_type == 17:
            raise ValueError(f"{PREFIX}: Y must be float32, float16 or bfloat16")
        if out is not None and (out.shape != rows + (N,) or not out.is_contiguous()
                                or out.device != device or out.data_ptr() % 16 != 0):
            raise ValueError(f"{PREFIX}: out must be contiguous {list(rows + (N,))} on {device}, "
                             "aligned to 16 bytes")
        elsewhere = _elsewhere(device, stream)
        if elsewhere is not None:
            with elsewhere:
                return self(A, scales, out, out_dtype)
        if not A.is_contiguous():
            A = A.contiguous()
        address = A.data_ptr()
        if address % 16 != 0:
            A = A.clone()
            address = A.data_ptr()
        if scales is not None and not scales.is_contiguous():
            scales = scales.contiguous()
        M = A.numel() // K
        if out is None:
            out = torch.empty(rows + (N,), dtype=dtype, device=device)
        need = self._needs.get((M, a_type))
        if need is None:
            need = self._remember(M, A.dtype)
        work = self._stream_workspace(need, device) if need else None
        status = _lib.mnb_fp8_run(self._plan, M, a_type, address,
                                  None if scales is None else scales.data_ptr(), y_type,
                                  out.data_ptr(), None if work is None else work.data_ptr(), need,
                                  _raw_stream(device))
        if status != 0:
            _check(status, "run")
        return out

    def _remember(self, M, dtype):
        if len(self._needs) > 256:
            self._needs = {}
        need = self._needs[M, _types[dtype]] = self.workspace_bytes(M, dtype)
        return need

    run = __call__

    def workspace_bytes(self, M: int, dtype) -> int:
        """Device workspace of a call of M rows of `dtype` (mnb_fp8_workspace_bytes)."""
        n = ctypes.c_size_t()
        _check(_library().mnb_fp8_workspace_bytes(self._plan, M, _types[dtype], ctypes.byref(n)),
               "workspace_bytes")
        return n.value

    def kernel_name(self, M: int) -> str:
        """The kernel that multiplies M rows into a bfloat16 Y."""
        return _library().mnb_fp8_kernel_name(self._plan, M).decode()

    def device_bytes(self) -> int:
        """Device memory the plan owns (mnb_fp8_plan_device_bytes)."""
        n = ctypes.c_size_t()
        _check(_library().mnb_fp8_plan_device_bytes(self._plan, ctypes.byref(n)), "device_bytes")
        return n.value
