"""A whole mixture-of-experts layer on 4-bit weights (include/mnb_moe.h).

``MatMulNBitsMoE`` does for a layer of experts what ``GateUpSiLU`` and a
``MatMulNBits`` node do for a dense one: the router's product, the choice of
top_k experts for each token, their gated MLPs and the weighted sum, for few
tokens at a time. Its weights are MatMulNBits weights with the experts as their
first axis. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import MatMulNBits, _check, _raw_stream, library
from .fp8 import _elsewhere, _laid_out, _shared_works

PREFIX = "onnx_light_cpu_amd::MatMulNBitsMoE"


class MoeDesc(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int64), ("intermediate", ctypes.c_int64),
                ("experts", ctypes.c_int32), ("top_k", ctypes.c_int32), ("bits", ctypes.c_int32),
                ("block_size", ctypes.c_int32), ("normalize", ctypes.c_int32),
                ("has_zero_points", ctypes.c_int32)]


class MoeWeight(ctypes.Structure):
    _fields_ = [("B", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("zero_points", ctypes.c_void_p)]


_lib = None
_types = None  # torch dtype -> MNB_TYPE_* of include/mnb_fp8.h


def _library():
    """libmnb.so with the expert layer's entry points' signatures."""
    global _lib, _types
    if _lib is None:
        import torch
        L = library()
        vp, i64, i32, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t
        desc, weight = ctypes.POINTER(MoeDesc), ctypes.POINTER(MoeWeight)
        for name in ("mnb_moe_plan_create", "mnb_moe_plan_create_device"):
            getattr(L, name).argtypes = [desc, vp, weight, weight, weight, ctypes.POINTER(vp)]
        L.mnb_moe_plan_destroy.argtypes = [vp]
        L.mnb_moe_plan_device_bytes.argtypes = [vp, ctypes.POINTER(sz)]
        L.mnb_moe_workspace_bytes.argtypes = [vp, i64, i32, ctypes.POINTER(sz)]
        L.mnb_moe_run.argtypes = [vp, i64, i32, vp, vp, vp, vp, vp, vp, sz, vp]
        _types = {torch.float32: 1, torch.float16: 10, torch.bfloat16: 16}
        _lib = L
    return _lib


class MatMulNBitsMoE:
    """One mixture-of-experts layer: Y[..., H] of X[..., H], each token through
    the top_k of `experts` gated MLPs (SiLU, width `intermediate`) that its router
    logits choose, weighted by the softmax over the chosen (normalize) or over all.
    Calls of one object on several streams or threads may overlap."""

    op_type = "MatMulNBitsMoE"

    def __init__(self, hidden: int, intermediate: int, experts: int, top_k: int, bits: int = 4,
                 block_size: int = 32, normalize: bool = True):
        self.desc = MoeDesc(hidden, intermediate, experts, top_k, bits, block_size,
                            int(bool(normalize)), 0)
        self._plan = ctypes.c_void_p()
        self._device = None
        self._router = False
        self._needs = {}  # workspace bytes by (tokens, type)

    _works = _shared_works
    _stream_workspace = MatMulNBits._stream_workspace

    # -- constants ---------------------------------------------------------
    def _check_sizes(self, router, gate, up, down):
        d = self.desc
        if min(d.hidden, d.intermediate, d.experts) <= 0 or d.block_size < 2:
            return  # the C ABI reports it
        arrays = []
        for name, w, n, k in (("gate", gate, d.intermediate, d.hidden),
                              ("up", up, d.intermediate, d.hidden),
                              ("down", down, d.hidden, d.intermediate)):
            nb = -(-k // d.block_size)
            for what, a, last in zip(("B", "scales", "zero_points"), w,
                                     ([nb, d.block_size // 2], [nb], [(nb + 1) // 2])):
                arrays.append((f"{name}'s {what}", a, [d.experts, n] + last))
        arrays.append(("router", router, [d.experts, d.hidden]))
        arrays = [(name, a, want) for name, a, want in arrays if a is not None]
        for name, a, want in arrays:
            if math.prod(a.shape) != math.prod(want):
                raise ValueError(f"{PREFIX}: {name} has {math.prod(a.shape)} elements, expected "
                                 f"{math.prod(want)}")
        for name, a, want in arrays:
            if not _laid_out(a.shape, want):
                raise ValueError(f"{PREFIX}: {name} must be {want}, got {list(a.shape)}")

    def _weights(self, gate, up, down):
        ws = [tuple(w) + (None,) * (3 - len(w)) for w in (gate, up, down)]
        if len({w[2] is None for w in ws}) != 1:
            raise ValueError(f"{PREFIX}: all three weights must have zero points, or none")
        self.desc.has_zero_points = int(ws[0][2] is not None)
        return ws

    def prepare(self, router, gate, up, down):
        """Uploads host (numpy) constants once, to the current device. gate, up and
        down: (B, scales, zero_points or None), MatMulNBits weights with the experts
        as first axis, gate and up [experts, intermediate, ...] over hidden, down
        [experts, hidden, ...] over intermediate; router float32 [experts, hidden],
        or None where every call brings its logits. Axes may be joined, as in flat
        arrays."""
        import torch
        self.release()
        ws = [tuple(None if a is None else np.ascontiguousarray(a, dtype=t)
                    for a, t in zip(w, (np.uint8, np.float32, np.uint8)))
              for w in self._weights(gate, up, down)]
        r = None if router is None else np.ascontiguousarray(router, dtype=np.float32)
        self._check_sizes(r, *ws)
        self._create("mnb_moe_plan_create", r, ws, lambda a: a.ctypes.data)
        self._device = torch.device("cuda", torch.cuda.current_device())
        return self

    def prepare_device(self, router, gate, up, down):
        """Lays out device (torch) constants once, as prepare's. They may be freed
        afterwards."""
        import torch
        self.release()
        ws = self._weights(gate, up, down)
        device = ws[0][0].device
        for w in ws:
            for a, t in zip(w, (torch.uint8, torch.float32, torch.uint8)):
                if a is not None and (a.dtype != t or a.device != device or not a.is_cuda):
                    raise ValueError(f"{PREFIX}: weights must be uint8, scales float32 and zero "
                                     "points uint8 tensors on one device")
        if router is not None and (router.dtype != torch.float32 or router.device != device):
            raise ValueError(f"{PREFIX}: router must be a float32 tensor on the weights' device")
        self._check_sizes(router, *ws)
        with torch.cuda.device(device):
            ws = [tuple(None if a is None else a.contiguous() for a in w) for w in ws]
            r = None if router is None else router.contiguous()
            self._create("mnb_moe_plan_create_device", r, ws, lambda a: a.data_ptr())
        self._device = device
        return self

    def _create(self, entry, router, ws, address):
        structs = [MoeWeight(*(None if a is None else address(a) for a in w)) for w in ws]
        _check(getattr(_library(), entry)(
            ctypes.byref(self.desc), None if router is None else address(router),
            *(ctypes.byref(s) for s in structs), ctypes.byref(self._plan)), "prepare")
        self._router = router is not None

    def release(self):
        if self._plan:
            _library().mnb_moe_plan_destroy(self._plan)
            self._plan = ctypes.c_void_p()
        self._needs = {}

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass

    # -- compute -----------------------------------------------------------
    def __call__(self, X, logits=None, routing: bool = False, out=None, stream=None):
        """Y[..., H] of X's type (a float32, float16 or bfloat16 device tensor
        [..., H]). logits: float32 [..., experts] to choose by in the router's place.
        With routing: (Y, experts int32 [..., top_k], weights float32 [..., top_k])."""
        import torch
        if not self._plan:
            raise ValueError(f"{PREFIX}: prepare() was not called")
        d = self.desc
        x_type, device = _types.get(X.dtype), X.device
        if x_type is None or device != self._device:
            raise ValueError(f"{PREFIX}: X must be a float32, float16 or bfloat16 tensor on "
                             f"{self._device}")
        H, k, shape = d.hidden, d.top_k, X.shape
        if not shape or shape[-1] != H:
            raise ValueError(f"{PREFIX}: X must be [..., {H}], got {list(shape)}")
        rows = shape[:-1]
        if logits is None:
            if not self._router:
                raise ValueError(f"{PREFIX}: a layer without a router needs logits")
        elif (logits.shape != rows + (d.experts,) or logits.dtype != torch.float32
                or logits.device != device):
            raise ValueError(f"{PREFIX}: logits must be float32 {list(rows) + [d.experts]} on "
                             f"{device}")
        if out is not None and (out.shape != shape or out.dtype != X.dtype
                                or out.device != device or not out.is_contiguous()):
            raise ValueError(f"{PREFIX}: out must be contiguous, of X's shape, type and device")
        elsewhere = _elsewhere(device, stream)
        if elsewhere is not None:
            with elsewhere:
                return self(X, logits, routing, out)
        if not X.is_contiguous():
            X = X.contiguous()
        if logits is not None and not logits.is_contiguous():
            logits = logits.contiguous()
        if out is None:
            out = torch.empty(shape, dtype=X.dtype, device=device)
        ids = weights = None
        if routing:
            ids = torch.empty(rows + (k,), dtype=torch.int32, device=device)
            weights = torch.empty(rows + (k,), dtype=torch.float32, device=device)
        T = X.numel() // H
        need = self._needs.get((T, x_type))
        if need is None:
            if len(self._needs) > 256:
                self._needs = {}
            need = self._needs[T, x_type] = self.workspace_bytes(T, X.dtype)
        work = self._stream_workspace(need, device) if need else None
        status = _lib.mnb_moe_run(self._plan, T, x_type, X.data_ptr(),
                                  None if logits is None else logits.data_ptr(), out.data_ptr(),
                                  None if ids is None else ids.data_ptr(),
                                  None if weights is None else weights.data_ptr(),
                                  None if work is None else work.data_ptr(), need,
                                  _raw_stream(device))
        if status != 0:
            _check(status, "run")
        return (out, ids, weights) if routing else out

    run = __call__

    def workspace_bytes(self, T: int, dtype) -> int:
        """Device workspace of a call of T tokens of `dtype` (mnb_moe_workspace_bytes)."""
        n = ctypes.c_size_t()
        _check(_library().mnb_moe_workspace_bytes(self._plan, T, _types[dtype], ctypes.byref(n)),
               "workspace_bytes")
        return n.value

    def device_bytes(self) -> int:
        """Device memory the plan owns (mnb_moe_plan_device_bytes)."""
        n = ctypes.c_size_t()
        _check(_library().mnb_moe_plan_device_bytes(self._plan, ctypes.byref(n)), "device_bytes")
        return n.value
