"""Rotary positions with several axes (include/mnb_rotary.h).

``Rotary`` turns the query and key heads of a QKV projection by their tokens'
positions: one axis for text, three (time, row, column) for images and video.
The frequencies are kept as turns in 64-bit fixed point: the product with a position is
not rounded, and the frequency's own rounding moves position p by 2^-65 |p| turns, less than
fp32 results show up to 2^38. There is no CPU fallback, and no gradient: backward() through
a result raises.
"""
from __future__ import annotations

import ctypes
import math
from . import _check, _raw_stream, library
from .fp8 import _elsewhere, _without_gradient

PREFIX = "onnx_light_cpu_amd::Rotary"
MAX_PAIRS, MAX_AXES = 256, 8
# 2^256 / (2 pi), of pi's first 60 digits
_PI_DIGITS = 314159265358979323846264338327950288419716939937510582097494
_PER_TURN = 2 ** 256 * 10 ** 59 // (2 * _PI_DIGITS)

_lib = None
_types = None  # torch dtype -> MNB_TYPE_* of include/mnb_fp8.h
_positions = None  # torch dtype -> MNB_TYPE_* of include/mnb_rotary.h


class RotaryDesc(ctypes.Structure):
    _fields_ = [("head_dim", ctypes.c_int32), ("rotary_dim", ctypes.c_int32),
                ("axes", ctypes.c_int32), ("interleaved", ctypes.c_int32),
                ("turns", ctypes.POINTER(ctypes.c_uint64)), ("axis", ctypes.POINTER(ctypes.c_uint8))]


class RotaryHeads(ctypes.Structure):
    _fields_ = [("heads", ctypes.c_int32), ("x", ctypes.c_void_p),
                ("x_token_stride", ctypes.c_int64), ("x_head_stride", ctypes.c_int64),
                ("y", ctypes.c_void_p), ("y_token_stride", ctypes.c_int64),
                ("y_head_stride", ctypes.c_int64)]


def _library():
    """libmnb.so with the rotation's signature."""
    global _lib, _types, _positions
    if _lib is None:
        import torch
        L = library()
        vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
        heads = ctypes.POINTER(RotaryHeads)
        L.mnb_rotary.argtypes = [ctypes.POINTER(RotaryDesc), i64, i32, vp, i64, i32, heads, heads,
                                 vp]
        _types = {torch.float32: 1, torch.float16: 10, torch.bfloat16: 16}
        _positions = {torch.int32: 6, torch.int64: 7}
        _lib = L
    return _lib


class Rotary:
    """Rotation of the first `rotary_dim` values (default: all) of heads of `head_dim`.

    sections: how many of the rotary_dim / 2 frequencies each axis has, in their
    order (default: one axis); axes: or each frequency's axis. inv_freq: the
    frequencies in radians a position (default: base ** (-2 j / rotary_dim)).
    Pair j is (x[j], x[j + rotary_dim / 2]), or (x[2j], x[2j + 1]) if interleaved.
    Calls of one object on several streams or threads may overlap."""

    op_type = "Rotary"

    def __init__(self, head_dim: int, sections=None, base: float = 10000.0, rotary_dim=None,
                 interleaved: bool = False, inv_freq=None, axes=None):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        pairs = self.rotary_dim // 2
        if (self.rotary_dim % 2 or not 1 <= pairs <= MAX_PAIRS
                or not self.rotary_dim <= self.head_dim <= 4096):
            raise ValueError(f"{PREFIX}: rotary_dim must be even, 2 .. {2 * MAX_PAIRS} and at most "
                             f"head_dim (at most 4096), got {self.rotary_dim} of {self.head_dim}")
        if sections is not None and axes is not None:
            raise ValueError(f"{PREFIX}: sections or axes, not both")
        if axes is None:
            sections = (pairs,) if sections is None else tuple(int(n) for n in sections)
            if min(sections, default=-1) < 0 or sum(sections) != pairs:
                raise ValueError(f"{PREFIX}: sections must add up to rotary_dim / 2 = {pairs}, got "
                                 f"{list(sections)}")
            axes = [a for a, n in enumerate(sections) for _ in range(n)]
            self.axes = len(sections)
        else:
            axes = [int(a) for a in axes]
            if len(axes) != pairs or min(axes) < 0:
                raise ValueError(f"{PREFIX}: axes must be one axis for each of the {pairs} "
                                 "frequencies")
            self.axes = max(axes) + 1
        if self.axes > MAX_AXES:
            raise ValueError(f"{PREFIX}: at most {MAX_AXES} axes, got {self.axes}")
        if inv_freq is None:
            if not 0.0 < base < math.inf:
                raise ValueError(f"{PREFIX}: base must be positive, got {base}")
            inv_freq = [math.exp(-2.0 * j / self.rotary_dim * math.log(base))
                        for j in range(pairs)]
        self.inv_freq = [float(f) for f in inv_freq]
        if len(self.inv_freq) != pairs or not all(map(math.isfinite, self.inv_freq)):
            raise ValueError(f"{PREFIX}: inv_freq must be {pairs} finite numbers")
        # f / (2 pi) modulo 1 in units of 2^-64, from the double as the ratio that it is
        turns = []
        for f in self.inv_freq:
            over, under = f.as_integer_ratio()
            turns.append(((over * _PER_TURN // under >> 191) + 1 >> 1) % 2 ** 64)
        self._turns = (ctypes.c_uint64 * pairs)(*turns)
        self._axis = (ctypes.c_uint8 * pairs)(*axes)
        self.desc = RotaryDesc(self.head_dim, self.rotary_dim, self.axes, int(bool(interleaved)),
                               self._turns, self._axis)
        self._ref = ctypes.byref(self.desc)

    @staticmethod
    def _strides(x, shape):
        """(between tokens, between heads) of x [..., H, D] in values, None where its heads
        are not whole or its tokens not evenly apart, or the same memory several times."""
        strides = x.stride()
        H, D = shape[-2:]
        sh = strides[-2] if H > 1 else D
        if len(shape) == 3:
            st = strides[0] if shape[0] > 1 else H * D
        else:
            st = apart = None
            for n, d in zip(shape[-3::-1], strides[-3::-1]):  # the axes of tokens, last first
                if n == 1:
                    continue
                if st is None:
                    st = apart = d
                elif d != apart:
                    return None
                apart *= n
            if st is None:
                st = H * D
        if st < D or sh < D or (D > 1 and strides[-1] != 1):
            return None
        return st, sh

    def __call__(self, Q, K, positions, out=None, stream=None):
        """(Q', K') of Q [..., Hq, head_dim] and K [..., Hkv, head_dim] (float32, float16
        or bfloat16 device tensors of one type, of any strides with whole heads; K may be
        None: then Q' alone). positions: int32 or int64, [...] the tokens' axes, or [axes,
        ...] where there are several. out: the results' tensors, which may be Q and K
        themselves, and overlap nothing else."""
        import torch
        L = _lib or _library()
        device, dtype, D = Q.device, Q.dtype, self.head_dim
        x_type = _types.get(dtype)
        if x_type is None or not Q.is_cuda:
            raise ValueError(f"{PREFIX}: Q must be a float32, float16 or bfloat16 device tensor")
        shapes = (Q.shape,) if K is None else (Q.shape, K.shape)
        tokens = shapes[0][:-2]
        for name, shape in zip("QK", shapes):
            if len(shape) < 2 or shape[-1] != D or shape[:-2] != tokens:
                raise ValueError(f"{PREFIX}: {name} must be [..., heads, {D}] of the same tokens, "
                                 f"got {list(shape)}")
        if K is not None and (K.dtype != dtype or K.device != device):
            raise ValueError(f"{PREFIX}: K must be of Q's type and device")
        pos_type, where = _positions.get(positions.dtype), positions.shape
        if (pos_type is None or positions.device != device
                or (where != (self.axes,) + tokens and (self.axes > 1 or where != tokens))):
            want = ([] if self.axes == 1 else [self.axes]) + list(tokens)
            raise ValueError(f"{PREFIX}: positions must be int32 or int64 {want} on {device}, "
                             f"got {positions.dtype} {list(where)}")
        parts = (Q,) if K is None else (Q, K)
        if out is not None:
            out = (out,) if K is None and isinstance(out, torch.Tensor) else tuple(out)
            if len(out) != len(parts):
                raise ValueError(f"{PREFIX}: out must be {len(parts)} tensors")
            for name, shape, y in zip("QK", shapes, out):
                if (y.shape != shape or y.dtype != dtype or y.device != device
                        or (y.numel() and self._strides(y, shape) is None)):
                    raise ValueError(f"{PREFIX}: out must have {name}'s shape, type and device, "
                                     "and whole heads")
        if (Q.requires_grad or (K is not None and K.requires_grad)) and torch.is_grad_enabled():
            if out is not None:
                raise ValueError(f"{PREFIX}: with out, Q and K must not require a gradient")
            return _without_gradient(PREFIX, lambda: self(Q, K, positions, stream=stream), *parts)
        elsewhere = _elsewhere(device, stream)
        if elsewhere is not None:
            with elsewhere:
                return self(Q, K, positions, out)
        T = tokens[0] if len(tokens) == 1 else math.prod(tokens)
        if T == 0:
            results = [torch.empty_like(x) for x in parts] if out is None else out
            return results[0] if K is None else tuple(results)
        heads, results, keep = [], [], []
        for x, shape in zip(parts, shapes):
            strides, address = self._strides(x, shape), x.data_ptr()
            if out is None:
                y = torch.empty_like(x, memory_format=torch.contiguous_format)
                to, address_y = (shape[-2] * D, D), y.data_ptr()
            else:
                y = out[len(results)]
                to, address_y = self._strides(y, shape), y.data_ptr()
            if strides is None or (address == address_y and strides != to):
                x = x.clone(memory_format=torch.contiguous_format)
                keep.append(x)
                strides, address = (shape[-2] * D, D), x.data_ptr()
            heads.append(RotaryHeads(shape[-2], address, *strides, address_y, *to))
            results.append(y)
        if not positions.is_contiguous():
            positions = positions.contiguous()
        status = L.mnb_rotary(self._ref, T, pos_type, positions.data_ptr(), T, x_type,
                              ctypes.byref(heads[0]),
                              ctypes.byref(heads[1]) if K is not None else None,
                              _raw_stream(device))
        if status != 0:
            _check(status, "rotary")
        return results[0] if K is None else tuple(results)

    run = __call__
