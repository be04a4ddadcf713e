"""A paged key/value cache in 8 bits and the attention over it (include/mnb_kv.h).

``Fp8KVCache`` holds keys and values as e4m3 codes with a power-of-two scale for
each page of tokens and head. ``append`` writes a call's new tokens, ``attend`` is
the causal attention of their queries over the cache, from one token of each
sequence to chunks of prompts, in one call for all sequences. Between them and a
QKV projection stands ``Rotary``. There is no CPU fallback, and no gradient: the cache
holds values alone, and backward() through a result of ``attend`` raises.
"""
from __future__ import annotations

import ctypes
import math

from . import MatMulNBits, _check, _raw_stream, library
from .fp8 import _elsewhere, _shared_works, _without_gradient

PREFIX = "onnx_light_cpu_amd::Fp8KVCache"
PAGE_SIZES = (16, 32, 64, 128, 256)


class KvCache(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_int64), ("kv_heads", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scales", ctypes.c_void_p),
                ("v_scales", ctypes.c_void_p)]


class KvBatch(ctypes.Structure):
    _fields_ = [("sequences", ctypes.c_int64), ("tokens", ctypes.c_int64),
                ("max_tokens", ctypes.c_int64), ("table_width", ctypes.c_int64),
                ("table", ctypes.c_void_p), ("lengths", ctypes.c_void_p),
                ("starts", ctypes.c_void_p)]


class KvRows(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64)]


_lib = None
_types = None  # torch dtype -> MNB_TYPE_* of include/mnb_fp8.h
_int32 = _current_device = None  # torch.int32, torch's query of the current device


def _library():
    """libmnb.so with the cache's signatures."""
    global _lib, _types, _int32, _current_device
    if _lib is None:
        import torch
        L = library()
        vp, i64, i32, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t
        cache, batch = ctypes.POINTER(KvCache), ctypes.POINTER(KvBatch)
        rows = ctypes.POINTER(KvRows)
        L.mnb_kv_append.argtypes = [cache, batch, i32, rows, rows, vp]
        L.mnb_kv_workspace_bytes.argtypes = [cache, batch, i32, i32, ctypes.POINTER(sz)]
        L.mnb_kv_attend.argtypes = [cache, batch, i32, i32, rows, ctypes.c_float, i64, vp, vp, sz,
                                    vp]
        _types = {torch.float32: 1, torch.float16: 10, torch.bfloat16: 16}
        _int32, _current_device = torch.int32, torch._C._cuda_getDevice
        _lib = L
    return _lib


class Fp8KVCache:
    """Keys and values of `pages` pages of `page_size` tokens (16, 32, 64, 128 or 256) and
    `kv_heads` heads of `head_dim` (a multiple of 16, at most 256), all pages free. Calls on several
    streams or threads may overlap where they touch different pages, or only read.

    k, v: float8_e4m3fn [pages, kv_heads, page_size, head_dim]; k_scales, v_scales:
    float32 [pages, kv_heads]; value = code * scale.

    The calls share their description of the sequences. Tensors of tokens are [tokens,
    heads, head_dim], or [sequences, tokens of each, heads, head_dim]. table: int32
    [sequences, width], the pages of each sequence in their order; lengths: int32
    [sequences], each sequence's tokens with those of the call, which are its last;
    starts: int32 [sequences + 1], the first row of each sequence where they have
    different numbers of rows, and the end; max_tokens: the largest number (kernels are
    chosen by it; without it, all rows might be one sequence's). All are device tensors
    but max_tokens: a captured call can be replayed as they change."""

    op_type = "Fp8KVCache"

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device=None):
        import torch
        self._check_sizes(pages, kv_heads, head_dim, page_size)
        shape = (pages, kv_heads, page_size, head_dim)
        device = torch.device("cuda" if device is None else device)
        self._set(*(torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device)
                    for _ in range(2)),
                  *(torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2)))

    @classmethod
    def from_tensors(cls, k, v, k_scales, v_scales):
        """A cache of tensors that exist (held, not copied); scales may be any
        numbers from 2^-100 to 2^100 (powers of two to 2^120), or 0 for a page of codes of
        0. append makes powers of two, but a page that it continues keeps a larger scale."""
        import torch
        if k.dim() != 4:
            raise ValueError(f"{PREFIX}: k must be [pages, kv_heads, page_size, head_dim], got "
                             f"{list(k.shape)}")
        cls._check_sizes(k.shape[0], k.shape[1], k.shape[3], k.shape[2])
        for name, x, shape, dtype in (("k", k, k.shape, torch.float8_e4m3fn),
                                      ("v", v, k.shape, torch.float8_e4m3fn),
                                      ("k_scales", k_scales, k.shape[:2], torch.float32),
                                      ("v_scales", v_scales, k.shape[:2], torch.float32)):
            if (x.dtype != dtype or x.shape != shape or x.device != k.device
                    or not x.is_contiguous() or x.data_ptr() % 16 != 0):
                raise ValueError(f"{PREFIX}: {name} must be a contiguous {dtype} tensor "
                                 f"{list(shape)} on k's device, aligned to 16 bytes")
        self = cls.__new__(cls)
        self._set(k, v, k_scales, v_scales)
        return self

    @staticmethod
    def _check_sizes(pages, kv_heads, head_dim, page_size):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"{PREFIX}: page_size must be one of {list(PAGE_SIZES)}, got "
                             f"{page_size}")
        if head_dim % 16 != 0 or not 16 <= head_dim <= 256:
            raise ValueError(f"{PREFIX}: head_dim must be a multiple of 16 up to 256, got "
                             f"{head_dim}")
        if not 1 <= kv_heads <= 1024 or not 1 <= pages < 2 ** 31:
            raise ValueError(f"{PREFIX}: kv_heads must be 1 .. 1024 and pages 1 .. 2^31 - 1, got "
                             f"{kv_heads} and {pages}")

    # The calls hold these tensors' addresses: they cannot be replaced.
    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scales = property(lambda self: self._tensors[2])
    v_scales = property(lambda self: self._tensors[3])

    def _set(self, k, v, k_scales, v_scales):
        self._tensors = (k, v, k_scales, v_scales)
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.device = k.device
        self._cache = KvCache(self.pages, self.kv_heads, self.page_size, self.head_dim,
                              k.data_ptr(), v.data_ptr(), k_scales.data_ptr(),
                              v_scales.data_ptr())
        self._cache_ref = ctypes.byref(self._cache)
        self._needs = {}  # workspace bytes by the call's sizes

    _works = _shared_works
    _stream_workspace = MatMulNBits._stream_workspace

    # -- what the calls share ----------------------------------------------
    # The smallest calls are bound by these functions, not by their 4 us of kernels: an
    # attribute of a tensor costs 50 to 100 ns, so each is read once.
    def _check_tokens(self, shape, dtype, device, name, heads):
        if (len(shape) not in (3, 4) or shape[-1] != self.head_dim
                or (heads is not None and shape[-2] != heads)):
            raise ValueError(f"{PREFIX}: {name} must be [..., "
                             f"{'heads' if heads is None else heads}, {self.head_dim}], got "
                             f"{list(shape)}")
        if dtype not in _types or device != self.device:
            raise ValueError(f"{PREFIX}: {name} must be a float32, float16 or bfloat16 tensor on "
                             f"{self.device}")

    def _batch(self, shape, table, lengths, starts, max_tokens):
        """(the C struct of the sequences of tokens of this shape, what it points to)."""
        device = self.device
        sizes = table.shape
        if len(sizes) != 2 or table.dtype != _int32 or table.device != device:
            raise ValueError(f"{PREFIX}: table must be int32 [sequences, width] on {device}")
        B, width = sizes
        if lengths.shape != (B,) or lengths.dtype != _int32 or lengths.device != device:
            raise ValueError(f"{PREFIX}: lengths must be int32 [{B}] on {device}")
        each = 0
        if len(shape) == 3:
            tokens = even = shape[0]
            if starts is None and (even % B if B else even):
                even = -1
        else:
            tokens, even = shape[0] * shape[1], 0 if shape[0] == B else -1
        if max_tokens is not None and max_tokens < 0:
            raise ValueError(f"{PREFIX}: max_tokens must not be negative, got {max_tokens}")
        first = None
        if starts is not None:
            if len(shape) != 3:
                raise ValueError(f"{PREFIX}: with starts, tokens must be [tokens, heads, "
                                 f"{self.head_dim}], got {list(shape)}")
            if starts.shape != (B + 1,) or starts.dtype != _int32 or starts.device != device:
                raise ValueError(f"{PREFIX}: starts must be int32 [{B + 1}] on {device}")
            if not starts.is_contiguous():
                starts = starts.contiguous()
            # the C struct's field would cut a larger number to its low 64 bits
            first, each = starts.data_ptr(), min(max_tokens or 0, tokens)
        elif even < 0:
            raise ValueError(f"{PREFIX}: {list(shape[:-2])} tokens are not the same number for each "
                             f"of {B} sequences")
        if device.type != "cuda":
            raise ValueError(f"{PREFIX}: the cache is on {device}; there is no CPU fallback")
        if not table.is_contiguous():
            table = table.contiguous()
        if not lengths.is_contiguous():
            lengths = lengths.contiguous()
        return KvBatch(B, tokens, each, width, table.data_ptr(), lengths.data_ptr(),
                       first), (table, lengths, starts)

    @staticmethod
    def _rows(X, shape):
        """(the C struct of X [..., heads, head_dim], the tensor it points into): X, or a
        copy where its rows are not evenly apart or not aligned to 16 bytes."""
        strides, address, even = X.stride(), X.data_ptr(), True
        if len(shape) == 3:
            n, H, D = shape
            st = strides[0] if n > 1 else H * D
        else:
            n, t, H, D = shape
            st = strides[1] if t > 1 else strides[0] if n > 1 else H * D
            even = n <= 1 or t <= 1 or strides[0] == t * strides[1]
        sh = strides[-2] if H > 1 else D
        # 8 values of any of the types are whole 16 bytes
        if (not even or strides[-1] != 1 or st < D or sh < D or st % 8 or sh % 8
                or address % 16):
            X = X.clone() if X.is_contiguous() else X.contiguous()
            st, sh, address = H * D, D, X.data_ptr()
        return KvRows(address, st, sh), X

    # -- compute -----------------------------------------------------------
    def append(self, K, V, table, lengths, starts=None, max_tokens=None, stream=None):
        """Writes the keys K and values V [..., kv_heads, head_dim] (float32, float16 or
        bfloat16, of one type, any strides) behind what the sequences hold. A page's
        scale is the least power of two that its largest magnitude allows; it grows
        as the page fills, and then the page's codes are rounded again."""
        L = _lib or _library()
        shape, dtype, device = K.shape, K.dtype, K.device
        self._check_tokens(shape, dtype, device, "K", self.kv_heads)
        if V.shape != shape or V.dtype != dtype or V.device != device:
            self._check_tokens(V.shape, V.dtype, V.device, "V", self.kv_heads)
            raise ValueError(f"{PREFIX}: K and V must be of one shape and type")
        if stream is not None or (device.index is not None and device.index != _current_device()):
            self._batch(shape, table, lengths, starts, max_tokens)  # its refusals first
            elsewhere = _elsewhere(device, stream)
            if elsewhere is not None:
                with elsewhere:
                    return self.append(K, V, table, lengths, starts, max_tokens)
        batch, keep = self._batch(shape, table, lengths, starts, max_tokens)
        k, K = self._rows(K, shape)
        v, V = self._rows(V, shape)
        status = L.mnb_kv_append(self._cache_ref, ctypes.byref(batch), _types[dtype],
                                 ctypes.byref(k), ctypes.byref(v), _raw_stream(device))
        if status != 0:
            _check(status, "append")
        return self

    def attend(self, Q, table, lengths, starts=None, max_tokens=None, scale=None, window: int = 0,
               out=None, stream=None):
        """Y of Q's shape and type: for each token and query head the softmax of scale q .
        k (default 1 / sqrt(head_dim)) over its sequence's tokens up to itself, or
        the last `window` of them (0: all), times their values. Q [..., heads, head_dim],
        heads a multiple of kv_heads: neighbouring heads share a cache head. A row
        that sees nothing is 0. Rows of no sequence are 0, or stay as they are in out."""
        import torch
        L = _lib or _library()
        shape, dtype, device = Q.shape, Q.dtype, Q.device
        self._check_tokens(shape, dtype, device, "Q", None)
        heads, x_type = shape[-2], _types[dtype]
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"{PREFIX}: Q's heads must be a multiple of {self.kv_heads}, got "
                             f"{heads}")
        if window < 0:
            raise ValueError(f"{PREFIX}: window must not be negative, got {window}")
        window = min(window, 2 ** 31)  # more than any table reaches, and the C argument holds
        if scale is None:
            scale = self.head_dim ** -0.5
        elif not math.isfinite(scale):
            raise ValueError(f"{PREFIX}: scale must be finite, got {scale}")
        if out is not None and (out.shape != shape or out.dtype != dtype or out.device != device
                                or not out.is_contiguous() or out.data_ptr() % 16 != 0):
            raise ValueError(f"{PREFIX}: out must be contiguous, of Q's shape, type and device, "
                             "aligned to 16 bytes")
        if Q.requires_grad and torch.is_grad_enabled():
            if out is not None:
                raise ValueError(f"{PREFIX}: with out, Q must not require a gradient")
            return _without_gradient(PREFIX, lambda: self.attend(
                Q, table, lengths, starts, max_tokens, scale, window, stream=stream), Q)
        if stream is not None or (device.index is not None and device.index != _current_device()):
            self._batch(shape, table, lengths, starts, max_tokens)  # its refusals first
            elsewhere = _elsewhere(device, stream)
            if elsewhere is not None:
                with elsewhere:
                    return self.attend(Q, table, lengths, starts, max_tokens, scale, window, out)
        batch, keep = self._batch(shape, table, lengths, starts, max_tokens)
        q, X = self._rows(Q, shape)
        if out is None:
            if starts is not None:
                out = torch.zeros(shape, dtype=dtype, device=device)
            else:
                out = torch.empty_like(Q, memory_format=torch.contiguous_format)
        key = (batch.sequences, batch.tokens, batch.max_tokens, batch.table_width, heads, x_type,
               starts is None)
        need = self._needs.get(key)
        if need is None:
            if len(self._needs) > 256:
                self._needs = {}
            n = ctypes.c_size_t()
            _check(L.mnb_kv_workspace_bytes(self._cache_ref, ctypes.byref(batch), heads, x_type,
                                            ctypes.byref(n)), "workspace_bytes")
            need = self._needs[key] = n.value
        work = self._stream_workspace(need, device) if need else None
        status = L.mnb_kv_attend(self._cache_ref, ctypes.byref(batch), heads, x_type,
                                 ctypes.byref(q), scale, window, out.data_ptr(),
                                 None if work is None else work.data_ptr(), need,
                                 _raw_stream(device))
        if status != 0:
            _check(status, "attend")
        return out
