"""The 8-bit cache without a GPU: the C ABI's exports, its refusals and sizes, and
the object's checks of its arguments."""
import ctypes
import math
import re

import pytest

OK, NULLP, SHAPE, ATTR, UNSUP, WORK = range(6)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.kv._library()


def test_every_header_function_is_exported(pkg, lib):
    text = (pkg.ROOT / "include" / "mnb_kv.h").read_text()
    names = set(re.findall(r"^\s*int (mnb_\w+)\s*\(", text, re.M))
    assert names == {"mnb_kv_append", "mnb_kv_attend", "mnb_kv_workspace_bytes"}
    for name in names:
        assert hasattr(lib, name), name


CACHE = dict(pages=8, kv_heads=2, page_size=64, head_dim=64, k=16, v=16, k_scales=16, v_scales=16)
BATCH = dict(sequences=2, tokens=4, max_tokens=0, table_width=3, table=16, lengths=16, starts=None)
ROWS = dict(x=16, token_stride=128, head_stride=64)


def _call(pkg, lib, cache=(), batch=(), rows=(), heads=2, x_type=1, scale=1.0, window=0, Y=16,
          work=16, bytes_=1 << 30):
    """(append's status, attend's, workspace_bytes'): pointers (all 16) are never followed."""
    c = pkg.kv.KvCache(*dict(CACHE, **dict(cache)).values())
    b = pkg.kv.KvBatch(*dict(BATCH, **dict(batch)).values())
    r = pkg.kv.KvRows(*dict(ROWS, **dict(rows)).values())
    n = ctypes.c_size_t()
    c, b, r = ctypes.byref(c), ctypes.byref(b), ctypes.byref(r)
    return (lib.mnb_kv_append(c, b, x_type, r, r, None),
            lib.mnb_kv_attend(c, b, heads, x_type, r, scale, window, Y, work, bytes_, None),
            lib.mnb_kv_workspace_bytes(c, b, heads, x_type, ctypes.byref(n)))


@pytest.mark.parametrize("change,status", [
    ({"cache": {"pages": 0}}, SHAPE), ({"cache": {"pages": 1 << 31}}, SHAPE),
    ({"cache": {"kv_heads": 0}}, SHAPE), ({"cache": {"kv_heads": 1025}}, SHAPE),
    ({"cache": {"head_dim": 0}}, SHAPE), ({"cache": {"head_dim": 72}}, SHAPE),
    ({"cache": {"head_dim": 272}}, SHAPE), ({"cache": {"page_size": 8}}, ATTR),
    ({"cache": {"page_size": 48}}, ATTR), ({"cache": {"page_size": 512}}, ATTR),
    ({"cache": {"page_size": -16}}, ATTR), ({"batch": {"sequences": -1}}, SHAPE),
    ({"batch": {"sequences": 65536, "tokens": 65536}}, SHAPE), ({"batch": {"tokens": -2}}, SHAPE),
    ({"batch": {"tokens": (1 << 24) + 2}}, SHAPE), ({"batch": {"tokens": 3}}, SHAPE),
    ({"batch": {"max_tokens": -1}}, SHAPE), ({"batch": {"table_width": -1}}, SHAPE),
    ({"batch": {"table_width": (1 << 24) + 1}}, SHAPE), ({"x_type": 17}, ATTR)])
def test_shapes(pkg, lib, change, status):
    assert _call(pkg, lib, **change) == (status,) * 3


@pytest.mark.parametrize("change,status", [
    ({"cache": {"k": None}}, NULLP), ({"cache": {"v": None}}, NULLP),
    ({"cache": {"k_scales": None}}, NULLP), ({"cache": {"v_scales": None}}, NULLP),
    ({"batch": {"table": None}}, NULLP), ({"batch": {"lengths": None}}, NULLP),
    ({"rows": {"x": None}}, NULLP), ({"cache": {"k": 24}}, SHAPE), ({"cache": {"v": 24}}, SHAPE),
    ({"cache": {"k_scales": 18}}, SHAPE), ({"cache": {"v_scales": 18}}, SHAPE),
    ({"batch": {"table": 18}}, SHAPE), ({"batch": {"lengths": 18}}, SHAPE),
    ({"batch": {"starts": 18}}, SHAPE), ({"rows": {"x": 24}}, SHAPE),
    ({"rows": {"token_stride": 63}}, SHAPE), ({"rows": {"token_stride": 130}}, SHAPE),
    ({"rows": {"head_stride": 66}}, SHAPE), ({"rows": {"head_stride": 0}}, SHAPE),
    ({"rows": {"token_stride": 132}, "x_type": 10}, SHAPE)])
def test_pointers_and_strides(pkg, lib, change, status):
    assert _call(pkg, lib, **change) == (status, status, OK)


@pytest.mark.parametrize("change,status", [
    ({"heads": 0}, SHAPE), ({"heads": 3}, SHAPE), ({"heads": (1 << 16) + 2}, SHAPE),
    ({"heads": 18, "batch": {"tokens": 1 << 23}}, SHAPE)])
def test_heads(pkg, lib, change, status):
    bad = dict(change, cache={"k": None})
    assert _call(pkg, lib, **bad)[1:] == (status, status)


@pytest.mark.parametrize("change,status", [
    ({"scale": math.nan}, ATTR), ({"scale": math.inf}, ATTR), ({"window": -1}, ATTR),
    ({"Y": None}, NULLP), ({"Y": 24}, SHAPE), ({"work": 24}, SHAPE)])
def test_attention(pkg, lib, change, status):
    assert _call(pkg, lib, **change)[1] == status


def test_workspace(pkg, lib):
    """Long tables are shared out over workgroups, whose parts need room; short ones not."""
    n = ctypes.c_size_t()
    c = pkg.kv.KvCache(*CACHE.values())
    long = dict(BATCH, table_width=4096, sequences=1, tokens=1)
    for batch, some in ((BATCH, False), (long, True)):
        b = pkg.kv.KvBatch(*batch.values())
        assert lib.mnb_kv_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 2, 1,
                                          ctypes.byref(n)) == OK
        assert (n.value > 0) == some
    assert _call(pkg, lib, batch=long, bytes_=n.value - 1)[1] == WORK
    assert _call(pkg, lib, batch=long, work=None)[1] == WORK
    assert lib.mnb_kv_workspace_bytes(None, ctypes.byref(b), 2, 1, ctypes.byref(n)) == NULLP
    assert lib.mnb_kv_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 2, 1, None) == NULLP
    assert lib.mnb_kv_append(ctypes.byref(c), None, 1, None, None, None) == NULLP
    assert lib.mnb_kv_append(ctypes.byref(c), ctypes.byref(b), 1, None, None, None) == NULLP


def test_nothing_to_do(pkg, lib):
    for batch in ({"sequences": 0, "tokens": 0}, {"tokens": 0}):
        empty = dict(batch, table=None, lengths=None)
        assert _call(pkg, lib, batch=empty, Y=None) == (OK, OK, OK)


def test_python_refusals(pkg):
    import torch
    i32 = torch.int32
    make = pkg.Fp8KVCache
    for args, match in (((0, 2, 64), "pages"), ((4, 0, 64), "kv_heads"), ((4, 2, 72), "head_dim"),
                        ((4, 2, 64, 40), "page_size")):
        with pytest.raises(ValueError, match=match):
            make(*args, device="cpu")
    c = make(4, 2, 64, 32, device="cpu")
    assert c.k.shape == (4, 2, 32, 64) and c.v_scales.shape == (4, 2)
    codes, scales = c.k, c.k_scales
    for tensors, match in (((codes[0], codes, scales, scales), "k must be"),
                           ((codes, codes[:2], scales, scales), "v must be"),
                           ((codes, codes.view(torch.uint8), scales, scales), "v must be"),
                           ((codes, codes, scales[:, :1], scales), "k_scales must be"),
                           ((codes, codes, scales, scales.double()), "v_scales must be"),
                           ((codes.transpose(0, 1).contiguous().transpose(0, 1), codes, scales,
                             scales), "k must be")):
        with pytest.raises(ValueError, match=match):
            make.from_tensors(*tensors)
    x, table, lengths = torch.zeros(6, 2, 64), torch.zeros(2, 3, dtype=i32), torch.zeros(2, dtype=i32)
    starts = torch.zeros(3, dtype=i32)
    cases = [
        ((x[0], table, lengths), {}, r"must be \[..., "),
        ((x[..., :32], table, lengths), {}, r"must be \[..., "),
        ((x.double(), table, lengths), {}, "must be a float32"),
        ((x, table.long(), lengths), {}, "table must be int32"),
        ((x, table[0], lengths), {}, "table must be int32"),
        ((x, table, lengths[:1]), {}, "lengths must be int32"),
        ((x, table, lengths.long()), {}, "lengths must be int32"),
        ((x[:5], table, lengths), {}, "not the same number"),
        ((x.reshape(3, 2, 2, 64), table, lengths), {}, "not the same number"),
        ((x, table, lengths), {"starts": lengths}, "starts must be int32"),
        ((x.reshape(2, 3, 2, 64), table, lengths), {"starts": starts}, "with starts"),
        ((x, table, lengths), {"starts": starts, "max_tokens": -1}, "max_tokens"),
        ((x, table, lengths), {}, "no CPU fallback")]
    for (X, *rest), kwargs, match in cases:
        with pytest.raises(ValueError, match=match):
            c.append(X, X, *rest, **kwargs)
        with pytest.raises(ValueError, match=match):
            c.attend(X, *rest, **kwargs)
    with pytest.raises(ValueError, match="K must be"):
        c.append(x[:, :1], x, table, lengths)
    with pytest.raises(ValueError, match="one shape and type"):
        c.append(x, x.half(), table, lengths)
    for kwargs, match in (({"scale": math.inf}, "scale must be finite"),
                          ({"window": -1}, "window"), ({"out": x[:3]}, "out must be"),
                          ({"out": x.half()}, "out must be")):
        with pytest.raises(ValueError, match=match):
            c.attend(x, table, lengths, **kwargs)
    with pytest.raises(ValueError, match="multiple of 2"):
        c.attend(torch.zeros(6, 3, 64), table, lengths)
