"""Rotary positions without a GPU: the C ABI's exports and refusals, and the
object's frequencies and arguments."""
import ctypes
import math
import re

import pytest

OK, NULLP, SHAPE, ATTR, UNSUP, WORK = range(6)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.rotary._library()


def test_every_header_function_is_exported(pkg, lib):
    text = (pkg.ROOT / "include" / "mnb_rotary.h").read_text()
    assert set(re.findall(r"^\s*int (mnb_\w+)\s*\(", text, re.M)) == {"mnb_rotary"}
    assert hasattr(lib, "mnb_rotary")


def _call(pkg, lib, desc=(), query=(), key=(), turns=True, axis=(0, 0, 1, 1), **change):
    """The status of a call whose device pointers (all 16) are never followed."""
    d = dict(head_dim=8, rotary_dim=8, axes=2, interleaved=0)
    d.update(desc)
    turns_ = (ctypes.c_uint64 * 4096)()
    axis_ = (ctypes.c_uint8 * 4096)(*axis)
    D = pkg.rotary.RotaryDesc(*d.values(), turns_ if turns else None, axis_ if axis else None)
    heads = dict(heads=2, x=16, xt=16, xh=8, y=16, yt=16, yh=8)
    q, k = dict(heads, **dict(query)), dict(heads, **dict(key))
    a = dict(T=4, pos_type=7, pos=16, axis_stride=4, x_type=1)
    a.update(change)
    H = pkg.rotary.RotaryHeads
    return lib.mnb_rotary(ctypes.byref(D), *a.values(), ctypes.byref(H(*q.values())),
                          ctypes.byref(H(*k.values())), None)


@pytest.mark.parametrize("change,status", [
    ({"desc": {"head_dim": 0}}, SHAPE), ({"desc": {"head_dim": 4097}}, SHAPE),
    ({"desc": {"rotary_dim": 7}}, SHAPE), ({"desc": {"rotary_dim": 0}}, SHAPE),
    ({"desc": {"rotary_dim": 10}}, SHAPE), ({"desc": {"head_dim": 1024, "rotary_dim": 514}}, SHAPE),
    ({"desc": {"axes": 0}}, ATTR), ({"desc": {"axes": 9}}, ATTR), ({"desc": {"axes": 1}}, ATTR),
    ({"desc": {"interleaved": 2}}, ATTR), ({"axis": (0, 0, 1, 2)}, ATTR), ({"turns": False}, NULLP),
    ({"axis": ()}, NULLP), ({"T": -1}, SHAPE), ({"T": (1 << 24) + 1}, SHAPE),
    ({"axis_stride": 3}, SHAPE), ({"pos_type": 1}, ATTR), ({"x_type": 17}, ATTR),
    ({"pos": None}, NULLP), ({"pos": 20}, SHAPE), ({"pos_type": 6, "pos": 18}, SHAPE),
    ({"query": {"x": None}}, NULLP), ({"key": {"y": None}}, NULLP), ({"query": {"x": 18}}, SHAPE),
    ({"key": {"y": 17}, "x_type": 10}, SHAPE), ({"query": {"xh": 7}}, SHAPE),
    ({"key": {"yt": 7}}, SHAPE), ({"key": {"heads": -1}}, SHAPE), ({"query": {"yt": 32}}, UNSUP),
    ({"query": {"heads": (1 << 16) + 1}}, SHAPE), ({"T": 0}, OK),
    ({"T": 0, "pos": None, "query": {"x": None}}, OK),
    ({"query": {"heads": 0}, "key": {"heads": 0}, "pos": None}, OK)])
def test_refusals(pkg, lib, change, status):
    assert _call(pkg, lib, **change) == status


def test_null_descriptions(pkg, lib):
    H = pkg.rotary.RotaryHeads(0)
    assert lib.mnb_rotary(None, 0, 7, None, 0, 1, ctypes.byref(H), None, None) == NULLP
    r = pkg.Rotary(8)
    assert lib.mnb_rotary(ctypes.byref(r.desc), 0, 7, None, 0, 1, None, None, None) == NULLP
    assert lib.mnb_rotary(ctypes.byref(r.desc), 3, 7, None, 0, 1, ctypes.byref(H), None, None) == OK


def test_turns_are_frequencies_over_two_pi(pkg):
    """A turn is 2^64 units, off by half a unit and the double's own rounding."""
    r = pkg.Rotary(64, base=500000.0)
    for j, f in enumerate(r.inv_freq):
        assert f == math.exp(-2.0 * j / 64 * math.log(500000.0))
        assert abs(r._turns[j] / 2.0 ** 64 - f / (2.0 * math.pi)) <= 2.0 ** -52 * f + 2.0 ** -64
    r = pkg.Rotary(8, inv_freq=[2.0 * math.pi, 7.0, -1.0, 0.0])
    # 2 pi rounded to a double is 2.4e-16 short of a turn
    assert (2 ** 64 - r._turns[0]) % 2 ** 64 < 2 ** 64 * 1e-16
    assert abs(r._turns[1] / 2.0 ** 64 - (7.0 / (2.0 * math.pi) - 1.0)) < 1e-15
    assert r._turns[2] + pkg.Rotary(8, inv_freq=[1.0] * 4)._turns[0] == 2 ** 64
    assert r._turns[3] == 0


def test_turns_are_the_nearest(pkg):
    """Half a unit of 2^-64 of a turn is all that a frequency, a double, loses: 2^-65 |p| turns at
    position p."""
    from fractions import Fraction
    two_pi = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494")
    for r in (pkg.Rotary(128), pkg.Rotary(64, base=5e5),
              pkg.Rotary(8, inv_freq=[1e-9, 3.0, -2.5e4, 1e12])):
        for f, turn in zip(r.inv_freq, r._turns):
            off = (Fraction(f) / two_pi * 2 ** 64 - turn) % 2 ** 64
            assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + Fraction(1, 1000)


def test_axes_of_frequencies(pkg):
    assert list(pkg.Rotary(16, sections=(2, 3, 3))._axis) == [0, 0, 1, 1, 1, 2, 2, 2]
    r = pkg.Rotary(16, rotary_dim=8, axes=(0, 1, 2, 0))
    assert list(r._axis) == [0, 1, 2, 0] and r.axes == 3 and r.desc.rotary_dim == 8
    assert pkg.Rotary(16, sections=(0, 8)).axes == 2


@pytest.mark.parametrize("kwargs,match", [
    ({"head_dim": 7}, "rotary_dim must be even"), ({"head_dim": 8, "rotary_dim": 10}, "rotary_dim"),
    ({"head_dim": 8, "rotary_dim": 0}, "rotary_dim"), ({"head_dim": 514}, "rotary_dim"),
    ({"head_dim": 8, "sections": (2, 3)}, "sections must add up"),
    ({"head_dim": 8, "sections": (5, -1)}, "sections must add up"),
    ({"head_dim": 8, "sections": ()}, "sections must add up"),
    ({"head_dim": 8, "sections": (4,), "axes": (0,) * 4}, "not both"),
    ({"head_dim": 8, "axes": (0, 1)}, "one axis for each"),
    ({"head_dim": 8, "axes": (0, 1, -1, 0)}, "one axis for each"),
    ({"head_dim": 8, "axes": (0, 1, 8, 0)}, "at most 8 axes"),
    ({"head_dim": 8, "base": 0.0}, "base must be"), ({"head_dim": 8, "base": math.nan}, "base"),
    ({"head_dim": 8, "inv_freq": [1.0]}, "inv_freq must be 4"),
    ({"head_dim": 8, "inv_freq": [1.0, 1.0, math.inf, 1.0]}, "inv_freq must be 4")])
def test_python_refusals(pkg, kwargs, match):
    with pytest.raises(ValueError, match=match):
        pkg.Rotary(**kwargs)


def test_strides_of_tokens_of_several_axes(pkg):
    """Token axes that can be walked with one stride, and those that cannot: expanded ones (a
    stride of 0, innermost or not), transposed and sliced ones. Every value that the strides
    lead to is the tensor's own."""
    import torch
    H, D = 4, 8
    x = torch.arange(6 * H * D, dtype=torch.float32).reshape(2, 3, H, D)
    row = x[0, :, None]  # [3, 1, H, D]
    cases = [(x, True), (x.view(6, H, D), True), (x.view(1, 2, 3, H, D), True), (x[:, :1], True),
             (x[:, 1:2], True), (x[:, 0], True), (x[:1], True), (x[:1, :1], True), (x[..., :2, :], True),
             (x.view(2, 3, 1, H, D), True), (x[0, 0], True),
             (x.transpose(0, 1), False), (x[:, :2], False), (x[:, ::2], False),
             (row.expand(3, 2, H, D), False), (row.expand(3, 5, H, D)[:1], False),
             (row[:1].expand(3, 2, H, D), False), (x[:1].expand(2, 3, H, D), False),
             (row[None].expand(2, 3, 1, H, D), False), (row[:, :, None].expand(3, 1, 2, H, D), False),
             (x[0, :1].expand(3, H, D), False), (x[0, :, :1].expand(3, H, D), False),
             (x[0, 0].expand(3, H, D), False)]
    for n, (t, even) in enumerate(cases):
        got = pkg.Rotary._strides(t, t.shape)
        assert (got is not None) == even, (n, t.shape, t.stride(), got)
        if got is not None:
            T = t.numel() // (t.shape[-2] * D)
            at = (torch.arange(T)[:, None, None] * got[0] + torch.arange(t.shape[-2])[:, None] * got[1]
                  + torch.arange(D) + t.storage_offset())
            assert torch.equal(x.flatten()[at], t.reshape(T, -1, D)), n


def test_no_cpu_fallback(pkg):
    import torch
    with pytest.raises(ValueError, match="device tensor"):
        pkg.Rotary(8)(torch.zeros(1, 2, 8), None, torch.zeros(1, dtype=torch.int64))
