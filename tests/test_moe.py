"""The expert layer's C ABI and Python object without a GPU: exports, and the
refusals that come before any device call."""
import ctypes
import re

import numpy as np
import pytest

OK, NULLP, SHAPE, ATTR, UNSUP, WORK = range(6)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.moe._library()


def _weights(pkg, zeros=False):
    return [pkg.moe.MoeWeight(16, 16, 16 if zeros else None) for _ in range(3)]


def _create(pkg, lib, weights=None, router=16, **change):
    """Both creations' common status; the pointers (all 16) are never followed."""
    fields = dict(hidden=64, intermediate=32, experts=4, top_k=2, bits=4, block_size=32,
                  normalize=1, has_zero_points=0)
    fields.update(change)
    d = pkg.moe.MoeDesc(*(fields[n] for n, _ in pkg.moe.MoeDesc._fields_))
    got = set()
    for entry in (lib.mnb_moe_plan_create, lib.mnb_moe_plan_create_device):
        plan = ctypes.c_void_p(7)
        ws = weights or _weights(pkg, fields["has_zero_points"] == 1)
        got.add(entry(ctypes.byref(d), router, *(w and ctypes.byref(w) for w in ws),
                      ctypes.byref(plan)))
        assert not plan.value
    assert len(got) == 1
    return got.pop()


def test_every_header_function_is_exported(pkg, lib):
    text = (pkg.ROOT / "include" / "mnb_moe.h").read_text()
    names = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(mnb_moe_\w+)\s*\(", text, re.M))
    assert names == {"mnb_moe_plan_create", "mnb_moe_plan_create_device", "mnb_moe_plan_destroy",
                     "mnb_moe_plan_device_bytes", "mnb_moe_workspace_bytes", "mnb_moe_run"}
    for name in names:
        assert hasattr(lib, name), name


@pytest.mark.parametrize("change,status", [
    ({"bits": 8}, UNSUP), ({"block_size": 8}, ATTR), ({"block_size": 48}, ATTR),
    ({"normalize": 2}, ATTR), ({"has_zero_points": 2}, ATTR), ({"hidden": 0}, SHAPE),
    ({"intermediate": -3}, SHAPE), ({"hidden": (1 << 20) + 1}, SHAPE),
    ({"hidden": 1 << 20, "intermediate": 1 << 20}, SHAPE), ({"experts": 0}, SHAPE),
    ({"experts": 1025}, SHAPE), ({"top_k": 0}, ATTR), ({"top_k": 5}, ATTR),
    ({"experts": 64, "top_k": 33}, ATTR)])
def test_bad_descriptions(pkg, lib, change, status):
    assert _create(pkg, lib, **change) == status


def test_pointers_and_zero_points(pkg, lib):
    for i in range(3):
        for field in ("B", "scales"):
            ws = _weights(pkg)
            setattr(ws[i], field, None)
            assert _create(pkg, lib, ws) == NULLP
        ws = _weights(pkg)
        ws[i] = None
        assert _create(pkg, lib, ws) == NULLP
        ws = _weights(pkg, True)
        ws[i].zero_points = None
        assert _create(pkg, lib, ws, has_zero_points=1) == NULLP
        ws = _weights(pkg)
        ws[i].zero_points = 16
        assert _create(pkg, lib, ws) == UNSUP
    n = ctypes.c_size_t()
    assert lib.mnb_moe_plan_destroy(None) == OK
    assert lib.mnb_moe_plan_device_bytes(None, ctypes.byref(n)) == NULLP
    assert lib.mnb_moe_workspace_bytes(None, 1, 1, ctypes.byref(n)) == NULLP
    assert lib.mnb_moe_run(None, 1, 1, 16, None, 16, None, None, 16, 0, None) == NULLP


def test_python_refusals(pkg):
    import torch
    op = pkg.MatMulNBitsMoE(64, 32, 4, 2)
    with pytest.raises(ValueError, match=r"prepare\(\) was not called"):
        op(torch.zeros(1, 64))
    gate = (np.zeros((4, 32, 2, 16), np.uint8), np.zeros((4, 32, 2), np.float32))
    down = (np.zeros((4, 64, 1, 16), np.uint8), np.zeros((4, 64, 1), np.float32))
    router = np.zeros((4, 64), np.float32)
    with pytest.raises(ValueError, match="all three weights"):
        op.prepare(router, gate + (np.zeros((4, 32, 1), np.uint8),), gate, down)
    with pytest.raises(ValueError, match="down's B has"):
        op.prepare(router, gate, gate, (down[0][:3], down[1]))
    with pytest.raises(ValueError, match="router has"):
        op.prepare(router[:3], gate, gate, down)
    with pytest.raises(ValueError, match="tensors on one device"):
        op.prepare_device(None, *(tuple(torch.from_numpy(a) for a in w) for w in (gate, gate, down)))
    with pytest.raises(ValueError, match="bad attribute"):
        pkg.MatMulNBitsMoE(64, 32, 4, 5).prepare(router, gate, gate, down)


def test_shapes_of_constants(pkg):
    """Weights, zero points and a router with the right number of elements in the wrong
    order."""
    op = pkg.MatMulNBitsMoE(64, 128, 4, 2)
    up = (np.zeros((4, 128, 2, 16), np.uint8), np.zeros((4, 128, 2), np.float32),
          np.zeros((4, 128, 1), np.uint8))
    down = (np.zeros((4, 64, 4, 16), np.uint8), np.zeros((4, 64, 4), np.float32),
            np.zeros((4, 64, 2), np.uint8))
    router = np.zeros((4, 64), np.float32)
    for args, match in (
            ((router, down, up, down), r"gate's B must be \[4, 128, 2, 16\], got \[4, 64, 4, 16\]"),
            ((router, up, up, (up[0],) + down[1:]), "down's B must be"),
            ((router, up, (up[0].transpose(1, 0, 2, 3),) + up[1:], down), "up's B must be"),
            ((router, up, up, (down[0], down[1].transpose(0, 2, 1), down[2])),
             r"down's scales must be \[4, 64, 4\], got \[4, 4, 64\]"),
            ((router, up, up, down[:2] + (down[2].transpose(0, 2, 1),)), "down's zero_points must"),
            ((router.T, up, up, down), r"router must be \[4, 64\], got \[64, 4\]")):
        with pytest.raises(ValueError, match=match):
            op.prepare(*args)
    assert not op._plan


@pytest.mark.parametrize("hidden,intermediate", [
    ((1 << 18) + 1, 32), (64, (1 << 18) + 1), (1 << 18, (1 << 16) + 1), ((1 << 16) + 1, 1 << 18)])
def test_width_limits(pkg, lib, hidden, intermediate):
    """One past each width's limit, which keeps offsets in 32 bits, and past the
    product's, with both widths inside theirs."""
    assert _create(pkg, lib, hidden=hidden, intermediate=intermediate) == SHAPE


@pytest.mark.parametrize("hidden,intermediate", [(1 << 18, 1 << 16), (1 << 16, 1 << 18)])
def test_widths_at_their_limits(pkg, lib, hidden, intermediate):
    """The limits themselves pass the description's check: what is refused next is
    the missing weight."""
    ws = _weights(pkg)
    ws[2] = None
    assert _create(pkg, lib, ws, hidden=hidden, intermediate=intermediate) == NULLP
