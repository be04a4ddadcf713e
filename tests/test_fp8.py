"""The 8-bit product's C ABI and Python objects without a GPU: exports, and the
refusals that come before any device call."""
import ctypes
import re

import numpy as np
import pytest

OK, NULLP, SHAPE, ATTR, UNSUP, WORK = range(6)


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.fp8._library()


def test_every_header_function_is_exported(pkg, lib):
    text = (pkg.ROOT / "include" / "mnb_fp8.h").read_text()
    names = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(mnb_fp8_\w+)\s*\(", text, re.M))
    assert names == {"mnb_fp8_quantize", "mnb_fp8_plan_create", "mnb_fp8_plan_create_device",
                     "mnb_fp8_plan_destroy", "mnb_fp8_plan_device_bytes",
                     "mnb_fp8_workspace_bytes", "mnb_fp8_run", "mnb_fp8_kernel_name"}
    for name in names:
        assert hasattr(lib, name), name


@pytest.mark.parametrize("K,N,status", [(0, 8, SHAPE), (8, -1, SHAPE), ((1 << 22) + 1, 8, SHAPE),
                                        (8, (1 << 26) + 1, SHAPE)])
def test_plan_shapes(lib, K, N, status):
    plan = ctypes.c_void_p(7)
    W, S = np.zeros(64, np.uint8), np.zeros(4, np.float32)
    for create in (lib.mnb_fp8_plan_create, lib.mnb_fp8_plan_create_device):
        assert create(K, N, W.ctypes.data, S.ctypes.data, ctypes.byref(plan)) == status
        assert not plan.value


def test_plan_null_pointers(lib):
    plan = ctypes.c_void_p()
    W, S = np.zeros(64, np.uint8), np.zeros(4, np.float32)
    assert lib.mnb_fp8_plan_create(8, 8, None, S.ctypes.data, ctypes.byref(plan)) == NULLP
    assert lib.mnb_fp8_plan_create(8, 8, W.ctypes.data, None, ctypes.byref(plan)) == NULLP
    assert lib.mnb_fp8_plan_create(8, 8, W.ctypes.data, S.ctypes.data, None) == NULLP
    assert lib.mnb_fp8_plan_destroy(None) == OK
    n = ctypes.c_size_t()
    assert lib.mnb_fp8_plan_device_bytes(None, ctypes.byref(n)) == NULLP
    assert lib.mnb_fp8_workspace_bytes(None, 1, 1, ctypes.byref(n)) == NULLP
    assert lib.mnb_fp8_run(None, 1, 17, 16, 16, 1, 16, None, 0, None) == NULLP
    assert lib.mnb_fp8_kernel_name(None, 1) == b""


@pytest.mark.parametrize("args,status", [
    # M, K, type, X, ldx, Q, scales: the pointers are never followed
    ((1, 8, 17, 16, 8, 16, 16), ATTR), ((1, 8, 2, 16, 8, 16, 16), ATTR),
    ((-1, 8, 1, 16, 8, 16, 16), SHAPE), ((1, 0, 1, 16, 8, 16, 16), SHAPE),
    ((1, 8, 1, 16, 7, 16, 16), SHAPE), ((1, 8, 1, None, 8, 16, 16), NULLP),
    ((1, 8, 1, 16, 8, None, 16), NULLP), ((1, 8, 1, 16, 8, 16, None), NULLP),
    ((1, 8, 1, 18, 8, 16, 16), SHAPE), ((1, 8, 10, 17, 8, 16, 16), SHAPE),
    ((1, 8, 1, 16, 8, 16, 18), SHAPE), ((0, 8, 1, None, 8, None, None), OK)])
def test_quantize_refusals(lib, args, status):
    assert lib.mnb_fp8_quantize(*args, None) == status


def test_python_refusals(pkg):
    import torch
    with pytest.raises(ValueError, match="device tensor"):
        pkg.quantize_fp8(torch.zeros(2, 8))
    op = pkg.MatMulFp8(8, 8)
    with pytest.raises(ValueError, match=r"prepare\(\) was not called"):
        op(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="W has 4 values"):
        op.prepare(np.zeros(4, np.uint8), np.zeros(1, np.float32))
    with pytest.raises(ValueError, match="scales has 2 elements"):
        op.prepare(np.zeros((8, 8), np.uint8), np.zeros(2, np.float32))
    with pytest.raises(ValueError, match="device tensor"):
        op.prepare_device(torch.zeros(8, 8, dtype=torch.uint8), torch.zeros(1, 1))
    with pytest.raises(ValueError, match="bad shape"):
        pkg.MatMulFp8(0, 8).prepare(np.zeros(1, np.uint8), np.zeros(1, np.float32))


def test_shapes_of_constants(pkg):
    """A weight or scales with the right number of values in the wrong order."""
    import torch
    op = pkg.MatMulFp8(256, 384)
    W, S = np.zeros((384, 256), np.uint8), np.zeros((3, 2), np.float32)
    for w, s, match in ((W.T, S, r"W must be \[N, K\] = \[384, 256\], got \[256, 384\]"),
                        (W.reshape(192, 512), S, "W must be"), (W.reshape(768, 128), S, "W must"),
                        (W, S.T, r"scales must be .* = \[3, 2\], got \[2, 3\]")):
        with pytest.raises(ValueError, match=match):
            op.prepare(w, s)
    assert not op._plan
    laid_out = pkg.fp8._laid_out
    for shape in ((2, 3, 4), (6, 4), (2, 12), (24,), (1, 2, 3, 1, 4), (24, 1)):
        assert laid_out(shape, [2, 3, 4])
    for shape in ((3, 2, 4), (4, 6), (12, 2), (2, 4, 3), (2, 2, 6), (2, 3), (2, 3, 4, 2), ()):
        assert not laid_out(shape, [2, 3, 4])
    assert laid_out((1, 1), [1]) and laid_out((5,), [1, 5, 1]) and laid_out((), [1, 1])
