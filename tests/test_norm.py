"""The RMS norm's C ABI and Python functions without a GPU: exports, and the
refusals that come before any device call."""
import math
import re

import pytest

OK, NULLP, SHAPE, ATTR, UNSUP, WORK = range(6)
F32, F16, BF16, E4M3 = 1, 10, 16, 17


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.norm._library()


def test_every_header_function_is_exported(pkg, lib):
    text = (pkg.ROOT / "include" / "mnb_norm.h").read_text()
    names = set(re.findall(r"^\s*int (mnb_\w+)\s*\(", text, re.M))
    assert names == {"mnb_rms_norm"}
    assert hasattr(lib, "mnb_rms_norm")


def _call(lib, **change):
    """The status of a call whose pointers (all 16) are never followed."""
    a = dict(M=1, K=8, x_type=F32, X=16, ldx=8, R=16, ldr=8, gamma=16, eps=1e-5, y_type=E4M3, Y=16,
             scales=16, H=16)
    a.update(change)
    return lib.mnb_rms_norm(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    ({"x_type": 17}, ATTR), ({"x_type": 2}, ATTR), ({"y_type": F16}, ATTR), ({"y_type": 0}, ATTR),
    ({"x_type": BF16, "y_type": F32}, ATTR), ({"eps": -1e-9}, ATTR), ({"eps": math.nan}, ATTR),
    ({"eps": math.inf}, ATTR), ({"M": -1}, SHAPE), ({"M": (1 << 30) + 1}, SHAPE),
    ({"K": 0}, SHAPE), ({"K": (1 << 22) + 1, "ldx": 1 << 23, "ldr": 1 << 23}, SHAPE),
    ({"ldx": 7}, SHAPE), ({"ldr": 7}, SHAPE), ({"ldx": (1 << 40) + 1}, SHAPE),
    ({"X": None}, NULLP), ({"gamma": None}, NULLP), ({"Y": None}, NULLP),
    ({"scales": None}, NULLP), ({"H": None}, NULLP), ({"R": None}, UNSUP),
    ({"y_type": F32}, UNSUP), ({"X": 18}, SHAPE), ({"R": 18}, SHAPE), ({"H": 18}, SHAPE),
    ({"gamma": 18}, SHAPE), ({"scales": 18}, SHAPE), ({"x_type": F16, "X": 17}, SHAPE),
    ({"y_type": F32, "scales": None, "Y": 18}, SHAPE), ({"M": 0}, OK),
    ({"M": 0, "X": None, "R": None, "H": None, "Y": None, "gamma": None, "scales": None}, OK)])
def test_refusals(lib, change, status):
    assert _call(lib, **change) == status


def test_python_refusals(pkg):
    import torch
    x, g = torch.zeros(2, 8), torch.ones(8)
    for f in (pkg.rms_norm, pkg.rms_norm_fp8):
        with pytest.raises(ValueError, match="X must be a float32, float16 or bfloat16 device"):
            f(x, g)
        with pytest.raises(ValueError, match="X must be a float32, float16 or bfloat16 device"):
            f(x.double(), g)
    with pytest.raises(ValueError, match="X must be a float32"):
        pkg.MatMulFp8(8, 8).run_rmsnorm(x, g)
