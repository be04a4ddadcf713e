"""Rotary positions on the GPU, against angles in exact arithmetic.

Tolerances, fixed before the first run. The angle in turns is exact but for 2^-33
of a turn (its lower word), 2^-30 in radians; as fp32 it is off by 2^-24 relative,
2^-24 for x <= pi / 4; cos and sin are polynomials that are off by 2e-9 and by the
roundings of their last two steps, 2^-23. Together below 2^-22. An output u c - v s
adds its products' and its sum's roundings, 2^-23 of |u| + |v|: below 2^-21 of |u| +
|v|, and half a step (eps / 2) of the value for its type.
"""
import math
from fractions import Fraction

import pytest

pytestmark = pytest.mark.gpu

TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494")


def _reference(x, pos, inv_freq, axes, rotary_dim, interleaved):
    """(y, |u| + |v| of each value) in 64 bits; pos [axes, T], x [T, H, D] on the CPU."""
    import torch
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    half = rotary_dim // 2
    for t in range(x.shape[0]):
        for j in range(half):
            turn = Fraction(inv_freq[j]) * int(pos[axes[j], t]) / TWO_PI
            angle = float((turn - math.floor(turn)) * TWO_PI)
            i0, i1 = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
            u, v = x[t, :, i0].double(), x[t, :, i1].double()
            y[t, :, i0] = u * math.cos(angle) - v * math.sin(angle)
            y[t, :, i1] = v * math.cos(angle) + u * math.sin(angle)
            size[t, :, i0] = size[t, :, i1] = u.abs() + v.abs()
    return y, size


def _check(got, x, pos, op, axes=None, interleaved=False):
    import torch
    axes = list(op._axis) if axes is None else axes
    y, size = _reference(x.cpu(), pos.cpu().reshape(op.axes, -1), op.inv_freq, axes, op.rotary_dim,
                         interleaved)
    info = torch.finfo(x.dtype)
    tol = 2.0 ** -21 * size + info.eps / 2 * y.abs() + info.smallest_normal * info.eps
    assert ((got.cpu().double() - y).abs() <= tol).all()
    kept = got[..., op.rotary_dim:]
    assert torch.equal(kept, x[..., op.rotary_dim:])


def _heads(T, H, D, dtype, device, seed):
    import torch
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return torch.randn(T, H, D, device=device, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,R", [(1, 1, 1, 2, 2), (3, 4, 2, 64, 64), (2, 3, 1, 80, 80),
                                          (5, 8, 2, 128, 128), (2, 2, 1, 100, 66), (2, 5, 5, 40, 16),
                                          (1, 2, 1, 512, 512), (2, 2, 2, 24, 6), (1, 40, 8, 96, 48)])
def test_one_axis(pkg, cuda, T, Hq, Hkv, D, R, interleaved, dtype):
    import torch
    dtype = getattr(torch, dtype)
    op = pkg.Rotary(D, rotary_dim=R, interleaved=interleaved, base=500000.0)
    q, k = _heads(T, Hq, D, dtype, cuda, T + D), _heads(T, Hkv, D, dtype, cuda, T + D + 1)
    pos = torch.tensor([0, 1, 7, 100, 131071][:T], device=cuda)
    Q, K = op(q, k, pos)
    _check(Q, q, pos, op, interleaved=interleaved)
    _check(K, k, pos, op, interleaved=interleaved)
    assert torch.equal(op(q, None, pos), Q)
    assert torch.equal(op(q, k, pos.int())[1], K)


@pytest.mark.parametrize("pos", [2 ** 20 + 1, 2 ** 31 - 1, -5, 2 ** 31, 2 ** 40 + 12345, 2 ** 62,
                                 -2 ** 63])
def test_far_positions(pkg, cuda, pos):
    """No position is too far for the angle: as exact as near ones."""
    import torch
    op = pkg.Rotary(128)
    q = _heads(1, 2, 128, torch.float32, cuda, 3)
    p = torch.tensor([pos], device=cuda)
    # The frequency is rounded to 2^-65 of a turn: seen from here, 2^-65 |pos| turns.
    Q = op(q, None, p)
    y, size = _reference(q.cpu(), p.cpu()[None], op.inv_freq, [0] * 64, 128, False)
    tol = (2.0 ** -21 + 2 * math.pi * 2.0 ** -65 * abs(pos)) * size + 2.0 ** -24 * y.abs()
    assert ((Q.cpu().double() - y).abs() <= tol).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pos", [2 ** 31 - 1, 2 ** 40 + 12345, 2 ** 62, 2 ** 63 - 1, -2 ** 63, -7])
def test_turns_of_far_positions(pkg, cuda, pos, interleaved):
    """The angle is the position times the frequency as the object holds it, in units of 2^-64 of
    a turn, with no rounding: the same tolerance at any position."""
    import torch
    op = pkg.Rotary(128, interleaved=interleaved)
    q = _heads(1, 2, 128, torch.float32, cuda, 18)
    got = op(q, None, torch.tensor([pos], device=cuda)).cpu().double()
    x = q.cpu().double()
    for j in range(64):
        angle = float(Fraction(op._turns[j] * pos % 2 ** 64, 2 ** 64) * TWO_PI)
        i0, i1 = (2 * j, 2 * j + 1) if interleaved else (j, j + 64)
        u, v = x[0, :, i0], x[0, :, i1]
        for i, y in ((i0, u * math.cos(angle) - v * math.sin(angle)),
                     (i1, v * math.cos(angle) + u * math.sin(angle))):
            tol = 2.0 ** -21 * (u.abs() + v.abs()) + 2.0 ** -24 * y.abs()
            assert ((got[0, :, i] - y).abs() <= tol).all(), j


def test_axes_by_sections_and_by_list(pkg, cuda):
    import torch
    T, D = 6, 64
    q, k = _heads(T, 4, D, torch.bfloat16, cuda, 4), _heads(T, 2, D, torch.bfloat16, cuda, 5)
    pos = torch.tensor([[0, 0, 0, 1, 1, 1], [5, 5, 6, 900, 901, 2], [0, 7, 3, 70000, 1, 33]],
                       device=cuda)
    op = pkg.Rotary(D, sections=(8, 12, 12))
    axes = [0] * 8 + [1] * 12 + [2] * 12
    Q, K = op(q, k, pos)
    _check(Q, q, pos, op, axes)
    _check(K, k, pos, op, axes)
    turns = [j % 3 for j in range(32)]
    op = pkg.Rotary(D, axes=turns)
    _check(op(q, k, pos)[0], q, pos, op, turns)
    same = pos[:1].expand(3, T)
    assert torch.equal(op(q, k, same)[0], pkg.Rotary(D)(q, k, pos[0])[0])


@pytest.mark.parametrize("D", [128, 100])
def test_views_in_place_and_shapes(pkg, cuda, D):
    """Views of a QKV projection's rows, batches of sequences, and results in place:
    what lies beside the heads stays as it was."""
    import torch
    T, Hq, Hkv = 6, 3, 2
    op = pkg.Rotary(D, rotary_dim=D // 4 * 2)
    qkv = _heads(T, Hq + 2 * Hkv, D, torch.float16, cuda, 6)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:].clone()
    pos = torch.arange(T, device=cuda) * 11
    want = op(q.contiguous(), k.contiguous(), pos)
    for a, b in zip(op(q, k, pos), want):
        assert torch.equal(a, b)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(op(by_head, k, pos)[0], want[0])
    batched = op(q.contiguous().reshape(2, 3, Hq, D), k.contiguous().reshape(2, 3, Hkv, D),
                 pos.reshape(2, 3))
    assert torch.equal(batched[1].reshape(T, Hkv, D), want[1])
    assert torch.equal(op(q[2], k[2], pos[2])[0], want[0][2])
    odd = torch.zeros(T * Hq * D + 1, dtype=torch.float16, device=cuda)[1:].view(T, Hq, D)
    odd.copy_(q)
    assert torch.equal(op(odd, k, pos)[0], want[0])
    Q, K = op(q, k, pos, out=(q, k))
    assert Q.data_ptr() == qkv.data_ptr()
    assert torch.equal(qkv[:, :Hq], want[0]) and torch.equal(qkv[:, Hq:Hq + Hkv], want[1])
    assert torch.equal(qkv[:, Hq + Hkv:], v)


def test_expanded_tokens(pkg, cuda):
    """One row for several tokens (stride 0, of the inner or the outer axis): read as their
    copies are; a result that would lie on itself is refused."""
    import torch
    D = 64
    op = pkg.Rotary(D)
    q, k = _heads(3, 4, D, torch.bfloat16, cuda, 13), _heads(3, 2, D, torch.bfloat16, cuda, 14)
    for axis, shape in ((1, (3, 2)), (0, (2, 3))):
        pos = torch.arange(6, device=cuda).reshape(shape) * 13
        Q, K = (x.unsqueeze(axis).expand(*shape, *x.shape[1:]) for x in (q, k))
        want = op(Q.contiguous(), K.contiguous(), pos)
        for a, b in zip(op(Q, K, pos), want):
            assert torch.equal(a, b)
        fresh = [torch.empty(shape + x.shape[1:], dtype=x.dtype, device=cuda) for x in (q, k)]
        for a, b in zip(op(Q, K, pos, out=fresh), want):
            assert torch.equal(a, b)
        with pytest.raises(ValueError, match="whole heads"):
            op(Q, K, pos, out=(fresh[0], K))
        with pytest.raises(ValueError, match="whole heads"):
            op(Q, K, pos, out=(Q, fresh[1]))


def test_many_tokens(pkg, cuda):
    """More tokens than a workgroup has, against the same tokens a few at a time."""
    import torch
    op = pkg.Rotary(64, sections=(16, 16))
    q, k = _heads(3001, 2, 64, torch.bfloat16, cuda, 7), _heads(3001, 1, 64, torch.bfloat16, cuda, 8)
    pos = torch.randint(0, 10 ** 6, (2, 3001), device=cuda)
    Q, K = op(q, k, pos)
    for t in (0, 63, 64, 1000, 3000):
        a, b = op(q[t:t + 1], k[t:t + 1], pos[:, t:t + 1])
        assert torch.equal(Q[t:t + 1], a) and torch.equal(K[t:t + 1], b)
    empty = op(q[:0], k[:0], pos[:, :0])
    assert empty[0].shape == (0, 2, 64)


def test_most_tokens(pkg, cuda):
    """As many tokens as a call may have, each with so many heads that a workgroup has only
    one: more workgroups than one launch takes. Against the same tokens a few at a time."""
    import torch
    T, H, D = 2 ** 24, 300, 2
    op = pkg.Rotary(D, sections=(0, 1))
    g = torch.Generator(device=cuda)
    g.manual_seed(15)
    x = torch.empty(T, H, D, dtype=torch.float16, device=cuda)  # 20 GB
    x.view(-1, 4)[:] = torch.randn(4, device=cuda, generator=g).half()
    x[:, :, 0] += (torch.arange(T, device=cuda) % 1009)[:, None].half() / 1024
    pos = torch.randint(0, 10 ** 6, (2, T), dtype=torch.int32, device=cuda, generator=g)
    at = torch.tensor([0, 1, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 1, T - 2, T - 1], device=cuda)
    want = op(x[at], x[at, :1], pos[:, at])
    K = x[:, :1].clone()
    assert op(x, K, pos, out=(x, K))[0] is x
    assert torch.equal(x[at], want[0]) and torch.equal(K[at], want[1])
    del x, K
    torch.cuda.empty_cache()


def test_refusals(pkg, cuda):
    import torch
    op = pkg.Rotary(64, sections=(16, 16))
    q, k = _heads(4, 2, 64, torch.float32, cuda, 9), _heads(4, 1, 64, torch.float32, cuda, 10)
    pos = torch.zeros(2, 4, dtype=torch.int64, device=cuda)
    for args, kwargs, match in (((q[..., :32], k, pos), {}, "Q must be"),
                                ((q, k[:3], pos), {}, "K must be"),
                                ((q, k.half(), pos), {}, "K must be of Q's type"),
                                ((q, k, pos[0]), {}, "positions must be"),
                                ((q, k, pos.float()), {}, "positions must be"),
                                ((q, k, pos.cpu()), {}, "positions must be"),
                                ((q, k, pos), {"out": (q,)}, "out must be 2"),
                                ((q, k, pos), {"out": (q, k.half())}, "out must have K's"),
                                ((q, k, pos), {"out": (q, k[:, :, :1].expand(4, 1, 64))}, "whole")):
        with pytest.raises(ValueError, match=match):
            op(*args, **kwargs)


def test_stream_and_graph(pkg, cuda):
    import torch
    op = pkg.Rotary(128)
    q, k = _heads(9, 4, 128, torch.bfloat16, cuda, 11), _heads(9, 2, 128, torch.bfloat16, cuda, 12)
    pos = torch.arange(9, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = op(q, k, pos, stream=side)
    side.synchronize()
    assert torch.equal(got[0], op(q, k, pos)[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op(q, k, pos)
    for n in range(3):
        pos += 1000 * n + 1
        graph.replay()
        torch.cuda.synchronize()
        want = op(q, k, pos)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_no_gradient(pkg, cuda):
    """Q and K that require a gradient are turned all the same; backward() says that there is
    none, and their own memory is not written behind the graph's back."""
    import torch
    op = pkg.Rotary(64)
    q, k = _heads(5, 4, 64, torch.float32, cuda, 16), _heads(5, 2, 64, torch.float32, cuda, 17)
    pos = torch.arange(5, device=cuda)
    want = op(q, k, pos)
    for leaf in (q, k):
        leaf.requires_grad_()
        got = op(q, k, pos)
        assert all(torch.equal(a, b) and a.requires_grad for a, b in zip(got, want))
        for y in got:
            with pytest.raises(RuntimeError, match="no gradient"):
                y.sum().backward(retain_graph=True)
        with pytest.raises(ValueError, match="must not require a gradient"):
            op(q, k, pos, out=(torch.empty_like(q), torch.empty_like(k)))
        with torch.no_grad():
            assert not op(q, k, pos)[0].requires_grad
        leaf.requires_grad_(False)
    q.requires_grad_()
    alone = op(q, None, pos)
    assert torch.equal(alone, want[0])
    with pytest.raises(RuntimeError, match="no gradient"):
        alone.sum().backward()
    with torch.no_grad():
        op(q, k, pos, out=(q, k))
    assert torch.equal(q, want[0])
