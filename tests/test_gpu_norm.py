"""The RMS norm on the GPU, against its definition in 64 bits.

Tolerances, fixed before the first run. A thread adds up the squares of at most 8 n
values, n the units that it holds (4, or K / 8192 of a longer row), then a tree of 6
and a sum of 16 add to them: with half a unit (2^-24) lost in each of these and in
each square, the sum is off by (8 n + 23) 2^-24 relative, its root by half of that,
and division, root, reciprocal and two products add 2^-24 (2^-23 for the root
and the reciprocal) each. With n <= 6 here that is below 2^-18 of y. The output's
rounding is half a step (eps / 2) of the value more. A code stands for y within
2^-4 of it or, below e4m3's normal values, half its least step, 2^-10, of the scale.
"""
import pytest

pytestmark = pytest.mark.gpu

FP32 = 2.0 ** -18


def _problem(M, K, dtype, device, seed=0):
    import torch
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    x, r = (torch.randn(M, K, device=device, generator=g)
            * torch.exp(torch.randn(M, 1, device=device, generator=g)) for _ in range(2))
    gamma = 1.0 + 0.3 * torch.randn(K, device=device, generator=g)
    return x.to(dtype), r.to(dtype), gamma


def _norm64(h, gamma, eps):
    import torch
    h = h.double()
    return h / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + eps) * gamma.double()


def _check_codes(codes, scales, y):
    """Codes and scales [M, nb] against y [M, K] in 64 bits."""
    import torch
    M, K = y.shape
    nb = -(-K // 128)
    pad = torch.nn.functional.pad(y, (0, nb * 128 - K)).reshape(M, nb, 128)
    want = pad.abs().amax(dim=-1).clamp(min=2.0 ** -100) / 448.0
    assert codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32
    assert ((scales.double() - want).abs() <= (FP32 + 2.0 ** -23) * want).all()
    s = scales.double().repeat_interleave(128, dim=1)[:, :K]
    got = codes.float().double() * s
    tol = (2.0 ** -4 + 2 * FP32) * y.abs() + (2.0 ** -10 + 2 * FP32) * s
    assert ((got - y).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 8), (2, 7), (3, 127), (5, 128), (2, 129), (3, 1000),
                                 (4, 1001), (1, 4096), (600, 512), (530, 2048), (520, 4104),
                                 (7, 8192), (2, 16392), (3, 32768), (2, 32776), (1, 40001)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(pkg, cuda, M, K, dtype, residual):
    import torch
    dtype = getattr(torch, dtype)
    x, r, gamma = _problem(M, K, dtype, cuda, M + K)
    r = r if residual else None
    h = x if r is None else (x.float() + r.float()).to(dtype)
    y = _norm64(h, gamma, 1e-5)
    Y = pkg.rms_norm(x, gamma, 1e-5, residual=r)
    C = pkg.rms_norm_fp8(x, gamma, 1e-5, residual=r)
    if residual:
        Y, H = Y
        assert torch.equal(H, h) and torch.equal(C[2], h)
    assert Y.dtype == dtype
    info = torch.finfo(dtype)
    tol = (info.eps / 2 + FP32) * y.abs() + info.smallest_normal * info.eps
    assert ((Y.double() - y).abs() <= tol).all()
    _check_codes(C[0], C[1], y)


@pytest.mark.parametrize("K", [512, 513])
def test_strided_rows(pkg, cuda, K):
    """Rows of a wider tensor, on any side; the values beside them do not count."""
    import torch
    x, r, gamma = _problem(9, K, torch.bfloat16, cuda, 3)
    wide, wide_r = (torch.full((9, K + 24), float("nan"), dtype=torch.bfloat16, device=cuda)
                    for _ in range(2))
    wide[:, 8:8 + K] = x
    wide_r[:, 16:16 + K] = r
    want = pkg.rms_norm_fp8(x, gamma, residual=r)
    got = pkg.rms_norm_fp8(wide[:, 8:8 + K], gamma, residual=wide_r[:, 16:16 + K])
    for a, b in zip(got, want):
        assert torch.equal(a.float(), b.float())
    shaped = pkg.rms_norm(x.reshape(3, 3, K).transpose(0, 1), gamma)
    assert torch.equal(shaped, pkg.rms_norm(x, gamma).reshape(3, 3, K).transpose(0, 1))


def test_special_rows(pkg, cuda):
    """Zeros give zeros, an infinity or a NaN spoils its own row alone."""
    import torch
    x, _, gamma = _problem(6, 384, torch.float32, cuda, 4)
    x[1] = 0.0
    x[2, 5] = float("inf")
    x[3, 200] = float("nan")
    Y = pkg.rms_norm(x, gamma)
    codes, scales = pkg.rms_norm_fp8(x, gamma)
    assert (Y[1] == 0).all() and (codes[1].float() == 0).all()
    # 1 / sqrt(inf) = 0: the infinity becomes NaN, its row's other values 0
    assert Y[2, 5].isnan() and Y[3].isnan().all() and codes[3].float().isnan().all()
    assert (scales[2] * codes[2].float().reshape(3, 128)[:, 5])[0].isnan()
    good = [0, 4, 5]
    y = _norm64(x[good], gamma, 1e-5)
    assert ((Y[good].double() - y).abs() <= (2.0 ** -24 + FP32) * y.abs()).all()
    _check_codes(codes[good], scales[good], y)


def test_epsilon_and_empty(pkg, cuda):
    import torch
    x, r, gamma = _problem(2, 64, torch.float32, cuda, 5)
    y = _norm64(x * 1e-3, gamma, 0.25)
    Y = pkg.rms_norm(x * 1e-3, gamma, 0.25)
    assert ((Y.double() - y).abs() <= 2 * FP32 * y.abs()).all()
    assert pkg.rms_norm(x[:0], gamma).shape == (0, 64)
    codes, scales, h = pkg.rms_norm_fp8(x[:0], gamma, residual=r[:0])
    assert codes.shape == (0, 64) and scales.shape == (0, 1) and h.shape == (0, 64)


def test_refusals(pkg, cuda):
    import torch
    x, r, gamma = _problem(2, 64, torch.float32, cuda, 6)
    for args, kwargs, match in (((x, gamma.half()), {}, "gamma"), ((x, gamma[:63]), {}, "gamma"),
                                ((x, gamma.cpu()), {}, "gamma"), ((x, gamma, -1.0), {}, "epsilon"),
                                ((x, gamma, float("nan")), {}, "epsilon"),
                                ((x, gamma), {"residual": r.half()}, "residual"),
                                ((x, gamma), {"residual": r[:1]}, "residual"),
                                ((x[:, :0], gamma), {}, "K >= 1")):
        for f in (pkg.rms_norm, pkg.rms_norm_fp8):
            with pytest.raises(ValueError, match=match):
                f(*args, **kwargs)


def test_stream_and_graph(pkg, cuda):
    """On another stream, and captured: replays read the inputs of their time."""
    import torch
    x, r, gamma = _problem(33, 1024, torch.bfloat16, cuda, 7)
    want = pkg.rms_norm_fp8(x, gamma, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = pkg.rms_norm_fp8(x, gamma, residual=r, stream=side)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.float(), b.float())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.rms_norm_fp8(x, gamma, residual=r)
    for k in range(3):
        x.copy_(_problem(33, 1024, torch.bfloat16, cuda, 20 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, pkg.rms_norm_fp8(x, gamma, residual=r)):
            assert torch.equal(a.float(), b.float())


def test_norm_of_a_projection(pkg, cuda):
    """MatMulFp8.run_rmsnorm is the norm and the product, and returns the sum."""
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(8)
    K, N = 512, 384
    W = (torch.randn(N, K, device=cuda, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(3, 4, device=cuda, generator=g) + 0.5
    op = pkg.MatMulFp8(K, N).prepare_device(W, s)
    x, r, gamma = _problem(17, K, torch.bfloat16, cuda, 9)
    codes, scales, h = pkg.rms_norm_fp8(x, gamma, residual=r)
    Y, H = op.run_rmsnorm(x, gamma, residual=r)
    assert torch.equal(H, h)
    assert torch.equal(Y, op(codes, scales=scales, out_dtype=torch.bfloat16))
    Y = op.run_rmsnorm(x.reshape(17, 1, K), gamma, out_dtype=torch.float32)
    codes, scales = pkg.rms_norm_fp8(x, gamma)
    assert torch.equal(Y.reshape(17, N), op(codes, scales=scales))


@pytest.mark.parametrize("which", ["x", "gamma", "residual"])
def test_no_gradient(pkg, cuda, which):
    """What requires a gradient is taken, with the same results; backward() says that there is
    none, and nothing is recorded where none is wanted."""
    import torch
    x, r, gamma = _problem(3, 256, torch.float32, cuda, 10)
    W = torch.ones(128, 256, device=cuda).to(torch.float8_e4m3fn)
    op = pkg.MatMulFp8(256, 128).prepare_device(W, torch.ones(1, 2, device=cuda))
    calls = (lambda: pkg.rms_norm(x, gamma, residual=r), lambda: op.run_rmsnorm(x, gamma, residual=r),
             lambda: pkg.rms_norm_fp8(x, gamma, residual=r)[1:],
             lambda: (pkg.rms_norm(x, gamma, residual=r, stream=torch.cuda.current_stream())[0],))
    want = [call() for call in calls]
    {"x": x, "gamma": gamma, "residual": r}[which].requires_grad_()
    for call, ys in zip(calls, want):
        got = call()
        assert len(got) == len(ys) and all(torch.equal(a, b) for a, b in zip(got, ys))
        for y in got:
            assert y.requires_grad
            with pytest.raises(RuntimeError, match="no gradient"):
                (y * 2.0).sum().backward(retain_graph=True)
        with torch.no_grad():
            assert not any(y.requires_grad for y in call())
    if which != "residual":
        y = pkg.rms_norm(x, gamma)
        y += 1.0  # a result may be changed in place
        with pytest.raises(RuntimeError, match="no gradient"):
            y.sum().backward()
    assert x.grad is None and gamma.grad is None


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("M,K", [(1, 4096), (4096, 2048), (600, 5000), (64, 40001)])
def test_codes_are_the_nearest(pkg, cuda, M, K, dtype):
    """Every code is the one nearest to 448 y / amax as 64 bits have it, unless that lies
    within 2^-45 of the middle of two: 64 bits themselves do not decide there. (The row's own
    factor is y's and amax's, and drops out.)"""
    import torch
    x, r, gamma = _problem(M, K, getattr(torch, dtype), cuda, 11)
    codes, _, h = pkg.rms_norm_fp8(x, gamma, residual=r)
    nb = -(-K // 128)
    u = torch.nn.functional.pad(h.double() * gamma.double(), (0, nb * 128 - K)).reshape(M, nb, 128)
    q = 448.0 * u / u.abs().amax(dim=-1, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -7))).clamp(min=-6.0) - 3.0)
    got = torch.nn.functional.pad(codes.float(), (0, nb * 128 - K)).reshape(M, nb, 128).double()
    assert ((got - q).abs() <= step / 2 + 2.0 ** -45 * q.abs()).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("K", [128, 512, 4096, 9999, 32776])
def test_factor_of_a_row(pkg, cuda, K, dtype):
    """Rows of powers of two, whose squares and their sums (below 2^24) are exact: a value of 1 is
    the row's factor, rounded once, half a unit, 2^-24; a scale is four times it over 448, rounded
    again. Of 16-bit results half a step more."""
    import torch
    dtype = getattr(torch, dtype)
    g = torch.Generator(device=cuda)
    g.manual_seed(13)
    share = torch.rand(700, 1, device=cuda, generator=g)  # another mean for each row
    x = torch.where(torch.rand(700, K, device=cuda, generator=g) < share, 1.0, 2.0)
    x[:, ::128] = -4.0
    ones = torch.ones(K, device=cuda)
    norm = torch.rsqrt((x.double() ** 2).mean(dim=1, keepdim=True) + 2.0 ** -16)
    Y = pkg.rms_norm(x.to(dtype), ones, 2.0 ** -16).double()
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -24)
    want = x.double() * norm
    assert ((Y - want).abs() <= (2.0 ** -24 + half) * want.abs()).all()
    _, scales = pkg.rms_norm_fp8(x.to(dtype), ones, 2.0 ** -16)
    want = 4.0 * norm / 448.0
    assert ((scales.double() - want).abs() <= (2.0 ** -23 + 2.0 ** -48) * want).all()
