"""The mixture-of-experts layer on the GPU, against its definition in 64 bits.

Tolerances, fixed before the first run. Activations enter the products rounded
to 2^-22 (fp32) or 2^-14 (16-bit types) of the largest magnitude of their block
of 128, at most half a step of 2^(e - 21) or 2^(e - 13) with 2^e <= that
magnitude. A product's sum is then off by at most u times the sum over its
blocks of (largest |x|) (sum of |w|), u that 2^-22 or 2^-14, plus fp32's
rounding of two scalings and one addition per weight block, (folds + 4) 2^-24 of
the sum of magnitudes, which the same sum bounds. _layer64 carries these bounds
through the layer: through silu (slope at most 1.1), the product with up, the
second rounding, down, and the weighted sum; the choice's weights are off by at
most 2^-19 (fp32 exp, one ulp, and a sum of at most E terms). The output's own
rounding is at most half a step of it. (16-bit types are rounded to 2^-22 too:
test_outliers_leave_the_other_values holds them to that.)
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -22, "float16": 2.0 ** -14, "bfloat16": 2.0 ** -14}


def _weight(E, N, K, bs, zp, gen, device):
    import torch
    nb = -(-K // bs)
    B = torch.randint(0, 256, (E, N, nb, bs // 2), dtype=torch.uint8, device=device, generator=gen)
    S = (torch.rand((E, N, nb), device=device, generator=gen) + 0.5) * (0.2 / K ** 0.5)
    Z = torch.randint(0, 256, (E, N, (nb + 1) // 2), dtype=torch.uint8, device=device,
                      generator=gen) if zp else None
    return B, S, Z


def _dense(W, K):
    """W [E, N, K] in 64 bits."""
    import torch
    B, S, Z = W
    q = torch.stack((B & 15, B >> 4), dim=-1).flatten(-2).double()      # [E, N, nb, bs]
    z = 8.0
    if Z is not None:
        z = torch.stack((Z & 15, Z >> 4), dim=-1).flatten(-2)[..., :S.shape[-1], None].double()
    return ((q - z) * S[..., None].double()).flatten(-2)[..., :K].contiguous()


def _problem(T, H, I, E, bs, zp, dtype, seed, device):
    import torch
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    x = torch.randn(T, H, device=device, generator=g).to(getattr(torch, dtype))
    router = torch.randn(E, H, device=device, generator=g) * (1.5 / H ** 0.5)
    return x, router, [_weight(E, n, k, bs, zp, g, device) for n, k in ((I, H), (I, H), (H, I))]


def _choice(logits, k, normalize):
    """(ids, weights) in 64 bits from fp32 logits, ties to the lowest index."""
    import torch
    l = torch.where(logits.isnan(), torch.full_like(logits, -np.inf), logits)
    ids = torch.argsort(l, dim=-1, descending=True, stable=True)[:, :k]
    p = torch.softmax(l.double(), dim=-1).gather(1, ids)
    return ids, p / p.sum(dim=-1, keepdim=True) if normalize else p


def _blocks(x):
    """Largest magnitude of each value's block of 128, spread over the block."""
    import torch
    n = x.shape[-1]
    pad = torch.nn.functional.pad(x.abs(), (0, -n % 128)).reshape(x.shape[0], -1, 128)
    return pad.amax(-1, keepdim=True).expand(pad.shape).reshape(x.shape[0], -1)[:, :n].contiguous()


def _layer64(x, ids, p, dense, bs, u):
    """(Y, bound on its error) in 64 bits."""
    import torch
    Wg, Wu, Wd = dense
    x = x.double()
    y, err = torch.zeros_like(x), torch.zeros_like(x)

    def product(v, ve, W):
        """v W^T and its bound, v off by at most ve."""
        Wt = W.t().contiguous()
        top = _blocks(v.abs() + ve)
        round_off = u + (-(-v.shape[1] // bs) + 4) * 2.0 ** -24
        return v @ Wt, (ve + round_off * top) @ Wt.abs()

    for e in sorted(set(ids.flatten().tolist())):
        t, s = torch.nonzero(ids == e, as_tuple=True)
        zero = torch.zeros_like(x[t])
        g, ge = product(x[t], zero, Wg[e])
        v, ve = product(x[t], zero, Wu[e])
        silu = g * torch.sigmoid(g)
        se = 1.1 * ge + 2.0 ** -20 * (silu.abs() + 1.1 * ge)
        h, he = silu * v, se * (v.abs() + ve) + silu.abs() * ve
        d, de = product(h, he + 2.0 ** -23 * (h.abs() + he), Wd[e])
        w = p[t, s][:, None]
        y[t] += w * d
        err[t] += w * de + w * 2.0 ** -18 * (d.abs() + de)
    return y, err


def _check(Y, ref, err):
    import torch
    info = torch.finfo(Y.dtype)
    tol = err * (1 + info.eps) + info.eps / 2 * ref.abs() + info.tiny * info.eps / 2
    off = (Y.double() - ref).abs()
    bad = torch.nonzero(~(off <= tol))
    assert bad.numel() == 0, (bad[:4].tolist(), float((off / tol).max()))
    return float((off / tol).max())


SHAPES = [
    # T, H, I, E, k, bs, zp, dtype, normalize
    (1, 128, 128, 4, 2, 128, True, "float32", True),
    (1, 2048, 768, 64, 6, 128, True, "bfloat16", True),
    (1, 1, 1, 1, 1, 16, True, "float32", True),
    (2, 17, 129, 3, 3, 16, True, "float32", False),
    (3, 130, 16, 5, 1, 32, False, "float16", True),
    (4, 1024, 512, 8, 2, 16, False, "bfloat16", True),
    (5, 700, 333, 10, 4, 32, True, "float32", True),
    (6, 256, 384, 8, 8, 64, True, "float32", False),
    (7, 1500, 701, 10, 3, 16, True, "float32", False),
    (8, 512, 256, 160, 8, 64, False, "float16", False),
    (9, 384, 640, 4, 1, 256, True, "bfloat16", True),
    (16, 1024, 512, 128, 8, 32, True, "bfloat16", True),
    (17, 640, 200, 6, 2, 128, False, "float32", True),
    (33, 512, 300, 1024, 32, 64, True, "bfloat16", True),
    (40, 256, 128, 2, 2, 512, True, "float32", True),
    (64, 896, 1000, 8, 2, 128, False, "float16", True),
    (64, 300, 260, 1, 1, 16, True, "float32", False),
    (65, 256, 256, 12, 4, 32, True, "bfloat16", True),
    (150, 200, 140, 5, 2, 16, False, "float32", True),
    # one token: of more experts than a workgroup chooses from, 32 of 256, on wide
    # experts (down in parts), with few blocks and with many
    (1, 260, 200, 300, 4, 16, True, "bfloat16", False),
    (1, 128, 64, 256, 32, 64, False, "float32", False),
    (1, 256, 8200, 9, 8, 32, True, "float32", True),
    (1, 300, 8200, 9, 8, 16, False, "bfloat16", True),
    (1, 512, 2200, 9, 8, 16, True, "float16", True),
    (1, 33, 2200, 12, 8, 256, False, "float32", True),
    # the last number of tokens whose sums stay in down's workgroups, and the next
    (8, 512, 2200, 9, 3, 16, True, "bfloat16", True),
    (8, 130, 700, 32, 32, 32, True, "float32", True),
    (8, 256, 4400, 24, 8, 64, False, "float32", True),
    (9, 512, 2200, 9, 3, 16, False, "float32", True),
    # several tokens on either side of narrow workgroups
    (4, 300, 1000, 64, 4, 128, True, "bfloat16", True),
    (2, 640, 2000, 16, 2, 32, False, "float32", True),
    (8, 200, 120, 100, 12, 16, True, "float32", False),
    (8, 200, 120, 100, 11, 64, True, "bfloat16", True),
    # two and four column groups with every width of block
    (64, 200, 260, 4, 2, 16, True, "bfloat16", True),
    (64, 200, 260, 4, 2, 32, False, "bfloat16", True),
    (64, 300, 130, 4, 2, 64, True, "float32", False),
    (64, 130, 300, 3, 3, 128, True, "float32", True),
    (48, 700, 200, 16, 4, 32, True, "bfloat16", True),
    (24, 700, 333, 8, 2, 64, False, "float32", True),
    (30, 256, 128, 16, 2, 16, True, "float32", True),
]


@pytest.mark.parametrize("T,H,I,E,k,bs,zp,dtype,normalize", SHAPES)
def test_layer(pkg, cuda, T, H, I, E, k, bs, zp, dtype, normalize):
    import torch
    x, router, ws = _problem(T, H, I, E, bs, zp, dtype, T + H + I + E, cuda)
    op = pkg.MatMulNBitsMoE(H, I, E, k, block_size=bs, normalize=normalize)
    op.prepare_device(router, *ws)
    print(f"case moe T={T} H={H} I={I} E={E} k={k} bs={bs} zp={zp} {dtype}", flush=True)
    y, ids, p = op(x, routing=True)
    logits = (x.double() @ router.double().t().contiguous()).float()
    want_ids, want_p = _choice(logits, k, normalize)
    assert ids.dtype == torch.int32 and torch.equal(ids.long(), want_ids)
    assert bool(((p.double() - want_p).abs() <= 2.0 ** -19 * want_p).all())
    ref, err = _layer64(x, want_ids, want_p, [_dense(w, n) for w, n in zip(ws, (H, H, I))], bs,
                        U[dtype])
    print(f"  worst / bound {_check(y, ref, err):.3f}", flush=True)
    assert torch.equal(y, op(x))                    # no order changes it
    assert torch.equal(y, op(x, logits=logits))


def test_given_logits_ties_and_order(pkg, cuda):
    """Equal logits go to the lowest expert, -0 equals 0, infinities and NaN have
    their place, and a layer without a router needs logits."""
    import torch
    T, H, I, E, k = 6, 128, 128, 9, 4
    x, _, ws = _problem(T, H, I, E, 32, True, "float32", 1, cuda)
    op = pkg.MatMulNBitsMoE(H, I, E, k, block_size=32).prepare_device(None, *ws)
    with pytest.raises(ValueError, match="needs logits"):
        op(x)
    inf, nan = float("inf"), float("nan")
    logits = torch.zeros(T, E, device=cuda)
    logits[1] = torch.tensor([0.0, -0.0, 1, 1, -1, 1, 0, 2, 2])
    logits[2, :] = -0.0
    logits[2, 5] = 0.0
    logits[3] = torch.tensor([nan, 1, nan, -inf, 3, nan, 2, -inf, -5])
    logits[4, :] = -1e30
    logits[4, 8] = 1e30
    logits[5] = torch.arange(E).flip(0)
    y, ids, p = op(x, logits=logits, routing=True)
    print("case moe ties", flush=True)
    assert ids.tolist() == [[0, 1, 2, 3], [7, 8, 2, 3], [0, 1, 2, 3], [4, 6, 1, 8], [8, 0, 1, 2],
                            [0, 1, 2, 3]]
    want_ids, want_p = _choice(logits, k, True)
    assert bool(((p.double() - want_p).abs() <= 2.0 ** -19 * want_p + 2.0 ** -149).all())
    ref, err = _layer64(x, want_ids, want_p, [_dense(w, n) for w, n in zip(ws, (H, H, I))], 32,
                        U["float32"])
    _check(y, ref, err)
    logits[0, :] = nan                 # nothing to choose by: the first experts, no weights
    y2, ids2, p2 = op(x, logits=logits, routing=True)
    assert ids2[0].tolist() == [0, 1, 2, 3] and bool(p2[0].isnan().all())
    assert bool(y2[0].isnan().all()) and torch.equal(y2[1:], y[1:])


def test_every_token_on_one_expert(pkg, cuda):
    """The longest list an expert can have, and all others empty."""
    import torch
    for dtype in ("float32", "bfloat16"):
        T, H, I, E = 64, 256, 200, 7
        x, _, ws = _problem(T, H, I, E, 64, True, dtype, 5, cuda)
        op = pkg.MatMulNBitsMoE(H, I, E, 1, block_size=64).prepare_device(None, *ws)
        logits = torch.zeros(T, E, device=cuda)
        logits[:, 4] = 1
        y, ids, p = op(x, logits=logits, routing=True)
        print("case moe one expert", dtype, flush=True)
        assert bool((ids == 4).all()) and bool((p == 1).all())
        ref, err = _layer64(x, ids.long(), p.double(),
                            [_dense(w, n) for w, n in zip(ws, (H, H, I))], 64, U[dtype])
        _check(y, ref, err)


def test_workspace_serves_every_launch_of_a_run(pkg, cuda):
    """39 tokens of this layer need more than 64 (down in more parts), and a run of
    103 ends with them."""
    import torch
    H, I, E = 3328, 2048, 16
    x, router, ws = _problem(103, H, I, E, 128, False, "bfloat16", 43, cuda)
    op = pkg.MatMulNBitsMoE(H, I, E, 1, block_size=128).prepare_device(router, *ws)
    for dtype in (torch.bfloat16, torch.float32):
        needs = [op.workspace_bytes(T, dtype) for T in range(130)]
        assert needs == sorted(needs) and needs[0] == 0 and len(set(needs[64:])) == 1
    print("case moe 64 + 39 tokens", flush=True)
    y = op(x)
    assert torch.equal(y[:64], op(x[:64])) and torch.equal(y[64:], op(x[64:]))


def test_nonfinite_tokens_stay_alone(pkg, cuda):
    import torch
    for T in (3, 40):
        x, router, ws = _problem(T, 300, 140, 6, 32, True, "float32", 9, cuda)
        op = pkg.MatMulNBitsMoE(300, 140, 6, 2, block_size=32).prepare_device(None, *ws)
        logits = torch.randn(T, 6, device=cuda)
        clean = op(x, logits=logits)
        for bad in (float("inf"), -float("inf"), float("nan")):
            dirty = x.clone()
            dirty[1, 299] = bad
            y = op(dirty, logits=logits)
            assert bool(y[1].isnan().all())
            keep = [t for t in range(T) if t != 1]
            assert torch.equal(y[keep], clean[keep])


def test_large_and_small_tokens(pkg, cuda):
    """Each token has scales of its own: powers of two between tokens change
    nothing but the power, and a zero token gives zeros."""
    import torch
    x, _, ws = _problem(6, 256, 128, 4, 128, True, "float32", 3, cuda)
    op = pkg.MatMulNBitsMoE(256, 128, 4, 2, block_size=128).prepare_device(None, *ws)
    logits = torch.randn(6, 4, device=cuda)
    x[2] = 0
    x[3] *= 2.0 ** -60
    x[4] *= 2.0 ** 20
    y, ids, p = op(x, logits=logits, routing=True)
    assert bool((y[2] == 0).all())
    ref, err = _layer64(x, ids.long(), p.double(),
                        [_dense(w, n) for w, n in zip(ws, (256, 256, 128))], 128, U["float32"])
    # below 2^-90 the fixed point stands still: the tiny token's expert rows
    # (about 2^-120) count as zero, within the output's least normal
    off = (y.double() - ref).abs()
    assert bool((off <= err + 2.0 ** -24 * ref.abs() + 2.0 ** -100).all())


def test_host_and_device_plans_agree(pkg, cuda):
    import torch
    for zp in (True, False):
        x, router, ws = _problem(5, 200, 90, 4, 32, zp, "float32", 13, cuda)
        dev = pkg.MatMulNBitsMoE(200, 90, 4, 2, block_size=32).prepare_device(router, *ws)
        host = pkg.MatMulNBitsMoE(200, 90, 4, 2, block_size=32).prepare(
            router.cpu().numpy(),
            *(tuple(None if a is None else a.cpu().numpy() for a in w) for w in ws))
        want = dev(x)
        for a in [router] + [a for w in ws for a in w if a is not None]:
            a.zero_()  # the plan keeps copies
        assert torch.equal(dev(x), want) and torch.equal(host(x), want)
        assert dev.device_bytes() == host.device_bytes()


def test_strides_batches_and_out(pkg, cuda):
    import torch
    x, router, ws = _problem(12, 128, 128, 4, 32, True, "bfloat16", 15, cuda)
    op = pkg.MatMulNBitsMoE(128, 128, 4, 2, block_size=32).prepare_device(router, *ws)
    y, ids, p = op(x, routing=True)
    y3, ids3, p3 = op(x.reshape(3, 4, 128), routing=True)
    assert y3.shape == (3, 4, 128) and ids3.shape == p3.shape == (3, 4, 2)
    assert torch.equal(y3.reshape(12, 128), y) and torch.equal(ids3.reshape(12, 2), ids)
    assert torch.equal(op(x.t().contiguous().t()), y)
    odd = torch.zeros(12 * 128 + 1, dtype=x.dtype, device=cuda)[1:].view(12, 128)
    odd.copy_(x)
    assert torch.equal(op(odd), y)
    buf = torch.full((14, 128), 7.0, dtype=x.dtype, device=cuda)
    assert op(x, out=buf[:12]).data_ptr() == buf.data_ptr()
    assert torch.equal(buf[:12], y) and bool((buf[12:] == 7).all())
    e = op(x[:0], routing=True)
    assert [tuple(t.shape) for t in e] == [(0, 128), (0, 2), (0, 2)]


def test_refusals(pkg, cuda):
    import torch
    x, router, ws = _problem(4, 64, 32, 4, 32, False, "float32", 17, cuda)
    op = pkg.MatMulNBitsMoE(64, 32, 4, 2).prepare_device(router, *ws)
    for call, match in (
            (lambda: op(x.double()), "X must be a float32"),
            (lambda: op(x.cpu()), "X must be a float32"),
            (lambda: op(x[:, :32]), r"X must be \[..., 64\]"),
            (lambda: op(x, logits=torch.zeros(4, 5, device=cuda)), "logits must be"),
            (lambda: op(x, logits=torch.zeros(4, 4, device=cuda).half()), "logits must be"),
            (lambda: op(x, out=torch.empty(4, 64, device=cuda).half()), "out must be"),
            (lambda: op(x, out=torch.empty(64, 4, device=cuda).t()), "out must be")):
        with pytest.raises(ValueError, match=match):
            call()
    L = pkg.moe._library()
    P = lambda t, o=0: ctypes.c_void_p(t.data_ptr() + o)
    need = op.workspace_bytes(4, torch.float32)
    work, y = torch.empty(need, dtype=torch.uint8, device=cuda), torch.empty_like(x)
    run = lambda *a: L.mnb_moe_run(op._plan, *a, None)
    assert run(4, 2, P(x), None, P(y), None, None, P(work), need) == 3
    assert run(-1, 1, P(x), None, P(y), None, None, P(work), need) == 2
    assert run((1 << 24) + 1, 1, P(x), None, P(y), None, None, P(work), need) == 2
    assert run(4, 1, None, None, P(y), None, None, P(work), need) == 1
    assert run(4, 1, P(x), None, None, None, None, P(work), need) == 1
    assert run(4, 1, P(x, 2), None, P(y), None, None, P(work), need) == 2
    assert run(4, 1, P(x), None, P(y), P(work, 2), None, P(work), need) == 2
    assert run(4, 1, P(x), None, P(y), None, None, P(work), need - 1) == 5
    assert run(4, 1, P(x), None, P(y), None, None, None, 0) == 5
    assert run(0, 1, None, None, None, None, None, None, 0) == 0


def test_streams_and_graph(pkg, cuda):
    """One object's calls on several streams, and captured ones replayed between
    eager calls: every result equals the serial one."""
    import torch
    x, router, ws = _problem(64, 512, 256, 16, 32, True, "bfloat16", 21, cuda)
    op = pkg.MatMulNBitsMoE(512, 256, 16, 4, block_size=32).prepare_device(router, *ws)
    xs = [x[:1], x[1:8], x[8:40], x]
    want = [op(v, routing=True) for v in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = [op(v, routing=True, stream=s) for v, s in zip(xs, streams)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs = []
    for v in (x[:3].clone(), x[3:40].clone()):  # two graphs of one object
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = op(v, routing=True)
        graphs.append((g, v, out))
    for scale in (1.0, -1.0, 0.5):
        for g, v, out in graphs:
            v.copy_(x[:v.shape[0]] * scale)
            g.replay()
        for g, v, out in graphs:
            eager = op(v, routing=True)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, eager))


def test_decoder_half_layer(pkg, orc, cuda):
    """The operators as a model runs them: rows through an 8-bit projection, the
    residual, and the expert layer on the sum; against the same in 64 bits, each
    operator fed what the one before gave."""
    import torch
    T, H, I, E, k = 9, 512, 384, 8, 2
    g = torch.Generator(device=cuda)
    g.manual_seed(31)
    x = torch.randn(T, H, device=cuda, generator=g)
    W = (torch.randn(H, H, device=cuda, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    sw = (torch.rand(4, 4, device=cuda, generator=g) + 0.5) * (0.01 / H ** 0.5)
    _, router, ws = _problem(1, H, I, E, 128, True, "float32", 33, cuda)
    proj = pkg.MatMulFp8(H, H).prepare_device(W, sw)
    moe = pkg.MatMulNBitsMoE(H, I, E, k, block_size=128).prepare_device(router, *ws)
    codes, scales = pkg.quantize_fp8(x)
    o = proj(x)
    hidden = x + o
    y, ids, p = moe(hidden, routing=True)
    a = codes.double() * scales.double().repeat_interleave(128, 1)
    w = W.double() * sw.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    ref = a @ w.t().contiguous()
    bound = (132 + 4) * 2.0 ** -23 * (a.abs() @ w.abs().t().contiguous()) + 2.0 ** -24 * ref.abs()
    assert bool(((o.double() - ref).abs() <= bound).all())
    logits = (hidden.double() @ router.double().t().contiguous()).float()
    want_ids, want_p = _choice(logits, k, True)
    assert torch.equal(ids.long(), want_ids)
    ref, err = _layer64(hidden, want_ids, want_p,
                        [_dense(v, n) for v, n in zip(ws, (H, H, I))], 128, U["float32"])
    _check(y, ref, err)


def test_threads(pkg, cuda):
    """Calls of four threads on one stream, each with a workspace of its own."""
    import threading
    import torch
    x, router, ws = _problem(70, 256, 300, 12, 32, True, "float16", 37, cuda)
    op = pkg.MatMulNBitsMoE(256, 300, 12, 3, block_size=32).prepare_device(router, *ws)
    xs = [x[:1], x[1:9], x[9:40], x]
    want = [op(v) for v in xs]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        got[i] = [op(xs[i]) for _ in range(8)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for ys, w in zip(got, want):
        assert all(torch.equal(y, w) for y in ys)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,H,I,E,bs,zp", [
    (1, 256, 128, 4, 32, True), (1, 512, 4224, 8, 128, False), (4, 256, 128, 4, 16, False),
    (8, 384, 200, 4, 128, True), (9, 384, 200, 8, 64, True), (30, 256, 128, 4, 32, False),
    (64, 256, 300, 4, 256, True)])
def test_outliers_leave_the_other_values(pkg, cuda, T, H, I, E, bs, zp, dtype):
    """Every 128th activation is 2^12, every 128th channel of the experts 2^12 times as
    large, and their weights are zero: the result is that of the other values.

    Beside 2^12 the fixed point's step is 2^-9. The other activations are multiples of
    2^-6 below 2: exact. Their products are off by the fp32 scalings and additions
    alone, (blocks + 4) 2^-24 of the digits' magnitudes: a value's digits add up to at
    most four times its size and two halves of a digit, 2^8 steps. The experts' rows
    are off by half a step, 2^-22 of their block's largest, more. The rest is
    _layer64's."""
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(T + H + I)
    x = torch.randint(-127, 128, (T, H), device=cuda, generator=g).float() / 64
    x[:, ::128] = torch.where(torch.arange(T, device=cuda) % 2 == 0, 4096.0, -4096.0)[:, None]
    x = x.to(getattr(torch, dtype))
    _, _, ws = _problem(1, H, I, E, bs, zp, "float32", 7, cuda)
    for B, S, Z in ws:
        if Z is not None:
            Z.fill_(0x88)
        row = B.flatten(2)  # zero weights for every 128th value
        row[:, :, ::64] = row[:, :, ::64] & 0xF0 | 8
        B.copy_(row.reshape(B.shape))
    ws[1][1][:, ::128] *= 4096.0
    dense = [_dense(w, n) for w, n in zip(ws, (H, H, I))]
    logits = torch.randn(T, E, device=cuda, generator=g)
    ids, p = _choice(logits, 2, True)
    op = pkg.MatMulNBitsMoE(H, I, E, 2, block_size=bs).prepare_device(None, *ws)
    y = op(x, logits=logits)
    print(f"case moe outliers T={T} H={H} I={I} E={E} bs={bs} zp={zp} {dtype}", flush=True)
    v = x.double()
    ref, err = torch.zeros_like(v), torch.zeros_like(v)

    def product(v, ve, W, exact):
        Wt, top = W.t().contiguous(), _blocks(v.abs() + ve)
        digits = 4 * (v.abs() + ve) + 2.0 ** -13 * top
        off = ve + (0 if exact else 2.0 ** -22 * top) + (-(-v.shape[1] // bs) + 4) * 2.0 ** -24 * digits
        return v @ Wt, off @ Wt.abs()

    for e in sorted(set(ids.flatten().tolist())):
        t, s = torch.nonzero(ids == e, as_tuple=True)
        zero = torch.zeros_like(v[t])
        gate, ge = product(v[t], zero, dense[0][e], True)
        up, ue = product(v[t], zero, dense[1][e], True)
        silu = gate * torch.sigmoid(gate)
        se = 1.1 * ge + 2.0 ** -20 * (silu.abs() + 1.1 * ge)
        h, he = silu * up, se * (up.abs() + ue) + silu.abs() * ue
        d, de = product(h, he + 2.0 ** -23 * (h.abs() + he), dense[2][e], False)
        w = p[t, s][:, None]
        ref[t] += w * d
        err[t] += w * de + w * 2.0 ** -18 * (d.abs() + de)
    print(f"  worst / bound {_check(y, ref, err):.3f}", flush=True)


def test_joined_axes_of_constants(pkg, cuda):
    """Weights with their axes joined give the same plan; other orders are refused."""
    import torch
    x, router, ws = _problem(3, 64, 96, 4, 32, True, "float32", 47, cuda)
    want = pkg.MatMulNBitsMoE(64, 96, 4, 2).prepare_device(router, *ws)(x)
    flat = [tuple(a.flatten(1) for a in w) for w in ws]
    op = pkg.MatMulNBitsMoE(64, 96, 4, 2).prepare_device(router.reshape(-1), *flat)
    assert torch.equal(op(x), want)
    with pytest.raises(ValueError, match="router must be"):
        op.prepare_device(router.t(), *ws)
    with pytest.raises(ValueError, match="gate's scales must be"):
        op.prepare_device(router, (ws[0][0], ws[0][1].transpose(1, 2), ws[0][2]), ws[1], ws[2])


def test_layers_share_a_workspace(pkg, cuda):
    """Layers that run one after another on a stream take turns at one workspace, which
    the 8-bit products have too."""
    import torch
    pkg.release_workspaces()
    layers = []
    for i in range(4):
        x, router, ws = _problem(40, 256, 384, 8, 32, True, "bfloat16", 61 + i, cuda)
        layers.append((pkg.MatMulNBitsMoE(256, 384, 8, 2).prepare_device(router, *ws), x,
                       torch.empty_like(x)))
    W = torch.ones(256, 300, device=cuda).to(torch.float8_e4m3fn)
    proj = pkg.MatMulFp8(300, 256).prepare_device(W, torch.ones(2, 3, device=cuda))
    v, o = torch.ones(100, 300, device=cuda), torch.empty(100, 256, device=cuda)
    need = layers[0][0].workspace_bytes(40, torch.bfloat16)
    assert need > proj.workspace_bytes(100, torch.float32) > 0
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for op, x, y in layers:
        op(x, out=y)
        proj(v, out=o)
    assert torch.cuda.memory_allocated() - before <= need + 512
    for op, x, y in layers:
        assert torch.equal(op(x), y)
    assert bool((o == 300).all())
