"""A decoder layer of the package's operators, as a program would write it: the RMS norm
with the residual into an 8-bit QKV projection, rotary positions in place on views of
its rows, the new keys and values into the cache, the attention, the 8-bit output
projection, the norm with the residual and a layer of experts.

Each step is held to its own definition on the inputs that it was given, with the
tolerances of its own test module; the whole layer, captured into a graph, to itself run
eagerly, bit for bit.
"""
import pytest

from test_gpu_kv import _append64, _attend64, _i32, _spans, _state, _values
from test_gpu_norm import FP32, _check_codes, _norm64
from test_gpu_rotary import _check as _check_rotary

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, DIM, PAGE = 512, 8, 2, 64, 32


class Layer:
    def __init__(self, pkg, device, seed=0):
        import torch
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def randn(*shape):
            return torch.randn(shape, device=device, generator=g)

        def fp8(K, N):
            W = (randn(N, K) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
            scales = torch.full((-(-N // 128), -(-K // 128)), 0.01 / K ** 0.5, device=device)
            return pkg.MatMulFp8(K, N).prepare_device(W, scales)

        def experts(K, N):
            B = torch.randint(0, 256, (4, N, K // 32, 16), dtype=torch.uint8, device=device,
                              generator=g)
            return B, torch.full((4, N, K // 32), 0.2 / K ** 0.5, device=device)

        self.pkg = pkg
        self.gamma = [1.0 + 0.1 * randn(HIDDEN) for _ in range(2)]
        self.qkv, self.out = fp8(HIDDEN, (HQ + 2 * HKV) * DIM), fp8(HQ * DIM, HIDDEN)
        self.rotary = pkg.Rotary(DIM, base=500000.0)
        self.cache = pkg.Fp8KVCache(12, HKV, DIM, PAGE, device=device)
        self.moe = pkg.MatMulNBitsMoE(HIDDEN, 256, 4, 2).prepare_device(
            randn(4, HIDDEN) * 0.05, experts(HIDDEN, 256), experts(HIDDEN, 256), experts(256, HIDDEN))

    def __call__(self, x, residual, positions, table, lengths, starts=None, max_tokens=None,
                 seen=None):
        """(the layer's output, the residual stream); seen: a list for each step's result."""
        rows, residual = self.qkv.run_rmsnorm(x, self.gamma[0], residual=residual)
        heads = rows.view(-1, HQ + 2 * HKV, DIM)
        if seen is not None:
            seen.append((residual.clone(), heads.clone()))
        q, k, v = heads.split([HQ, HKV, HKV], dim=1)
        self.rotary(q, k, positions, out=(q, k))
        self.cache.append(k, v, table, lengths, starts=starts, max_tokens=max_tokens)
        y = self.cache.attend(q, table, lengths, starts=starts, max_tokens=max_tokens)
        if seen is not None:
            seen.append((heads, y))
        y = self.out(y.view(-1, HQ * DIM))
        y, residual = self.pkg.rms_norm(y, self.gamma[1], residual=residual)
        if seen is not None:
            seen.append((y, residual))
        return self.moe(y), residual


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_each_step(pkg, cuda, dtype):
    """A prompt and a decoded token beside the end of another prompt."""
    import torch
    dtype = getattr(torch, dtype)
    layer = Layer(pkg, cuda)
    table = [[7, 2, 9], [4, 0, 11]]
    state = _state(layer.cache)
    lengths = [0, 0]
    for news in ([37, 20], [1, 44]):
        lengths = [a + b for a, b in zip(lengths, news)]
        starts = [0, news[0], sum(news)]
        positions = torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, news)]).to(cuda)
        x, r = (torch.randn(sum(news), HIDDEN, device=cuda).to(dtype) for _ in range(2))
        seen = []
        args = (_i32(table, cuda), _i32(lengths, cuda))
        Y, stream = layer(x, r, positions, *args, _i32(starts, cuda), max(news), seen)
        (h, heads), (turned, y), (z, h2) = seen
        info = torch.finfo(dtype)

        # norm and projection
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
        codes, scales = pkg.rms_norm_fp8(h, layer.gamma[0])
        _check_codes(codes, scales, _norm64(h, layer.gamma[0], 1e-5))
        assert torch.equal(heads.view(sum(news), -1),
                           layer.qkv(codes, scales=scales, out_dtype=dtype))
        # positions, in place; values as they were
        _check_rotary(turned[:, :HQ], heads[:, :HQ], positions, layer.rotary)
        _check_rotary(turned[:, HQ:HQ + HKV], heads[:, HQ:HQ + HKV], positions, layer.rotary)
        assert torch.equal(turned[:, HQ + HKV:], heads[:, HQ + HKV:])
        # cache
        spans = _spans(sum(news), lengths, starts)
        new = turned[:, HQ:].cpu()
        for (values, s), rows, codes, got in zip(state, (new[:, :HKV], new[:, HKV:]),
                                                 (layer.cache.k, layer.cache.v),
                                                 (layer.cache.k_scales, layer.cache.v_scales)):
            _append64(values, s, rows, table, spans, PAGE)
            assert torch.equal(_values(codes), values) and torch.equal(got.cpu().double(), s)
        # attention
        c = layer.cache
        want, tol = _attend64(turned[:, :HQ].cpu(), _values(c.k, c.k_scales),
                              _values(c.v, c.v_scales), table, spans, DIM ** -0.5, 0, dtype)
        assert ((y.cpu().double() - want).abs() <= tol).all()
        # the second norm, of the sum
        assert torch.equal(stream, h2)
        want = _norm64(h2, layer.gamma[1], 1e-5)
        assert ((z.double() - want).abs() <= (info.eps / 2 + FP32) * want.abs()).all()
        assert torch.equal(Y, layer.moe(z)) and Y.isfinite().all()


def test_decoding_from_a_graph(pkg, cuda):
    """Three sequences, a token each: one captured step, replayed as they grow past pages,
    against the same steps run eagerly on a second cache."""
    import torch
    layers = [Layer(pkg, cuda, 3) for _ in range(2)]
    table = _i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]], cuda)
    lengths = [30, 1, 62]
    x, r = (torch.randn(3, HIDDEN, device=cuda).bfloat16() for _ in range(2))
    for layer in layers:
        prompt = torch.randn(sum(lengths), HIDDEN, device=cuda,
                             generator=torch.Generator(device=cuda).manual_seed(5)).bfloat16()
        positions = torch.cat([torch.arange(n) for n in lengths]).to(cuda)
        layer(prompt, prompt, positions, table, _i32(lengths, cuda),
              _i32([0, 30, 31, 93], cuda), 62)
    n, positions = _i32(lengths, cuda), torch.tensor(lengths, device=cuda)
    for layer in layers:
        layer(x, r, positions, table, n)  # warm up, both alike
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    n += 1
    with torch.cuda.graph(graph):
        out, stream = layers[0](x, r, positions, table, n)
    for step in range(5):
        if step:
            n += 1
            positions += 1
        x.copy_(torch.randn_like(x) * 2.0 ** step)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), stream.clone()
        side = torch.tanh(torch.randn(256, 256, device=cuda) @ torch.randn(256, 256, device=cuda))
        want = layers[1](x, r, positions, table, n)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), step
        for a, b in ((layers[0].cache.k, layers[1].cache.k), (layers[0].cache.v, layers[1].cache.v)):
            assert torch.equal(a.float(), b.float()), step
    del side
