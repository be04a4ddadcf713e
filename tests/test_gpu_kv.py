"""The 8-bit cache and its attention on the GPU, against definitions in 64 bits.

Tolerances, fixed before the first run. What append writes is exact: scales are
powers of two, so a code is the value's own rounding. For an output of attend, with
p the exact weights, A = sum p |v| and S the largest |scale| sum |q k| of the
row's keys:
  - a score adds D exact products in fp32 (half a unit, 2^-24, lost in each addition
    of magnitudes up to S), is scaled twice and shifted; a fp32 query is two fp16 terms,
    2^-22 of each value; together (D + 16) 2^-24 S + 2^-22 S, and the exponent's
    own rounding, 2^-24 of at most (S + 128) / ln 2, twice. A weight is off by that,
    and by 2^-21 for the hardware's exponential;
  - the weights of a row are divided by their sum, which has the same errors: twice;
  - a weight is rounded to fp16, 2^-11 relative, for 16-bit queries, to 2^-22 for fp32,
    and where it is below fp16's normal values by 2^-25 at most; the largest weight (times its
    value scale) is 2^12 or, as a factor of 2 is left above it when it is found, 2^11 at
    least: 2^-36 of it, n 2^-35 max|v| for n keys, max|v| by channel;
  - sums of n weighted values in fp32: n 2^-24 A; joins and the division, 2^-20 A;
  - the output's rounding, half a step (eps / 2) of the value.
"""
import itertools
import math

import pytest

pytestmark = pytest.mark.gpu


# ---- definitions ------------------------------------------------------------

def _e4m3(v):
    """v (float64) rounded to the nearest e4m3 value, ties to even."""
    import torch
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -7))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(v / step) * step


def _spans(tokens, lengths, starts):
    """[(first row, rows, length)] of each sequence."""
    B = len(lengths)
    if starts is None:
        n = tokens // B
        return [(b * n, n, max(0, lengths[b])) for b in range(B)]
    return [(starts[b], starts[b + 1] - starts[b], max(0, lengths[b])) for b in range(B)]


def _append64(values, scales, X, table, spans, page):
    """values [pages, H, page, D] (code values) and scales [pages, H], in 64 bits, in place."""
    import torch
    for b, (row, n, length) in enumerate(spans):
        at = length - n
        rows = X[row + max(0, -at):row + n].double()
        at = max(0, at)
        while len(rows):
            p, slot = at // page, at % page
            part, rows = rows[:page - slot], rows[page - slot:]
            at += len(part)
            if p >= len(table[b]) or not 0 <= table[b][p] < len(values):
                continue
            p = table[b][p]
            finite = torch.where(part.isfinite(), part, 0.0)
            amax = finite.abs().amax(dim=(0, 2))
            e = torch.ceil(torch.log2(amax / 448.0)).clamp(min=-64.0)
            scale = torch.exp2(e)
            if slot:
                scale = torch.maximum(scale, scales[p])
                values[p] = torch.where(values[p].isnan(), values[p],
                                        _e4m3(values[p] * (scales[p] / scale)[:, None, None]))
            scales[p] = scale
            q = _e4m3(finite / scale[:, None])
            q = torch.where(part.isfinite(), q, math.nan)
            values[p, :, slot:slot + len(part)] = q.transpose(0, 1)


def _attend64(Q, k, v, table, spans, scale, window, dtype):
    """(y, tolerance) in 64 bits; k, v [pages, H, page, D] values."""
    import torch
    T, Hq, D = Q.shape
    H, page = k.shape[1:3]
    eps = torch.finfo(dtype).eps
    y, tol = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    for b, (row, n, length) in enumerate(spans):
        for i in range(n):
            pos = length - n + i
            keys = [t for t in range(max(0, pos - window + 1) if window else 0, pos + 1)
                    if t // page < len(table[b]) and 0 <= table[b][t // page] < len(k)]
            if not keys:
                continue
            at = torch.tensor([[table[b][t // page], t % page] for t in keys]).t()
            for h in range(Hq):
                kk, vv = k[at[0], h * H // Hq, at[1]], v[at[0], h * H // Hq, at[1]]
                q = Q[row + i, h].double()
                s = scale * (kk @ q)
                p = torch.softmax(s, dim=0)
                S = abs(scale) * (kk.abs() @ q.abs()).max().item()
                A = p @ vv.abs()
                m = len(keys)
                e = 2 * ((D + 16) * 2.0 ** -24 * S + 2.0 ** -22 * S + 2.0 ** -22 * (S + 128)
                         + 2.0 ** -21)
                w = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
                y[row + i, h] = p @ vv
                tol[row + i, h] = ((e + w + m * 2.0 ** -24 + 2.0 ** -20) * A
                                   + m * 2.0 ** -35 * vv.abs().amax(dim=0))
    tol += eps / 2 * (y.abs() + tol) + torch.finfo(dtype).smallest_normal * eps
    return y, tol


# ---- problems ---------------------------------------------------------------

def _rand(shape, seed, device, size=1.0):
    import torch
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return torch.randn(shape, device=device, generator=g) * size


def _table(B, width, spare, seed):
    """A table of different pages in no order, and how many pages there are."""
    import torch
    g = torch.Generator()
    g.manual_seed(seed)
    pages = B * width + spare
    return torch.randperm(pages, generator=g)[:B * width].reshape(B, width).tolist(), pages


def _cache(pkg, pages, H, page, D, device, seed, exponents=(-8, -3)):
    """A cache of random values and what they are; some scales no powers of two."""
    import torch
    tensors = []
    for n in range(2):
        codes = (_rand((pages, H, page, D), seed + n, device, 100.0).clamp(-448, 448)
                 .to(torch.float8_e4m3fn))
        g = torch.Generator(device=device)
        g.manual_seed(seed + 5 + n)
        e = torch.randint(*exponents, (pages, H), device=device, generator=g)
        tensors += [codes, torch.exp2(e.double()).float() * 1.25 ** (n * (seed % 2))]
    return pkg.Fp8KVCache.from_tensors(tensors[0], tensors[2], tensors[1], tensors[3])


def _values(codes, scales=None):
    v = codes.cpu().float().double()
    return v if scales is None else v * scales.cpu().double()[..., None, None]


def _i32(x, device):
    import torch
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=device)


def _check_attend(pkg, cuda, Hq, H, D, page, lengths, news, dtype, window=0, seed=0, ragged=True,
                  scale=None, spoil=None, q_size=1.0, exponents=(-8, -3), max_tokens=None):
    """attend against the definition; unseen slots and pages hold NaN codes. spoil(table,
    cache, Q): changes before the call."""
    import torch
    dtype = getattr(torch, dtype)
    B, T = len(lengths), sum(news)
    width = max(1, -(-max(lengths) // page))
    table, pages = _table(B, width, 2, seed)
    cache = _cache(pkg, pages, H, page, D, cuda, seed, exponents)
    Q = _rand((T, Hq, D), seed + 9, cuda, q_size).to(dtype)
    hold = torch.zeros(pages, page, dtype=torch.bool, device=cuda)
    for b in range(B):
        for t in range(lengths[b]):
            hold[table[b][t // page], t % page] = True
    for codes in (cache.k, cache.v):
        codes.view(torch.uint8).masked_fill_(~hold[:, None, :, None], 0x7F)
    if spoil is not None:
        spoil(table, cache, Q)
    starts = [sum(news[:b]) for b in range(B + 1)] if ragged else None
    got = cache.attend(Q, _i32(table, cuda), _i32(lengths, cuda), starts=_i32(starts, cuda),
                       scale=scale, window=window, max_tokens=max_tokens)
    y, tol = _attend64(Q.cpu(), _values(cache.k, cache.k_scales), _values(cache.v, cache.v_scales),
                       table, _spans(T, lengths, starts), D ** -0.5 if scale is None else scale,
                       window, dtype)
    assert got.dtype == dtype and got.shape == Q.shape
    got = got.cpu().double()
    nan = y.isnan()
    assert torch.equal(got.isnan(), nan)
    assert ((got - y).abs() <= tol)[~nan].all()
    return got


# ---- attention --------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("Hq,H", [(1, 1), (6, 2), (20, 1)])
def test_one_token(pkg, cuda, D, Hq, H, dtype):
    _check_attend(pkg, cuda, Hq, H, D, 32, [100, 7, 1, 33], [1] * 4, dtype, seed=D + Hq)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 63, 64, 65, 127, 300])
def test_lengths_and_pages(pkg, cuda, page, length):
    _check_attend(pkg, cuda, 4, 2, 64, page, [length], [1], "bfloat16", seed=length, ragged=False)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D", [64, 112, 256])
@pytest.mark.parametrize("Hq,H,news", [(2, 2, [2, 17, 40]), (8, 2, [5, 1, 9]), (7, 1, [30, 3, 1])])
def test_several_tokens(pkg, cuda, Hq, H, D, news, dtype):
    _check_attend(pkg, cuda, Hq, H, D, 32, [70, 17, 130], news, dtype, seed=D + Hq)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 1000, 1 << 40])
@pytest.mark.parametrize("news", [[1, 1], [40, 90]])
def test_windows(pkg, cuda, window, news):
    _check_attend(pkg, cuda, 4, 2, 64, 32, [200, 90], news, "float16", window=window, seed=window % 91)


@pytest.mark.parametrize("news,lengths", [([3, 1, 2], [3, 0, 1]), ([1, 1], [0, 0]), ([5, 70], [2, 0]),
                                          ([0, 4, 0], [10, 4, 0]), ([1], [1])])
@pytest.mark.parametrize("window", [0, 2])
def test_empty_rows(pkg, cuda, news, lengths, window):
    """Sequences of no tokens, of fewer tokens than rows, and of no rows."""
    got = _check_attend(pkg, cuda, 4, 2, 64, 16, lengths, news, "float32", window=window, seed=3)
    row = 0
    for n, length in zip(news, lengths):
        for i in range(n):
            assert (got[row + i] == 0).all() == (length - n + i < 0)
        row += n


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("news", [[1], [3], [150]])
@pytest.mark.parametrize("D", [64, 128])
def test_long(pkg, cuda, news, dtype, D):
    """Long enough for the keys to be shared out over workgroups."""
    _check_attend(pkg, cuda, 2, 1, D, 64, [2500], news, dtype, seed=D)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [0, 900])
def test_prompts_beside_decoded_sequences(pkg, cuda, window, dtype):
    """One call of sequences with one row and with many, both long enough to be shared out,
    and an empty slot."""
    _check_attend(pkg, cuda, 4, 1, 64, 64, [2100, 1500, 0, 700, 1300], [60, 1, 1, 3, 20], dtype,
                  window=window, seed=16, max_tokens=60)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("group", [17, 32, 33, 40, 48, 64, 65, 72])
def test_many_heads_beside_a_prompt(pkg, cuda, group, dtype):
    """Ragged calls with many query heads to a cache head: one token's rows are as many as a
    tile of few rows, or more than any; long enough to be shared out."""
    _check_attend(pkg, cuda, 2 * group, 2, 32, 64, [700, 1100, 0, 330], [12, 1, 1, 2], dtype,
                  seed=group, max_tokens=12)


def _many(B):
    """Rows and lengths of B sequences: one row, mostly, or none, and a few prompts."""
    news = [0 if b % 11 == 3 else 75 if b == B - 30 else 20 if b % 50 == 7 else 1 for b in range(B)]
    return news, [n + (b * 7) % 40 - 1 if b % 9 else n for b, n in enumerate(news)]


@pytest.mark.parametrize("D,dtype", [(64, "bfloat16"), (128, "float32"), (256, "bfloat16"),
                                     (256, "float32")])
@pytest.mark.parametrize("B,max_tokens", [(64, None), (65, 75), (150, None)])
def test_many_sequences(pkg, cuda, B, max_tokens, D, dtype):
    """More sequences than a wavefront has lanes."""
    news, lengths = _many(B)
    _check_attend(pkg, cuda, 4, 1, D, 16, lengths, news, dtype, seed=19, max_tokens=max_tokens)


@pytest.mark.parametrize("max_tokens", [1, 3, 20])
def test_max_tokens_too_small(pkg, cuda, max_tokens):
    """Rows past what the caller gave as the most are left out, in bounds; the others of
    their sequence, and other sequences, are not the worse for it."""
    import torch
    table, pages = _table(2, 30, 1, 17)
    cache = _cache(pkg, pages, 2, 64, 64, cuda, 17)
    Q = _rand((45, 8, 64), 18, cuda)
    args = (_i32(table, cuda), _i32([1900, 1800], cuda))
    starts = _i32([0, 40, 45], cuda)
    want = cache.attend(Q, *args, starts=starts)
    got = cache.attend(Q, *args, starts=starts, max_tokens=max_tokens, out=torch.full_like(Q, 7.0))
    most = _values(cache.v, cache.v_scales).abs().max().item()
    for row, n in ((0, 40), (40, 5)):
        seen = min(n, max_tokens)
        assert ((got - want)[row:row + seen].abs() <= 2.0 ** -16 * most).all()
        assert (got[row + seen:row + n] == 7.0).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("q_size,scale", [(1e-4, 1e3), (300.0, 1e-3), (30.0, None), (1.0, 0.0),
                                          (1.0, -0.2)])
def test_sizes_of_queries(pkg, cuda, q_size, scale, dtype):
    """Sharp and flat weights; queries that fp16 alone could not hold."""
    _check_attend(pkg, cuda, 4, 2, 64, 32, [150, 3], [1, 3], dtype, seed=5, q_size=q_size,
                  scale=scale)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sizes_of_values(pkg, cuda, dtype):
    """Pages of very different scales: their weights have to keep up."""
    _check_attend(pkg, cuda, 2, 1, 64, 16, [130], [5], dtype, seed=6, exponents=(-30, 20),
                  scale=1e-6)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("news", [[1, 3], [40, 90]])
def test_pages_of_zeros(pkg, cuda, news, dtype):
    """Scales of 0, as a quantizer may give a page of zeros: its tokens still have their
    weights."""
    def zeros(table, cache, Q):
        for p in (table[0][1], table[1][0], table[1][3]):
            cache.v[p].zero_()
            cache.v_scales[p] = 0.0
        for p in (table[0][0], table[1][3], table[1][4]):
            cache.k_scales[p] = 0.0

    _check_attend(pkg, cuda, 4, 2, 64, 32, [110, 200], news, dtype, seed=35, spoil=zeros)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news,lengths", [([1, 1, 1, 1], [2, 3, 4, 7]), ([9], [12]), ([40], [40]),
                                          ([150], [150])])
def test_weights_of_float16_rows(pkg, cuda, D, news, lengths):
    """A float16 result is as exact as its own rounding: half a step of the value, and what an
    fp32 result may be off by (its weights have 22 bits as well). Positive values, so that no
    weight's rounding is undone by another's, of few keys."""
    import torch
    page, B = 16, len(lengths)
    table, pages = _table(B, -(-max(lengths) // page), 1, D)
    cache = _cache(pkg, pages, 1, page, D, cuda, D)
    cache.v.view(torch.uint8).bitwise_and_(0x7F)
    Q = _rand((sum(news), 4, D), D + 1, cuda, 0.3).to(torch.float16)
    starts = [sum(news[:b]) for b in range(B + 1)]
    got = cache.attend(Q, _i32(table, cuda), _i32(lengths, cuda), starts=_i32(starts, cuda))
    y, tol = _attend64(Q.cpu(), _values(cache.k, cache.k_scales), _values(cache.v, cache.v_scales),
                       table, _spans(len(Q), lengths, starts), D ** -0.5, 0, torch.float32)
    half = torch.exp2(torch.floor(torch.log2(y.abs() + tol)).clamp(min=-14.0) - 11.0)
    assert ((got.cpu().double() - y).abs() <= half + tol).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("news", [1, 100, 150])
@pytest.mark.parametrize("exponent", [-100, -64, 0, 100, 120])
def test_ends_of_value_scales(pkg, cuda, exponent, news, dtype):
    """The least and the largest value scales, 2^18 keys of one weight: the weights' sum, which
    is divided by the scale, neither overflows nor vanishes. Values of 1, so that all sums are
    whole multiples of one power of two: only the division and Y round."""
    import torch
    page, D, width = 256, 64, 1024
    cache = pkg.Fp8KVCache(1, 1, D, page, device=cuda)
    cache.k.view(torch.uint8).fill_(0x38)  # 1.0
    cache.v.view(torch.uint8).fill_(0x38)
    cache.k_scales.fill_(1.0)
    cache.v_scales.fill_(2.0 ** exponent)
    table = torch.zeros(1, width, dtype=torch.int32, device=cuda)  # one page for all
    Q = _rand((news, 1, D), 90, cuda).to(getattr(torch, dtype))
    got = cache.attend(Q, table, _i32([width * page], cuda), scale=0.0).double()
    assert ((got - 2.0 ** exponent).abs() <= 2.0 ** (exponent - 22)).all()


def test_huge_queries(pkg, cuda):
    """fp32 and bf16 queries far beyond fp16's range, undone by the scale."""
    for dtype in ("float32", "bfloat16"):
        _check_attend(pkg, cuda, 2, 1, 64, 16, [40], [2], dtype, seed=7, q_size=1e20, scale=1e-21)


# ---- what must leave no trace ---------------------------------------------------

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("news", [[4], [40]])
def test_nan_in_later_tokens(pkg, cuda, D, news, window):
    """A NaN value reaches the rows that see it and no others, by channel; a NaN key
    the whole of those rows."""
    import torch

    def spoil(table, cache, Q):
        for which, t, d in (("v", 97, 3), ("v", 98, 5), ("k", 99, 1), ("v", 70, 7)):
            code = getattr(cache, which).view(torch.uint8)
            code[table[0][t // 32], 0, t % 32, d] = 0xFF

    got = _check_attend(pkg, cuda, 4, 2, D, 32, [100], news, "bfloat16", window=window, seed=8,
                        spoil=spoil)
    first = got[news[0] - 4]  # position 96: sees none of the last three
    assert first[:2, [3, 5]].isfinite().all() and first[2:].isfinite().all()
    assert got[news[0] - 3, :2, 3].isnan().all() and got[news[0] - 1, :2].isnan().all()


@pytest.mark.parametrize("dtype,D", [("bfloat16", 64), ("float16", 128), ("float32", 128),
                                     ("bfloat16", 256)])
@pytest.mark.parametrize("news", [[1, 2], [40, 30], [150, 9]])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, -1.0])
def test_scales_of_unseen_pages(pkg, cuda, news, bad, dtype, D):
    """Pages that lie before the window, in its first tile, hold anything: codes and scales."""
    lengths, window, page = [300, 180], 37, 16

    def spoil(table, cache, Q):
        for b, (n, length) in enumerate(zip(news, lengths)):
            for p in range((length - n - window + 1) // page):
                for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
                    codes.view(torch.uint8)[table[b][p]] = 0x7F
                    scales[table[b][p]] = bad

    import torch
    got = _check_attend(pkg, cuda, 4, 2, D, page, lengths, news, dtype, window=window, seed=45,
                        spoil=spoil)
    assert got.isfinite().all()


@pytest.mark.parametrize("dtype,D", [("bfloat16", 64), ("float32", 128), ("bfloat16", 256)])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("new", [40, 150])
@pytest.mark.parametrize("which", ["k_scales", "v_scales"])
def test_nan_scales_of_later_pages(pkg, cuda, which, new, window, dtype, D):
    """A page whose scale is NaN is the trouble of the rows that see it, and of no other."""
    length, page, at = 170, 16, 10

    def spoil(table, cache, Q):
        getattr(cache, which)[table[0][at], 0] = math.nan

    got = _check_attend(pkg, cuda, 4, 2, D, page, [length], [new], dtype, window=window, seed=46,
                        spoil=spoil)
    for i in range(new):
        pos = length - new + i
        sees = pos >= at * page and (window == 0 or pos - window < (at + 1) * page - 1)
        assert got[i, :2].isnan().all() == sees and got[i, 2:].isfinite().all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,new,length,window", [(1, 600, 632, 0), (1, 600, 1000, 300), (1, 120, 400, 290),
                                                  (4, 150, 400, 290), (4, 150, 182, 0)])
def test_nan_in_many_tiles(pkg, cuda, Hq, new, length, window, D, dtype):
    """NaN values in tile after tile that some of a workgroup's rows see and others do not,
    five to nine of them: rows and channels of each are its own."""
    def spoil(table, cache, Q):
        v = cache.v.view(torch.uint8)
        for t in range(5, length, 61):
            v[table[0][t // 32], 0, t % 32, t * 7 % D] = 0x7F

    import torch
    got = _check_attend(pkg, cuda, Hq, 1, D, 32, [length], [new], dtype, window=window, seed=49,
                        spoil=spoil)
    assert got.isnan().any() and got.isfinite().any(dim=2).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("new", [100, 150])
@pytest.mark.parametrize("q_size,scale,exponents", [(1e-4, 1e3, (-8, -3)), (300.0, 1e-3, (-8, -3)),
                                                    (30.0, None, (-8, -3)), (1.0, 0.0, (-8, -3)),
                                                    (1.0, -0.2, (-8, -3)), (1.0, 1e-6, (-30, 20))])
def test_sizes_of_queries_and_values_of_prompts(pkg, cuda, q_size, scale, exponents, new, dtype):
    """Sharp and flat weights, negative scales and pages of very different ones, where rows are
    many: more than 64 and more than 128 to a cache head. Values up to 448 2^19 pass float16's
    largest, 65504: from half a step above it, 65520, on a result is an infinity, and a result
    that is within its tolerance of 65520 may be."""
    import torch
    dtype, page, D = getattr(torch, dtype), 16, 64
    table, pages = _table(1, -(-(new + 30) // page), 2, 50)
    cache = _cache(pkg, pages, 2, page, D, cuda, 50, exponents)
    Q = _rand((new, 2, D), 59, cuda, q_size).to(dtype)
    got = cache.attend(Q, _i32(table, cuda), _i32([new + 30], cuda), scale=scale).cpu().double()
    y, tol = _attend64(Q.cpu(), _values(cache.k, cache.k_scales), _values(cache.v, cache.v_scales),
                       table, [(0, new, new + 30)], D ** -0.5 if scale is None else scale, 0, dtype)
    good = (got - y).abs() <= tol
    if dtype == torch.float16:
        inf = got == torch.copysign(torch.full_like(y, math.inf), y)
        good = torch.where(y.abs() - tol >= 65520.0, inf, good | (inf & (y.abs() + tol >= 65520.0)))
    assert good.all()


@pytest.mark.parametrize("new", [100, 150])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_huge_queries_of_prompts(pkg, cuda, new, dtype):
    _check_attend(pkg, cuda, 1, 1, 64, 16, [new + 30], [new], dtype, seed=51, q_size=1e20,
                  scale=1e-21)


@pytest.mark.parametrize("new", [100, 150])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_infinite_queries_of_prompts(pkg, cuda, new, dtype):
    """Rows whose queries are not finite leave the others' bits alone."""
    import torch
    dtype = getattr(torch, dtype)
    table, pages = _table(1, 6, 0, 52)
    cache = _cache(pkg, pages, 1, 32, 64, cuda, 52)
    args = (_i32(table, cuda), _i32([180], cuda))
    Q = _rand((new, 2, 64), 53, cuda).to(dtype)
    want = cache.attend(Q, *args)
    bad = torch.zeros(new, 2, dtype=torch.bool, device=cuda)
    for row, head, value in ((1, 0, math.inf), (2, 1, math.nan), (40, 0, -math.inf), (99, 1, math.nan)):
        Q[row, head, row % 64] = value
        bad[row, head] = True
    got = cache.attend(Q, *args)
    assert torch.equal(got[~bad], want[~bad])
    assert got[2, 1].isnan().all() and got[99, 1].isnan().all()


def test_infinite_queries(pkg, cuda):
    """A row whose query is not finite is its own trouble."""
    import torch

    def spoil(table, cache, Q):
        Q[1, 0, 3] = float("inf")
        Q[2, 1, 0] = float("nan")

    import torch as _t
    dtype, lengths = _t.float32, [60]
    clean = _check_attend(pkg, cuda, 2, 1, 64, 32, lengths, [4], "float32", seed=9)
    table, pages = _table(1, 2, 2, 9)
    cache = _cache(pkg, pages, 1, 32, 64, cuda, 9)
    Q = _rand((4, 2, 64), 18, cuda).to(dtype)
    spoil(table, cache, Q)
    got = cache.attend(Q, _i32(table, cuda), _i32(lengths, cuda)).cpu().double()
    assert got[2, 1].isnan().all() and not got[1, 0].isfinite().all()
    good = torch.ones(4, 2, dtype=torch.bool)
    good[1, 0] = good[2, 1] = False
    assert torch.equal(got[good], clean[good])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("new", [3, 40, 150])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_of_minus_infinity(pkg, cuda, D, new, dtype):
    """A query with an infinity where all keys are negative: only scores of -inf, a row of
    0, however large the query's other values; where all are positive, NaN."""
    import torch
    dtype, length, page = getattr(torch, dtype), 160, 32
    table, pages = _table(1, 5, 1, 47)
    cache = _cache(pkg, pages, 1, page, D, cuda, 47)
    cache.k.view(torch.uint8)[..., 3] = 0xB8  # -1.0
    cache.k.view(torch.uint8)[..., 4] = 0x38  # 1.0
    Q = _rand((new, 4, D), 48, cuda).to(dtype)
    Q[:, 1, 3] = math.inf
    Q[:, 2, 3] = math.inf
    Q[:, 2, 5:9] = 60000.0 if dtype == torch.float16 else 1e6
    Q[:, 3, 4] = math.inf
    args = (_i32(table, cuda), _i32([length], cuda))
    got = cache.attend(Q, *args)
    assert got[:, 0].isfinite().all() and (got[:, 1:3] == 0).all() and got[:, 3].isnan().all()
    got = cache.attend(Q, *args, scale=-0.1)  # the signs the other way round
    assert got[:, 0].isfinite().all() and got[:, 1:3].isnan().all() and (got[:, 3] == 0).all()


@pytest.mark.parametrize("news", [[1, 1], [30, 60]])
def test_pages_outside_the_cache(pkg, cuda, news):
    """Pages that the cache does not have are not seen: nothing is read there."""
    import torch

    def spoil(table, cache, Q):
        table[0][1], table[0][2], table[1][0] = -1, cache.pages, -2 ** 31
        table[1][1] = 2 ** 31 - 1

    _check_attend(pkg, cuda, 4, 2, 64, 32, [100, 90], news, "float16", seed=10, spoil=spoil)
    # every page of one sequence: a row of nothing
    def gone(table, cache, Q):
        table[0][:] = [cache.pages] * len(table[0])

    got = _check_attend(pkg, cuda, 4, 2, 64, 32, [100, 90], news, "float32", seed=11, spoil=gone)
    assert (got[:news[0]] == 0).all()
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("lengths,starts", [
    ([10 ** 9, -5], [0, 3, 6]), ([2 ** 31 - 1, -2 ** 31], [0, 3, 6]), ([20, 20], [0, 100, 200]),
    ([20, 20], [-5, 2, -7]), ([20, 20], [6, 3, 0]), ([20, 20], [2 ** 31 - 1, -2 ** 31, 5])])
def test_lengths_and_starts_out_of_range(pkg, cuda, lengths, starts):
    """What the device memory holds may be anything: rows outside stay as they are."""
    import torch
    table, pages = _table(2, 2, 1, 12)
    cache = _cache(pkg, pages, 1, 32, 64, cuda, 12)
    Q = _rand((6, 2, 64), 13, cuda)
    args = (_i32(table, cuda), _i32(lengths, cuda))
    out = torch.full_like(Q, 7.0)
    cache.attend(Q, *args, starts=_i32(starts, cuda), out=out)
    cache.append(Q[:, :1], Q[:, 1:], *args, starts=_i32(starts, cuda))
    cache.attend(Q, *args, out=out)
    torch.cuda.synchronize()
    if starts == [0, 100, 200]:
        # one sequence of six rows
        want = cache.attend(Q, args[0][:1], args[1][:1])
        out = torch.full_like(Q, 7.0)
        cache.attend(Q, *args, starts=_i32(starts, cuda), out=out)
        assert torch.equal(out, want)


@pytest.mark.parametrize("lengths,starts", [
    ([10 ** 9, -5], [0, 3, 6]), ([2 ** 31 - 1, -2 ** 31], [0, 3, 6]), ([20, 30], [0, 100, 200]),
    ([20, 30], [-5, 2, 4]), ([70, 64], [1, 4, 9]), ([2, 0], [0, 3, 5]), ([20, 20], [-5, 2, -7]),
    ([20, 20], [6, 3, 0]), ([20, 20], [2 ** 31 - 1, -2 ** 31, 5])])
def test_rows_and_pages_outside_of_all_spans(pkg, cuda, lengths, starts):
    """starts are held to 0 .. tokens, positions to the table: what lies outside stays as it
    is, bit for bit, and the rows inside are those of a call of their own. (Falling starts may
    leave rows out.)"""
    import torch
    page, width, T = 32, 2, 6
    table, pages = _table(2, width, 1, 77)
    cache = _cache(pkg, pages, 1, page, 64, cuda, 77)
    X = [_rand((T, 1, 64), 78 + n, cuda) for n in range(2)]
    Q = _rand((T, 2, 64), 80, cuda)
    falling = any(a > b for a, b in zip(starts, starts[1:]))
    spans = []
    for b in range(2):
        row = min(max(starts[b], 0), T)
        spans.append((row, max(0, min(starts[b + 1], T) - row), max(0, lengths[b])))
    args = (_i32(table, cuda), _i32(lengths, cuda))
    state, before = _state(cache), [cache.k.view(torch.uint8).clone(), cache.v.view(torch.uint8).clone(),
                                    cache.k_scales.clone(), cache.v_scales.clone()]
    cache.append(*X, *args, starts=_i32(starts, cuda))
    touched = torch.zeros(pages, dtype=torch.bool, device=cuda)
    for b, (row, n, length) in enumerate(spans):
        for i in range(n):
            if 0 <= length - n + i < width * page:
                touched[table[b][(length - n + i) // page]] = True
    after = (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scales, cache.v_scales)
    for a, b in zip(before, after):
        assert torch.equal(a[~touched], b[~touched])
    if not falling:
        for (values, scales), x, codes, s in zip(state, X, (cache.k, cache.v),
                                                 (cache.k_scales, cache.v_scales)):
            _append64(values, scales, x.cpu(), table, spans, page)
            assert torch.equal(_values(codes), values) and torch.equal(s.cpu().double(), scales)

    out = torch.full_like(Q, 7.0)
    cache.attend(Q, *args, starts=_i32(starts, cuda), out=out)
    inside = torch.zeros(T, dtype=torch.bool, device=cuda)
    most = _values(cache.v, cache.v_scales).abs().max().item()
    for b, (row, n, length) in enumerate(spans):
        inside[row:row + n] = True
        for i in range(0 if falling else n):
            sees = min(length - n + i, width * page - 1) + 1
            want = (cache.attend(Q[row + i:row + i + 1], args[0][b:b + 1], _i32([sees], cuda))[0]
                    if sees > 0 else torch.zeros(2, 64, device=cuda))
            assert ((out[row + i] - want).abs() <= 2.0 ** -16 * most).all()
    assert (out[~inside] == 7.0).all()


@pytest.mark.parametrize("split", [False, True])
def test_rows_of_no_sequence(pkg, cuda, split):
    """Rows before the first, behind the last sequence: kept in out, 0 without it."""
    import torch
    width = 40 if split else 1
    table, pages = _table(2, width, 0, 14)
    cache = _cache(pkg, pages, 2, 64, 64, cuda, 14)
    Q = _rand((10, 4, 64), 15, cuda).to(torch.bfloat16)
    lengths = [64 * width, 64 * width - 3]
    args = (_i32(table, cuda), _i32(lengths, cuda))
    out = torch.full_like(Q, 7.0)
    cache.attend(Q, *args, starts=_i32([2, 5, 7], cuda), out=out)
    fresh = cache.attend(Q, *args, starts=_i32([2, 5, 7], cuda), max_tokens=3)
    assert (out[:2] == 7).all() and (out[7:] == 7).all()
    assert (fresh[:2] == 0).all() and (fresh[7:] == 0).all()
    alone = cache.attend(Q[2:5], args[0][:1], args[1][:1])
    # Other bounds may choose another kernel: each result is off by half a step (2^-8) of its
    # value, and by 2^-10 of the largest value for its weights' rounding (2^-11) and sums.
    most = _values(cache.v, cache.v_scales).abs().max().item()
    for a, b in ((out[2:7], fresh[2:7]), (out[2:5], alone)):
        a, b = a.float(), b.float()
        assert ((a - b).abs() <= 2.0 ** -8 * (a.abs() + b.abs()) + 2.0 ** -9 * most).all()


# ---- append -----------------------------------------------------------------

def _check_append(pkg, cuda, cache, state, X, table, lengths, starts, page):
    """One append, on both sides; everything else stays as it was, bit for bit."""
    import torch
    spans = _spans(X[0].shape[0], lengths, starts)
    cache.append(*X, _i32(table, cuda), _i32(lengths, cuda), starts=_i32(starts, cuda))
    for (values, scales), x, codes, s in zip(state, X, (cache.k, cache.v),
                                             (cache.k_scales, cache.v_scales)):
        _append64(values, scales, x.cpu(), table, spans, page)
        assert torch.equal(s.cpu().double(), scales)
        got = _values(codes)
        assert torch.equal(got.isnan(), values.isnan())
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(values))


def _state(cache):
    return [[_values(cache.k), cache.k_scales.cpu().double()],
            [_values(cache.v), cache.v_scales.cpu().double()]]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("H,D", [(1, 16), (3, 80), (2, 128), (2, 256)])
def test_append(pkg, cuda, dtype, page, H, D):
    """A prompt, tokens one by one with values that grow, and a chunk, of two
    sequences: the scales and codes of every step."""
    import torch
    dtype = getattr(torch, dtype)
    table, pages = _table(2, 4 * 64 // page + 2, 1, 20)
    cache = _cache(pkg, pages, H, page, D, cuda, 20)
    state = _state(cache)
    lengths = [0, 0]
    for step, news in enumerate([[20, 37], [1, 1], [1, 1], [1, 0], [70, 30], [1, 1]]):
        lengths = [a + b for a, b in zip(lengths, news)]
        starts = [0, news[0], sum(news)]
        X = [_rand((sum(news), H, D), 30 + 2 * step + n, cuda, 4.0 ** step).to(dtype) for n in (0, 1)]
        _check_append(pkg, cuda, cache, state, X, table, lengths, starts, page)


def test_append_borders_of_scales(pkg, cuda):
    """Magnitudes just below, at and above 448 times a power of two, zeros, fp32's
    ends, ties of codes, infinities and NaN."""
    import torch
    tops = [448.0, math.nextafter(448.0, 500.0), 0.0, 2.0 ** -55, 448 * 2.0 ** -64, 2.0 ** -140, 1.75,
            3.4e38, float("inf"), float("nan"), 1.0]
    table, pages = _table(len(tops), 1, 0, 21)
    cache = _cache(pkg, pages, 1, 16, 16, cuda, 21)
    X = []
    for n in range(2):
        x = _rand((len(tops), 1, 16), 22 + n, cuda, 1e-3).abs()
        for i, top in enumerate(tops):
            top = torch.tensor(top, dtype=torch.float32).item()
            x[i] = torch.nan_to_num(x[i] * (top if 0 < top < 1e38 else 1.0))
            x[i, 0, 5] = top
            # halves of a code's last place: 1.0625 and 1.1875 lie between two codes
            x[i, 0, 6:8] = torch.tensor([1.0625, -1.1875], device=cuda) * (0.5 if top == 1.0 else 0)
        X.append(x.contiguous())
    _check_append(pkg, cuda, cache, _state(cache), X, table, [1] * len(tops), None, 16)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [1.0, 1.25, 1.375, 1.75, 1.1, 3.0 * 2.0 ** -9])
def test_append_beside_other_scales(pkg, cuda, scale, dtype):
    """A continued page keeps a scale that is no power of two: codes are the fp32 quotients',
    halves of a code's last place to the even one."""
    import torch
    D, page = 64, 16
    scale = torch.tensor(scale, dtype=torch.float32)
    cache = pkg.Fp8KVCache(1, 1, D, page, device=cuda)
    for s in (cache.k_scales, cache.v_scales):
        s.fill_(scale.item())
    # 17 / 16 and on: between two codes, at eight powers of two, below 448
    halves = (torch.arange(17, 32, 2)[:, None] / 16 * torch.exp2(torch.arange(-2.0, 6.0))).reshape(1, D)
    X = [(sign * halves * scale).to(getattr(torch, dtype)).repeat(4, 1)[:, None] for sign in (1, -1)]
    cache.append(*(x.to(cuda) for x in X), _i32([[0]], cuda), _i32([9], cuda))
    for x, codes, s in zip(X, (cache.k, cache.v), (cache.k_scales, cache.v_scales)):
        assert s.item() == scale.item()
        want = _e4m3((x.float() / scale).double())
        assert torch.equal(_values(codes)[0, 0, 5:9], want[:, 0])


def test_append_of_strided_and_batched_rows(pkg, cuda):
    """Views of a QKV projection's rows, misaligned rows, [sequences, tokens, ...]."""
    import torch
    H, D, page, T = 2, 48, 16, 12
    table, pages = _table(3, 2, 0, 23)
    qkv = _rand((T, 8 + 2 * H, D), 24, cuda).to(torch.bfloat16)
    k, v = qkv[:, 8:8 + H], qkv[:, 8 + H:]
    odd = torch.zeros(T * H * D + 1, dtype=torch.bfloat16, device=cuda)[1:].view(T, H, D)
    odd.copy_(k)
    lengths = [4, 20, 3]
    codes = []
    for K, V in ((k.contiguous(), v.contiguous()), (k, v), (odd, v),
                 (k.reshape(3, 4, H, D), v.reshape(3, 4, H, D)),
                 (k.transpose(0, 1).contiguous().transpose(0, 1), v)):
        cache = _cache(pkg, pages, H, page, D, cuda, 25)
        cache.append(K, V, _i32(table, cuda), _i32(lengths, cuda))
        codes.append([t.view(torch.uint8) for t in (cache.k, cache.v)]
                     + [cache.k_scales, cache.v_scales])
    for other in codes[1:]:
        assert all(torch.equal(a, b) for a, b in zip(codes[0], other))


def test_append_outside_the_table_and_cache(pkg, cuda):
    """Positions below 0 or past the table, pages outside: dropped; the rest is written."""
    import torch
    H, D, page = 1, 32, 16
    table, pages = _table(3, 2, 1, 26)
    table[1][0], table[2][1] = -1, pages
    cache = _cache(pkg, pages, H, page, D, cuda, 26)
    X = [_rand((60, H, D), 27 + n, cuda) for n in range(2)]
    _check_append(pkg, cuda, cache, _state(cache), X, table, [10, 25, 45], None, page)


@pytest.mark.parametrize("B", [64, 65, 150])
def test_append_of_many_sequences(pkg, cuda, B):
    news, lengths = _many(B)
    H, D, page = 2, 32, 16
    table, pages = _table(B, 8, 1, 33)
    cache = _cache(pkg, pages, H, page, D, cuda, 33)
    X = [_rand((sum(news), H, D), 34 + n, cuda) for n in range(2)]
    _check_append(pkg, cuda, cache, _state(cache), X, table, lengths,
                  [sum(news[:b]) for b in range(B + 1)], page)


def test_append_twice_is_append_once(pkg, cuda):
    import torch
    table, pages = _table(2, 3, 0, 28)
    cache = _cache(pkg, pages, 2, 32, 64, cuda, 28)
    X = [_rand((10, 2, 64), 29 + n, cuda, 100.0) for n in range(2)]
    args = (*X, _i32(table, cuda), _i32([40, 66], cuda))
    cache.append(*args)
    once = [cache.k.clone(), cache.v.clone(), cache.k_scales.clone(), cache.v_scales.clone()]
    cache.append(*args)
    for a, b in zip(once, (cache.k, cache.v, cache.k_scales, cache.v_scales)):
        assert torch.equal(a.float(), b.float())


# ---- streams, graphs, sizes ---------------------------------------------------

def test_offsets_past_32_bits(pkg, cuda):
    """A cache of more than 4 GiB of codes: pages at its very end."""
    import torch
    pages, H, page, D = 40000, 4, 256, 128  # 5.2 GB of keys, as much of values
    cache = pkg.Fp8KVCache(pages, H, D, page)
    table = [[pages - 1, 3], [pages - 2, 32768]]
    lengths = [300, 260]
    X = [_rand((520, H, D), 40 + n, cuda) for n in range(2)]
    starts = [0, 300, 520]
    lengths[1] = 220
    cache.append(*X, _i32(table, cuda), _i32(lengths, cuda), starts=_i32(starts, cuda))
    small = pkg.Fp8KVCache(4, H, D, page)
    small.append(*X, _i32([[0, 1], [2, 3]], cuda), _i32(lengths, cuda), starts=_i32(starts, cuda))
    for p, r in ((pages - 1, 0), (3, 1), (pages - 2, 2)):
        assert torch.equal(cache.k[p].float(), small.k[r].float())
        assert torch.equal(cache.v_scales[p], small.v_scales[r])
    assert (cache.k_scales > 0).sum().item() == 3 * H
    Q = _rand((2, 8, D), 42, cuda)
    got = cache.attend(Q, _i32(table, cuda), _i32(lengths, cuda))
    want = small.attend(Q, _i32([[0, 1], [2, 3]], cuda), _i32(lengths, cuda))
    assert torch.equal(got, want)
    del cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("ragged,max_tokens", [(False, None), (True, 1), (True, None)])
def test_most_sequences(pkg, cuda, ragged, max_tokens):
    """As many sequences as a call may have, of one token each: its value comes back. A code is
    off by half a step (2^-4) of the value or of the least normal (2^-6 scale); scores are
    below 128, so a weight and the sum are off by 2^-11 (above), and everything else by less."""
    import torch
    B, D, page = 65535, 16, 16
    cache = pkg.Fp8KVCache(B, 1, D, page, device=cuda)
    g = torch.Generator(device=cuda)
    g.manual_seed(36)
    table = torch.randperm(B, device=cuda, generator=g).int()[:, None]
    lengths = torch.ones(B, dtype=torch.int32, device=cuda)
    starts = torch.arange(B + 1, dtype=torch.int32, device=cuda) if ragged else None
    K, V, Q = (_rand((B, 1, D), 37 + n, cuda).clamp(-4, 4) for n in range(3))
    cache.append(K, V, table, lengths, starts=starts, max_tokens=max_tokens)
    got = cache.attend(Q, table, lengths, starts=starts, max_tokens=max_tokens)
    scale = cache.v_scales[table[:, 0].long()][:, :, None]
    held = cache.v[table[:, 0].long(), :, 0].float() * scale
    assert ((held - V).abs() <= 2.0 ** -4 * V.abs() + 2.0 ** -10 * scale).all()
    assert ((got - held).abs() <= 2.0 ** -10 * held.abs()).all()


def test_streams_and_threads(pkg, cuda):
    """Calls that overlap, each with a workspace of its own."""
    import threading

    import torch
    table, pages = _table(3, 30, 0, 43)
    cache = _cache(pkg, pages, 2, 64, 64, cuda, 43)
    args = (_i32(table, cuda), _i32([1900, 1500, 3], cuda))
    Qs = [_rand((3, 4, 64), 44 + n, cuda) for n in range(4)]
    want = [cache.attend(Q, *args) for Q in Qs]
    torch.cuda.synchronize()
    got = [[] for _ in Qs]

    def work(n):
        stream = torch.cuda.Stream()
        for _ in range(20):
            got[n].append(cache.attend(Qs[n], *args, stream=stream))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for n in range(4):
        assert len(got[n]) == 20 and all(torch.equal(y, want[n]) for y in got[n])


def test_graphs(pkg, cuda):
    """A captured append and attention replayed as the sequences grow; two graphs on
    one cache do not share a workspace."""
    import torch
    H, Hq, D, page = 2, 8, 64, 64
    table, pages = _table(2, 40, 0, 50)
    cache, plain = (_cache(pkg, pages, H, page, D, cuda, 50) for _ in range(2))
    table_, lengths = _i32(table, cuda), _i32([2400, 60], cuda)
    K, V = (_rand((2, H, D), 51 + n, cuda).to(torch.bfloat16) for n in range(2))
    Q = _rand((2, Hq, D), 53, cuda).to(torch.bfloat16)
    R = _rand((2, Hq, D), 54, cuda).to(torch.bfloat16)
    for c in (cache, plain):
        c.append(K, V, table_, lengths)
        c.attend(Q, table_, lengths)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in (Q, R):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.append(K, V, table_, lengths)
            outs.append(cache.attend(q, table_, lengths))
        graphs.append(graph)
    for step in range(4):
        lengths += 1
        for n, x in enumerate((K, V, Q, R)):
            x.copy_(_rand(x.shape, 60 + 4 * step + n, cuda, 2.0 ** step))
        plain.append(K, V, table_, lengths)
        want = [plain.attend(q, table_, lengths) for q in (Q, R)]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.k.float(), plain.k.float())
        assert torch.equal(cache.v_scales, plain.v_scales)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_graph_of_ragged_calls(pkg, cuda):
    """A captured ragged call replayed as rows go from one sequence to another, to none, and
    as lengths and pages change."""
    import torch
    H, Hq, D, page, T = 2, 8, 64, 16, 64
    table, pages = _table(3, 100, 0, 55)
    cache, plain = (_cache(pkg, pages, H, page, D, cuda, 55) for _ in range(2))
    table_, lengths, starts = _i32(table, cuda), _i32([1500, 300, 64], cuda), _i32([0, 60, 61, 64], cuda)
    K, V = (_rand((T, H, D), 56 + n, cuda).to(torch.bfloat16) for n in range(2))
    Q = _rand((T, Hq, D), 58, cuda).to(torch.bfloat16)
    args = (table_, lengths, starts)
    for c in (cache, plain):
        c.append(K, V, *args)
        c.attend(Q, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(K, V, *args)
        got = cache.attend(Q, *args)
    for s, l, swap in (([0, 60, 61, 64], [1500, 300, 64], False), ([0, 1, 2, 64], [1501, 301, 130], False),
                       ([5, 5, 64, 64], [1501, 360, 0], True), ([0, 64, 64, 64], [20, 0, 130], False),
                       ([0, 0, 0, 0], [1600, 1600, 1600], False), ([0, 20, 41, 64], [1600, 21, 24], True)):
        starts.copy_(_i32(s, cuda))
        lengths.copy_(_i32(l, cuda))
        if swap:
            table_.copy_(table_.flip(0).clone())
        plain.append(K, V, *args)
        want = plain.attend(Q, *args)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.k.float().nan_to_num(), plain.k.float().nan_to_num())
        assert torch.equal(cache.k_scales, plain.k_scales)
        assert torch.equal(got, want)


def test_same_bits_again(pkg, cuda):
    import torch
    table, pages = _table(2, 32, 0, 70)
    cache = _cache(pkg, pages, 2, 64, 128, cuda, 70)
    for n in (1, 6, 200):
        Q = _rand((2 * n, 8, 128), 71, cuda).to(torch.bfloat16)
        args = (Q, _i32(table, cuda), _i32([2048, 1111], cuda))
        want = cache.attend(*args)
        assert all(torch.equal(cache.attend(*args), want) for _ in range(5))


def test_shapes_of_queries(pkg, cuda):
    """[sequences, tokens, heads, head_dim], strides, and rows of nothing."""
    import torch
    table, pages = _table(2, 3, 0, 72)
    cache = _cache(pkg, pages, 2, 32, 64, cuda, 72)
    args = (_i32(table, cuda), _i32([90, 40], cuda))
    qkv = _rand((2, 3, 12, 64), 73, cuda).to(torch.float16)
    Q = qkv[:, :, :8]
    want = cache.attend(Q.contiguous().reshape(6, 8, 64), *args)
    assert torch.equal(cache.attend(Q, *args).reshape(6, 8, 64), want)
    swapped = Q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(cache.attend(swapped, *args).reshape(6, 8, 64), want)
    assert cache.attend(Q[:, :0], *args).shape == (2, 0, 8, 64)
    none = cache.attend(Q[:0], args[0][:0], args[1][:0])
    assert none.shape == (0, 3, 8, 64)
    out = torch.empty(6, 8, 64, dtype=torch.float16, device=cuda)
    assert cache.attend(want, *args, out=out) is out


def test_values_come_back(pkg, cuda):
    """A sequence of one token: its value, whatever the query. Its weight w is 2^14 but
    for the rounding of a difference; an fp32 value is multiplied by two fp16 terms, w (1 +
    2^-22) at most, divided by w as a product with a reciprocal (two roundings, 2^-24
    each, and 2^-24 of the sum): within 2^-21. The one term of a 16-bit Y is off by as little."""
    import torch
    for dtype, D in itertools.product((torch.float32, torch.bfloat16), (64, 256)):
        cache = pkg.Fp8KVCache(3, 2, D, 16)
        v = (torch.randint(-7, 8, (1, 2, D), device=cuda) * 2.0).to(dtype)
        table, lengths = _i32([[1]], cuda), _i32([1], cuda)
        cache.append(v * 0.5, v, table, lengths)
        y = cache.attend(_rand((1, 6, D), 80, cuda).to(dtype), table, lengths)
        v = v.repeat_interleave(3, dim=1)
        assert ((y - v).abs() <= (2.0 ** -21 if dtype == torch.float32 else 0.0) * v.abs()).all()


def test_no_gradient(pkg, cuda):
    """Queries that require a gradient have their results; backward() says that there is none."""
    import torch
    table, pages = _table(2, 3, 0, 74)
    cache = _cache(pkg, pages, 2, 32, 64, cuda, 74)
    args = (_i32(table, cuda), _i32([90, 40], cuda))
    Q = _rand((6, 8, 64), 75, cuda)
    K = _rand((6, 2, 64), 76, cuda)
    cache.append(K, K, *args)
    want = cache.attend(Q, *args, window=30, scale=0.3)
    Q.requires_grad_()
    K.requires_grad_()
    cache.append(K, K, *args)  # the cache holds values alone
    assert not cache.k_scales.requires_grad
    got = cache.attend(Q, *args, window=30, scale=0.3)
    assert torch.equal(got, want) and got.requires_grad
    with pytest.raises(RuntimeError, match="no gradient"):
        got.sum().backward()
    with pytest.raises(ValueError, match="must not require a gradient"):
        cache.attend(Q, *args, out=torch.empty_like(want))
    with torch.no_grad():
        out = torch.empty_like(want)
        assert cache.attend(Q, *args, window=30, scale=0.3, out=out) is out
    assert torch.equal(out, want) and not out.requires_grad and Q.grad is None


@pytest.mark.parametrize("more", [2 ** 31, 2 ** 63, 2 ** 64, 2 ** 64 + 1, 10 ** 30])
def test_numbers_past_64_bits(pkg, cuda, more):
    """A window and a largest number of tokens beyond anything mean no limit, whatever is left of
    them in 64 bits."""
    import torch
    table, pages = _table(2, 30, 0, 81)
    cache = _cache(pkg, pages, 2, 64, 64, cuda, 81)
    Q = _rand((7, 4, 64), 82, cuda)
    args = (Q, _i32(table, cuda), _i32([1900, 60], cuda))
    starts = _i32([0, 3, 7], cuda)
    want = cache.attend(*args, starts=starts)
    assert torch.equal(cache.attend(*args, starts=starts, window=more), want)
    assert torch.equal(cache.attend(*args, starts=starts, max_tokens=more), want)
