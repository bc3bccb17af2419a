"""Weights in four bits: quantising, reading back and the linear layer, against their formulas in 64 bits.

What a result may be off. u = 2^-24 is half a step of fp32. The linear layer adds K products (and the bias, and a scale per group) in fp32; the tensor cores cut
off where others round, so an addition is off by 2 u of what has been added up so far, which A = sum |x w'| + |b| bounds: 2 u (K + 2 G + 4) A in all. fp32 rows are
split into three bf16 terms that miss up to 2^-23 of x in all (a bit more than 24 bits): 2^-22 A covers it. The GELU has a slope below 1.13, erf and the rest of it are a few u of the value. bf16 results:
half a step, 2^-8 of the value. With weights rounded to bf16 (bf16 x and y, more rows than int4.linear's docstring says): 2^-8 A for every element, and for the
whole result, whose weights' roundings are independent and spread over their steps, the 2-norm goes by their variance: a step's width below 2^-7 of a value's, so below 2^-8 / sqrt 3 of
|x| |w'| in quadrature, and the result's own rounding as much again.
"""
import math

import pytest
import torch

from pragnosia_b200 import int4, ops
from pragnosia_b200._lib import graph_capture, warm_up

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
ROWS = 16                                                             # up to here weights are not rounded


def levels(w, group, zeros):
    """The formulas' levels, scales and zeros, one fp32 operation after the other."""
    N, K = w.shape
    G = -(-K // group)
    f = torch.nn.functional.pad(w.float(), (0, G * group - K)).view(N, G, group)
    lo, hi = f.amin(2).clamp_max(0.0), f.amax(2).clamp_min(0.0)
    top = hi - lo if zeros else torch.maximum(hi, -lo)
    s = (top / torch.full_like(top, 15.0 if zeros else 7.0)).to(w.dtype)      # by a tensor: by a number torch multiplies with its reciprocal
    t = s.float()
    safe = torch.where(t > 0, t, torch.ones_like(t))
    z = torch.where(t > 0, torch.round(-lo / safe).clamp(0, 15), torch.zeros_like(t)) if zeros else torch.full_like(t, 8.0)
    q = (torch.round(f / safe[..., None]) + z[..., None]).clamp(0, 15)
    q = torch.where(t[..., None] > 0, q, z[..., None].expand_as(q))
    return q.view(N, -1)[:, :K].to(torch.uint8), s, z.to(torch.uint8)


def packed(q):
    return q[:, 0::2] | (q[:, 1::2] << 4)


def spread(t, w, K):
    return t.double().repeat_interleave(w.group, 1)[:, :K]


def value(w):
    """scale (q - zero) in 64 bits."""
    N, K = w.shape
    q = torch.stack([w.q & 15, w.q >> 4], 2).view(N, K).double()
    return spread(w.scales, w, K) * (q - (8.0 if w.zeros is None else spread(w.zeros, w, K)))


def random_weight(N, K, group, zeros, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 16, (N, K), device="cuda", generator=g, dtype=torch.uint8)
    G = -(-K // group)
    s = (0.02 * torch.rand(N, G, device="cuda", generator=g) + 0.005).to(dtype)
    z = torch.randint(0, 17, (N, G), device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    return int4.Int4Weight(packed(q), s, z, group)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (1, 32, 128), (3, 96, 64), (17, 704, 128), (2328, 768, 64), (5, 4096, 32), (1, 160, 128)])
def test_quantize(N, K, group, zeros, dtype):
    g = torch.Generator(device="cuda").manual_seed(N + K)
    w = (torch.randn(N, K, device="cuda", generator=g) * torch.exp(torch.randn(N, 1, device="cuda", generator=g))).to(dtype)
    w[0, :32] = 0.0                                                   # a stretch (at group 32 a group) without range
    if N > 2:
        w[1] = w[1].abs()                                             # one side of zero
        w[2] = -w[2].abs()
    got, (q, s, z) = int4.quantize(w, group, not zeros), levels(w, group, zeros)
    assert torch.equal(got.scales, s) and torch.equal(got.q, packed(q)) and (got.zeros is None if not zeros else torch.equal(got.zeros, z))
    for out in (BF, F32):
        back, v = int4.dequantize(got, out), value(got)
        # exact in fp32 for bf16 scales (8 + 5 bits), else one rounding; then one to the result's type
        assert back.dtype == out and torch.all((back.double() - v).abs() <= (2.0 ** -8 if out == BF else 0.0 if dtype == BF else U) * v.abs() * (1 + 2 * U) + (U * v.abs() if out == BF else 0))
    step = spread(s, got, K)
    # nearest level: half a step and the fp32 quotient's rounding, and at the ends what rounding the scale took from the range (15 levels of 2^-8 of a step)
    assert torch.all((value(got) - w.double()).abs() <= (0.5 + (16 * 2.0 ** -8 if dtype == BF else 32 * U) + 1e-6) * step + (0 if zeros else 0))


@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_ties_and_extremes(dtype, zeros):
    """Quotients that are ties, next to ties, huge and subnormal: the formulas' own levels."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = [torch.arange(128, device="cuda") % 31 - 15.0]             # ends at +-15: quotients of halves and wholes
    rows[0] = rows[0] / 2
    rows += [torch.where(torch.rand(128, device="cuda", generator=g) < 0.5, 7.0, 3.5) * s for s in (1.0, 2.0 ** -130, 2.0 ** 100, 3e-45)]
    rows += [torch.randint(-40, 41, (128,), device="cuda", generator=g).float() * s for s in (2.0 ** -149, 2.0 ** -133, 2.0 ** -126, 1e-30, 1e37 / 4)]
    rows += [(torch.randint(-64, 65, (128,), device="cuda", generator=g).float() + 0.5) / 9.0, torch.randn(128, device="cuda", generator=g).to(BF).float()]
    w = torch.stack(rows).repeat(64, 1)
    w[::7] *= torch.randint(1, 256, (w[::7].shape[0], 1), device="cuda", generator=g)
    w = w.clamp(-1e37, 1e37).to(dtype)
    for group in (32, 128):
        got, (q, s, z) = int4.quantize(w, group, not zeros), levels(w, group, zeros)
        assert torch.equal(got.scales, s) and torch.equal(got.q, packed(q)) and (not zeros or torch.equal(got.zeros, z))


def test_quantize_what_is_no_number():
    w = torch.randn(4, 128, device="cuda")
    w[0, 3], w[1, 70], w[2, 127] = math.inf, math.nan, -math.inf
    w[3, 0], w[3, 1] = 3e38, -3e38                                    # a range that leaves fp32
    for dtype, zeros in ((F32, True), (BF, True), (F32, False)):
        got = int4.quantize(w.to(dtype), 64, not zeros)
        back = int4.dequantize(got)
        want = torch.zeros(4, 2, dtype=torch.bool, device="cuda")
        want[0, 0] = want[1, 1] = want[2, 1] = True
        want[3, 0] = zeros
        assert torch.equal(back.isnan(), want.repeat_interleave(64, 1)) and torch.equal(got.scales.isnan(), want)


def check_linear(x, w, bias, act, out, y):
    N, K = w.shape
    v, x64 = value(w), x.reshape(-1, K).double()
    y64, A = x64 @ v.t(), x64.abs() @ v.abs().t()
    if bias is not None:
        y64, A = y64 + bias.double(), A + bias.double().abs()
    G = w.scales.shape[1]
    tol = 2 * U * (K + 2 * G + 4) * A + (2.0 ** -22 * A if x.dtype == F32 else 0.0)
    M, rounded = x64.shape[0], x.dtype == BF and out == BF and x64.shape[0] > ROWS
    lin = y64
    if act:
        y64 = y64 * torch.special.ndtr(y64)
        tol = 1.13 * tol + 16 * U * lin.abs() + 2.0 ** -126
    half = 2.0 ** -8 if out == BF else U
    d = (y.reshape(-1, N).double() - y64).abs()
    assert y.dtype == out and y.shape == (*x.shape[:-1], N)
    if not rounded:
        assert torch.all(d <= tol + half * (y64.abs() + tol)), float((d / (tol + half * y64.abs())).max())
        return
    wide = tol + (1.13 if act else 1.0) * 2.0 ** -8 * A
    if act:
        wide = wide + 3.4e-5                                          # the tensor-core kernel's GELU against the erf form
    assert torch.all(d <= wide + half * (y64.abs() + wide)), float((d / wide).max())
    var = (x64 ** 2 @ (v ** 2).t()).sum() * (2.0 ** -8) ** 2 / 3 * (1.13 ** 2 if act else 1.0) + (y64 ** 2).sum() * (2.0 ** -8) ** 2 / 3 + (M * N * 3.4e-5 ** 2 if act else 0)
    if M * N >= 4096:                                                 # enough values for their mean
        assert float(d.norm()) <= 1.3 * float(var.sqrt()) + float(tol.norm())


SHAPES = [(1, 768, 768), (1, 32, 1), (1, 64, 7), (2, 96, 33), (7, 704, 2816), (8, 2816, 704), (9, 160, 65), (16, 768, 2328), (17, 768, 100), (33, 1024, 129), (64, 2048, 512),
          (65, 96, 300), (127, 704, 257), (128, 768, 768), (129, 416, 130), (300, 768, 513), (513, 2048, 1000)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("x_dtype,scale_dtype,out", [(BF, BF, BF), (BF, BF, F32), (F32, F32, F32), (BF, F32, BF), (F32, BF, BF)])
def test_linear(M, K, N, x_dtype, scale_dtype, out):
    i = SHAPES.index((M, K, N))
    group, zeros, act, with_bias = (32, 64, 128)[i % 3], i % 2 == 0, (None, "gelu")[(i // 2) % 2], i % 4 != 1
    w = random_weight(N, K, group, zeros, scale_dtype, i)
    g = torch.Generator(device="cuda").manual_seed(100 + i)
    x = torch.randn(M, K, device="cuda", generator=g).to(x_dtype)
    bias = torch.randn(N, device="cuda", generator=g).to(x_dtype) if with_bias else None
    y = int4.linear(x, w, bias, act=act, out_dtype=out)
    check_linear(x, w, bias, act, out, y)
    assert torch.equal(y, int4.linear(x, w, bias, act=act, out_dtype=out))


LARGE = [(4096, 160, 1900), (129, 96, 28500), (8197, 416, 1000), (16384, 32, 1001), (256, 704, 50257), (2000, 2048, 4099), (896, 128, 16384)]


@pytest.mark.parametrize("M,K,N", LARGE)
@pytest.mark.parametrize("scale_dtype", [BF, F32])
def test_linear_of_many_tiles(M, K, N, scale_dtype):
    """From one to several tiles a CTA, ends that fill no tile, one stretch of columns and many."""
    i = LARGE.index((M, K, N))
    w = random_weight(N, K, (64, 32, 128)[i % 3], i % 2 == 0, scale_dtype, i)
    g = torch.Generator(device="cuda").manual_seed(200 + i)
    x = torch.randn(M, K, device="cuda", generator=g).to(BF)
    bias = torch.randn(N, device="cuda", generator=g).to(BF) if i % 3 != 1 else None
    act = "gelu" if i % 2 else None
    y = int4.linear(x, w, bias, act=act)
    check_linear(x, w, bias, act, BF, y)
    assert torch.equal(y, int4.linear(x, w, bias, act=act))


EXACT = [(9, 2048, 4100), (17, 96, 60001), (20, 14048, 410), (33, 1024, 5000), (200, 416, 2003), (2000, 32, 4099), (129, 160, 8190), (64, 768, 50257), (1000, 4096, 130), (4100, 704, 704), (11000, 4096, 40)]


@pytest.mark.parametrize("M,K,N", EXACT)
@pytest.mark.parametrize("x_dtype,scale_dtype,out", [(BF, BF, F32), (F32, BF, F32), (F32, F32, F32), (BF, F32, F32), (F32, BF, BF)])
def test_linear_in_full_precision(M, K, N, x_dtype, scale_dtype, out):
    """Many rows, x or the result in float32: no weight is rounded. From one share of K to eight, ends that fill no tile."""
    i = EXACT.index((M, K, N))
    w = random_weight(N, K, (64, 32, 128)[(i + (scale_dtype == F32)) % 3], i % 2 == 0, scale_dtype, i)
    g = torch.Generator(device="cuda").manual_seed(300 + i)
    x = torch.randn(M, K, device="cuda", generator=g).to(x_dtype)
    bias = torch.randn(N, device="cuda", generator=g).to(x_dtype) if i % 3 != 1 else None
    act = "gelu" if i % 2 else None
    y = int4.linear(x, w, bias, act=act, out_dtype=out)
    check_linear(x, w, bias, act, out, y)
    assert torch.equal(y, int4.linear(x, w, bias, act=act, out_dtype=out))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_linear_groups_in_full_precision(group, zeros, dtype):
    K, N, M = 416, 1000, 2000
    w = random_weight(N, K, group, zeros, dtype, 3)
    rows = torch.arange(M, device="cuda")
    cols, f = rows * 7 % K, (1.0 + rows * 2.0 ** -13)                 # in float32 twelve bits and more, which only the sum of a value's terms has
    for x_dtype in (F32, BF):
        x = torch.zeros(M, K, device="cuda", dtype=x_dtype)
        x[rows, cols] = f.to(x_dtype)
        want = value(w).t()[cols] * x[rows, cols].double()[:, None]
        y = int4.linear(x, w, out_dtype=F32).double()
        assert torch.all((y - want).abs() <= 2.0 ** -23 * want.abs())     # the product of x and the whole number, and that by the scale, are rounded


def test_full_precision_carries_what_is_no_number():
    M, K, N = 100, 704, 3000
    w = random_weight(N, K, 64, False, BF, 5)
    x = torch.randn(M, K, device="cuda")
    x[3, 7], x[50, 700], x[99, 0] = math.inf, math.nan, -math.inf
    x[7] *= 1e-30
    w.scales[5, 2] = math.nan
    q = w.q.clone()
    q[:, 3] |= 0x90                                                   # no weight of column 7 is 0
    w = w._replace(q=q)
    y, v = int4.linear(x, w), value(w)
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[50], bad[:, 5] = True, True
    bad[99] |= v[:, 0] == 0
    want = x.double() @ v.t()
    assert torch.equal(y.isnan(), bad)
    inf = torch.zeros_like(bad)
    inf[3] = inf[99] = True
    inf &= ~bad
    assert torch.equal(y.isinf(), inf) and torch.equal(y[inf].double(), want[inf])
    rest = ~(bad | inf)
    A = x.double().abs().nan_to_num(0, 0, 0) @ v.abs().nan_to_num(0).t()
    assert torch.all((y.double() - want).abs()[rest] <= (2 * U * (K + 2 * 11 + 4) * A + 2.0 ** -22 * A)[rest])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [True, False])
def test_linear_groups_of_many_tiles(group, zeros):
    K, N, M = 416, 4000, 2000
    w = random_weight(N, K, group, zeros, BF, 3)
    x = torch.zeros(M, K, device="cuda", dtype=BF)
    cols = (torch.arange(M, device="cuda") * 7) % K
    x[torch.arange(M, device="cuda"), cols] = 1.0
    v = value(w).t()[cols]
    assert torch.all((int4.linear(x, w).double() - v).abs() <= 2.0 ** -8 * v.abs())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("M", [1, 5, 12, 40, 200])
def test_linear_groups(M, group, zeros):
    """Every column and group has its own weight in the result: rows of x that are unit vectors read the weight back."""
    K, N = 416, 70
    w = random_weight(N, K, group, zeros, BF, 3)
    x = torch.zeros(M, K, device="cuda", dtype=BF)
    cols = (torch.arange(M, device="cuda") * 7) % K
    x[torch.arange(M, device="cuda"), cols] = 1.0
    y = int4.linear(x, w, out_dtype=F32 if M <= ROWS else None)
    v = value(w).t()[cols]
    assert torch.all((y.double() - v).abs() <= (0.0 if M <= ROWS else 2.0 ** -8) * v.abs())


def test_linear_views_strides_and_empty():
    K, N = 256, 72
    w = random_weight(N, K, 64, True, BF, 5)
    big = torch.randn(9, 2 * K + 8, device="cuda").to(BF)
    whole = torch.randn(40, K, device="cuda").to(BF)
    for x in (big[:, 3:3 + K], big[:, 8:8 + K], whole[::3], whole.view(4, 10, K), whole.t().contiguous().t(), whole[:0], whole[0], big.flatten()[1:1 + 4 * K].view(4, K)):
        y = int4.linear(x, w)
        assert y.shape == (*x.shape[:-1], N)
        if x.numel():
            assert torch.equal(y, int4.linear(x.contiguous().clone(), w))
            check_linear(x, w, None, None, BF, y)
    part = int4.Int4Weight(w.q[8:40], w.scales[8:40], w.zeros[8:40], 64)       # rows of a held weight are a held weight
    assert torch.equal(int4.linear(whole[:4], part), int4.linear(whole[:4], w)[:, 8:40])
    wide = torch.zeros(N, K, dtype=torch.uint8, device="cuda")                  # levels, scales and zeros in every second column of something, made dense just ahead of the kernel
    wide[:, ::2] = w.q
    assert torch.equal(int4.linear(whole[:4], w._replace(q=wide[:, ::2], scales=w.scales.t().contiguous().t()), constant=True), int4.linear(whole[:4], w))
    odd = torch.empty(N * K // 2 + 1, dtype=torch.uint8, device="cuda")[1:].view(N, K // 2).copy_(w.q)      # levels that begin at an odd address
    assert torch.equal(int4.linear(whole[:4], w._replace(q=odd)), int4.linear(whole[:4], w))


def test_linear_carries_what_is_no_number():
    K, N = 128, 40
    for M in (3, 50):
        w = random_weight(N, K, 32, True, BF, 6)
        x = torch.randn(M, K, device="cuda").to(BF)
        x[1, 5], x[2, 77] = math.nan, math.inf
        w.scales[7, 2] = math.nan
        y = int4.linear(x, w)
        assert y[1].isnan().all() and not y[2, torch.arange(N) != 7].isfinite().any() and y[:, 7].isnan().all()
        assert y[0, torch.arange(N) != 7].isfinite().all()


def test_linear_refusals():
    w = random_weight(40, 128, 64, True, BF)
    x = torch.randn(3, 128, device="cuda").to(BF)
    for bad, err in ((lambda: int4.linear(x[:, :96], w), ValueError), (lambda: int4.linear(x.half(), w), TypeError), (lambda: int4.linear(x, w, torch.zeros(39, device="cuda")), ValueError),
                     (lambda: int4.linear(x, w._replace(group=32)), ValueError), (lambda: int4.linear(x, w._replace(group=48)), ValueError),
                     (lambda: int4.linear(x, w._replace(zeros=w.zeros[:, :1])), ValueError), (lambda: int4.linear(x, w._replace(scales=w.scales.half())), TypeError),
                     (lambda: int4.linear(x, w._replace(q=w.q.int())), TypeError), (lambda: int4.linear(x, w._replace(q=w.q.cpu())), RuntimeError),
                     (lambda: int4.linear(x, w._replace(q=w.q[:, :56])), ValueError), (lambda: int4.quantize(x[:, :100]), ValueError), (lambda: int4.quantize(x.half()), TypeError),
                     (lambda: int4.quantize(x, 256), ValueError), (lambda: int4.quantize(x[0]), ValueError)):
        with pytest.raises(err):
            bad()
    with torch.enable_grad():
        for call in (lambda: int4.linear(x.clone().requires_grad_(), w), lambda: int4.linear(x, w, torch.zeros(40, device="cuda", requires_grad=True)),
                     lambda: int4.quantize(x.clone().requires_grad_()), lambda: int4.linear(x, w._replace(scales=w.scales.clone().requires_grad_())),
                     lambda: int4.dequantize(w._replace(scales=w.scales.clone().requires_grad_()))):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
    with torch.no_grad():
        assert int4.linear(x.clone().requires_grad_(), w).shape == (3, 40)


@pytest.mark.parametrize("M", [1, 12, 40, 300, 10000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_in_a_graph_and_on_another_stream(M, dtype):
    K, N = 768, 776
    w = random_weight(N, K, 64, True, BF, 8)
    x = torch.randn(M, K, device="cuda").to(dtype)
    want = int4.linear(x, w)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    held = torch.zeros_like(x)
    with warm_up(side):
        int4.linear(held, w)
    with graph_capture(graph, side):
        y = int4.linear(held, w)
        z = int4.linear(y[:, :K].contiguous(), w, constant=True)
    held.copy_(x)
    graph.replay()
    assert torch.equal(y, want) and torch.equal(z, int4.linear(want[:, :K].contiguous(), w))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = int4.linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)


def test_streams_side_by_side():
    """Clusters that exchange sums, on two streams at once and beside another kernel's with tensor memory of their own."""
    K, N = 2048, 1000
    w = random_weight(N, K, 64, True, BF, 12)
    g = torch.Generator(device="cuda").manual_seed(5)
    a, b = torch.randn(64, K, device="cuda", generator=g).to(BF), torch.randn(120, K, device="cuda", generator=g)
    W = (torch.randn(N, K, device="cuda", generator=g) * 0.02).to(BF)
    calls = (lambda: int4.linear(a, w, act="gelu"), lambda: int4.linear(b, w), lambda: ops.batch_linear(a[:16], W), lambda: int4.linear(a, w, out_dtype=F32))
    want = [f() for f in calls]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    out = [[] for _ in streams]
    for i in range(20):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                k = (i + j) % len(calls)
                out[j].append((k, calls[k]()))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[k]) for o in out for k, y in o)


@pytest.mark.parametrize("M", [1, 40, 2000])
def test_a_weight_made_just_ahead(M):
    """Levels, scales and activations that the kernels right ahead on the stream write: read behind them."""
    K, N = 2048, 4096
    x = torch.randn(M, K, device="cuda").to(BF)
    ws = [torch.randn(N, K, device="cuda").to(BF) for _ in range(4)]
    buf = int4.quantize(ws[0])
    for w in ws:
        new = int4.quantize(w)
        want = int4.linear(x, new).clone()
        torch.cuda.synchronize()
        for a, b in zip(buf[:3], new[:3]):
            a.fill_(1)
            a.copy_(b)
        assert torch.equal(int4.linear(x, buf), want)


def test_run_together():
    """A feed-forward block in four bits, quantised, stepped and read back, against the same block with the weights read back."""
    d, ff = 704, 2816
    g = torch.Generator(device="cuda").manual_seed(4)
    A, B = (torch.randn(*s, device="cuda", generator=g).mul_(0.03).to(BF) for s in ((ff, d), (d, ff)))
    wa, wb = int4.quantize(A, 64), int4.quantize(B, 128, symmetric=True)
    for M in (1, 5, 64):
        x = torch.randn(M, d, device="cuda", generator=g).to(BF)
        h = int4.linear(x, wa, act="gelu")
        y = int4.linear(h, wb, out_dtype=F32)
        check_linear(x, wa, None, "gelu", BF, h)
        check_linear(h, wb, None, None, F32, y)


def test_compiled():
    w = random_weight(200, 256, 64, True, BF, 9)
    x = torch.randn(5, 256, device="cuda").to(BF)

    def f(x):
        return int4.linear(x, w, act="gelu") + 1
    with torch.no_grad():
        assert torch.equal(torch.compile(f, fullgraph=True)(x), f(x))
