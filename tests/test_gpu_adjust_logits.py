"""Penalties, biases and masks on logits, against their definition in 64 bits. Every step is one rounded fp32 operation: a result is off by u = 2^-24 of what each
of the up to 2 + (biases of the word) + 3 steps holds, whose size the sum of the magnitudes bounds."""
import math

import pytest
import torch

from pragnosia_b200 import sampling
from pragnosia_b200._lib import graph_capture, warm_up

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def want(logits, prompt=None, prompt_lengths=None, generated=None, generated_lengths=None, repetition=1.0, frequency=0.0, presence=0.0, bias_ids=None, bias=None, mask=None):
    """(result, bound) on the CPU in 64 bits."""
    B, V = logits.shape
    cpu = lambda t: t.cpu() if torch.is_tensor(t) else t
    row = lambda t, b: t[b if t.shape[0] > 1 else 0]
    num = lambda v, b: float(cpu(v)[b].float()) if torch.is_tensor(v) else float(torch.tensor(v, dtype=F32))
    out, tol = logits.double().cpu().clone(), torch.zeros(B, V, dtype=torch.float64)
    for b in range(B):
        def count(ids, lengths):
            c = torch.zeros(V, dtype=torch.float64)
            if ids is None:
                return c
            r = row(cpu(ids), b).long()
            if lengths is not None:
                n = cpu(lengths).reshape(-1)
                r = r[:max(0, int(n[b if n.numel() > 1 else 0]))]
            r = r[(r >= 0) & (r < V)]
            return c + torch.bincount(r, minlength=V)
        n, m = count(generated, generated_lengths), count(prompt, prompt_lengths)
        r, f, p = num(repetition, b), num(frequency, b), num(presence, b)
        s = out[b]
        seen = (n + m) > 0
        s = torch.where(seen, torch.where(s > 0, s / r, s * r), s)
        size = s.abs() + (abs(f) * n + abs(p)) * (n > 0)
        s = torch.where(n > 0, s - f * n - p, s)
        steps = torch.full((V,), 6.0, dtype=torch.float64)
        if bias_ids is not None:
            for v, x in zip(row(cpu(bias_ids), b).tolist(), row(cpu(bias), b).double().tolist()):
                if 0 <= v < V:
                    s[v] += x
                    size[v] += abs(x)
                    steps[v] += 1
        if mask is not None:
            ok = row(cpu(mask), b)
            if ok.dtype == torch.int32:
                ok = ((ok.long()[:, None] >> torch.arange(32)) & 1).flatten()[:V].bool()
            s = torch.where(ok, s, torch.full_like(s, -math.inf))
        out[b], tol[b] = s.float().double(), (steps + 1) * U * size   # a result past fp32's range (its lowest value times a repetition) is an infinity
    return out, tol


def check(logits, got=None, **kw):
    ref, tol = want(logits, **kw)
    y = sampling.adjust_logits(logits, **kw) if got is None else got
    assert y.dtype == F32 and y.shape == logits.shape
    y = y.double().cpu()
    assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y.isinf(), ref.isinf()) and torch.equal(y[ref.isinf()], ref[ref.isinf()])
    fine = ref.isfinite()
    assert torch.all((y - ref).abs()[fine] <= tol[fine])


def make(B, V, n=40, k=5, seed=0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = lambda *s: torch.randint(-2, V + 2, s, device="cuda", generator=g)                # padding and ids past the end among them
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    ok = torch.rand(B, V, device="cuda", generator=g) < 0.4
    W = -(-V // 32)
    bits = (torch.nn.functional.pad(ok, (0, 32 * W - V)).view(B, W, 32).long() << torch.arange(32, device="cuda")).sum(2).to(torch.int32)
    return dict(logits=(4 * rnd(B, V)).to(dtype), prompt=ids(B, n), generated=ids(B, n // 2 + 1), bias_ids=ids(B, k), bias=rnd(B, k), ok=ok, bits=bits,
                rows=lambda lo, hi: lo + (hi - lo) * torch.rand(B, device="cuda", generator=g), ids=ids, rnd=rnd)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,V", [(1, 1), (1, 31), (2, 33), (3, 2048), (2, 2049), (1, 8192), (5, 4097), (2, 50257)])
def test_all_of_it(B, V, dtype):
    x = make(B, V, seed=V + B, dtype=dtype)
    one = dict(prompt=x["prompt"], generated=x["generated"], bias_ids=x["bias_ids"], bias=x["bias"])
    check(x["logits"])
    check(x["logits"], **one, repetition=1.3, frequency=0.4, presence=-0.2, mask=x["bits"])
    check(x["logits"], **one, repetition=x["rows"](0.5, 2), frequency=x["rows"](-1, 1), presence=x["rows"](-1, 1).to(BF), mask=x["ok"])
    check(x["logits"], mask=x["bits"][:1])
    check(x["logits"], mask=x["ok"][:1], prompt=x["prompt"][:1], repetition=2.0, bias_ids=x["bias_ids"][:1], bias=x["bias"][:1])


@pytest.mark.parametrize("n", [1, 255, 4096, 5000, 33000])
def test_histories_and_their_lengths(n):
    B, V = 3, 5003
    x = make(B, V, n=n, seed=n)
    gen = x["ids"](B, 4097) if n == 5000 else x["generated"]
    kw = dict(repetition=1.2, frequency=0.3, presence=0.1)
    lengths = torch.tensor([0, n // 2, n + 7], device="cuda")
    check(x["logits"], prompt=x["prompt"], prompt_lengths=lengths, generated=gen, generated_lengths=torch.tensor([gen.shape[1], 0, 1], device="cuda"), **kw)
    check(x["logits"], prompt=x["prompt"], prompt_lengths=-lengths, generated=gen.int(), generated_lengths=torch.tensor([1], device="cuda", dtype=torch.int32), **kw)
    check(x["logits"], prompt=x["prompt"][:, ::2], generated=x["prompt"].t().contiguous().t(), **kw)
    check(x["logits"], generated=torch.full((B, n), 17, device="cuda"), **kw)                 # one word, over and over
    check(x["logits"], prompt=x["prompt"][:, :0], generated=gen[:, :0], **kw)
    check(x["logits"], prompt=x["prompt"][1:2].expand(B, n), prompt_lengths=torch.tensor(n, device="cuda"), **kw)


def test_biases_of_the_same_word():
    """An id twice counts twice, in the order given: the same bits as adding them up one by one."""
    V = 3000
    l = torch.randn(2, V, device="cuda")
    ids = torch.tensor([[5, 2999, 5, -1, 5, 2999, V, 0] * 100, list(range(800))], device="cuda")
    b = torch.randn(2, 800, device="cuda") * 100
    y = sampling.adjust_logits(l, bias_ids=ids, bias=b)
    for v in (5, 2999, 0):
        s = torch.zeros((), device="cuda")
        for x in b[0][ids[0] == v]:
            s = s + x
        assert torch.equal(y[0, v], l[0, v] + s)
    check(l, got=y, bias_ids=ids, bias=b)
    check(l, bias_ids=torch.full((2, 1024), 7, device="cuda"), bias=torch.randn(2, 1024, device="cuda"))
    check(l, bias_ids=torch.full((1, 1), 7, device="cuda"), bias=torch.full((1, 1), -math.inf, device="cuda"))


def test_rows_without_a_word_and_what_is_no_number():
    V = 300
    l = torch.randn(4, V, device="cuda")
    l[0, 3], l[1, 4], l[2, 5], l[3, 6] = math.nan, math.inf, -math.inf, torch.finfo(F32).min
    ok = torch.ones(4, V, dtype=torch.bool, device="cuda")
    ok[0] = False
    ok[1, 4] = False
    every = torch.arange(V, device="cuda")[None]
    check(l, mask=ok, generated=every, repetition=1.5, frequency=0.1)
    y = sampling.adjust_logits(l, mask=ok)
    assert (y[0] == -math.inf).all() and y[1, 4] == -math.inf and y[2, 5] == -math.inf
    check(l, generated=every, repetition=1.5)


def test_rows_with_a_stride_and_in_place():
    V = 515
    big = torch.randn(3, 800, device="cuda")
    kw = dict(generated=torch.randint(0, V, (3, 20), device="cuda"), frequency=0.5)
    for l in (big[:, :V], big[:, 1:V + 1], big.t()[:V].t(), big[::2, :V][:, ::1][:2].expand(2, V), big.to(BF)[:, 3:V + 3]):
        check(l, **(kw if l.shape[0] == 3 else {}))
    l = big[:, :V].contiguous()
    ref = sampling.adjust_logits(l, **kw)
    out = torch.empty_like(l)
    assert sampling.adjust_logits(l, **kw, out=out) is not None and torch.equal(out, ref)
    got = sampling.adjust_logits(l, **kw, out=l)
    assert got.data_ptr() == l.data_ptr() and torch.equal(l, ref)
    both = torch.randn(2 * 3 * V, device="cuda")                      # rows that overlap where the result goes
    l, out = both[:3 * V].view(3, V), both[V:4 * V].view(3, V)
    ref = sampling.adjust_logits(l, **kw)
    assert torch.equal(sampling.adjust_logits(l, **kw, out=out), ref) and torch.equal(out, ref)
    one = big[0:1, :V]
    ref = sampling.adjust_logits(one, frequency=0.0, bias_ids=torch.zeros(1, 1, dtype=torch.long, device="cuda"), bias=torch.ones(1, 1, device="cuda"))
    assert torch.equal(sampling.adjust_logits(one, bias_ids=torch.zeros(1, 1, dtype=torch.long, device="cuda"), bias=torch.ones(1, 1, device="cuda"), out=one), ref)
    assert sampling.adjust_logits(big[:0]).shape == (0, 800)


def test_refusals():
    l = torch.randn(2, 50, device="cuda")
    ids, b = torch.zeros(2, 3, dtype=torch.long, device="cuda"), torch.zeros(2, 3, device="cuda")
    f = sampling.adjust_logits
    for bad, err in ((lambda: f(l[0]), ValueError), (lambda: f(l.half()), TypeError), (lambda: f(l, prompt=ids.float()), TypeError), (lambda: f(l, prompt=ids[0]), ValueError),
                     (lambda: f(l, prompt=ids.expand(2, 2, 3)), ValueError), (lambda: f(l, prompt=torch.zeros(3, 3, dtype=torch.long, device="cuda")), ValueError),
                     (lambda: f(l, prompt_lengths=ids[:, 0]), ValueError), (lambda: f(l, prompt=ids, prompt_lengths=torch.zeros(3, dtype=torch.long, device="cuda")), ValueError),
                     (lambda: f(l, repetition=0.0), ValueError), (lambda: f(l, repetition=-1.0), ValueError), (lambda: f(l, repetition=torch.ones(3, device="cuda")), ValueError),
                     (lambda: f(l, frequency=torch.ones(2, device="cuda", dtype=torch.long)), ValueError), (lambda: f(l, bias=b), ValueError), (lambda: f(l, bias_ids=ids), ValueError),
                     (lambda: f(l, bias_ids=ids, bias=b[:, :2]), ValueError), (lambda: f(l, bias_ids=ids.repeat(1, 400), bias=b.repeat(1, 400)), ValueError),
                     (lambda: f(l, mask=torch.zeros(2, 1, dtype=torch.int32, device="cuda")), ValueError), (lambda: f(l, mask=torch.zeros(2, 49, dtype=torch.bool, device="cuda")), ValueError),
                     (lambda: f(l, mask=torch.zeros(2, 2, device="cuda")), TypeError), (lambda: f(l, out=l.to(BF)), ValueError), (lambda: f(l, out=l.t().contiguous().t()), ValueError),
                     (lambda: f(l, prompt=ids.cpu()), RuntimeError), (lambda: f(l, mask=torch.zeros(2, 2, dtype=torch.int32)), RuntimeError)):
        with pytest.raises(err):
            bad()
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no gradient"):
        f(l.clone().requires_grad_())
    leaf = torch.ones(l.shape[0], device=l.device, requires_grad=True)
    for kw in (dict(repetition=leaf), dict(frequency=leaf), dict(presence=leaf), dict(bias_ids=torch.zeros(1, 1, dtype=torch.long, device=l.device), bias=leaf[:1, None])):
        with torch.enable_grad(), pytest.raises(RuntimeError, match="no gradient"):
            f(l, **kw)
        with torch.no_grad():
            assert f(l, **kw).shape == l.shape


def test_in_a_graph_with_a_counter_on_the_device():
    """The loop of a decoder: history and its length live on the device, and a replay sees what the last one left."""
    B, V = 2, 4099
    x = make(B, V, seed=3)
    hist, cnt = torch.randint(0, V, (B, 30), device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda")
    kw = dict(prompt=x["prompt"], generated=hist, generated_lengths=cnt, repetition=1.1, frequency=0.2, presence=0.1, mask=x["bits"])
    side, graph, buf = torch.cuda.Stream(), torch.cuda.CUDAGraph(), x["logits"].clone()
    with warm_up(side):
        sampling.adjust_logits(buf, **kw)
    with graph_capture(graph, side):
        y = sampling.adjust_logits(buf, **kw)
        cnt.add_(1)
    for i in range(5):
        cnt.fill_(7 * i)
        graph.replay()
        check(x["logits"], got=y, **{**kw, "generated_lengths": torch.tensor([7 * i])})


def test_compiled():
    x = make(2, 500, seed=9)
    f = lambda l, i, r: sampling.adjust_logits(l, generated=i, repetition=r, presence=0.5) * 2
    with torch.no_grad():
        r = x["rows"](1, 2)
        assert torch.equal(torch.compile(f, fullgraph=True)(x["logits"], x["generated"], r), f(x["logits"], x["generated"], r))
