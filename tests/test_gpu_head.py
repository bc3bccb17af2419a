"""The losses over the vocabulary and the embedding against their definitions in 64 bits, at the sizes and masks where they can go wrong.

Tolerances count roundings. A logit is a sum of d products whose fp32 partial sums, at most A = sum |h w|, are rounded once per 16
products (6 times as often with fp32 operands): ds <= (steps + 2) 2^-23 A. The loss is off by at most 2 ds and a few fp32 roundings of its
terms. ds_nv, the logits' gradient, is off by q 2 ds and by its rounding to bf16 (2^-8 of itself; fp32 operands: 2^-23); the gradients behind it
are sums of its products, rounded once more to their own type."""
import math

import pytest
import torch

from pragnosia_b200 import head
from pragnosia_b200._lib import check, host, lib
from pragnosia_b200.model import LM

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _grad_enabled_and_waits_fine():
    import ctypes
    with torch.enable_grad():
        yield
    flag = ctypes.c_int(-1)
    check(lib().pgb_tc_error_flag(ctypes.byref(flag)), "pgb_tc_error_flag")
    assert flag.value == 0


def operands(N, V, d, dtype, seed, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.randn(N, d, device=DEV, generator=g).to(dtype)
    w = (spread / math.sqrt(d) * torch.randn(V, d, device=DEV, generator=g)).to(dtype)
    return h, w, g


def dense(h, w, p, live, tau, c, reduction):
    """(loss, dh, dw) and what each may be off by. p (N,V): target distributions; live (N); c (N): weights of the rows (none)."""
    dtype, (N, d), V = h.dtype, h.shape, w.shape[0]
    h, w, p = h.double(), w.double(), p.double()
    s = h @ w.t()
    logq = torch.log_softmax(s / tau, 1)
    q = logq.exp()
    rows = tau * tau * (torch.special.xlogy(p, p) - p * logq).sum(1)
    rows = torch.where(live, rows, torch.zeros_like(rows))
    n = live.sum()
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / n}[reduction]
    cs = c.double() if reduction == "none" else torch.full((N,), 1.0 / max(1, int(n)) if reduction == "mean" else 1.0, device=DEV, dtype=torch.float64)
    cs = torch.where(live, cs, torch.zeros_like(cs)) * tau
    ds = cs[:, None] * (q - p)
    dh, dw = ds @ w, ds.t() @ h
    steps = (1 if dtype == BF else 6) * math.ceil(d / 16) + 2
    ds_s = steps * 2.0 ** -23 * (h.abs() @ w.abs().t()).amax(1, keepdim=True)      # of a logit, by row
    e_rows = (tau * 2 * ds_s[:, 0] + tau * tau * 2.0 ** -21 * (1 + logq.abs().amax(1))) * live
    e_loss = {"none": e_rows, "sum": e_rows.sum() + 2.0 ** -23 * rows.sum().abs(), "mean": (e_rows.sum() + 2.0 ** -23 * rows.sum().abs()) / max(1, int(n))}[reduction]
    half, half_ds = (2.0 ** -8, 2.0 ** -8) if dtype == BF else (2.0 ** -24, 2.0 ** -23)
    e_ds = cs.abs()[:, None] * q * (2 * ds_s / tau + 2.0 ** -20) + half_ds * ds.abs()
    acc = lambda k: ((1 if dtype == BF else 6) * math.ceil(k / 16) + 34) * 2.0 ** -23
    e_dh = (e_ds + acc(V) * ds.abs()) @ w.abs() + 1.01 * half * dh.abs() + 1e-37
    e_dw = (e_ds + acc(N) * ds.abs()).t() @ h.abs() + 1.01 * half * dw.abs() + 1e-37
    return (loss, dh, dw), (e_loss, e_dh, e_dw)


def within(got, want, off, names=("loss", "dh", "dw")):
    for name, a, b, e in zip(names, got, want, off):
        a = a.double()
        assert a.shape == b.shape, name
        assert torch.equal(torch.isnan(a), torch.isnan(b)), name
        over = ((a - b).abs() - e).nan_to_num(-1.0)
        assert (over <= 0).all(), f"{name}: off by {float((a - b).abs().nan_to_num(0).max()):.3e}, {int((over > 0).sum())} of {a.numel()} past their bound"


def xent(h, w, t, c, reduction, **kw):
    h, w = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = head.linear_cross_entropy(h, w, t, reduction=reduction, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, [h, w], c if reduction == "none" else None))


def one_hot(t, V, ignore=-100):
    live = t != ignore
    p = torch.zeros(t.numel(), V, device=DEV, dtype=torch.float64)
    p[torch.arange(t.numel(), device=DEV)[live], t[live]] = 1.0
    return p, live


SIZES = [(1, 1, 8), (3, 5, 8), (1, 257, 64), (2, 300, 24), (130, 1000, 72), (255, 256, 64), (256, 255, 128), (257, 513, 704), (511, 8192, 768), (64, 50257, 256),
         (1500, 130, 1536)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,d", SIZES)
def test_cross_entropy(N, V, d, dtype):
    h, w, g = operands(N, V, d, dtype, N + V)
    c = torch.rand(N, device=DEV, generator=g) - 0.3
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    for share, reduction in ((0.0, "mean"), (0.4, "none"), (0.4, "mean"), (0.2, "sum")):
        t2 = torch.where(torch.rand(N, device=DEV, generator=g) < share, torch.full_like(t, -100), t)
        p, live = one_hot(t2, V)
        if reduction == "mean" and not live.any():
            continue
        within(xent(h, w, t2, c, reduction), *dense(h, w, p, live, 1.0, c, reduction))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,d", [(9000, 6200, 64), (3000, 17000, 72)])
def test_cross_entropy_in_pieces(N, V, d, dtype):
    """More logits than the workspace takes at once: pieces along the rows, and along the vocabulary."""
    h, w, g = operands(N, V, d, dtype, 5)
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    t[::7] = -100
    c = torch.rand(N, device=DEV, generator=g)
    p, live = one_hot(t, V)
    for reduction in ("mean", "none"):
        within(xent(h, w, t, c, reduction), *dense(h, w, p, live, 1.0, c, reduction))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_cross_entropy_of_large_logits(dtype):
    """Logits of some hundreds: exponentials that overflow without the maximum, rows whose target holds all the probability or none of it."""
    h, w, g = operands(200, 700, 64, dtype, 3, spread=120.0)
    t = torch.randint(0, 700, (200,), device=DEV, generator=g)
    t[:50] = (h[:50].double() @ w.double().t()).argmax(1)
    p, live = one_hot(t, 700)
    within(xent(h, w, t, None, "mean"), *dense(h, w, p, live, 1.0, None, "mean"))


def test_no_row_counts():
    h, w, _ = operands(70, 300, 64, BF, 1)
    t = torch.full((70,), -100, device=DEV)
    loss, dh, dw = xent(h, w, t, None, "mean")
    assert math.isnan(float(loss)) and not dh.any() and not dw.any()
    loss, dh, dw = xent(h, w, t, None, "sum")
    assert float(loss) == 0.0 and not dh.any() and not dw.any()
    loss, dh, dw = xent(h, w, t, torch.ones(70, device=DEV), "none")
    assert not loss.any() and not dh.any() and not dw.any()
    for reduction, want in (("sum", 0.0), ("mean", math.nan)):
        loss, dh, dw = xent(h[:0], w, t[:0], None, reduction)
        assert (float(loss) == want or math.isnan(want) and math.isnan(float(loss))) and dh.shape == (0, 64) and not dw.any()


def test_targets_outside_the_vocabulary_give_nan():
    h, w, g = operands(300, 333, 64, BF, 2)
    t = torch.randint(0, 333, (300,), device=DEV, generator=g)
    for bad in (333, 340, 400, -1, 1 << 40, -(1 << 40)):
        t2 = t.clone(); t2[17] = bad
        loss, dh, dw = xent(h, w, t2, torch.ones(300, device=DEV), "none")
        assert math.isnan(float(loss[17])) and torch.isfinite(loss[:17]).all() and torch.isfinite(loss[18:]).all()
        assert torch.isnan(dh[17]).all() and torch.isfinite(dh[:17]).all() and torch.isfinite(dh[18:]).all() and torch.isnan(dw).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V", [(700, 300), (3000, 17000), (9000, 6200)])
def test_rows_that_do_not_count_may_hold_anything(N, V, dtype):
    """Infinities and NaN in ignored rows of h (padding that a kernel never wrote): the results are those with zeros there, to the bit."""
    h, w, g = operands(N, V, 72, dtype, 11)
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    dead = torch.rand(N, device=DEV, generator=g) < 0.2
    dead[-1] = True
    t[dead] = -100
    filled = h.clone()
    filled[dead] = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device=DEV)[torch.randint(0, 4, (int(dead.sum()), 72), device=DEV, generator=g)].to(dtype)
    h[dead] = 0
    ids, logits = lists(N, V, 3, g, False)
    ids[dead] = -1
    c = torch.rand(N, device=DEV, generator=g)
    for call in (lambda x: xent(x, w, t, c, "mean"), lambda x: xent(x, w, t, c, "none"), lambda x: distill(x, w, ids, logits, 2.0, c, "mean")):
        want, got = call(h), call(filled)
        assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(want, got))


def test_rows_past_32_bits():
    """h of more than 2^31 elements: its last rows are as they are by themselves."""
    N, V, d, n = 2_900_000, 70, 768, 300
    g = torch.Generator(device=DEV).manual_seed(3)
    h = torch.empty(N, d, device=DEV, dtype=BF).normal_(generator=g)
    w = (0.05 * torch.randn(V, d, device=DEV, generator=g)).to(BF)
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    c = torch.rand(N, device=DEV, generator=g)
    loss, dh, dw = xent(h, w, t, c, "none")
    p, live = one_hot(t[-n:], V)
    want, off = dense(h[-n:], w, p, live, 1.0, c[-n:], "none")
    within((loss[-n:], dh[-n:]), want[:2], off[:2])
    del loss, dh
    y, de = embed(t, w, h)
    assert torch.equal(y[-n:], w[t[-n:]])
    ref = torch.zeros(V, d, device=DEV, dtype=torch.float64)
    for a in range(0, N, 100_000):
        ref.index_add_(0, t[a:a + 100_000], h[a:a + 100_000].double())
    # chunks of 32 added one by one (32 roundings), their 1300 sums by eight threads: 163 + 8 roundings of sums of about 41400 normal numbers
    assert ((de.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 210 * 2.0 ** -24 * 41400 * 0.9).all()


def test_forms_of_the_call():
    """Leading axes, other strides and types of ids, a view off the 16-byte grid, one gradient alone, an ignore_index inside the vocabulary."""
    h, w, g = operands(12 * 31, 333, 64, BF, 4)
    t = torch.randint(0, 333, (12 * 31,), device=DEV, generator=g)
    c = torch.rand(12, 31, device=DEV, generator=g)
    want = xent(h, w, t, c.view(-1), "none")
    a = xent(h.view(12, 31, 64), w, t.view(12, 31).int(), c, "none")
    assert a[0].shape == (12, 31) and a[1].shape == (12, 31, 64)
    assert all(torch.equal(x.reshape(y.shape), y) for x, y in zip(a, want))
    # rows in another order, and one gradient alone: the K axis of the gradients' products is cut at other places, so the bits may differ
    p, live = one_hot(t, 333)
    ref, off = dense(h, w, p, live, 1.0, c.view(-1), "none")
    a = xent(h.view(12, 31, 64).transpose(0, 1), w.t().contiguous().t(), t.view(12, 31).t(), c.t(), "none")
    assert torch.equal(a[0].t().reshape(-1), want[0])
    within((want[0], a[1].transpose(0, 1).reshape(-1, 64), a[2]), ref, off)
    room = torch.empty(h.numel() + 1, device=DEV, dtype=BF)
    moved = room[1:].view_as(h).copy_(h)
    assert all(torch.equal(x, y) for x, y in zip(xent(moved, w, t, c.view(-1), "none"), want))
    for wrt in (0, 1):
        x = [h.clone(), w.clone()]
        x[wrt].requires_grad_()
        (got,) = torch.autograd.grad(head.linear_cross_entropy(*x, t, reduction="none"), [x[wrt]], c.view(-1))
        within((got,), ref[1 + wrt:2 + wrt], off[1 + wrt:2 + wrt])
    with torch.no_grad():
        assert torch.equal(head.linear_cross_entropy(h, w, t, reduction="none"), want[0])
    ig = int(t[5])
    got = xent(h, w, t, c.view(-1), "none", ignore_index=ig)
    p, live = one_hot(t, 333, ig)
    within(got, *dense(h, w, p, live, 1.0, c.view(-1), "none"))


def test_same_bits_every_time_and_in_a_graph():
    h, w, g = operands(700, 3000, 128, BF, 6)
    t = torch.randint(0, 3000, (700,), device=DEV, generator=g)
    want = xent(h, w, t, None, "mean")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(xent(h, w, t, None, "mean"), want))
    hs, ws, ts = h.clone().requires_grad_(), w.clone().requires_grad_(), t.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            loss = head.linear_cross_entropy(hs, ws, ts)
            out = (loss.detach(), *torch.autograd.grad(loss, [hs, ws]))
    for s in (0, 1):
        with torch.no_grad():
            hs.copy_(h.flip(0) if s else h); ts.copy_(t.flip(0) if s else t)
        graph.replay()
        torch.cuda.synchronize()
        again = xent(hs.detach(), w, ts, None, "mean")
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_upstream_gradient_and_accumulation():
    h, w, g = operands(300, 500, 64, F32, 7)
    t = torch.randint(0, 500, (300,), device=DEV, generator=g)
    one = xent(h, w, t, None, "mean")
    h2, w2 = h.clone().requires_grad_(), w.clone().requires_grad_()
    (3.0 * head.linear_cross_entropy(h2, w2, t)).backward()
    head.linear_cross_entropy(h2, w2, t).backward()
    assert torch.allclose(h2.grad, 4 * one[1], rtol=1e-6, atol=1e-9) and torch.allclose(w2.grad, 4 * one[2], rtol=1e-6, atol=1e-9)
    h2 = h.clone().requires_grad_()
    (gh,) = torch.autograd.grad(head.linear_cross_entropy(h2, w, t), [h2], create_graph=True)
    with pytest.raises(RuntimeError):
        gh.sum().backward()


def test_gradient_against_differences():
    """Along random directions, central differences of the fp32 loss: its error 2^-21 / step, the third derivative's step^2."""
    h, w, g = operands(40, 90, 32, F32, 8)
    t = torch.randint(0, 90, (40,), device=DEV, generator=g)
    _, dh, dw = xent(h, w, t, None, "mean")
    for x, dx, f in ((h, dh, lambda y: head.linear_cross_entropy(y, w, t)), (w, dw, lambda y: head.linear_cross_entropy(h, y, t))):
        u = torch.randn(x.shape, device=DEV, generator=g)
        u /= u.norm()
        step = 0.1
        with torch.no_grad():
            slope = (float(f(x + step * u)) - float(f(x - step * u))) / (2 * step)
        assert abs(slope - float((dx * u).sum())) < 2.0 ** -20 * 6 / step + step ** 2


# ------------------------------------------------------------------------------------------------ distillation
def lists(N, V, k, g, ragged):
    ids = torch.stack([torch.randperm(V, device=DEV, generator=g)[:k] for _ in range(N)])
    logits = 3.0 * torch.randn(N, k, device=DEV, generator=g)
    if ragged:
        n = torch.randint(0, k + 1, (N, 1), device=DEV, generator=g)
        gone = torch.arange(k, device=DEV).flip(0) >= n if k % 2 else torch.arange(k, device=DEV) >= n
        ids = torch.where(gone, torch.full_like(ids, -1), ids)
    return ids, logits


def teacher(ids, logits, V, tau):
    N, k = ids.shape
    z = torch.where(ids >= 0, logits.double() / tau, torch.full_like(logits, -math.inf, dtype=torch.float64))
    live = (z > -math.inf).any(1)
    p = torch.softmax(z, 1).nan_to_num(0.0)
    full = torch.zeros(N, V, device=DEV, dtype=torch.float64)
    full.scatter_add_(1, ids.clamp_min(0), p)
    return full, live, torch.special.xlogy(p, p).sum(1)


def distill(h, w, ids, logits, tau, c, reduction):
    h, w = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = head.linear_distill(h, w, ids, logits, temperature=tau, reduction=reduction)
    return (loss.detach(), *torch.autograd.grad(loss, [h, w], c if reduction == "none" else None))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,d,k", [(1, 8, 8, 1), (5, 40, 24, 40), (130, 1000, 72, 5), (257, 513, 704, 64), (300, 8192, 256, 33), (64, 50257, 128, 64), (20, 2000, 64, 1000)])
def test_distillation(N, V, d, k, dtype):
    h, w, g = operands(N, V, d, dtype, N + V + k)
    c = torch.rand(N, device=DEV, generator=g) - 0.3
    for tau, ragged, reduction in ((1.0, False, "mean"), (2.0, True, "none"), (0.5, True, "sum")):
        ids, logits = lists(N, V, k, g, ragged)
        p, live, _ = teacher(ids, logits, V, tau)
        want, off = dense(h, w, p, live, tau, c, reduction)
        # the teacher's probabilities are fp32: a few 2^-23 of themselves (exponential, sum, quotient: 2^-20 is enough)
        dp = 2.0 ** -20 * p
        cs = (c.abs() if reduction == "none" else torch.full_like(c, 1.0 / max(1, int(live.sum())) if reduction == "mean" else 1.0)).double()[:, None] * tau
        s = (h.double() @ w.double().t()).abs()
        e = tau * tau * ((dp * (s / tau + 20.0)).sum(1) + 2.0 ** -20 * (1 + (p * (p + 1e-300).log().abs()).sum(1)))
        e = {"none": e, "sum": e.sum(), "mean": e.sum() / max(1, int(live.sum()))}[reduction]
        off = (off[0] + e, off[1] + (cs * dp) @ w.double().abs(), off[2] + (cs * dp).t() @ h.double().abs())
        within(distill(h, w, ids, logits, tau, c, reduction), want, off)


def test_distillation_forms():
    """bf16 logits, int32 ids, leading axes, an entry twice, -inf entries, values behind absent ids that are not numbers, no rows."""
    h, w, g = operands(6 * 50, 400, 64, BF, 9)
    ids, logits = lists(300, 400, 7, g, False)
    logits = logits.to(BF).float()
    c = torch.rand(300, device=DEV, generator=g)
    want = distill(h, w, ids, logits, 1.5, c, "none")
    got = distill(h.view(6, 50, 64), w, ids.view(6, 50, 7).int(), logits.to(BF).view(6, 50, 7), 1.5, c.view(6, 50), "none")
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    # absent entries: by id or by logit, whatever stands beside them; order does not matter but for the sums' last bits
    pad_ids = torch.cat([ids, torch.full((300, 3), -1, device=DEV), torch.randint(0, 400, (300, 2), device=DEV, generator=g)], 1)
    pad_logits = torch.cat([logits, torch.tensor([math.nan, math.inf, 5.0], device=DEV).expand(300, 3), torch.full((300, 2), -math.inf, device=DEV)], 1)
    got = distill(h, w, pad_ids, pad_logits, 1.5, c, "none")
    assert all(torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-5) for a, b in zip(got, want))
    empty = ids.clone(); empty[::3] = -1
    logits2 = logits.clone(); logits2[1::3] = -math.inf
    loss, dh, dw = distill(h, w, empty, logits2, 1.5, c, "none")
    assert not loss[::3].any() and not loss[1::3].any() and not dh[::3].any() and not dh[1::3].any() and torch.equal(loss[2::3], want[0][2::3])
    # the same word twice is the word once with the probabilities added
    twice = torch.stack([ids[:, 0], ids[:, 1], ids[:, 0]], 1)
    z = logits[:, :3].contiguous()
    p, live, plogp = teacher(twice, z, 400, 1.0)
    ref, off = dense(h, w, p, live, 1.0, c, "none")
    ref = (ref[0] - torch.special.xlogy(p, p).sum(1) + plogp, *ref[1:])
    within(distill(h, w, twice, z, 1.0, c, "none"), ref, (off[0] + 1e-4, *(o + 1e-5 for o in off[1:])))
    assert torch.isnan(distill(h, w, torch.full_like(ids, 400), logits, 1.0, c, "none")[0]).all()
    loss, dh, dw = distill(h[:0], w, ids[:0], logits[:0], 1.0, None, "sum")
    assert float(loss) == 0.0 and dh.shape == (0, 64) and not dw.any()


# ------------------------------------------------------------------------------------------------ embedding
def embed(ids, w, gy, **kw):
    w = w.clone().requires_grad_()
    y = head.embedding(ids, w, **kw)
    return y.detach(), torch.autograd.grad(y, [w], gy)[0]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,d,how", [(1, 1, 1, "one"), (1, 8192, 768, "uniform"), (31, 7, 33, "uniform"), (33, 1000, 64, "one"), (1000, 8192, 768, "text"),
                                       (5000, 100, 72, "uniform"), (20000, 50257, 128, "text"), (4096, 333, 1100, "one"), (4097, 100000, 40, "uniform"),
                                       (777, 3, 2056, "uniform"),
                                       (256, 8192, 768, "text"), (257, 8192, 768, "text"), (255, 1, 2056, "one"), (100, 65, 31, "uniform"), (256, 33, 8, "one")])
def test_embedding(N, V, d, how, dtype):
    """One word for all tokens, words in equal parts, words as in a text; rows of 16-byte pieces and others."""
    g = torch.Generator(device=DEV).manual_seed(N + V)
    w = torch.randn(V, d, device=DEV, generator=g).to(dtype)
    gy = torch.randn(N, d, device=DEV, generator=g).to(dtype)
    if how == "one":
        ids = torch.full((N,), V // 2, device=DEV)
    elif how == "uniform":
        ids = torch.randint(0, V, (N,), device=DEV, generator=g)
    else:
        ids = (V * torch.rand(N, device=DEV, generator=g, dtype=torch.float64) ** 6).long().clamp_max(V - 1)
    half = 2.0 ** -8 if dtype == BF else 2.0 ** -24
    for scale, padding in ((1.0, None), (math.sqrt(d), int(ids[0]))):
        y, dw = embed(ids, w, gy, scale=scale, padding_idx=padding)
        scale32 = float(torch.tensor(scale, dtype=F32))                # the kernels' scale is fp32
        want = scale32 * w.double()[ids]
        assert y.dtype == dtype and ((y.double() - want).abs() <= 1.01 * half * want.abs()).all()
        if scale == 1.0:
            assert torch.equal(y, w[ids])
        use = ids != (-1 if padding is None else padding)
        ref = torch.zeros(V, d, device=DEV, dtype=torch.float64).index_add_(0, ids[use], gy[use].double()) * scale32
        mag = torch.zeros(V, d, device=DEV, dtype=torch.float64).index_add_(0, ids[use], gy[use].double().abs()) * scale32
        count = torch.bincount(ids[use], minlength=V)[:, None]
        # chunks of 32 added one by one, then their sums: at most 32 + count / 32 roundings of partial sums
        off = 1.01 * half * ref.abs() + (33 + count / 32) * 2.0 ** -24 * mag + 1e-38
        assert ((dw.double() - ref).abs() <= off).all()
        assert not dw[count[:, 0] == 0].any()
        again = embed(ids, w, gy, scale=scale, padding_idx=padding)
        assert torch.equal(again[0], y) and torch.equal(again[1], dw)


def test_embedding_forms():
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn(50, 64, device=DEV, generator=g).to(BF)
    ids = torch.randint(0, 50, (4, 30), device=DEV, generator=g)
    gy = torch.randn(4, 30, 64, device=DEV, generator=g).to(BF)
    y, dw = embed(ids, w, gy)
    for i in (ids.int(), ids.t().contiguous().t()):
        y2, dw2 = embed(i, w, gy)
        assert torch.equal(y, y2) and torch.equal(dw, dw2)
    y2, dw2 = embed(ids, w.t().contiguous().t(), gy[:, :1].expand(4, 30, 64))
    assert torch.equal(y, y2) and torch.equal(dw2, embed(ids, w, gy[:, :1].repeat(1, 30, 1))[1])
    room = torch.empty(w.numel() + 1, device=DEV, dtype=BF)
    assert torch.equal(embed(ids, room[1:].view_as(w).copy_(w), gy)[0], y)
    assert torch.equal(head.embedding(ids[0, 0], w), w[ids[0, 0]])
    y2, dw2 = embed(ids[:0], w, gy[:0])
    assert y2.shape == (0, 30, 64) and not dw2.any()
    bad = ids.clone(); bad[1, 3], bad[2, 5], bad[0, 0] = 50, -1, 1 << 40
    y2, dw2 = embed(bad, w, gy)
    out = (bad < 0) | (bad >= 50)
    assert torch.isnan(y2[out]).all() and torch.equal(y2[~out], y[~out])
    gz = gy.clone(); gz[out] = 0
    assert torch.equal(dw2, embed(ids, w, gz)[1])


def test_embedding_in_a_graph():
    g = torch.Generator(device=DEV).manual_seed(2)
    w = torch.randn(500, 64, device=DEV, generator=g).to(BF).requires_grad_()
    gy = torch.randn(900, 64, device=DEV, generator=g).to(BF)
    ids = torch.randint(0, 500, (900,), device=DEV, generator=g)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        y = head.embedding(ids, w)
        (dw,) = torch.autograd.grad(y, [w], gy)
    for s in range(3):
        ids.copy_(torch.randint(0, 500 >> (4 * s), (900,), device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        a, b = embed(ids, w.detach(), gy)
        assert torch.equal(y, a) and torch.equal(dw, b)


# ------------------------------------------------------------------------------------------------ the three together
def lm(mixer, dtype, vocab=333, d=128):
    torch.manual_seed(5)
    return LM(vocab=vocab, d=d, layers=2, mlp_mult=2, ctx=64, mixer=mixer, norm="rms").to(DEV).to(dtype)


@pytest.mark.parametrize("mixer,dtype,d", [("aspin", BF, 128), ("dspin", BF, 128), ("aspin", F32, 128), ("fspin", BF, 72), ("fspin", F32, 72)])
def test_language_model_loss(mixer, dtype, d):
    """LM.loss is the trunk with the three operators at its ends: loss, the trunk's gradients and the tied table's two shares of its own are
    what those operators give, to the bit; the operators are held to their definitions above."""
    m = lm(mixer, dtype, d=d)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randint(0, 333, (3, 70), device=DEV, generator=g)
    ids, logits = torch.randint(0, 333, (3, 70, 5), device=DEV, generator=g), torch.randn(3, 70, 5, device=DEV, generator=g)
    target = torch.cat([x[:, 1:], torch.full_like(x[:, :1], -100)], 1)
    for kw in ({}, dict(reduction="sum"), dict(teacher=(ids, logits), temperature=2.0, alpha=1.0)):
        m.zero_grad()
        loss = m.loss(x, **kw)
        loss.backward()
        e = m.e.weight.detach()[x].requires_grad_()
        h = m._add_norm(*m._layers(e + m.p(torch.arange(70, device=DEV) % 64), [None] * 2), m.n)[1]
        hd, wd = h.detach().requires_grad_(), m.e.weight.detach().requires_grad_()
        want = head.linear_distill(hd, wd, ids, logits, temperature=2.0) if "teacher" in kw else head.linear_cross_entropy(hd, wd, target, **kw)
        dh, dw = torch.autograd.grad(want, [hd, wd])
        others = [(n, p) for n, p in m.named_parameters() if n != "e.weight" and p.grad is not None]
        grads = torch.autograd.grad(h, [e] + [p for _, p in others], dh)
        assert torch.equal(loss.detach(), want.detach())
        assert all(".wi." in n and mixer == "dspin" for n, p in m.named_parameters() if p.grad is None)      # the delta rule has no write gate
        for (n, p), b in zip(others, grads[1:]):
            assert torch.equal(p.grad, b), n
        assert torch.equal(m.e.weight.grad, dw + host().embedding_bwd(x, grads[0], 1.0, -1, 333))
    with torch.no_grad():
        rows = m.loss(x, reduction="none")
        ref = torch.nn.functional.cross_entropy(torch.nn.functional.linear(m.trunk(x).double(), m.e.weight.double()).flatten(0, 1), target.flatten(), reduction="none")
        assert rows.shape == (3, 70) and ((rows.flatten().double() - ref).abs() < 1e-4).all()
        both = m.loss(x, teacher=(ids, logits), temperature=2.0, alpha=0.25)
        assert abs(float(both) - 0.75 * float(m.loss(x)) - 0.25 * float(m.loss(x, teacher=(ids, logits), temperature=2.0, alpha=1.0))) < 1e-5
        assert m.loss(x[:, :1], target[:, :1], reduction="none").shape == (3, 1)
    with pytest.raises(ValueError):
        m.loss(x[:, :1])


def test_compiled_callers_take_the_operators():
    """Under torch.compile and under a dispatch mode the same calls are the registered operators, with the same results."""
    h, w, g = operands(100, 300, 64, F32, 1)
    t = torch.randint(0, 300, (100,), device=DEV, generator=g)
    ids, logits = lists(100, 300, 6, g, True)

    def f(h, w):
        z = head.embedding(t, w, scale=2.0)
        return head.linear_cross_entropy(h + z, w, t) + head.linear_distill(h + z, w, ids, logits, temperature=2.0, reduction="none").sum()

    want = torch.autograd.grad(f(*(a := [h.clone().requires_grad_(), w.clone().requires_grad_()])), a)
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(*(a := [h.clone().requires_grad_(), w.clone().requires_grad_()])), a)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        names = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Seen.names.add(func.name())
            return func(*args, **(kwargs or {}))
    with Seen():
        got = torch.autograd.grad(f(*(a := [h.clone().requires_grad_(), w.clone().requires_grad_()])), a)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert {f"pragnosia_b200::{n}" for n in ("linear_xent", "linear_xent_bwd", "linear_distill", "linear_distill_bwd", "teacher_lists", "embedding", "embedding_bwd")} <= Seen.names


def test_streams():
    """Two streams at once, and tensors made on another stream than the one that uses them."""
    h, w, g = operands(600, 2000, 128, BF, 3)
    t = torch.randint(0, 2000, (600,), device=DEV, generator=g)
    want = xent(h, w, t, None, "mean")
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(xent(h, w, t, None, "mean"))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, want))


def test_a_capture_beside_an_eager_pass_of_the_same_leaves_is_refused():
    h, w, g = operands(50, 60, 64, BF, 3)
    w = w.requires_grad_()
    t = torch.randint(0, 60, (50,), device=DEV, generator=g)
    alive = head.linear_cross_entropy(h, w, t), head.embedding(t, w)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    errors = []
    with torch.cuda.graph(graph, stream=side):
        for call in (lambda: head.linear_cross_entropy(h, w, t), lambda: head.embedding(t, w), lambda: head.linear_distill(h, w, t[:, None], h[:, :1].float())):
            try:
                call()
            except RuntimeError as e:
                errors.append(str(e))
        with torch.no_grad():
            loss = head.linear_cross_entropy(h, w, t)
    assert len(errors) == 3 and all("still alive" in e for e in errors)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, alive[0].detach())


def test_what_the_forward_pass_leaves_is_checked():
    """The registered operators' backward passes read what a caller hands them: other sizes, types or places are refused before a launch."""
    ops = torch.ops.pragnosia_b200
    h, w, g = operands(6, 70, 16, BF, 3)
    t = torch.randint(0, 70, (6,), device=DEV, generator=g)
    ids, logits = torch.randint(0, 70, (6, 3), device=DEV, generator=g), torch.randn(6, 3, device=DEV, generator=g)
    loss, L, stats = ops.linear_xent(h, w.clone().requires_grad_(), t, -100, 0)
    assert loss.requires_grad and not L.requires_grad and not stats.requires_grad       # no gradient passes through these
    one = torch.ones(6, device=DEV)
    good = dict(L=L, stats=stats, grad=one)
    for name, bad in (("L", L[:5]), ("L", L.double()), ("L", L.cpu()), ("L", torch.empty(2, 6, device=DEV).t()), ("stats", stats[:1]), ("grad", one[:5]), ("grad", one.cpu())):
        with pytest.raises(ValueError):
            ops.linear_xent_bwd(h, w, t, -100, *(good | {name: bad}).values(), 0, True, True)
    lists, marks, ent = ops.teacher_lists(ids, logits, 1.0, 70)
    loss, L, stats, kept = ops.linear_distill(h, w, lists, marks, ent, 1.0, 0)
    for bad in ((lists[:5], marks, ent), (lists.long(), marks, ent), (lists, marks[:, :1], ent), (lists, marks, ent[:5]), (lists.view(6, 6), marks, ent)):
        with pytest.raises(ValueError):
            ops.linear_distill(h, w, *bad, 1.0, 0)
    for bad in ((lists, ent, kept[:, :2]), (lists[:, :2], ent, kept), (lists, ent.double(), kept)):
        with pytest.raises(ValueError):
            ops.linear_distill_bwd(h, w, *bad, 1.0, L, stats, one, 0, True, True)


def test_sizes_that_an_entry_point_cannot_hold_are_refused():
    """2^32 + 8 words or columns would be 8 to a 32-bit size; nothing of that size is read or copied on the way."""
    many = (1 << 32) + 8
    row, t = torch.zeros(1, 8, device=DEV, dtype=BF), torch.zeros(1, device=DEV, dtype=torch.long)
    tall, wide = row.expand(many, 8), row[:, :1].expand(1, many)
    for call in (lambda: head.linear_cross_entropy(row, tall, t), lambda: head.linear_cross_entropy(wide, wide, t), lambda: head.embedding(t, tall), lambda: head.embedding(t, wide),
                 lambda: head.linear_distill(row, tall, t[:, None], t[:, None].float()), lambda: torch.ops.pragnosia_b200.teacher_lists(t[:, None], t[:, None].float(), 1.0, many),
                 lambda: torch.ops.pragnosia_b200.embedding_bwd(t, row, 1.0, -1, many)):
        with pytest.raises(ValueError):
            call()


def test_distillation_keeps_little_for_its_gradient():
    """From the forward pass to the backward pass: the lists and the entries' logits (12 k bytes a row), 16 bytes a row, and nothing that grows with the vocabulary."""
    N, V, k = 2048, 8192, 16
    h, w, g = operands(N, V, 64, BF, 3)
    ids, logits = torch.randint(0, V, (N, k), device=DEV, generator=g), torch.randn(N, k, device=DEV, generator=g)
    h.requires_grad_()
    head.linear_distill(h, w, ids, logits).backward()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = head.linear_distill(h, w, ids, logits)
    kept = torch.cuda.memory_allocated() - before
    assert kept <= N * (12 * k + 16) + 8 * 512                        # blocks are handed out in multiples of 512 bytes
    del loss


def test_first_calls_inside_a_capture():
    """A process whose first calls of all are captured: kernels are loaded, and their residency asked for, during the capture."""
    import subprocess
    import sys
    code = """
import torch
from pragnosia_b200 import head
g = torch.Generator(device="cuda").manual_seed(3)
h, w = torch.randn(300, 64, device="cuda", generator=g).bfloat16(), torch.randn(500, 64, device="cuda", generator=g).bfloat16()
t = torch.randint(0, 500, (300,), device="cuda", generator=g)
x = torch.randn(300, 4, device="cuda", generator=g)
ids = torch.randint(0, 500, (300, 4), device="cuda", generator=g)
def step():
    h.grad = w.grad = None
    h.requires_grad_(); w.requires_grad_()
    y = head.embedding(t, w) + h
    loss = head.linear_cross_entropy(y, w, t) + head.linear_distill(y, w, ids, x)
    loss.backward()
    out = loss.detach(), h.grad, w.grad
    return out
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
got = [a.clone() for a in got]
want = step()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


def test_refusals():
    """Each with a message, before a launch: the process goes on."""
    h, w, g = operands(6, 70, 16, BF, 3)
    t = torch.randint(0, 70, (6,), device=DEV, generator=g)
    x = torch.randn(6, 3, device=DEV, generator=g)
    ids = torch.randint(0, 70, (6, 3), device=DEV, generator=g)
    ce, kd, emb = head.linear_cross_entropy, head.linear_distill, head.embedding
    bad = [(lambda: ce(h, w[:, :8], t), ValueError), (lambda: ce(h, w, t[:5]), ValueError), (lambda: ce(h, w.float(), t), TypeError), (lambda: ce(h.half(), w.half(), t), TypeError),
           (lambda: ce(h, w, t.float()), TypeError), (lambda: ce(h[:, :12], w[:, :12], t), ValueError), (lambda: ce(h, w[:0], t), ValueError), (lambda: ce(h, w[0], t), ValueError),
           (lambda: ce(h, w, t.cpu()), RuntimeError), (lambda: kd(h, w, ids, x[:5]), ValueError), (lambda: kd(h, w, ids[:5], x[:5]), ValueError),
           (lambda: kd(h, w, ids, x, temperature=0.0), ValueError), (lambda: kd(h, w, ids, x, temperature=float("nan")), ValueError), (lambda: kd(h, w, ids[:, :0], x[:, :0]), ValueError),
           (lambda: kd(h, w, ids[:, :1].expand(6, 1025), x[:, :1].expand(6, 1025)), ValueError), (lambda: kd(h, w, x, x), TypeError), (lambda: emb(x, w), TypeError),
           (lambda: emb(t, w.half()), TypeError), (lambda: emb(t, w[0]), ValueError), (lambda: emb(t, w[:0]), ValueError), (lambda: emb(t, w.cpu()), RuntimeError)]
    for grad in (False, True):
        h.requires_grad_(grad)
        w.requires_grad_(grad)
        for i, (call, error) in enumerate(bad):
            with pytest.raises(error):
                call()
                pytest.fail(f"call {i} was taken")
    assert torch.isfinite(ce(h, w, t))
