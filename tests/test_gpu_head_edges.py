"""The head's losses where the other tests do not reach: what a caller hands to the registered operators and the C entry points, lists in several
pieces, temperatures without an exact reciprocal, rows whose loss is next to nothing, teachers whose axes are not those of the hidden states,
masked batches of the language model and its gradients against the formulas on its own logits, padding of a size that a launch takes long to copy."""
import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

from pragnosia_b200 import head
from pragnosia_b200._lib import check, host, lib
from test_gpu_head import BF, DEV, F32, _grad_enabled_and_waits_fine, dense, distill, lm, operands, teacher, within, xent  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
def test_marks_of_longer_lists_write_nothing_past_a_row(dtype):
    """Marks say where in its list a word's logit goes. Those of lists of 40 beside lists of 3 point behind the end: what lies behind `kept` stays as it
    was, and so does the result of entries that the lists have."""
    N, V, d, k = 70, 300, 64, 3
    h, w, g = operands(N, V, d, dtype, 1)
    ids, logits = torch.rand(N, V, device=DEV, generator=g).argsort(1)[:, :40].contiguous(), torch.randn(N, 40, device=DEV, generator=g)
    marks = host().teacher_lists(ids, logits, 1.0, V)[1]
    first = host().teacher_lists(ids.sort(1).values[:, :k].contiguous(), logits[:, :k].contiguous(), 1.0, V)       # of the same rows, the first k words
    room = torch.full((N * k + 4096,), 7.0, device=DEV)
    loss, L, stats = torch.empty(N, device=DEV), torch.empty(N, 2, device=DEV), torch.empty(2, device=DEV)
    n = lib().pgb_head_loss_fwd_scratch_bytes(N, V, d, int(dtype == BF))
    scratch = torch.empty(n, device=DEV, dtype=torch.uint8)
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    check(lib().pgb_linear_distill_fwd(at(h), at(w), int(dtype == BF), at(first[0]), at(marks), at(first[2]), at(room), k, 1.0, at(loss), None, at(stats), at(L),
                                       at(scratch), n, 0, N, V, d, stream), "pgb_linear_distill_fwd")
    torch.cuda.synchronize()
    assert (room[N * k:] == 7.0).all()
    assert torch.equal(loss, host().linear_distill_fwd(h, w, *first, 1.0, 0)[0])


def test_long_padding_without_numbers():
    """Millions of rows, a fifth of them ignored and no numbers: the copy of h without them takes milliseconds, which no wait of the launch that makes it may
    count. The results are those of zeros there, to the bit."""
    N, V, d = 2_900_000, 70, 768
    g = torch.Generator(device=DEV).manual_seed(3)
    h = torch.empty(N, d, device=DEV, dtype=BF).normal_(generator=g)
    w = (0.05 * torch.randn(V, d, device=DEV, generator=g)).to(BF)
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    dead = torch.rand(N, device=DEV, generator=g) < 0.2
    t[dead] = -100
    h[dead] = 0
    want = xent(h, w, t, None, "mean")
    h[dead] = math.nan
    got = xent(h, w, t, None, "mean")
    assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(want, got))


def test_a_teacher_of_other_axes_is_refused_everywhere():
    """A teacher of (T, B) beside hidden states of (B, T) has as many rows: refused eagerly, under a dispatch mode and under a compiler alike."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    h, w, g = operands(6 * 5, 70, 16, BF, 3)
    h = h.view(6, 5, 16)
    ids, logits = torch.randint(0, 70, (6, 5, 3), device=DEV, generator=g), torch.randn(6, 5, 3, device=DEV, generator=g)
    turned = ids.transpose(0, 1).contiguous(), logits.transpose(0, 1).contiguous()
    for bad in (turned, (ids.flatten(0, 1), logits.flatten(0, 1)), (ids, logits[..., :2]), (ids[..., 0], logits[..., 0])):
        with pytest.raises(ValueError):
            head.linear_distill(h, w, *bad)
        with Mode(), pytest.raises(ValueError):
            head.linear_distill(h, w, *bad)
        torch._dynamo.reset()
        with pytest.raises(Exception, match="teacher"):
            torch.compile(head.linear_distill, backend="eager")(h, w, *bad)
    with Mode():
        seen = head.linear_distill(h, w, ids, logits)
    assert torch.equal(seen, head.linear_distill(h, w, ids, logits))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_certain_word_loses_nothing(dtype):
    """Logits of hundreds, the target ahead of all others by 30: its loss is below 700 e^-30, and what is left of it is the rounding of one exponential
    (two units, 2^-22) and of the sum, not of the logits' own size. No loss is negative."""
    h, w, _ = operands(400, 700, 64, dtype, 3, spread=120.0)
    top = (h.double() @ w.double().t()).topk(2, 1)
    sure = top.values[:, 0] - top.values[:, 1] > 30
    assert int(sure.sum()) > 100
    with torch.no_grad():
        loss = head.linear_cross_entropy(h, w, top.indices[:, 0], reduction="none")
    assert (loss >= 0).all() and (loss[sure] <= 2.0 ** -21).all(), (float(loss.min()), float(loss[sure].max()))


@pytest.mark.parametrize("tau", [1e-60, 1e-40, 1e-38, -1.0, 1e300, math.inf])
def test_temperatures_that_fp32_cannot_divide_by_are_refused(tau):
    h, w, g = operands(6, 70, 16, BF, 3)
    ids, logits = torch.randint(0, 70, (6, 3), device=DEV, generator=g), torch.randn(6, 3, device=DEV, generator=g)
    for grad in (False, True):
        h.requires_grad_(grad)
        with pytest.raises(ValueError, match="temperature"):
            head.linear_distill(h, w, ids, logits, temperature=tau)


def spread_lists(N, V, k, g, ragged):
    """k different words a row, evenly apart from a random one on, in an order of their own; ragged: 0 .. k of them."""
    j = torch.rand(N, k, device=DEV, generator=g).argsort(1)
    ids = (torch.randint(0, V, (N, 1), device=DEV, generator=g) + j * (V // k)) % V
    logits = 3.0 * torch.randn(N, k, device=DEV, generator=g)
    if ragged:
        ids = torch.where(torch.rand(N, k, device=DEV, generator=g) < torch.rand(N, 1, device=DEV, generator=g), ids, torch.full_like(ids, -1))
        ids[::11] = -1
    return ids, logits


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,V,d,tau", [(9000, 6200, 64, 3.5), (3000, 17000, 72, 0.7)])
def test_distillation_in_pieces(N, V, d, tau, dtype):
    """More logits than the workspace takes at once, pieces along the rows and along the vocabulary: every piece finds its rows' lists and its words."""
    h, w, g = operands(N, V, d, dtype, N + V)
    c = torch.rand(N, device=DEV, generator=g) - 0.3
    ids, logits = spread_lists(N, V, 24, g, True)
    p, live, _ = teacher(ids, logits, V, tau)
    # an entry's logit / tau and the largest one are off by two roundings each (the reciprocal, the product), 2^-23 |z|, and so is what they are divided by;
    # the rest (exponential, sum, quotient) by 2^-20
    dp = (2.0 ** -20 + 2.0 ** -21 * float(logits.abs().max()) / tau) * p
    s = (h.double() @ w.double().t()).abs()
    for reduction in ("mean", "none"):
        want, off = dense(h, w, p, live, tau, c, reduction)
        n = max(1, int(live.sum()))
        cs = (c.abs() if reduction == "none" else torch.full_like(c, 1.0 / n)).double()[:, None] * tau
        e = tau * tau * ((dp * (s / tau + 20.0)).sum(1) + 2.0 ** -20 * (1 + (p * (p + 1e-300).log().abs()).sum(1)))
        off = (off[0] + (e if reduction == "none" else e.sum() / n), off[1] + (cs * dp) @ w.double().abs(), off[2] + (cs * dp).t() @ h.double().abs())
        within(distill(h, w, ids, logits, tau, c, reduction), want, off)


# ------------------------------------------------------------------------------------------------ the language model's loss
def masked_batch(g, B=3, T=70, k=5, vocab=333):
    x = torch.randint(0, vocab, (B, T), device=DEV, generator=g)
    ids, logits = torch.rand(B, T, vocab, device=DEV, generator=g).argsort(2)[..., :k].contiguous(), 2.0 * torch.randn(B, T, k, device=DEV, generator=g)
    targets = torch.cat([x[:, 1:], torch.full_like(x[:, :1], -100)], 1)
    targets[:, :9] = -100                                             # a prompt
    targets[1, 40:] = -100                                            # padding
    return x, targets, ids, logits


def reference_loss(m, x, targets, ids, logits, tau, alpha):
    """The formulas in 64 bits on the model's own hidden states, differentiable through its layers and both uses of the table."""
    z = m.trunk(x).double() @ m.e.weight.double().t()
    ce = F.cross_entropy(z.flatten(0, 1), targets.flatten(), ignore_index=-100)
    p = torch.softmax(logits.double() / tau, -1)
    rows = tau * tau * (p * (p.log() - torch.log_softmax(z / tau, -1).gather(2, ids))).sum(-1)
    live = targets != -100
    return (1.0 - alpha) * ce + alpha * torch.where(live, rows, torch.zeros_like(rows)).sum() / live.sum()


@pytest.mark.parametrize("mixer,d", [("aspin", 128), ("dspin", 128), ("fspin", 72)])
@pytest.mark.parametrize("alpha", [0.0, 0.3, 1.0])
def test_language_model_loss_of_a_masked_batch(mixer, d, alpha):
    """Tokens without a target count in neither term, and the gradients are those of the formulas on the model's logits. fp32: the head's two gradients are
    off by some (6 d / 16 + 34) 2^-23 of what they add up, 1e-5, and go through the same layers on either side; a gradient may lose a factor of a hundred to
    cancellation. The associative layers' backward pass takes the gradient behind it as bf16 (2^-8), whose roundings fall differently for gradients that differ
    at all: two layers, 2^-7, of which a weight's gradient may lose a factor of four."""
    m = lm(mixer, F32, d=d)
    x, targets, ids, logits = masked_batch(torch.Generator(device=DEV).manual_seed(2))
    params = [(n, p) for n, p in m.named_parameters()]
    want = reference_loss(m, x, targets, ids, logits, 2.0, alpha)
    ref = torch.autograd.grad(want, [p for _, p in params], allow_unused=True)
    loss = m.loss(x, targets, teacher=(ids, logits), temperature=2.0, alpha=alpha)
    got = torch.autograd.grad(loss, [p for _, p in params], allow_unused=True)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-4
    size = math.sqrt(sum(float(r.norm()) ** 2 for r in ref if r is not None))
    rel, part = (1e-3, 1e-5) if mixer == "fspin" else (2.0 ** -5, 2.0 ** -8)
    for (n, _), a, b in zip(params, got, ref):
        assert (a is None) == (b is None), n
        if a is not None:
            assert float((a - b).norm()) <= rel * float(b.norm()) + part * size, n


def test_masked_tokens_of_a_language_model_may_have_any_teacher():
    """Lists of masked tokens change nothing, to the bit; int32 lists as int64; the caller's lists stay as they are."""
    m = lm("aspin", BF)
    x, targets, ids, logits = masked_batch(torch.Generator(device=DEV).manual_seed(4))
    dead = targets == -100
    other = torch.where(dead[..., None], (ids + 7) % 333, ids).int()
    kept = other.clone()
    for reduction in ("mean", "sum", "none"):
        a, b = (m.loss(x, targets, teacher=(t, logits), temperature=1.5, alpha=0.4, reduction=reduction) for t in (ids, other))
        assert torch.equal(a, b) and (reduction != "none" or not a[dead].any())
    assert torch.equal(other, kept)


def test_a_teacher_of_no_weight_is_left_out():
    """alpha 0 is the cross entropy, even where no token has an entry (whose mean would be 0 / 0)."""
    m = lm("aspin", BF)
    x, targets, ids, logits = masked_batch(torch.Generator(device=DEV).manual_seed(5))
    with torch.no_grad():
        assert torch.equal(m.loss(x, targets, teacher=(torch.full_like(ids, -1), logits), alpha=0.0), m.loss(x, targets))
    with pytest.raises(ValueError):
        m.loss(x, targets[0], teacher=(ids, logits), alpha=1.0)


def test_a_captured_training_step_of_the_language_model():
    """The layers and the three operators as one graph: a replay with other tokens, targets and lists gives what an eager step gives, to the bit."""
    g = torch.Generator(device=DEV).manual_seed(6)
    for mixer, dtype, d in (("aspin", BF, 128), ("dspin", BF, 128), ("fspin", F32, 72)):
        m = lm(mixer, dtype, d=d)
        x, targets, ids, logits = masked_batch(g)
        params = [p for n, p in m.named_parameters() if not (".wi." in n and mixer == "dspin")]

        def step():
            loss = m.loss(x, targets, teacher=(ids, logits), temperature=2.0, alpha=0.3)
            return [loss.detach(), *torch.autograd.grad(loss, params)]
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        with torch.cuda.graph(graph, stream=side):
            out = step()
        for _ in range(2):
            for a, b in zip((x, targets, ids, logits), masked_batch(g)):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_a_capture_beside_an_eager_step_of_the_same_model_is_refused():
    """Through the tied table, through the layers where the table is frozen, and through the fused up-projection by itself."""
    from pragnosia_b200 import ops
    m = lm("aspin", BF)
    x, targets, _, _ = masked_batch(torch.Generator(device=DEV).manual_seed(7))
    frozen = lm("aspin", BF)
    frozen.e.weight.requires_grad_(False)
    rows, a = torch.randn(130, 128, device=DEV).to(BF), m.mlp[0].a
    for call in (lambda: m.loss(x, targets), lambda: frozen.loss(x, targets), lambda: ops.linear_act(rows, a.weight, a.bias)):
        alive = call()
        side, graph, said = torch.cuda.Stream(), torch.cuda.CUDAGraph(), []
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            try:
                call()
            except RuntimeError as e:
                said.append(str(e))
            with torch.no_grad():
                seen = call()
        assert len(said) == 1 and "still alive" in said[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(seen, alive.detach()) or abs(float(seen.float().mean()) - float(alive.detach().float().mean())) < 1e-2     # no_grad fuses the norms
        del alive


def test_threads():
    """Training steps of two threads at once, each on a stream of its own."""
    import threading
    h, w, g = operands(700, 3000, 128, BF, 6)
    t = torch.randint(0, 3000, (700,), device=DEV, generator=g)
    ids, logits = torch.randint(0, 3000, (700, 9), device=DEV, generator=g), torch.randn(700, 9, device=DEV, generator=g)
    want = [xent(h, w, t, None, "mean"), distill(h, w, ids, logits, 2.0, None, "mean")]
    torch.cuda.synchronize()
    got, errors = [], []

    def work(kind):
        try:
            with torch.enable_grad(), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got.append((kind, xent(h, w, t, None, "mean") if kind == 0 else distill(h, w, ids, logits, 2.0, None, "mean")))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                        # noqa: BLE001  (told below)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors and len(got) == 40
    assert all(torch.equal(a, b) for k, o in got for a, b in zip(o, want[k]))
