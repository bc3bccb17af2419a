"""The two ends of a language model in training, as cases that can be timed and compared: the embedding lookup and its gradient,
softmax cross entropy against given tokens and distillation from a teacher's top logits, both of them straight from the hidden
states and the (tied) head's weight, without the logits of the whole batch in memory.

    listed()            the fixed cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program has in hand before the call
    run(state)          one pass: the plain form, or (own) the framework's operators
    work(case)          the bytes and operations one pass cannot do without
    exact(case, seed)   the outputs from the definitions, in 64 bits

The sizes are the benchmark's (width 768, vocabulary 8192, 16 x 2048 tokens), the fspin width 704, the larger vocabulary 50257 that the
decode step is timed with, and odd ones between.
"""
import math

import torch

own = False

DEV = "cuda"
IGNORE = -100


def listed():
    return [
        # One token's probability under the model: the smallest call (a constrained decoder, a verifier).
        dict(name="ce_score_1", kind="ce", train=False, reduction="none", dtype="bf16", N=1, V=8192, d=768, ignored=0.0),
        # Scoring texts: per-token losses of a batch of documents, padded.
        dict(name="ce_score_8191", kind="ce", train=False, reduction="none", dtype="bf16", N=8191, V=50257, d=768, ignored=0.1),
        # Training on one window of one sequence, its last token without a target.
        dict(name="ce_train_511", kind="ce", train=True, reduction="mean", dtype="bf16", N=511, V=8192, d=768, ignored=0.0),
        # The headline batch in training: 16 sequences of 2048.
        dict(name="ce_train_32768", kind="ce", train=True, reduction="mean", dtype="bf16", N=32768, V=8192, d=768, ignored=0.0),
        # A larger vocabulary of odd size and a padded batch, summed loss (gradients accumulated over micro-batches).
        dict(name="ce_train_vocab", kind="ce", train=True, reduction="sum", dtype="bf16", N=8192, V=50257, d=768, ignored=0.05),
        # A model kept in fp32 (the constructor's default), the diagonal carrier's width.
        dict(name="ce_train_fp32", kind="ce", train=True, reduction="mean", dtype="fp32", N=2000, V=8192, d=704, ignored=0.05),
        # Distillation of the benchmark's model from stored top logits.
        dict(name="kd_train_8192", kind="kd", train=True, reduction="mean", dtype="bf16", N=8192, V=8192, d=768, k=64, tau=2.0, ragged=False),
        # The larger vocabulary, lists of different lengths (top-p truncated), rows without any.
        dict(name="kd_train_vocab", kind="kd", train=True, reduction="mean", dtype="bf16", N=4095, V=50257, d=768, k=32, tau=1.0, ragged=True),
        # A small fp32 model and a short list: per-row losses, weighted by the caller.
        dict(name="kd_train_fp32", kind="kd", train=True, reduction="none", dtype="fp32", N=333, V=8192, d=768, k=8, tau=1.5, ragged=True),
        # A decode batch's tokens looked up.
        dict(name="embed_64", kind="embed", train=False, dtype="bf16", N=64, V=8192, d=768, scale=1.0, padding=-1),
        # The headline batch's embedding, forward and gradient; word frequencies fall as in a text.
        dict(name="embed_train_32768", kind="embed", train=True, dtype="bf16", N=32768, V=8192, d=768, scale=1.0, padding=-1),
        # Most words of the larger vocabulary unseen, scaled by sqrt(d), padding left out of the gradient, fp32 table.
        dict(name="embed_train_vocab", kind="embed", train=True, dtype="fp32", N=8191, V=50257, d=768, scale=math.sqrt(768.0), padding=0),
    ]


def _log(rng, lo, hi):
    """A whole number from lo..hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "kd", "embed"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    d = rng.choice([64, 128, 256, 512, 704, 768, 1024, 1536, 8 * rng.randint(8, 128)])
    V = _log(rng, 100, 50257)
    if kind == "embed":
        train = rng.random() < 0.7
        N = _log(rng, 1, min(65536, (32768 * 768) // d))
        return dict(kind=kind, train=train, dtype=dtype, N=N, V=V, d=d, scale=rng.choice([1.0, 1.0, math.sqrt(d)]),
                    padding=rng.choice([-1, -1, 0]))
    # no more work than the largest listed case; fp32 does the same work in full precision, so a smaller part of it
    most = 32768 * 8192 * 768 // (1 if dtype == "bf16" else 12)
    N = _log(rng, 1, max(1, min(32768, most // (V * d))))
    if kind == "ce":
        return dict(kind=kind, train=rng.random() < 0.7, reduction=rng.choice(["mean", "sum", "none"]), dtype=dtype, N=N, V=V, d=d,
                    ignored=rng.choice([0.0, 0.05, 0.3]))
    return dict(kind=kind, train=rng.random() < 0.8, reduction=rng.choice(["mean", "sum", "none"]), dtype=dtype, N=min(N, 16384), V=V, d=d,
                k=_log(rng, 1, 64), tau=rng.choice([1.0, 2.0, 3.5]), ragged=rng.random() < 0.5)


def _words(case, g):
    """Ids whose frequencies fall with their rank, as a text's do: rank r is drawn about as often as 1 / (r + 3)."""
    V = case["V"]
    u = torch.rand(case["N"], device=DEV, generator=g, dtype=torch.float64)
    return ((3.0 * ((V + 3.0) / 3.0) ** u - 3.0).long()).clamp_(0, V - 1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=DEV, generator=g)
    N, V, d = case["N"], case["V"], case["d"]
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    ids = _words(case, g)
    if case["kind"] == "embed":
        s = dict(case=case, ids=ids, weight=(0.02 * rn(V, d)).to(dt))
        if case["train"]:
            s["gy"] = rn(N, d).to(dt)                                 # what the layers above hand back
            s["weight"].requires_grad_(True)
        return s
    # hidden states behind the final norm (unit mean square), a head whose logits spread over a few units
    s = dict(case=case, h=rn(N, d).to(dt), weight=(2.0 / math.sqrt(d) * rn(V, d)).to(dt))
    if case["kind"] == "ce":
        drop = torch.rand(N, device=DEV, generator=g) < case["ignored"]
        s["target"] = torch.where(drop, torch.full_like(ids, IGNORE), ids)
    else:
        k = min(case["k"], V)
        j = torch.arange(k, device=DEV)
        step = 1 + (torch.rand(N, 1, device=DEV, generator=g) * max(1, V // k - 1)).long()
        s["ids"] = (ids[:, None] + j * step) % V                      # k different words a row
        s["logits"] = (rn(N, k) * 2.0).sort(dim=1, descending=True).values
        if case["ragged"]:                                            # lists cut to 0..k entries
            n = (torch.rand(N, 1, device=DEV, generator=g) * (k + 1)).long()
            s["ids"] = torch.where(j < n, s["ids"], torch.full_like(s["ids"], -1))
    if case["train"]:
        if case["reduction"] == "none":
            s["gl"] = torch.rand(N, device=DEV, generator=g)          # the caller's weight of each row
        s["h"].requires_grad_(True)
        s["weight"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ the framework's operators
def _run_own(s):
    from pragnosia_b200 import head
    case = s["case"]
    with torch.set_grad_enabled(case["train"]):
        if case["kind"] == "embed":
            y = head.embedding(s["ids"], s["weight"], scale=case["scale"], padding_idx=None if case["padding"] < 0 else case["padding"])
            if not case["train"]:
                return [y]
            return [y.detach(), *torch.autograd.grad(y, [s["weight"]], s["gy"])]
        if case["kind"] == "ce":
            loss = head.linear_cross_entropy(s["h"], s["weight"], s["target"], ignore_index=IGNORE, reduction=case["reduction"])
        else:
            loss = head.linear_distill(s["h"], s["weight"], s["ids"], s["logits"], temperature=case["tau"], reduction=case["reduction"])
        if not case["train"]:
            return [loss]
        return [loss.detach(), *torch.autograd.grad(loss, [s["h"], s["weight"]], s.get("gl"))]


# ------------------------------------------------------------------------------------------------ the plain form
def _soft_targets(s):
    """(ids, probabilities, rows that count): the target distribution as k entries a row, those without a word at probability 0."""
    case = s["case"]
    if case["kind"] == "ce":
        t = s["target"][:, None]
        live = t != IGNORE
        return t.clamp_min(0), live.float(), live[:, 0]
    live = s["ids"] >= 0
    z = torch.where(live, s["logits"].float() / case["tau"], torch.full_like(s["logits"], -math.inf))
    top = z.amax(1, keepdim=True)
    e = torch.where(live, torch.exp(z - torch.where(torch.isfinite(top), top, torch.zeros_like(top))), torch.zeros_like(z))
    return s["ids"].clamp_min(0), e / e.sum(1, keepdim=True).clamp_min(1e-30), live.any(1)


def _run_plain(s):
    case = s["case"]
    weight = s["weight"].detach()
    dt = weight.dtype
    if case["kind"] == "embed":
        ids, scale = s["ids"], case["scale"]
        y = (weight[ids].float() * scale).to(dt)
        if not case["train"]:
            return [y]
        g = s["gy"].float()
        if case["padding"] >= 0:
            g = g * (ids != case["padding"])[:, None]
        dw = torch.zeros(weight.shape, device=DEV).index_add_(0, ids, g)
        return [y, (dw * scale).to(dt)]
    tau = case.get("tau", 1.0)
    ids, p, live = _soft_targets(s)
    h, w = s["h"].detach().float(), weight.float()
    z = h @ w.t()
    if tau != 1.0:
        z = z / tau
    top = z.amax(1, keepdim=True)
    q = torch.exp(z - top)
    total = q.sum(1, keepdim=True)
    lse = top + torch.log(total)
    logp = torch.where(p > 0, torch.log(p.clamp_min(1e-38)), torch.zeros_like(p))
    row = tau * tau * (p * (logp - (z.gather(1, ids) - lse))).sum(1)
    row = torch.where(live, row, torch.zeros_like(row))
    count = live.sum().float()
    loss = {"none": row, "sum": row.sum(), "mean": row.sum() / count}[case["reduction"]]
    if not case["train"]:
        return [loss]
    c = s["gl"] if case["reduction"] == "none" else 1.0 / count if case["reduction"] == "mean" else torch.ones((), device=DEV)
    q = (q / total).scatter_add_(1, ids, -p)
    ds = q * (tau * torch.where(live, c.expand_as(row), torch.zeros_like(row)))[:, None]
    return [loss, (ds @ w).to(dt), (ds.t() @ h).to(dt)]


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    N, V, d = case["N"], case["V"], case["d"]
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "embed":
        rows = min(N, V)
        fwd = 8 * N + rows * d * e + N * d * e
        return {"bytes": fwd + (N * d * e + V * d * e if case["train"] else 0), "flops": N * d * (2 if case["train"] else 1)}
    lists = 8 * N if case["kind"] == "ce" else N * case["k"] * 12
    out = 4 * (N if case["reduction"] == "none" else 1)
    read = (N + V) * d * e
    live = N * (1.0 - case.get("ignored", 0.0))
    # logits; in training the two gradients' products as well, and h and the weight's gradients out
    return {"bytes": int(read * (2 if case["train"] else 1) + lists + out), "flops": int((6 if case["train"] else 2) * live * V * d)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    N, V = case["N"], case["V"]
    w = s["weight"].detach().double()
    if case["kind"] == "embed":
        y = case["scale"] * w.index_select(0, s["ids"])
        if not case["train"]:
            return [y]
        order = torch.argsort(s["ids"], stable=True)                  # every word's tokens next to one another: differences of running sums
        g = s["gy"].double().index_select(0, order)
        run_sum = torch.cat([g.new_zeros(1, g.shape[1]), g.cumsum(0)])
        ends = torch.searchsorted(s["ids"].index_select(0, order), torch.arange(V + 1, device=DEV))
        dw = case["scale"] * (run_sum[ends[1:]] - run_sum[ends[:-1]])
        if case["padding"] >= 0:
            dw[case["padding"]] = 0.0
        return [y, dw]
    tau, k = float(case.get("tau", 1.0)), (1 if case["kind"] == "ce" else s["ids"].shape[1])
    if case["kind"] == "ce":
        want, teach = s["target"].view(N, 1), torch.zeros(N, 1, device=DEV, dtype=torch.float64)
        has = want != IGNORE
    else:
        want, teach = s["ids"], s["logits"].double() / tau
        has = want >= 0
    live = has.any(1)
    n_live = int(live.sum())
    scale = {"none": None, "sum": 1.0, "mean": 1.0 / n_live if n_live else math.nan}[case["reduction"]]
    rows = torch.zeros(N, device=DEV, dtype=torch.float64)
    dh = torch.zeros(N, w.shape[1], device=DEV, dtype=torch.float64)
    dw = torch.zeros_like(w)
    step = max(1, (1 << 28) // V)
    for a in range(0, N, step):
        b = min(N, a + step)
        h = s["h"].detach()[a:b].double()
        logq = torch.log_softmax(h.matmul(w.t()) / tau, dim=1)
        t = teach[a:b].masked_fill(~has[a:b], -math.inf)
        p = torch.softmax(t, dim=1).nan_to_num(0.0)                   # a row without entries has none
        at = want[a:b].clamp(0, V - 1)
        plogp = torch.special.xlogy(p, p)
        rows[a:b] = tau ** 2 * (plogp - p * logq.gather(1, at)).sum(1)
        if case["train"]:
            c = (s["gl"][a:b].double() if scale is None else torch.full((b - a,), scale, device=DEV, dtype=torch.float64))
            c = tau * c.masked_fill(~live[a:b], 0.0)
            ds = logq.exp_()
            ds.scatter_add_(1, at, -p)
            ds *= c.unsqueeze(1)
            dh[a:b] = ds.matmul(w)
            dw += ds.t().matmul(h)
    loss = rows if scale is None else rows.sum() * scale
    return [loss, dh, dw] if case["train"] else [loss]
