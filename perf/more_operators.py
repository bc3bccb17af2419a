"""Serving with four-bit weights and controlled draws, as cases that can be timed and compared: the linear layer whose weight is held in
four bits with a scale per group, quantising a weight to that form and reading it back, and what stands between a model's logits and the
draw: penalties for tokens seen before, biases of single tokens and a mask of the tokens that a grammar allows.

    listed()            the fixed cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program has in hand before the call
    run(state)          one pass: the plain form, or (own) the framework's operators
    work(case)          the bytes and operations one pass cannot do without
    exact(case, seed)   the outputs from the definitions, in 64 bits

A weight (N, K) is held as bytes (N, K / 2), the even column in the low half of a byte, a scale and, unless it is symmetric, a whole number 0 .. 15 (its
zero) for each group of 32, 64 or 128 columns of a row, and stands for scale (q - zero); without zeros for scale (q - 8).

The sizes are the benchmark's (width 768, vocabulary 8192, fused projection 2328), the diagonal carrier's width 704 with its MLP of 2816, the larger vocabulary
50257 that the decode step is timed with, wider layers of generic size, and odd ones between.
"""
import math

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # One token through the smallest layer (output projection of the benchmark's width): latency.
        dict(name="int4_token_768", kind="linear", M=1, K=768, N=768, group=64, zeros=True, dtype="bf16", out="bf16", bias=False, act=""),
        # One token's logits over the larger vocabulary, left in fp32 for the draw.
        dict(name="int4_token_head", kind="linear", M=1, K=768, N=50257, group=64, zeros=False, dtype="bf16", out="fp32", bias=False, act=""),
        # One token through the up-projection of a wide model.
        dict(name="int4_token_wide", kind="linear", M=1, K=4096, N=16384, group=128, zeros=True, dtype="bf16", out="bf16", bias=True, act="gelu"),
        # A few sequences, small groups, the diagonal carrier's down-projection.
        dict(name="int4_batch_5", kind="linear", M=5, K=2816, N=704, group=32, zeros=True, dtype="bf16", out="bf16", bias=True, act=""),
        # A decode batch.
        dict(name="int4_batch_64", kind="linear", M=64, K=2048, N=8192, group=64, zeros=True, dtype="bf16", out="bf16", bias=True, act="gelu"),
        # Prompts, where the product itself is the time.
        dict(name="int4_prompt_4096", kind="linear", M=4096, K=2048, N=8192, group=64, zeros=False, dtype="bf16", out="bf16", bias=True, act="gelu"),
        # A model kept in fp32.
        dict(name="int4_fp32_9", kind="linear", M=9, K=704, N=2816, group=64, zeros=True, dtype="fp32", out="fp32", bias=True, act=""),
        # A layer's weight quantised and read back (what a program does to see what four bits cost it): the fused projection, then a wide layer.
        dict(name="quant_2328", kind="quant", N=2328, K=768, group=64, zeros=True, dtype="bf16"),
        dict(name="quant_16384", kind="quant", N=16384, K=4096, group=128, zeros=False, dtype="bf16"),
        # One sequence, a short text, repetition alone: latency.
        dict(name="logits_1", kind="logits", B=1, V=8192, dtype="fp32", prompt=64, made=17, per_row=False, freq=False, nb=0, mask=""),
        # A batch of requests with settings of their own, biases, and a grammar for each.
        dict(name="logits_64", kind="logits", B=64, V=50257, dtype="fp32", prompt=512, made=512, per_row=True, freq=True, nb=32, mask="bits"),
        # Long texts.
        dict(name="logits_long", kind="logits", B=4, V=50257, dtype="bf16", prompt=32768, made=4096, per_row=False, freq=True, nb=3, mask=""),
    ]


def _log(rng, lo, hi):
    """A whole number from lo..hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "linear", "quant", "logits", "logits"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    group, zeros = rng.choice([32, 64, 128]), rng.random() < 0.6
    if kind == "logits":
        B = _log(rng, 1, 128)
        V = _log(rng, 100, 50257)
        return dict(kind=kind, B=B, V=V, dtype=dtype, prompt=_log(rng, 1, min(32769, (1 << 18) // B)) - 1, made=_log(rng, 1, 4097) - 1, per_row=rng.random() < 0.5,
                    freq=rng.random() < 0.6, nb=rng.choice([0, 0, 1, 16, 300]), mask=rng.choice(["", "bits", "bits", "bytes"]))
    K = 32 * _log(rng, 2, 512)
    if kind == "quant":
        return dict(kind=kind, N=_log(rng, 1, (1 << 26) // K), K=K, group=group, zeros=zeros, dtype=dtype)
    N = _log(rng, 1, min(50257, (1 << 26) // K))
    most = 4096 * 2048 * 8192 // (1 if dtype == "bf16" else 16)       # no more work than the largest listed case, in full precision a part of it
    M = _log(rng, 1, max(1, min(4096, most // (N * K))))
    if rng.random() < 0.4:
        M = min(M, rng.randint(1, 64))
    out = "fp32" if dtype == "fp32" or (M <= 256 and rng.random() < 0.2) else "bf16"
    return dict(kind=kind, M=M, K=K, N=N, group=group, zeros=zeros, dtype=dtype, out=out, bias=rng.random() < 0.6, act=rng.choice(["", "", "gelu"]))


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _words(n, V, g):
    """Ids whose frequencies fall with their rank, as a text's do: rank r is drawn about as often as 1 / (r + 3)."""
    u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
    return ((3.0 * ((V + 3.0) / 3.0) ** u - 3.0).long()).clamp_(0, V - 1)


def _levels(w, group, zeros):
    """(levels 0..15 (N, K) uint8, scales (N, G) in w's type, zeros (N, G) uint8 or None) of a weight, in 32 bits: every step is a single
    correctly rounded operation."""
    N, K = w.shape
    G = -(-K // group)
    f = torch.nn.functional.pad(w.float(), (0, G * group - K)).view(N, G, group)      # zeros change no group's range
    if zeros:
        lo = f.amin(2).clamp_max(0.0)
        top = f.amax(2).clamp_min(0.0) - lo
    else:
        top = f.abs().amax(2)
    s = (top / torch.full_like(top, 15.0 if zeros else 7.0)).to(w.dtype)              # by a tensor: by a number torch multiplies with its reciprocal
    t = s.float()
    safe = torch.where(t > 0, t, torch.ones_like(t))
    z = torch.round(-lo / safe).clamp(0, 15) if zeros else torch.full_like(t, 8.0)
    q = (torch.round(f / safe.unsqueeze(2)) + z.unsqueeze(2)).clamp(0, 15)
    q = q.to(torch.uint8).view(N, G * group)[:, :K]
    return q, s, z.to(torch.uint8) if zeros else None


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=DEV, generator=g)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    if case["kind"] == "logits":
        B, V = case["B"], case["V"]
        ids = lambda n: _words(B * n, V, g).view(B, n)
        some = lambda n: (torch.rand(B, device=DEV, generator=g) * (n + 1)).long()    # texts of different lengths, padded
        s = dict(case=case, logits=(4.0 * rn(B, V)).to(dt), prompt=ids(case["prompt"]), made=ids(case["made"]), bias=None, mask=None)
        s["prompt_n"], s["made_n"] = some(case["prompt"]), some(case["made"])
        one = lambda lo, hi: lo + (hi - lo) * torch.rand(B, device=DEV, generator=g)
        s["rep"] = one(1.0, 1.5) if case["per_row"] else 1.1
        s["freq"], s["pres"] = ((one(-0.5, 1.0), one(-0.5, 1.0)) if case["per_row"] else (0.3, 0.2)) if case["freq"] else (0.0, 0.0)
        if case["nb"]:
            s["bias"] = (ids(case["nb"]), 5.0 * rn(B, case["nb"]))    # an id may come twice: both count
        if case["mask"]:
            ok = torch.rand(B, V, device=DEV, generator=g) < 0.2
            ok[0] = False                                             # a grammar at its end allows nothing
            s["mask"] = ok
            if case["mask"] == "bits":                                # 32 tokens a word, bit set: allowed
                W = -(-V // 32)
                bits = torch.nn.functional.pad(ok, (0, 32 * W - V)).view(B, W, 32).long() << torch.arange(32, device=DEV)
                s["mask"] = bits.sum(2).to(torch.int32)
        return s
    N, K = case["N"], case["K"]
    w = rn(N, K).mul_(0.05)
    if case["kind"] == "quant":
        return dict(case=case, weight=w.to(dt))
    q, scales, zeros = _levels(w.to(dt), case["group"], case["zeros"])
    s = dict(case=case, x=rn(case["M"], K).to(dt), q=q[:, 0::2] | (q[:, 1::2] << 4), scales=scales, zeros=zeros, bias=None)
    if case["bias"]:
        s["bias"] = rn(N).to(dt)
    return s


# ------------------------------------------------------------------------------------------------ the framework's operators
def _run_own(s):
    case = s["case"]
    if case["kind"] == "logits":
        from pragnosia_b200 import sampling
        ids, bias = s["bias"] if s["bias"] is not None else (None, None)
        return [sampling.adjust_logits(s["logits"], prompt=s["prompt"], prompt_lengths=s["prompt_n"], generated=s["made"], generated_lengths=s["made_n"],
                                       repetition=s["rep"], frequency=s["freq"], presence=s["pres"], bias_ids=ids, bias=bias, mask=s["mask"])]
    from pragnosia_b200 import int4
    if case["kind"] == "quant":
        w = int4.quantize(s["weight"], group=case["group"], symmetric=not case["zeros"])
        return [int4.dequantize(w), w.scales]
    return [int4.linear(s["x"], int4.Int4Weight(s["q"], s["scales"], s["zeros"], case["group"]), s["bias"], act=case["act"] or None,
                        out_dtype=torch.float32 if case["out"] == "fp32" else torch.bfloat16)]


# ------------------------------------------------------------------------------------------------ the plain form
def _values(q, scales, zeros, group):
    """scale (q - zero) of levels (N, K), in 32 bits."""
    z = 8.0 if zeros is None else zeros.float().repeat_interleave(group, 1)[:, :q.shape[1]]
    return (q.float() - z) * scales.float().repeat_interleave(group, 1)[:, :q.shape[1]]


def _gelu(y):
    return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))


def _counts(ids, n, V):
    """How often each word stands among the first n[b] ids of row b."""
    live = torch.arange(ids.shape[1], device=DEV) < n[:, None]
    return torch.zeros(ids.shape[0], V, device=DEV).scatter_add_(1, ids, live.float())


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "logits":
        l = s["logits"].float()
        V = l.shape[1]
        made = _counts(s["made"], s["made_n"], V)
        seen = made + _counts(s["prompt"], s["prompt_n"], V)
        col = lambda v: v[:, None] if torch.is_tensor(v) else v
        l = torch.where(seen > 0, torch.where(l > 0, l / col(s["rep"]), l * col(s["rep"])), l)
        if case["freq"]:
            l = l - col(s["freq"]) * made - col(s["pres"]) * (made > 0)
        if s["bias"] is not None:
            l = l + torch.zeros_like(l).scatter_add_(1, *s["bias"])
        if s["mask"] is not None:
            ok = s["mask"]
            if case["mask"] == "bits":
                v = torch.arange(V, device=DEV)
                ok = ((ok[:, v // 32] >> (v % 32)) & 1) > 0
            l = torch.where(ok, l, torch.full_like(l, -math.inf))
        return [l]
    if case["kind"] == "quant":
        q, scales, zeros = _levels(s["weight"], case["group"], case["zeros"])
        return [_values(q, scales, zeros, case["group"]).to(s["weight"].dtype), scales]
    q = torch.stack([s["q"] & 15, s["q"] >> 4], 2).view(case["N"], case["K"])
    y = s["x"].float() @ _values(q, s["scales"], s["zeros"], case["group"]).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["act"]:
        y = _gelu(y)
    return [y.to(torch.float32 if case["out"] == "fp32" else torch.bfloat16)]


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "logits":
        B, V = case["B"], case["V"]
        ids = 4 * B * (case["prompt"] + case["made"])                 # half of what is there, on average
        mask = {"": 0, "bits": B * 4 * -(-V // 32), "bytes": B * V}[case["mask"]]
        return {"bytes": B * V * (e + 4) + ids + 12 * B * case["nb"] + mask, "flops": 2 * B * V}
    N, K = case["N"], case["K"]
    held = N * K // 2 + N * -(-K // case["group"]) * (e + (1 if case["zeros"] else 0))
    if case["kind"] == "quant":
        return {"bytes": 2 * N * K * e + 2 * held, "flops": 4 * N * K}
    M = case["M"]
    return {"bytes": held + M * K * e + M * N * (4 if case["out"] == "fp32" else 2) + (N * e if case["bias"] else 0), "flops": 2 * M * N * K}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logits":
        l = s["logits"].double()
        B, V = l.shape
        rows = []
        for b in range(B):
            made = torch.bincount(s["made"][b, :int(s["made_n"][b])], minlength=V).double()
            old = torch.bincount(s["prompt"][b, :int(s["prompt_n"][b])], minlength=V).double()
            rep, freq, pres = (float(t[b]) if torch.is_tensor(t) else t for t in (s["rep"], s["freq"], s["pres"]))
            r = l[b].clone()
            at = (made + old).nonzero()[:, 0]
            r[at] = torch.maximum(r[at], r.new_zeros(())) / rep + torch.minimum(r[at], r.new_zeros(())) * rep
            r -= freq * made + pres * made.clamp_max(1.0)
            if s["bias"] is not None:
                r.index_add_(0, s["bias"][0][b], s["bias"][1][b].double())
            if s["mask"] is not None:
                ok = s["mask"][b]
                if case["mask"] == "bits":
                    ok = ((ok.view(-1, 1).long() >> torch.arange(32, device=DEV)) & 1).flatten()[:V].bool()
                r.masked_fill_(~ok, -math.inf)
            rows.append(r)
        return [torch.stack(rows)]
    g = case["group"]
    if case["kind"] == "quant":
        if case["dtype"] != "bf16":
            return None                                               # levels next to a border go by 32 bits' own rounding
        w = s["weight"].double()
        out, scales = torch.empty_like(w), []
        for k in range(0, case["K"], g):
            p = w[:, k:k + g]
            hi, lo = (p.amax(1).clamp_min(0), p.amin(1).clamp_max(0)) if case["zeros"] else (p.abs().amax(1), None)
            sc = ((hi - lo) / 15 if case["zeros"] else hi / 7).float().to(torch.bfloat16).double()
            z = (-lo / sc).round().clamp(0, 15) if case["zeros"] else torch.full_like(sc, 8.0)
            out[:, k:k + g] = sc[:, None] * (((p / sc[:, None]).round() + z[:, None]).clamp(0, 15) - z[:, None])
            scales.append(sc)
        return [out, torch.stack(scales, 1)]
    N, K, M = case["N"], case["K"], case["M"]
    y = torch.zeros(M, N, device=DEV, dtype=torch.float64)
    for i in range(-(-K // g)):                                       # group by group: the sum of whole numbers times x, then its scale
        k, n = i * g, min(g, K - i * g)
        b = s["q"][:, k // 2:(k + n) // 2].double()
        top = torch.floor(b / 16)
        z = 8.0 if s["zeros"] is None else s["zeros"][:, i:i + 1].double()
        xs = s["x"][:, k:k + n].double()
        part = xs[:, 0::2] @ (b - 16 * top - z).t() + xs[:, 1::2] @ (top - z).t()
        y += part * s["scales"][:, i].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"]:
        y = y * torch.special.ndtr(y)
    return [y]
