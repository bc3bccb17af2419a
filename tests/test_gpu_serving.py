"""A decoder with four-bit weights and with controlled draws, as a program runs it: prompt, steps, generated tokens, captured and not.

The four-bit step is the model with its layers' weights read back from four bits. In fp32 both sides form sums of a few hundred products in another order: 2^-24 each, a few hundred
operations deep through three layers, and the head: 1e-4 of the logits' norm is a thousand of them. In bf16 either side rounds a dozen times a layer (2^-8 of a value each); two
such runs of three layers differ by about as much as either does from fp32, which the tests of the other steps bound by 3e-2 of the norm."""
import copy

import pytest
import torch

from pragnosia_b200 import int4, sampling, synth
from pragnosia_b200.generate import Decoder
from pragnosia_b200.model import LM

from test_gpu_adjust_logits import want
from test_gpu_decode_token import healthy
from test_gpu_model import DEV

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def model(d=128, mixer="aspin", mult=2, vocab=500, layers=3, norm="rms", dtype=torch.float32):
    torch.manual_seed(d + layers)
    m = LM(vocab=vocab, d=d, layers=layers, mlp_mult=mult, ctx=64, mixer=mixer, norm=norm)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn_like(p) if p.dim() == 1 else 0.05 * torch.randn_like(p))
    return m.to(DEV).to(dtype).eval()


def read_back(m, group):
    """The model in fp32 with every weight that the four-bit step quantises read back from four bits."""
    r = copy.deepcopy(m).float()
    with torch.no_grad():
        for mx, my in zip(m.mix, r.mix):
            W = int4.dequantize(int4.quantize(mx._consts()["W"], group), torch.float32)
            d, H = mx.d, mx.h
            last = my.wb if mx.delta else my.wi
            for lin, rows in ((my.q, W[:d]), (my.k, W[d:2 * d]), (my.v, W[2 * d:3 * d]), (my.wa, W[3 * d:3 * d + H]), (last, W[3 * d + H:3 * d + 2 * H])):
                lin.weight.copy_(rows)
            my.o.weight.copy_(int4.dequantize(int4.quantize(mx._consts()["ow"], group), torch.float32) / torch.sigmoid(my.gate.float()))
        for mp, mq in zip(m.mlp, r.mlp):
            for a, b in ((mp.a, mq.a), (mp.b, mq.b)):
                b.weight.copy_(int4.dequantize(int4.quantize(a.weight, group), torch.float32))
    return r


def steps(dec, ids, states=None):
    lg = [dec.prefill(ids[:, :20])]
    if states is not None:                                            # the same prompt's states on both sides: the prompt keeps the model's own weights
        for st, S in zip(dec.states, states):
            st[0].copy_(S)
    kept = [st[0].clone() for st in dec.states]
    for t in range(20, 26):
        lg.append(dec.step(ids[:, t]).clone())
    return torch.stack(lg[1:], 1).double(), kept


@pytest.mark.parametrize("d,mixer,mult,group,norm", [(128, "aspin", 2, 64, "rms"), (256, "dspin", 3, 32, "ln"), (256, "hspin", 2, 128, "rms"), (704, "aspin", 4, 128, "rms")])
@pytest.mark.parametrize("B", [1, 5, 20])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_four_bit_steps(d, mixer, mult, group, norm, B, dtype):
    m = model(d, mixer, mult, norm=norm, dtype=dtype)
    ids = synth.token_ids(B, 30, 500, seed=B).to(DEV)
    got, S = steps(Decoder(m, batch=B, int4=group), ids)
    ref, _ = steps(Decoder(read_back(m, group), batch=B), ids, [s.float() for s in S])
    off = float((got - ref).norm() / ref.norm())
    assert off < (1e-4 if dtype == torch.float32 else 3e-2), off
    eager, _ = steps(Decoder(m, batch=B, int4=group, use_graph=False), ids)
    assert torch.equal(eager, got)
    assert healthy() == 0


def test_four_bit_weights_follow_the_model():
    m = model(dtype=BF)
    ids = synth.token_ids(2, 30, 500, seed=1).to(DEV)
    dec = Decoder(m, batch=2, int4=64)
    a, _ = steps(dec, ids)
    with torch.no_grad():
        m.mlp[1].b.weight.mul_(1.5)
        m.mlp[1].b.weight.data = m.mlp[1].b.weight.data.clone()       # moved: the stamp's addresses change
    b, _ = steps(dec, ids)
    assert torch.equal(b, steps(Decoder(m, batch=2, int4=64), ids)[0]) and not torch.equal(a, b)


def controls(B, V, kind):
    g = torch.Generator(device=DEV).manual_seed(5)
    per = lambda lo, hi: lo + (hi - lo) * torch.rand(B, device=DEV, generator=g)
    if kind == "numbers":
        return sampling.Controls(repetition=1.4, frequency=0.3, presence=0.2)
    ids = torch.randint(0, V, (B, 6), device=DEV, generator=g)
    ok = torch.rand(1 if kind == "mask" else B, V, device=DEV, generator=g) < 0.5
    c = sampling.Controls(repetition=per(1.0, 2.0), frequency=per(-1, 1), presence=per(-1, 1), bias=(ids, 3 * torch.randn(B, 6, device=DEV, generator=g)), mask=ok)
    return sampling.Controls(mask=ok) if kind == "mask" else c


@pytest.mark.parametrize("kind", ["numbers", "mask", "all"])
@pytest.mark.parametrize("B,dtype", [(1, BF), (2, torch.float32), (6, BF)])
def test_generated_tokens_under_controls(kind, B, dtype):
    V = 500
    m = model(256 if B == 6 else 128, dtype=dtype, vocab=V)
    c = controls(B, V, kind)
    ids = synth.token_ids(B, 40, V, seed=B).to(DEV)
    out = {}
    for use_graph in (True, False):
        dec = Decoder(m, batch=B, use_graph=use_graph, controls=c)
        out[use_graph] = dec.generate(ids, 24)
    assert torch.equal(out[True], out[False])
    # the same greedy tokens from the steps' own logits, controlled by the definition in 64 bits
    dec = Decoder(m, batch=B)
    lg, toks = dec.prefill(ids), []
    made = torch.full((B, 24), -1, dtype=torch.long, device=DEV)
    kw = dict(repetition=c.repetition, frequency=c.frequency, presence=c.presence, mask=c.mask)
    if c.bias is not None:
        kw.update(bias_ids=c.bias[0], bias=c.bias[1])
    for t in range(24):
        ref, tol = want(lg.float(), prompt=ids if c.sees_prompt else None, generated=made, **kw)
        tok = out[True][:, t].cpu()
        at = ref.gather(1, tok[:, None])[:, 0]
        assert torch.all(at >= ref.amax(1) - 2 * tol.amax(1)), t      # the largest, or within rounding of it
        made[:, t] = out[True][:, t]
        lg = dec.step(made[:, t]).clone()
    # the same decoder again, another prompt of another length and other values in the same settings: the same loop, and its own history
    dec = Decoder(m, batch=B, controls=c)
    assert torch.equal(dec.generate(ids, 24), out[True])
    graph = dec._gen_graph
    short = dec.generate(ids[:, :11], 24)
    assert dec._gen_graph is graph and torch.equal(short, Decoder(m, batch=B, controls=c).generate(ids[:, :11], 24))
    if torch.is_tensor(c.frequency):
        c.frequency.add_(1.0)
        assert torch.equal(dec.generate(ids, 24), Decoder(m, batch=B, controls=c, use_graph=False).generate(ids, 24)) and dec._gen_graph is graph
    dec.controls = None
    assert torch.equal(dec.generate(ids, 24), Decoder(m, batch=B).generate(ids, 24))


def test_a_captured_loop_reads_the_settings_of_its_own_call():
    """Settings that were others in between, while the loop was not in use."""
    V = 500
    m = model(dtype=BF, vocab=V)
    ids = synth.token_ids(2, 20, V, seed=7).to(DEV)
    one, other = sampling.Controls(frequency=torch.full((2,), 0.5, device=DEV)), sampling.Controls(mask=torch.arange(V, device=DEV)[None] < 50)
    dec = Decoder(m, batch=2, controls=one)
    first = dec.generate(ids, 24)
    for between in (other, None):
        dec.use_graph, dec.controls = False, between
        dec.generate(ids, 24)
        dec.use_graph, dec.controls = True, sampling.Controls(frequency=torch.full((2,), 3.0, device=DEV))
        assert torch.equal(dec.generate(ids, 24), Decoder(m, batch=2, controls=dec.controls).generate(ids, 24))
        dec.controls = one
        assert torch.equal(dec.generate(ids, 24), first)


def test_a_sampled_loop_keeps_to_its_mask():
    V, B = 500, 3
    m = model(dtype=BF, vocab=V)
    ids = synth.token_ids(B, 20, V, seed=2).to(DEV)
    ok = torch.zeros(B, V, dtype=torch.bool, device=DEV)
    ok[:, 100:117] = True
    bits = (torch.nn.functional.pad(ok, (0, 12)).view(B, 16, 32).long() << torch.arange(32, device=DEV)).sum(2).to(torch.int32)
    for mask in (ok, bits):
        got = Decoder(m, batch=B, int4=32, controls=sampling.Controls(mask=mask)).generate(ids, 64, temp=5.0, seed=3)
        assert bool(((got >= 100) & (got < 117)).all()) and got.unique().numel() > 8
    # nothing allowed: the draw takes id 0
    none = torch.zeros(1, V, dtype=torch.bool, device=DEV)
    assert bool((Decoder(m, batch=B, controls=sampling.Controls(mask=none)).generate(ids, 5, temp=1.0) == 0).all())


def test_refusals():
    m = model(dtype=BF)
    with pytest.raises(ValueError, match="group"):
        Decoder(m, batch=1, int4=48)
    with pytest.raises(ValueError, match="associative"):
        Decoder(LM(vocab=100, d=128, layers=1, mlp_mult=1, ctx=32, mixer="fspin").to(DEV), batch=1, int4=64)
    with pytest.raises(ValueError, match="device"):
        Decoder(m, batch=1, controls=sampling.Controls(mask=torch.ones(1, 500, dtype=torch.bool))).generate(torch.zeros(1, 4, dtype=torch.long, device=DEV), 2)
    assert Decoder(m, batch=1, controls=sampling.Controls()).generate(torch.zeros(1, 4, dtype=torch.long, device=DEV), 2).shape == (1, 2)
