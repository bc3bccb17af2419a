"""CPU-only checks of the four-bit weights and of the logits' adjustment: what is refused on the host, before a launch, by the C entry points and by
the Python ones, and the registered operators' shape functions."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from pragnosia_b200 import custom_ops, int4, sampling  # noqa: F401
from pragnosia_b200._lib import lib

OPS = torch.ops.pragnosia_b200
BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
at = ctypes.c_void_p
one, off1, off2, off4, off8 = (at(0x1000 + i) for i in (0, 1, 2, 4, 8))       # never dereferenced
NULL, SHAPE, ALIGN, DTYPE, LARGE = 1, 2, 4, 5, 7


def quantize(w=one, dtype=1, q=one, s=one, z=one, N=4, K=64, group=64):
    return lib().pgb_int4_quantize(w, dtype, q, s, z, N, K, group, None)


def dequantize(q=one, s=one, sd=1, z=one, w=one, dtype=1, N=4, K=64, group=64):
    return lib().pgb_int4_dequantize(q, s, sd, z, w, dtype, N, K, group, None)


def linear(x=one, xd=1, q=one, s=one, sd=1, z=None, b=None, act=0, y=one, od=1, sc=None, n=0, M=1, N=4, K=64, group=64, flags=0):
    return lib().pgb_int4_linear(x, xd, q, s, sd, z, b, act, y, od, sc, n, M, N, K, group, flags, None)


def adjust(l=one, dtype=0, stride=10, out=at(0x9000), p=None, ps=0, pn=0, pl=None, pls=0, g=None, gs=0, gn=0, gl=None, gls=0, rt=None, r=1.0, ft=None, pt=None,
           bi=None, bv=None, nb=0, mask=None, kind=0, B=2, V=10):
    return lib().pgb_adjust_logits(l, dtype, stride, out, p, ps, pn, pl, pls, g, gs, gn, gl, gls, rt, r, ft, 0.0, pt, 0.0, bi, bv, 0, nb, mask, kind, 0, B, V, None)


SIZES = [(dict(N=0), SHAPE), (dict(K=0), SHAPE), (dict(K=40), SHAPE), (dict(K=16), SHAPE), (dict(group=16), SHAPE), (dict(group=0), SHAPE), (dict(group=256), SHAPE),
         (dict(N=(1 << 24) + 1), LARGE), (dict(K=(1 << 24) + 32), LARGE), (dict(N=1 << 24, K=1 << 24), LARGE)]


@pytest.mark.parametrize("call,kw,code", [
    *[(f, kw, code) for f in (quantize, dequantize, linear) for kw, code in SIZES],
    *[(quantize, {n: None}, NULL) for n in ("w", "q", "s")], (quantize, dict(dtype=2), DTYPE), (quantize, dict(w=off8), ALIGN), (quantize, dict(q=off4), ALIGN),
    (quantize, dict(s=off1), ALIGN), (quantize, dict(s=off2, dtype=0), ALIGN),
    *[(dequantize, {n: None}, NULL) for n in ("w", "q", "s")], (dequantize, dict(dtype=2), DTYPE), (dequantize, dict(sd=-1), DTYPE), (dequantize, dict(w=off8), ALIGN),
    *[(linear, {n: None}, NULL) for n in ("x", "q", "s", "y")], (linear, dict(xd=2), DTYPE), (linear, dict(sd=2), DTYPE), (linear, dict(od=2), DTYPE),
    (linear, dict(M=0), SHAPE), (linear, dict(M=1 << 31), LARGE), (linear, dict(act=2), SHAPE), (linear, dict(act=-1), SHAPE), (linear, dict(flags=2), SHAPE),
    *[(linear, dict(xd=0, M=64, N=4096, K=768, **kw), code) for kw, code in ((dict(), NULL), (dict(sc=one, n=6 * 64 * 768 - 1), SHAPE), (dict(sc=off8, n=1 << 20), ALIGN))],
    (linear, dict(x=off8), ALIGN), (linear, dict(q=off8), ALIGN), (linear, dict(y=off8), ALIGN), (linear, dict(b=off1), ALIGN), (linear, dict(b=off2, xd=0), ALIGN),
    (adjust, dict(l=None), NULL), (adjust, dict(out=None), NULL), (adjust, dict(pn=3), NULL), (adjust, dict(gn=3), NULL), (adjust, dict(nb=3), NULL),
    (adjust, dict(nb=3, bi=one), NULL), (adjust, dict(kind=1), NULL), (adjust, dict(dtype=3), DTYPE), (adjust, dict(B=0), SHAPE), (adjust, dict(V=0), SHAPE),
    (adjust, dict(pn=-1), SHAPE), (adjust, dict(gn=-1), SHAPE), (adjust, dict(nb=-1), SHAPE), (adjust, dict(kind=3, mask=one), SHAPE), (adjust, dict(pls=2), SHAPE),
    (adjust, dict(gls=-1), SHAPE), (adjust, dict(r=0.0), SHAPE), (adjust, dict(r=-1.0), SHAPE), (adjust, dict(r=float("nan")), SHAPE),
    (adjust, dict(nb=1025, bi=one, bv=one), LARGE), (adjust, dict(V=(1 << 30) + 1), LARGE), (adjust, dict(B=1 << 31), LARGE), (adjust, dict(B=1 << 20, V=1 << 30), LARGE),
    (adjust, dict(l=off2), ALIGN), (adjust, dict(out=off2), ALIGN), (adjust, dict(p=off4, pn=1), ALIGN), (adjust, dict(gl=off4), ALIGN), (adjust, dict(rt=off2), ALIGN),
    (adjust, dict(bi=off4, bv=one, nb=1), ALIGN), (adjust, dict(mask=off2, kind=1), ALIGN), (adjust, dict(out=one, dtype=1), SHAPE), (adjust, dict(out=one, stride=12), SHAPE)])
def test_bad_calls(call, kw, code):
    assert call(**kw) == code


def test_scratch_of_the_linear_layer():
    n = lib().pgb_int4_linear_scratch_bytes
    assert n(0, 0, 64, 4096, 768) == n(0, 1, 64, 4096, 768) == 6 * 64 * 768 and n(0, 0, 1 << 20, 64, 4096) == 6 * 4096 * 10880 and n(0, 0, 1 << 20, 64, 1 << 24) == 6 * 64 << 24
    assert n(0, 0, 64, 1024, 768) == n(0, 0, 8, 1 << 20, 768) == n(1, 0, 64, 4096, 768) == n(1, 1, 64, 4096, 768) == 0     # few, or bf16
    assert n(0, 0, 0, 4096, 768) == n(0, 0, 1 << 31, 4096, 768) == n(0, 0, 64, 0, 768) == n(0, 0, 64, 4096, 100) == 0


def held(N=5, K=96, group=64, zeros=True, **kw):
    G = -(-K // group)
    return int4.Int4Weight(torch.zeros(N, K // 2, dtype=U8, **kw), torch.zeros(N, G, dtype=BF, **kw), torch.zeros(N, G, dtype=U8, **kw) if zeros else None, group)


def test_python_refusals():
    x, w = torch.zeros(2, 96), held()
    assert w.shape == (5, 96)
    for call in (lambda: int4.quantize(x), lambda: int4.dequantize(w), lambda: int4.linear(x, w), lambda: sampling.adjust_logits(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="act"):
        int4.linear(x, w, act="relu")
    for bad in (torch.float16, torch.int32):
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            int4.linear(x, w, out_dtype=bad)
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            int4.dequantize(w, bad)


def sig(t):
    return tuple(t.shape), t.dtype


def test_shape_functions():
    with FakeTensorMode():
        e = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device="cuda")
        for sym in (False, True):
            w = int4.quantize(e(5, 96), 64, sym)
            assert sig(w.q) == ((5, 48), U8) and sig(w.scales) == ((5, 2), BF) and (w.zeros is None if sym else sig(w.zeros) == ((5, 2), U8)) and w.shape == (5, 96)
            assert sig(int4.dequantize(w)) == ((5, 96), BF) and sig(int4.dequantize(w, F32)) == ((5, 96), F32)
            assert sig(int4.linear(e(2, 3, 96), w)) == ((2, 3, 5), BF) and sig(int4.linear(e(2, 96), w, e(5), act="gelu", out_dtype=F32)) == ((2, 5), F32)
        l, ids = e(2, 40), e(2, 7, dtype=torch.long)
        assert sig(sampling.adjust_logits(l, prompt=ids, repetition=1.1)) == ((2, 40), F32)
        assert sig(sampling.adjust_logits(l, generated=ids, frequency=e(2, dtype=F32), mask=e(2, 2, dtype=torch.int32))) == ((2, 40), F32)
    for name in ("int4_quantize", "int4_dequantize", "int4_linear", "adjust_logits"):
        schema = getattr(OPS, name).default._schema
        assert not any(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments), name
