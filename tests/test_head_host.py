"""CPU-only checks of the head's losses and the embedding: what is refused on the host, before a launch, by the C entry points and by the
Python ones, and the registered operators' shape functions."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from pragnosia_b200 import custom_ops, head  # noqa: F401
from pragnosia_b200._lib import HOST_PATH, lib

OPS = torch.ops.pragnosia_b200
BF, F32 = torch.bfloat16, torch.float32
one, odd = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1004)           # never dereferenced
BIG = 1 << 40


def xent_fwd(h=one, W=one, dtype=1, target=one, ignore=-100, rows=None, loss=one, stats=one, L=one, scratch=one, n=BIG, red=2, N=4, V=10, d=64):
    return lib().pgb_linear_xent_fwd(h, W, dtype, target, ignore, rows, loss, stats, L, scratch, n, red, N, V, d, None)


def xent_bwd(h=one, W=one, dtype=1, target=one, L=one, stats=one, grad=one, dh=one, dW=one, scratch=one, n=BIG, red=2, N=4, V=10, d=64):
    return lib().pgb_linear_xent_bwd(h, W, dtype, target, -100, L, stats, grad, dh, dW, scratch, n, red, N, V, d, None)


def distill_fwd(lists=one, marks=one, ent=one, kept=one, k=4, tau=1.0):
    return lib().pgb_linear_distill_fwd(one, one, 1, lists, marks, ent, kept, k, tau, None, one, one, one, one, BIG, 2, 4, 10, 64, None)


NULL, SHAPE, ALIGN, DTYPE, LARGE = 1, 2, 4, 5, 7


@pytest.mark.parametrize("call,kw,code", [
    *[(xent_fwd, {n: None}, NULL) for n in ("h", "W", "target", "loss", "stats", "L", "scratch")], (xent_fwd, dict(red=0), NULL),
    (xent_fwd, dict(dtype=2), DTYPE), (xent_fwd, dict(N=0), SHAPE), (xent_fwd, dict(V=0), SHAPE), (xent_fwd, dict(d=0), SHAPE), (xent_fwd, dict(d=60), SHAPE),
    (xent_fwd, dict(red=3), SHAPE), (xent_fwd, dict(red=-1), SHAPE), (xent_fwd, dict(n=100), SHAPE), (xent_fwd, dict(h=odd), ALIGN), (xent_fwd, dict(W=odd), ALIGN),
    (xent_fwd, dict(target=odd), ALIGN), (xent_fwd, dict(L=odd), ALIGN), (xent_fwd, dict(scratch=odd), ALIGN),
    (xent_fwd, dict(N=(1 << 30) + 1), LARGE), (xent_fwd, dict(V=(1 << 30) + 1), LARGE), (xent_fwd, dict(d=65544), LARGE), (xent_fwd, dict(N=1 << 30, V=1 << 24), LARGE),
    *[(xent_bwd, {n: None}, NULL) for n in ("h", "W", "target", "L", "stats", "grad", "scratch")], (xent_bwd, dict(dh=None, dW=None), NULL),
    (xent_bwd, dict(dh=odd), ALIGN), (xent_bwd, dict(dW=odd), ALIGN), (xent_bwd, dict(n=100), SHAPE), (xent_bwd, dict(d=12), SHAPE),
    *[(distill_fwd, {n: None}, NULL) for n in ("lists", "marks", "ent", "kept")], (distill_fwd, dict(k=0), SHAPE), (distill_fwd, dict(k=1025), LARGE),
    (distill_fwd, dict(tau=0.0), SHAPE), (distill_fwd, dict(tau=-1.0), SHAPE), (distill_fwd, dict(tau=float("inf")), SHAPE), (distill_fwd, dict(tau=float("nan")), SHAPE),
    (distill_fwd, dict(lists=odd), ALIGN), (distill_fwd, dict(marks=ctypes.c_void_p(0x1008)), ALIGN)])
def test_bad_calls_of_the_losses(call, kw, code):
    assert call(**kw) == code


def test_bad_calls_of_teacher_lists_and_embedding():
    L = lib()
    lists = lambda a=one, b=one, tau=1.0, o=one, m=one, e=one, N=4, V=9, k=3: L.pgb_teacher_lists(a, b, tau, o, m, e, N, V, k, None)
    assert all(lists(**{n: None}) == NULL for n in "abome")
    assert lists(k=0) == lists(N=0) == lists(V=0) == lists(tau=0.0) == SHAPE and lists(k=1025) == LARGE and lists(o=odd) == lists(m=odd) == lists(a=odd) == ALIGN
    fwd = lambda i=one, w=one, dt=1, y=one, N=3, V=5, d=7: L.pgb_embedding_fwd(i, w, dt, 1.0, y, N, V, d, None)
    assert fwd(i=None) == fwd(w=None) == fwd(y=None) == NULL and fwd(dt=3) == DTYPE and fwd(N=0) == fwd(V=0) == fwd(d=0) == SHAPE
    assert fwd(i=odd) == fwd(w=ctypes.c_void_p(0x1001)) == ALIGN and fwd(N=(1 << 30) + 1) == LARGE
    bwd = lambda i=one, g=one, dt=1, w=one, s=one, n=BIG, N=600, V=5, d=7: L.pgb_embedding_bwd(i, g, dt, 1.0, -1, w, s, n, N, V, d, None)
    assert bwd(i=None) == bwd(g=None) == bwd(w=None) == bwd(s=None) == NULL and bwd(n=10) == SHAPE and bwd(d=65537) == LARGE and bwd(s=odd) == ALIGN
    assert bwd(N=3, s=None, n=0, g=None) == NULL and bwd(N=3, s=None, n=0, d=65537) == LARGE       # few tokens need no scratch
    assert L.pgb_embedding_bwd_scratch_bytes(256, 9, 64) == 0 < L.pgb_embedding_bwd_scratch_bytes(257, 9, 64)
    assert L.pgb_head_loss_fwd_scratch_bytes(0, 5, 64, 1) == 0 and L.pgb_head_loss_bwd_scratch_bytes(5, 5, 63, 1, 1, 1) == 0 and L.pgb_embedding_bwd_scratch_bytes(1, 0, 4) == 0


@pytest.mark.parametrize("N,V,d,dtype", [(1, 1, 8, 1), (511, 8192, 768, 1), (32768, 8192, 768, 1), (8192, 50257, 768, 1), (2000, 8192, 704, 0), (100000, 300, 4096, 1),
                                         (7, 262144, 4096, 1), (1 << 20, 1 << 17, 4096, 1), (3, 1 << 24, 64, 0)])
def test_scratch_stays_far_below_the_logits(N, V, d, dtype):
    """The workspace of the backward pass: two pieces of 64 MiB (a block of 256 rows or columns where that is more), fp32 sums of the smaller
    gradient, split operands or a clean copy of h. Asked twice, the same."""
    L = lib()
    for want in ((1, 1), (1, 0), (0, 1)):
        n = L.pgb_head_loss_bwd_scratch_bytes(N, V, d, dtype, *want)
        assert n == L.pgb_head_loss_bwd_scratch_bytes(N, V, d, dtype, *want) > 0
        terms = 3 if dtype == 0 else 1
        pieces = 2 * max(64 << 20, 2 * terms * 256 * (min(N, V) + 512)) + (1 << 20)
        sums = 4 * 32 * d * 2 * (min(N, V) + 8192 + 512) if N * V < (1 << 27) else 4 * d * (min(N, V) + max(N, V)) * 4
        copies = 6 * d * (N + V) if dtype == 0 else 2 * d * N if want[1] else 0
        assert n <= pieces + sums + copies + 1024


def test_python_refusals():
    h, w, t = torch.randn(4, 16), torch.randn(9, 16), torch.zeros(4, dtype=torch.long)
    for call in (lambda: head.linear_cross_entropy(h, w, t), lambda: head.linear_distill(h, w, t[:, None], h[:, :1]), lambda: head.embedding(t, w)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="reduction"):
        head.linear_cross_entropy(h, w, t, reduction="avg")
    with pytest.raises(ValueError, match="reduction"):
        head.linear_distill(h, w, t[:, None], h[:, :1], reduction=None)
    for pad in (-1, 9):
        with pytest.raises(ValueError, match="padding_idx"):
            head.embedding(t, w, padding_idx=pad)


def sig(t):
    return tuple(t.shape), t.dtype


def test_shape_functions():
    with FakeTensorMode():
        e = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device="cuda")
        h, w, t = e(2, 5, 64), e(33, 64), e(2, 5, dtype=torch.long)
        for red, shape in ((0, (10,)), (1, ()), (2, ())):
            loss, L, stats = OPS.linear_xent(h, w, t, -100, red)
            assert sig(loss) == (shape, F32) and sig(L) == ((10, 2), F32) and sig(stats) == ((2,), F32)
        dh, dw = OPS.linear_xent_bwd(h, w, t, -100, L, stats, loss, 2, True, True)
        assert sig(dh) == ((2, 5, 64), BF) and sig(dw) == ((33, 64), BF)
        dh, dw = OPS.linear_xent_bwd(h, w, t, -100, L, stats, loss, 2, True, False)
        assert sig(dh) == ((2, 5, 64), BF) and dw.numel() == 0
        lists, marks, ent = OPS.teacher_lists(e(2, 5, 7, dtype=torch.long), e(2, 5, 7, dtype=F32), 2.0, 130)
        assert sig(lists) == ((10, 7, 2), torch.int32) and sig(marks) == ((10, 3, 4), torch.int32) and sig(ent) == ((10,), F32)
        loss, L, stats, kept = OPS.linear_distill(h, w, lists, marks, ent, 2.0, 0)
        assert sig(loss) == ((10,), F32) and sig(kept) == ((10, 7), F32)
        dh, dw = OPS.linear_distill_bwd(h, w, lists, ent, kept, 2.0, L, stats, loss, 0, True, True)
        assert sig(dh) == ((2, 5, 64), BF) and sig(dw) == ((33, 64), BF)
        assert sig(OPS.embedding(t, w, 1.0, -1)) == ((2, 5, 64), BF) and sig(OPS.embedding_bwd(t, h, 1.0, -1, 33)) == ((33, 64), BF)
        with torch.enable_grad():
            w.requires_grad_()
            y = head.embedding(t, w)
            assert sig(head.linear_cross_entropy(y, w, t, reduction="none")) == ((2, 5), F32) and head.linear_cross_entropy(y, w, t).requires_grad
            assert sig(head.linear_distill(y, w, e(2, 5, 3, dtype=torch.long), e(2, 5, 3, dtype=F32), reduction="none")) == ((2, 5), F32)
    for name in ("linear_xent", "linear_xent_bwd", "teacher_lists", "linear_distill", "linear_distill_bwd", "embedding", "embedding_bwd"):
        schema = getattr(OPS, name).default._schema
        assert not any(a.alias_info is not None and a.alias_info.is_write for a in schema.arguments), name


def test_the_module_shares_torch_s_cxx_library():
    """With a libstdc++ of its own in it, the check that refuses a call on a GPU crashes the process where it writes its message."""
    with open(HOST_PATH, "rb") as f:
        assert b"libstdc++.so.6\0" in f.read()
