"""CPU-only checks of the head's losses that stand beside test_head_host.py: what a traced call refuses, sizes of the workspace, temperatures."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from pragnosia_b200 import custom_ops, head  # noqa: F401
from pragnosia_b200._lib import lib
from test_head_host import BF, F32, SHAPE, distill_fwd, one, sig  # noqa: F401


def test_the_traced_call_refuses_a_teacher_of_other_axes():
    """As the eager one does: the operators behind it see rows only, and a teacher of (T, B) has as many as hidden states of (B, T)."""
    with FakeTensorMode():
        e = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device="cuda")
        h, w = e(2, 5, 64), e(33, 64)
        for ids, logits in (((5, 2, 3), (5, 2, 3)), ((10, 3), (10, 3)), ((2, 5, 3), (2, 5, 2)), ((2, 5), (2, 5)), ((2, 5, 1, 3), (2, 5, 1, 3))):
            with pytest.raises(ValueError, match="teacher"):
                head.linear_distill(h, w, e(*ids, dtype=torch.long), e(*logits, dtype=F32))
        assert sig(head.linear_distill(h, w, e(2, 5, 3, dtype=torch.long), e(2, 5, 3, dtype=F32), reduction="none")) == ((2, 5), F32)


@pytest.mark.parametrize("N,V,d", [(1 << 23, 1 << 23, 2048), (1 << 22, 1 << 22, 32768), (1 << 24, 3 << 20, 65536), (1 << 21, 1 << 22, 65536)])
def test_a_long_axis_is_summed_in_parts_that_a_wait_covers(N, V, d):
    """A gradient's product over millions of columns, whose tiles fill the GPU without a cut: its parts are 4096 blocks of 64 at most, 1.4 ms, since
    the wait for one that is not finished may end after some. A part's sums are an fp32 plane of the workspace, beside two pieces of 256 rows or columns
    of the longer axis and a copy of h."""
    by_rows, shorter = N >= V, min(N, V)
    n = lib().pgb_head_loss_bwd_scratch_bytes(N, V, d, 1, int(by_rows), int(not by_rows))
    assert n >= 2 * 2 * 256 * shorter + (0 if by_rows else 2 * N * d) + 4 * (shorter // 64 // 4096) * 256 * d


@pytest.mark.parametrize("tau", [1e-38, 1e-40, 1e-45, -1e-40])
def test_temperatures_whose_reciprocal_is_no_number_are_refused(tau):
    """log2(e) / temperature is what logits are multiplied with."""
    assert distill_fwd(tau=tau) == SHAPE
    assert lib().pgb_teacher_lists(one, one, tau, one, one, one, 4, 9, 3, None) == SHAPE
    assert lib().pgb_linear_distill_bwd(one, one, 1, one, one, one, 4, tau, one, one, one, one, one, one, 1 << 40, 2, 4, 10, 64, None) == SHAPE
