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
