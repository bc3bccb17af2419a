"""The two ends of the language model in training: its tokens' embedding, and the losses over the vocabulary straight from the
hidden states and the (tied) head's weight, without the logits in memory. The reference looks up with nn.Embedding (src/model.py:859)
and takes torch's cross entropy of whole logits (src/train.py:49); distillation has no counterpart there.

All three are differentiable, take CUDA tensors in float32 or bfloat16, launch on torch's current stream and never synchronise.
Eagerly they run as C++ autograd nodes (csrc/torch_host.cpp); under torch.compile, a tracer or a dispatch mode as the operators
of pragnosia_b200.custom_ops.
"""
from __future__ import annotations

import torch

from ._lib import host

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _reduction(name: str) -> int:
    if name not in _REDUCTIONS:
        raise ValueError(f"reduction is one of {sorted(_REDUCTIONS)}, got {name!r}")
    return _REDUCTIONS[name]


def _operators():
    from . import custom_ops  # noqa: F401  (registers them)
    return torch.ops.pragnosia_b200


def linear_cross_entropy(h, weight, target, *, ignore_index: int = -100, reduction: str = "mean"):
    """Softmax cross entropy of the logits h weight^T against `target`, which never lie in memory together.

    h (..., d); weight (V, d) of h's type, d a multiple of 8; target (...) int64 or int32. Returns float32: a loss per row (reduction
    "none", target's shape), their sum, or their mean over the rows whose target is not ignore_index (nan where there is none, as torch has it).
    Ignored rows lose 0 and have no gradient, whatever h holds there. Any other target outside 0 .. V-1 gives nan, in the loss and in the gradients of its row and of the weight.

    Without a gradient wanted (no_grad, or neither tensor requires one) this is the scoring of given tokens, one to many. bf16: products
    in bf16 with fp32 sums; the gradient of the logits is rounded to bf16 on its way into the two products behind it. float32: float32's own precision."""
    r = _reduction(reduction)
    if not torch.compiler.is_compiling():
        out = host().linear_xent(h, weight, target, int(ignore_index), r)
        if out is not None:
            return out
    loss = _operators().linear_xent(h, weight, target, int(ignore_index), r)[0]
    return loss.view(target.shape) if r == 0 else loss


def linear_distill(h, weight, teacher_ids, teacher_logits, *, temperature: float = 1.0, reduction: str = "mean"):
    """Distillation from a teacher's top logits: temperature^2 KL(p || softmax(h weight^T / temperature)), with p the softmax of the
    teacher's k logits at the same temperature (over those k words alone) and the student's softmax over the whole vocabulary.

    h, weight as in linear_cross_entropy; teacher_ids (..., k) int64 or int32, teacher_logits (..., k), k in 1 .. 1024, in any order.
    An entry with id < 0 or logit -inf is absent, so lists may differ in length; a row without any loses 0, has no gradient and
    does not count in the mean (nan where all are without). An id twice counts twice; an id >= V gives nan. No gradient goes to the teacher.

    bf16: the gradient of the logits, which has several large entries a row here, is rounded to bf16 on its way into the two products behind it, beside
    the gradients' own rounding (2-norm against 64 bits: 0.0023, where fp32 logits give 0.0017). Beside the results the call takes V / 4 bytes a row
    while it runs and keeps 12 k + 16 for the gradient. Sorting lists takes k^2: 4096 of 64 entries 10 us, of 256 60, of 1024 795."""
    r = _reduction(reduction)
    if not torch.compiler.is_compiling():
        out = host().linear_distill(h, weight, teacher_ids, teacher_logits, float(temperature), r)
        if out is not None:
            return out
    if teacher_ids.shape[:-1] != h.shape[:-1] or teacher_ids.dim() != h.dim() or teacher_logits.shape != teacher_ids.shape:     # the operators see rows only
        raise ValueError(f"linear_distill: k teacher entries per row of h, got {tuple(teacher_ids.shape)} and {tuple(teacher_logits.shape)} for {tuple(h.shape)}")
    ops = _operators()
    lists, marks, ent = ops.teacher_lists(teacher_ids, teacher_logits.detach(), float(temperature), weight.shape[0])
    loss = ops.linear_distill(h, weight, lists, marks, ent, float(temperature), r)[0]
    return loss.view(h.shape[:-1]) if r == 0 else loss


def embedding(ids, weight, *, scale: float = 1.0, padding_idx: int | None = None):
    """scale * weight[ids], rounded once to weight's type; ids of any shape, int64 or int32. An id outside 0 .. V-1 gives a row of nan.

    The weight's gradient is dense: every word's rows of the incoming gradient added up in float32 in the order of the tokens (the
    same bits every time), scaled and rounded once. padding_idx: a word that is looked up as any other and gets no gradient."""
    pad = -1 if padding_idx is None else int(padding_idx)
    if padding_idx is not None and not 0 <= pad < weight.shape[0]:
        raise ValueError(f"padding_idx is a word of the table (0 .. {weight.shape[0] - 1}), got {padding_idx}")
    if not torch.compiler.is_compiling():
        out = host().embedding(ids, weight, float(scale), pad)
        if out is not None:
            return out
    return _operators().embedding(ids, weight, float(scale), pad)
