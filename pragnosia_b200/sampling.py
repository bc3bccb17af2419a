"""What stands between a model's logits and the draw: penalties for words seen before, biases of single words, and a mask of the words that a
grammar allows. The reference draws from the logits as they are (src/bench.py:79-86).

CUDA tensors, torch's current stream, no synchronisation; no gradient (a call that would need one raises).
"""
from __future__ import annotations

import torch

from ._lib import host


def _split(v):
    """A setting as (one per row, one for all)."""
    return (v, 0.0) if torch.is_tensor(v) else (None, float(v))


def adjust_logits(logits, *, prompt=None, prompt_lengths=None, generated=None, generated_lengths=None, repetition=1.0, frequency=0.0, presence=0.0,
                  bias_ids=None, bias=None, mask=None, out=None):
    """logits (B, V), float32 or bfloat16, as a draw wants them: float32 (B, V). With n the times a word stands in a row's generated ids and m the times it
    stands in those and the prompt's, in this order:

        m > 0:  s / repetition where s > 0, else s repetition;      n > 0:  s - frequency n - presence;      + its biases;      -inf where the mask forbids

    prompt, generated: ids (B or 1, n), int64 (or int32), lengths (B,) or a single number on the device, how many of a row count (all without). Ids outside
    0 .. V-1 (padding) count nowhere. repetition (> 0), frequency, presence: numbers, or tensors (B,). bias_ids, bias: (B or 1, k), k up to 1024, an
    id twice counts twice. mask: int32 (B or 1, ceil(V / 32)), bit v % 32 of number v // 32 set where v is allowed, or bool (B or 1, V); a row that allows nothing
    is -inf throughout, from which the draw takes id 0. out: where the result goes, logits itself among others; one launch either way."""
    rt, r = _split(repetition)
    ft, f = _split(frequency)
    pt, p = _split(presence)
    if not torch.compiler.is_compiling():
        done = host().adjust_logits(logits, prompt, prompt_lengths, generated, generated_lengths, rt, r, ft, f, pt, p, bias_ids, bias, mask, out)
        if done is not None:
            return done
    from . import custom_ops  # noqa: F401  (registers the operator)
    done = torch.ops.pragnosia_b200.adjust_logits(logits, prompt, prompt_lengths, generated, generated_lengths, rt, r, ft, f, pt, p, bias_ids, bias, mask)
    return done if out is None else out.copy_(done)
