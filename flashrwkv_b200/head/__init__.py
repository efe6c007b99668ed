"""Losses of the head for training: the vocabulary projection fused with its softmax and the loss, forward and backward.

`x [...,C]` are the normalised rows behind the last block and `weight [V,C]` the head's weight, both bf16.  Logits are not
kept in fp32: while a call runs, a workspace holds one 16-bit value for each logit of a piece of the rows, at most 1 GiB.
The gradients of a scalar loss are made together with it, in the forward call, and only for the inputs that require one; the
upstream gradient scales them when the backward pass runs, which costs a pass over them and a second rounding to bf16 unless
it is 1 (powers of two round nothing).  A backward pass repeated over a retained graph, or captured apart from its forward
pass, makes them again, at the price of a whole step.  The gradients of row losses are made in the backward pass, which
repeats the forward's product.  The backward passes are not differentiable themselves.

The reference fuses its cross entropy with an L2 penalty of the largest logit (`csrc/sm90/head/l2wrap_ce`), which is not
part of these operators; it has no distillation.
"""
from __future__ import annotations

import torch

from .._ext import extension

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _check(reduction, **tensors) -> int:
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    return _REDUCTIONS[reduction]


def pretrain_head_cross_entropy_bf16(x, weight, targets, *, ignore_index: int = -100, reduction: str = "mean"):
    """Cross entropy of `softmax(x @ weight^T)` against `targets` (int32 or int64, x's leading shape), in fp32.

    Differentiable in x and weight.  Rows whose target is `ignore_index` take no part: their loss is 0, their gradient 0,
    and what x holds there reaches nothing.  `reduction="mean"` divides by the number of rows that take part (0 where there
    is none), `"none"` returns the losses of all rows in x's leading shape.  A target outside `[0,V)` makes its row's loss
    and the gradients NaN."""
    code = _check(reduction, x=x, weight=weight, targets=targets)
    if not isinstance(ignore_index, int) or isinstance(ignore_index, bool) or abs(ignore_index) >= 2 ** 63:
        raise ValueError("ignore_index must be an integer")
    return extension().pretrain_head_loss(x, weight, targets, None, ignore_index, 1.0, code)


def pretrain_head_distill_bf16(x, weight, teacher_logits, teacher_indices, *, temperature: float = 1.0,
                               reduction: str = "mean"):
    """Distillation from a teacher's highest logits: `temperature^2 * KL(p || softmax(x @ weight^T / temperature))` per row,
    in fp32, where p is the softmax of `teacher_logits / temperature` over the row's entries.

    `teacher_logits` (fp32, fp16 or bf16) and `teacher_indices` (int32 or int64) are `[...,K]`, K up to 512, with x's
    leading shape.  An entry of -inf is absent, whatever its index; a row without any entry takes no part, as a row without
    a label in `pretrain_head_cross_entropy_bf16`.  An index may occur more than once: each occurrence is
    an entry of its own in p and in the sum, and in the gradient their shares add up.  An index outside `[0,V)` makes its
    row's loss and the gradients NaN.  Differentiable in x and weight."""
    code = _check(reduction, x=x, weight=weight, teacher_logits=teacher_logits, teacher_indices=teacher_indices)
    if not isinstance(temperature, (int, float)) or isinstance(temperature, bool):
        raise ValueError("temperature must be positive")
    return extension().pretrain_head_loss(x, weight, teacher_indices, teacher_logits, -100, float(temperature), code)


__all__ = ["pretrain_head_cross_entropy_bf16", "pretrain_head_distill_bf16"]
