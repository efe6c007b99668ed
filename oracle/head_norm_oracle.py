"""Float64 restatements (torch, CPU or wherever the inputs are) of the block norms and the head's losses used in training.

Test infrastructure: formulas and their analytic gradients; `tests/test_head_norm_cpu.py` checks the gradients against
central differences.
"""
from __future__ import annotations

import torch


def layer_norm(s, weight, bias, eps):
    s, weight, bias = s.double(), weight.double(), bias.double()
    mean = s.mean(-1, keepdim=True)
    rstd = (((s - mean) ** 2).mean(-1, keepdim=True) + eps).rsqrt()
    return (s - mean) * rstd * weight + bias


def layer_norm_backward(grad, s, weight, eps):
    """`(d s, d weight, d bias)`."""
    grad, s, weight = grad.double(), s.double(), weight.double()
    mean = s.mean(-1, keepdim=True)
    rstd = (((s - mean) ** 2).mean(-1, keepdim=True) + eps).rsqrt()
    unit = (s - mean) * rstd
    h = grad * weight
    ds = rstd * (h - h.mean(-1, keepdim=True) - unit * (h * unit).mean(-1, keepdim=True))
    axes = tuple(range(grad.ndim - 1))
    return ds, (grad * unit).sum(axes), grad.sum(axes)


def teacher_shares(teacher_logits, temperature):
    """`(p, used)`: the teacher's renormalised probabilities (0 where an entry is absent, i.e. -inf) and which rows have any."""
    soft = teacher_logits.double() / temperature
    used = (soft > float("-inf")).any(-1)
    soft = torch.where(used[:, None], soft, torch.zeros_like(soft))
    return torch.softmax(soft, -1) * used[:, None], used


def head_losses(x, weight, labels, shares, temperature=1.0):
    """Per-row losses `T^2 sum_k p_k (log p_k - log q[label_k])`, q = softmax(x W^T / T); entries with p = 0 count nothing."""
    log_q = torch.log_softmax(x.double() @ weight.double().T / temperature, -1)
    picked = log_q.gather(1, torch.where(shares > 0, labels.long(), 0))
    return temperature ** 2 * (torch.special.xlogy(shares, shares) - shares * picked).sum(-1)


def head_backward(row_grads, x, weight, labels, shares, temperature=1.0):
    """`(d x, d weight)` of `sum(row_grads * head_losses)`; rows without any share contribute nothing."""
    x, weight = x.double(), weight.double()
    g = torch.softmax(x @ weight.T / temperature, -1) * shares.sum(-1, keepdim=True)
    g.scatter_add_(1, torch.where(shares > 0, labels.long(), 0), -shares)
    g *= temperature * row_grads.double()[:, None]
    return g @ weight, g.T @ x
