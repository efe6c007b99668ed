"""Training form of the block-level LayerNorm and of add + LayerNorm, with their backward passes, on bf16 tensors.

The reference has the inference forms only (`flashrwkv2/tmix/normalization/__init__.py:31-90`); the forward values here
are theirs, and the gradients of weight and bias are fixed-order fp32 sums over the rows.  Shapes, types, devices and
alignment are checked by the native layer (ValueError), which also holds the autograd functions.
"""
from __future__ import annotations

import torch

from ..._ext import extension


def _check_types(**tensors) -> None:
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")


def pretrain_tmix_layer_norm_bf16(x, weight, bias, *, eps: float = 1.0e-5):
    """`LayerNorm(x)` over the last axis of a bf16 `[...,C]` tensor, differentiable in x, weight and bias.  C is a
    multiple of 8 up to 16384."""
    from . import _check_eps

    _check_types(x=x, weight=weight, bias=bias)
    return extension().pretrain_tmix_layer_norm(x, weight, bias, _check_eps(eps))


def pretrain_tmix_add_layer_norm_bf16(x, residual, weight, bias, *, eps: float = 1.0e-5):
    """Returns `(x + residual, LayerNorm(x + residual))` on bf16 `[...,C]` tensors, differentiable in all four inputs;
    both outputs may carry a gradient (the sum is the residual stream that goes on to the next block).  The gradients of
    x and residual are the same tensor."""
    from . import _check_eps

    _check_types(x=x, residual=residual, weight=weight, bias=bias)
    return extension().pretrain_tmix_add_layer_norm(x, residual, weight, bias, _check_eps(eps))


__all__ = ["pretrain_tmix_layer_norm_bf16", "pretrain_tmix_add_layer_norm_bf16"]
