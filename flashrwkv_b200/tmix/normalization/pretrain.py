"""Training form of the block-level LayerNorm and of add + LayerNorm, with their backward passes, on bf16 tensors.

The reference has the inference forms only (`flashrwkv2/tmix/normalization/__init__.py:31-90`); the forward values here
are theirs, and the gradients of weight and bias are fixed-order fp32 sums over the rows.
"""
from __future__ import annotations

import torch

from ..._ext import extension
from .._checks import check_train_bf16


def _check(x, residual, weight, bias) -> None:
    tensors = {"x": x, "weight": weight, "bias": bias}
    if residual is not None:
        tensors["residual"] = residual
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    check_train_bf16(tensors)
    if x.ndim < 2 or x.numel() == 0:
        raise ValueError("x must have non-empty shape [...,C]")
    if x.shape[-1] % 8 or x.shape[-1] > 16384:
        raise ValueError("C must be a multiple of 8 up to 16384")
    if residual is not None and residual.shape != x.shape:
        raise ValueError("residual must have the same shape as x")
    for name, t in (("weight", weight), ("bias", bias)):
        if t.shape != (x.shape[-1],):
            raise ValueError(f"{name} must have shape [C]")
    for name, t in tensors.items():
        if t.data_ptr() % 16:
            raise ValueError(f"{name} must be 16-byte aligned")


def _ready(grad):
    """An upstream gradient as the kernels read it: packed and 16-byte aligned."""
    grad = grad.contiguous()
    return grad if grad.data_ptr() % 16 == 0 else grad.clone()


def _backward(ctx, grad_sum, grad_out):
    """`(gradient of the sum, of weight, of bias)`; None where nothing is asked or nothing arrives."""
    total, weight, mean, rstd = ctx.saved_tensors
    if grad_out is None:
        return grad_sum, None, None
    parameters = any(ctx.needs_input_grad[-3:-1])
    grads = extension().pretrain_tmix_layer_norm_backward(
        _ready(grad_out), None if grad_sum is None else _ready(grad_sum), total, weight, mean, rstd, parameters)
    return tuple(grads) if parameters else (grads[0], None, None)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        _, out, mean, rstd = extension().pretrain_tmix_layer_norm_forward(x, None, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        return (*_backward(ctx, None, grad_out), None)


class _AddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        total, out, mean, rstd = extension().pretrain_tmix_layer_norm_forward(x, residual, weight, bias, eps)
        ctx.save_for_backward(total, weight, mean, rstd)
        ctx.set_materialize_grads(False)
        return total, out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_sum, grad_out):
        grad_x, grad_weight, grad_bias = _backward(ctx, grad_sum, grad_out)
        return grad_x, grad_x, grad_weight, grad_bias, None


def pretrain_tmix_layer_norm_bf16(x, weight, bias, *, eps: float = 1.0e-5):
    """`LayerNorm(x)` over the last axis of a bf16 `[...,C]` tensor, differentiable in x, weight and bias."""
    from . import _check_eps

    _check(x, None, weight, bias)
    return _LayerNorm.apply(x, weight, bias, _check_eps(eps))


def pretrain_tmix_add_layer_norm_bf16(x, residual, weight, bias, *, eps: float = 1.0e-5):
    """Returns `(x + residual, LayerNorm(x + residual))` on bf16 `[...,C]` tensors, differentiable in all four inputs;
    both outputs may carry a gradient (the sum is the residual stream that goes on to the next block)."""
    from . import _check_eps

    if residual is None:
        raise TypeError("residual must be a torch.Tensor")
    _check(x, residual, weight, bias)
    return _AddLayerNorm.apply(x, residual, weight, bias, _check_eps(eps))


__all__ = ["pretrain_tmix_layer_norm_bf16", "pretrain_tmix_add_layer_norm_bf16"]
