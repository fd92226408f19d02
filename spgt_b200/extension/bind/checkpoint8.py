"""Layers that keep what their backward pass needs in 8 bits (ops.Checkpoint8), differentiable once.  Their values are those of the
plain layers; their gradients are those of the formulas at the rounded input.  The reference has no counterpart."""
import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ... import ops


class Activation8_Function(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, activation):
        Y, kept = ops.activation8(X.contiguous(), activation)
        ctx.args = (activation, X.shape, X.dtype)
        ctx.save_for_backward(kept.codes, kept.steps)
        return Y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        activation, shape, dtype = ctx.args
        kept = ops.Checkpoint8._of(*ctx.saved_tensors, shape, dtype)
        return ops.activation8_backward(grad_out.contiguous(), kept, activation), None


class Linear8_Function(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, weight, bias):
        ctx.args = (X.shape, X.dtype, bias is not None)
        if any(ctx.needs_input_grad[1:]):
            kept = ops.compress8(X.contiguous())
            ctx.save_for_backward(weight, kept.codes, kept.steps)
        else:                                               # a frozen layer
            ctx.save_for_backward(weight)
        return torch.nn.functional.linear(X, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        weight, *kept = ctx.saved_tensors
        shape, dtype, has_bias = ctx.args
        dX = dw = db = None
        if ctx.needs_input_grad[0]:
            dX = torch.matmul(grad_out, weight.to(grad_out.dtype)).to(dtype)
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dw, db = ops.weight_gradient8(grad_out.contiguous(), ops.Checkpoint8._of(*kept, shape, dtype), column_sums=has_bias)
            dw, db = dw.to(weight.dtype), None if db is None else db.to(weight.dtype)
        return dX, dw, db


def activation8(X: Tensor, activation) -> Tensor:
    """activation(X), of which the backward pass keeps X in 8 bits."""
    if torch.is_grad_enabled() and X.requires_grad:
        return Activation8_Function.apply(X, activation)
    return ops.activation8(X.contiguous(), activation)[0]


def linear8(X: Tensor, weight: Tensor, bias: Tensor = None) -> Tensor:
    """X weight^T + bias (torch's linear), of which the backward pass keeps X in 8 bits (nothing of X where weight and bias are
    frozen); 1 to ops.WEIGHT8_MOST features in and out."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (X, weight, bias)):
        if not 0 < min(weight.shape) <= max(weight.shape) <= ops.WEIGHT8_MOST:       # (not first in the backward pass)
            raise ValueError(f'linear8 takes 1 to {ops.WEIGHT8_MOST} features, got {tuple(weight.shape)}')
        return Linear8_Function.apply(X, weight, bias)
    return torch.nn.functional.linear(X, weight, bias)
