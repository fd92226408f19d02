"""Group normalisation with an activation, channels last, differentiable.  The reference has no counterpart."""
import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ... import ops


class Group_Norm_Act_Function(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, weight, bias, num_groups, eps, activation, activation_bits):
        X = X.contiguous()
        Y, stats, kept = ops.group_norm_forward(X, num_groups, weight, bias, eps, activation, activation_bits == 8)
        ctx.args = (num_groups, activation, X.shape, X.dtype)
        ctx.save_for_backward(weight, bias, stats, *((X,) if kept is None else (kept.codes, kept.steps)))
        return Y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        weight, bias, stats, *saved = ctx.saved_tensors
        num_groups, activation, shape, dtype = ctx.args
        X = saved[0] if len(saved) == 1 else ops.Checkpoint8._of(*saved, shape, dtype)
        dX, dw, db = ops.group_norm_backward(grad_out.contiguous(), X, num_groups, weight, bias, stats, activation)
        return dX, dw if weight is not None else None, db if bias is not None else None, None, None, None, None


def group_norm_act(X: Tensor, num_groups: int, weight: Tensor = None, bias: Tensor = None, eps: float = 1.0e-5, activation=None,
                   activation_bits: int = 32) -> Tensor:
    """activation(group_norm(X) * weight + bias) for X [N, ..., C], channels last (fp32, bf16 or fp16; weight, bias [C] fp32 or None);
    differentiable once in X, weight and bias.  activation_bits=8: the backward pass differentiates at X rounded to 8 bits
    (ops.Checkpoint8), with the forward's statistics, and X itself is not kept."""
    if activation_bits not in (8, 32):
        raise ValueError('activation_bits must be 8 or 32')
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (X, weight, bias)):
        return Group_Norm_Act_Function.apply(X, weight, bias, num_groups, eps, activation, activation_bits)
    return ops.group_norm_forward(X.contiguous(), num_groups, weight, bias, eps, activation, False)[0]
