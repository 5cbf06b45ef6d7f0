"""Gradients that cannot be differentiated again."""

from __future__ import annotations

import torch


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, mark, name):
        ctx.name = name
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise NotImplementedError(f"{ctx.name} has no second derivative")


def once(name, *grads):
    """``grads`` as a backward returns them: under ``create_graph`` they raise
    when they are differentiated (without this they would count as constants)."""
    if not torch.is_grad_enabled():
        return grads
    mark = torch.empty(0, requires_grad=True)
    return tuple(g if g is None else _Once.apply(g, mark, name) for g in grads)
