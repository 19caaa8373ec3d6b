"""Gradients that can be differentiated once, in a graph of the backward pass.

A kernel writes a gradient through a pointer, so what it returns has no graph of its own. Under
``create_graph=True`` torch would take it for a constant, and a penalty on it would leave its part
out of the next gradients without a word. An autograd node therefore passes its gradients through
:func:`once`, which ties them to what they were formed from; differentiating them again raises.
"""

from __future__ import annotations

import torch


class _Once(torch.autograd.Function):
    """A gradient as it is, between ``sources`` and those who differentiate it."""

    @staticmethod
    def forward(ctx, name, grad, *sources):
        ctx.name = name
        return grad.detach()

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"{ctx.name}: trying to differentiate twice; its gradients are formed by "
                           "kernels that have no gradient of their own")


def once(name: str, grads, sources) -> tuple:
    """``grads`` for a node's backward to return, ``sources`` the upstream gradients and saved
    tensors. A gradient that has a graph of its own, or is formed from constants, stays as it is."""
    grads = (grads,) if torch.is_tensor(grads) else tuple(grads)
    if not torch.is_grad_enabled():
        return grads
    sources = [t for t in sources if torch.is_tensor(t) and t.requires_grad]
    if not sources:
        return grads
    return tuple(_Once.apply(name, g, *sources) if torch.is_tensor(g) and not g.requires_grad else g
                 for g in grads)


def needs_tie(args, saved, outputs) -> bool:
    """Whether a saved tensor hides an argument that requires gradients and is not saved itself: one
    of as many elements (the copy of a strided argument, or what an activation has become)."""
    kept = [id(t) for t in saved]
    for arg in args:
        if not torch.is_tensor(arg) or not arg.requires_grad or id(arg) in kept:
            continue
        for t in saved:
            if (t.numel() == arg.numel() and t.is_floating_point()
                    and not any(t is known for known in (*args, *outputs))):
                return True
    return False


def tie() -> torch.Tensor:
    """An output without elements for such a node: saved among the others, it leads from the
    gradients back to the node's arguments and keeps no memory."""
    return torch.empty(0)
