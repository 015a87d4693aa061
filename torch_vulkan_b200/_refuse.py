"""Backward passes whose gradients cannot be differentiated again."""

from __future__ import annotations

import torch


class _Refuse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, name, n, *tensors):
        ctx.name = name
        return tuple(t.detach() for t in tensors[:n])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} cannot be differentiated twice")


def refuse_second(name, grads, sources):
    """The gradients of a backward. Where that is itself recorded (create_graph), the same values, whose differentiation along
    `sources`, the tensors that they depend on, raises an error: unrecorded they would count as constants."""
    if not torch.is_grad_enabled():
        return grads
    given = [t for t in grads if t is not None]
    if not given:
        return grads
    refused = iter(_Refuse.apply(name, len(given), *given, *sources))
    return [None if t is None else next(refused) for t in grads]
