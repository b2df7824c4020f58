"""Small host-side helpers shared by the ops (counterpart of flash_moe/ops/utils.py)."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .._lib import FmoeError


def contiguous(t):
    """The reference makes every tensor argument contiguous before a kernel sees it (ops/utils.py:35-45)."""
    return t.contiguous() if isinstance(t, torch.Tensor) else t


_grad_enabled, _tracing = torch.is_grad_enabled, torch._C._is_tracing


def plain_call() -> bool:
    """True where an op may run without its autograd node, which costs several microseconds of host time: no gradient is
    recorded, no forward-mode level is open (the node is what refuses tangents, which would be dropped silently) and
    torch.jit is not tracing (the node is what a trace records)."""
    return not _grad_enabled() and forward_ad._current_level < 0 and not _tracing()


def plain_call_without_gradient() -> bool:
    """The same for an op that has no gradient, whatever the grad mode."""
    return forward_ad._current_level < 0 and not _tracing()


def refuse_tangents(name, tensors):
    """For what has no autograd node to refuse them."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise FmoeError(f"{name} has no forward-mode derivative (jvp)")


def backward_once(backward):
    """``once_differentiable`` for the backward of an op: a second differentiation is refused.  Where no graph of the backward is
    recorded, which is nearly always, its bookkeeping (4 us of host time) is left out."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if _grad_enabled() else backward(ctx, *grads)

    return run
