"""Global norm of gradients and clipping: the layer's backward writes dense gradients of both expert tables, so the pass over them
is one of the longer ones of a training step (the reference leaves it to its caller)."""

from __future__ import annotations

import functools
from array import array
from typing import Iterable, List, Union

import torch

from .. import _lib
from .utils import refuse_tangents


def _dense(t: torch.Tensor) -> bool:
    """True where the tensor's values are one stretch of memory without gaps or repeats, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    step = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != step:
            return False
        step *= size
    return True


def _share_memory(dense: List[torch.Tensor]) -> bool:
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in dense)
    return any(a[1] > b[0] for a, b in zip(spans, spans[1:]))


def _call(name, grads: List[torch.Tensor], head, grad_scale) -> torch.Tensor:
    dev = grads[0].device
    scale, device_scale = grad_scale, None
    if isinstance(grad_scale, torch.Tensor):
        if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != dev:
            raise _lib.FmoeError("a grad_scale tensor must hold one float32 value on the device of the gradients")
        scale, device_scale = 1.0, grad_scale.data_ptr()
    elif not 0 <= grad_scale <= torch.finfo(torch.float32).max:
        raise _lib.FmoeError("grad_scale must be a finite float32 number that is not negative")
    n = len(grads)
    try:
        codes = array("i", [_lib.DTYPE_CODE[g.dtype] for g in grads])
    except KeyError:
        for g in grads:
            _lib.dtype_code(g)  # raises for the one that is not supported
        raise
    ptrs = array("Q", [g.data_ptr() for g in grads])
    numels = array("q", [g.numel() for g in grads])
    norm = grads[0].new_empty((), dtype=torch.float32)
    nbytes = _workspace_bytes(n)
    ws = grads[0].new_empty(nbytes, dtype=torch.uint8)
    rc = _lib.call(name, dev, ptrs.buffer_info()[0], numels.buffer_info()[0], codes.buffer_info()[0], n, *head, scale, device_scale,
                   norm.data_ptr(), ws.data_ptr(), nbytes)
    if rc == _lib.ERR_BAD_ARG and _share_memory(grads):
        raise _lib.FmoeError("two gradients share memory")
    if rc:
        _lib.check(rc, name)
    return norm


_workspace_bytes = functools.lru_cache(maxsize=256)(lambda n: _lib.lib().fmoe_grad_norm_workspace_bytes(n))


def _once(tensors: Iterable[torch.Tensor], what: str) -> List[torch.Tensor]:
    """Each tensor that has values once, however often it is given; all on one CUDA device and dense (`what`: the refusal of
    others, or "" where a copy will do)."""
    seen, dev = {}, None
    for t in tensors:
        if t.layout is not torch.strided:
            raise _lib.FmoeError("sparse gradients are not supported")
        n = t.numel()
        if not n:
            continue
        if dev is None:
            dev = _lib.require_cuda(t)
        elif t.device != dev:
            _lib.require_cuda(t)
            raise _lib.FmoeError(f"tensors on different devices: {dev} and {t.device}")
        key = (t.data_ptr(), n, t.dtype)
        if not t.is_contiguous() and not _dense(t):
            if what:
                raise _lib.FmoeError(what)
            key += (t.shape, t.stride())  # of the values given, not of their copy
            if key in seen:
                continue
            t = t.contiguous()
        seen.setdefault(key, t)
    return list(seen.values())


def grad_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], grad_scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """``grad_scale * sqrt(sum of all squares)`` over all tensors, a float32 scalar on their device (no synchronisation), as a constant:
    no graph is recorded through it.  A tensor given twice counts once; of two that overlap, each counts whole."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    refuse_tangents("grad_norm", tensors)
    grads = _once((t.detach() for t in tensors), "")
    if not grads:
        return torch.zeros((), device=tensors[0].device if tensors else None)
    return _call("fmoe_grad_norm", grads, (), grad_scale)


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float,
                    grad_scale: Union[float, torch.Tensor] = 1.0, eps: float = 1e-6) -> torch.Tensor:
    """Scale the gradients of `parameters` in place so that their global 2-norm is at most `max_norm`; returns that norm before
    clipping, a float32 scalar on their device (no synchronisation).

    With ``n = grad_scale * sqrt(sum of all squares)`` every gradient is multiplied by ``grad_scale * min(1, max_norm / (n + eps))``
    in float32 and rounded once; where that factor is 1 nothing is written.  `grad_scale` is a number or one float32 on the device:
    the inverse of a loss scale, or the number of ranks where averaged gradients are to be summed.  Parameters without a gradient
    are left out, one given twice counts once.  float32, bfloat16 and float16 gradients may be mixed; each must be dense, all on
    one device, and no two may share a part of their memory.  The norm is that of the gradients given: ranks that hold different
    parameters all-reduce the squares of their `grad_norm`s first and scale by the common factor, `max_norm=inf` and `grad_scale =
    min(1, max_norm / (n + eps))` as a tensor."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0 or not eps >= 0:
        raise _lib.FmoeError("max_norm and eps must not be negative")
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    refuse_tangents("clip_grad_norm_", grads)
    grads = _once(grads, "a gradient with gaps or repeated values cannot be scaled in place: make it contiguous")
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    norm = _call("fmoe_clip_grad_norm", grads, (max_norm, eps), grad_scale)
    torch.autograd.graph.increment_version(grads)
    return norm
