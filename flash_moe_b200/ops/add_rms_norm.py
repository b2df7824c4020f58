"""The residual's addition and the RMS pre-norm of a decoder block around the FlashMoE layer, with gradients, and with an output
in 8 bits for a product that takes one (the reference leaves both to its caller)."""

from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

from .. import _lib
from .utils import backward_once, contiguous, plain_call, plain_call_without_gradient

MAX_HIDDEN = 16384


def _arguments(x, residual, weight, eps):
    """Device, contiguous tensors, rows and columns of a call."""
    dev = _lib.require_cuda(x, residual, weight)
    shape = x.shape
    if not shape or not 0 < shape[-1] <= MAX_HIDDEN:
        raise _lib.FmoeError(f"expected x[..., hidden] with 1 to {MAX_HIDDEN} columns")
    H = shape[-1]
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
        raise _lib.FmoeError("residual must match x in shape and dtype")
    if weight is not None and (weight.shape != (H,) or weight.dtype != x.dtype):
        raise _lib.FmoeError("weight must be a [hidden] tensor in the dtype of x")
    if not eps >= 0:
        raise _lib.FmoeError("eps must not be negative")
    return dev, x.contiguous(), contiguous(residual), contiguous(weight), x.numel() // H, H


def _forward(x, residual, weight, eps):
    dev, x, r, w, rows, H = _arguments(x, residual, weight, eps)
    normed = torch.empty_like(x)
    summed = x if r is None else torch.empty_like(x)
    rc = _lib.call("fmoe_add_rms_norm", dev, x.data_ptr(), _lib.ptr(r), _lib.ptr(w), None if r is None else summed.data_ptr(),
                   normed.data_ptr(), _lib.dtype_code(x), rows, H, eps)
    if rc:
        _lib.check(rc, "fmoe_add_rms_norm")
    return normed, summed


_workspace_bytes = functools.lru_cache(maxsize=256)(lambda *shape: _lib.lib().fmoe_add_rms_norm_backward_workspace_bytes(*shape))


def _backward(dnormed, dsummed, summed, weight, eps, want_dweight):
    """(dx, dweight): the gradient of the sum, which x and the residual share, and of the weight."""
    # addresses go to the library: gradients may be views, and hooks may return saved tensors with other strides
    s, w = summed.contiguous(), contiguous(weight)
    dn, ds = (t if t is None or t.dtype == s.dtype else t.to(s.dtype) for t in (dnormed, dsummed))
    dn, ds = dn.contiguous(), contiguous(ds)
    dev, H = s.device, s.shape[-1]
    rows, code = s.numel() // H, _lib.dtype_code(s)
    dx = torch.empty_like(s)
    dw = ws = None
    nbytes = 0
    if want_dweight:
        dw = torch.empty_like(w)
        nbytes = _workspace_bytes(rows, H, code)
        ws = s.new_empty(nbytes, dtype=torch.uint8)
    rc = _lib.call("fmoe_add_rms_norm_backward", dev, dn.data_ptr(), _lib.ptr(ds), s.data_ptr(), _lib.ptr(w), dx.data_ptr(),
                   _lib.ptr(dw), code, rows, H, eps, _lib.ptr(ws), nbytes)
    if rc:
        _lib.check(rc, "fmoe_add_rms_norm_backward")
    return dx, dw


class AddRMSNormFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        normed, summed = _forward(x, residual, weight, eps)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(summed, weight)
        # without a residual the sum is x itself, which the caller has
        return (normed, summed) if residual is not None else normed

    @staticmethod
    @backward_once
    def backward(ctx, dnormed, dsummed=None):
        summed, weight = ctx.saved_tensors
        dw = None
        if dnormed is None:  # only the sum was used
            dx = dsummed
        else:
            dx, dw = _backward(dnormed, dsummed, summed, weight, ctx.eps, ctx.needs_input_grad[2])
        return dx, dx if ctx.needs_input_grad[1] else None, dw, None


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(normed, summed)``: ``summed = x + residual`` rounded to the dtype, ``normed = summed * rsqrt(mean(summed^2, -1) + eps) *
    weight`` over the last dimension, float32 inside, one rounding.

    What stands between two layers of a residual stack: x is a layer's output, residual the skip connection beside it, ``normed``
    the next layer's input and ``summed`` the next skip connection.  Without a residual ``summed`` is x.  Differentiable in x,
    residual and weight; x, residual and weight share one dtype, up to 16384 columns."""
    eps = float(eps)
    if plain_call():
        normed, summed = _forward(x, residual, weight, eps)
        return normed, x if residual is None else summed
    if residual is None:
        return AddRMSNormFunc.apply(x, None, weight, eps), x
    return AddRMSNormFunc.apply(x, residual, weight, eps)


def _forward_fp8(x, residual, weight, eps, group_size):
    dev, x, r, w, rows, H = _arguments(x, residual, weight, eps)
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
    scales = x.new_empty((*x.shape[:-1], 1 if group_size is None else -(-H // group_size)), dtype=torch.float32)
    summed = x if r is None else torch.empty_like(x)
    rc = _lib.call("fmoe_add_rms_norm_fp8", dev, x.data_ptr(), _lib.ptr(r), _lib.ptr(w), None if r is None else summed.data_ptr(),
                   q.data_ptr(), scales.data_ptr(), _lib.dtype_code(x), rows, H, group_size or 0, eps)
    if rc:
        _lib.check(rc, "fmoe_add_rms_norm_fp8")
    return q, scales, summed


class AddRMSNormFP8Func(torch.autograd.Function):
    """What refuses tangents and what a trace records; there is no gradient."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, group_size):
        q, scales, summed = _forward_fp8(x, residual, weight, eps, group_size)
        return (q, scales, summed) if residual is not None else (q, scales)


def add_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                     eps: float = 1e-6, group_size: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(quantised, scales, summed)``: the norm above in 8 bits, ``quantised * scales`` in its place (inference only).

    ``quantised`` is float8_e4m3fn in the shape of x; ``scales`` is float32, ``[..., 1]`` for one scale a row (``group_size=None``)
    or ``[..., ceil(hidden / group_size)]`` for one scale for each 32, 64 or 128 columns: the largest absolute value of the row or
    block / 448 (at least 2^-126).  The float32 value is divided by its scale, by an approximate reciprocal (2^-21), and rounded once, to
    8 bits."""
    if torch.is_grad_enabled() and (x.requires_grad or residual is not None and residual.requires_grad
                                    or weight is not None and weight.requires_grad):
        raise _lib.FmoeError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad(), or add_rms_norm")
    if group_size not in (None, 32, 64, 128):
        raise _lib.FmoeError("group_size must be None, 32, 64 or 128")
    eps = float(eps)
    if plain_call_without_gradient():
        q, scales, summed = _forward_fp8(x, residual, weight, eps, group_size)
        return q, scales, x if residual is None else summed
    if residual is None:
        return (*AddRMSNormFP8Func.apply(x, None, weight, eps, group_size), x)
    return AddRMSNormFP8Func.apply(x, residual, weight, eps, group_size)
