"""Selections per expert and the balance loss of the product-key router, on what the layer returns: its router logits and the ids
in ``last_indices`` (the reference leaves both to its caller)."""

from __future__ import annotations

import functools
from typing import Optional

import torch

from .. import _lib
from .utils import backward_once, contiguous, plain_call

MAX_KEYS = 2048


def _token_mask(mask, tokens, dev):
    if mask is None:
        return None
    if mask.dtype != torch.bool or mask.numel() != tokens:
        raise _lib.FmoeError("token_mask must hold one bool for each token")
    if mask.device != dev:
        raise _lib.FmoeError(f"tensors on different devices: {dev} and {mask.device}")
    return mask.reshape(-1).contiguous()


def expert_counts(indices: torch.Tensor, num_experts: int, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """How often each expert was selected: int64 ``[num_experts]`` for the ids ``indices[T, k]``.

    Empty slots (-1) and the tokens that ``token_mask`` (bool, one for each token, False for padding) leaves out are not counted;
    other ids outside ``[0, num_experts)`` are left out and raise the status flag that the expert ops raise."""
    dev = _lib.require_cuda(indices)
    if indices.dim() != 2 or num_experts < 0:
        raise _lib.FmoeError("expected indices[T,k] and a number of experts")
    if indices.dtype.is_floating_point or indices.dtype in (torch.bool, torch.complex64, torch.complex128):
        raise _lib.FmoeError("indices must be integers")
    T, k = indices.shape
    mask = _token_mask(token_mask, T, dev)
    idx = contiguous(indices)
    if idx.dtype != torch.int64:
        idx = idx.to(torch.int64)
    counts = idx.new_empty(num_experts)
    rc = _lib.call("fmoe_expert_counts", dev, idx.data_ptr(), _lib.ptr(mask), T, k, num_experts, counts.data_ptr(),
                   _lib.status_ptr(dev))
    if rc:
        _lib.check(rc, "fmoe_expert_counts")
    return counts


def _strided(logits):
    """The logits with values of a row next to each other, and their strides; the layer's own view needs no copy."""
    if logits.stride(2) != 1 and logits.shape[2] != 1:
        logits = logits.contiguous()
    return logits, logits.stride(1), logits.stride(0)


@functools.lru_cache(maxsize=256)
def _layout(T, nk):
    """Bytes of (what the backward needs of the counts, of the tokens, scratch), each rounded up to 256."""
    L = _lib.lib()
    sizes = L.fmoe_balance_loss_prepared_bytes(nk), 4 * L.fmoe_balance_loss_stats_floats(T, nk), L.fmoe_balance_loss_workspace_bytes(T, nk)
    return [(n + 255) // 256 * 256 for n in sizes]


def _loss_forward(logits, counts, mask):
    """(loss, state): the state is one allocation, for the backward."""
    dev = logits.device
    _, T, nk = logits.shape
    logits, ts, hs = _strided(logits)
    prepared, stats, scratch = _layout(T, nk)
    loss = counts.new_empty((), dtype=torch.float32)
    state = counts.new_empty(prepared + stats + scratch, dtype=torch.uint8)
    at = state.data_ptr()
    rc = _lib.call("fmoe_balance_loss_forward", dev, logits.data_ptr(), ts, hs, _lib.dtype_code(logits), counts.data_ptr(),
                   _lib.ptr(mask), T, nk, loss.data_ptr(), at + prepared, at, prepared, at + prepared + stats, scratch,
                   _lib.status_ptr(dev))
    if rc:
        _lib.check(rc, "fmoe_balance_loss_forward")
    return loss, state


def _loss_backward(logits, state, upstream):
    dev = logits.device
    _, T, nk = logits.shape
    logits, ts, hs = _strided(logits)
    prepared = _layout(T, nk)[0]
    # the rows of both halves of a token next to each other, as the router's product writes its logits
    dlogits = logits.new_empty((T, 2, nk))
    at = state.data_ptr()
    rc = _lib.call("fmoe_balance_loss_backward", dev, logits.data_ptr(), ts, hs, _lib.dtype_code(logits), T, nk, at + prepared, at,
                   prepared, upstream.data_ptr(), dlogits.data_ptr(), _lib.status_ptr(dev))
    if rc:
        _lib.check(rc, "fmoe_balance_loss_backward")
    return dlogits.transpose(0, 1)


class BalanceLossFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, router_logits, counts, mask):
        loss, state = _loss_forward(router_logits, counts, mask)
        ctx.save_for_backward(router_logits, state)
        return loss

    @staticmethod
    @backward_once
    def backward(ctx, upstream):
        logits, state = ctx.saved_tensors
        return _loss_backward(logits, state.contiguous(), upstream if upstream.dtype == torch.float32 else upstream.to(torch.float32)), None, None


def balance_loss(router_logits: torch.Tensor, counts: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The auxiliary loss that evens out the experts' load: a float32 scalar, differentiable in the router's logits.

    ``num_keys^2 * sum_e f_e P_e`` over the experts e = (i, j) of the product-key router, with ``f_e = counts_e / sum(counts)`` their
    share of the selections (a constant to the gradient) and ``P_e`` the mean over the tokens of ``softmax(logits[0])_i *
    softmax(logits[1])_j``.  1 where all experts are selected equally often.  The ``[T, num_experts]`` probabilities are never formed.

    ``router_logits`` is ``[2, T, num_keys]`` as the layer returns it (up to 2048 keys), ``counts`` what `expert_counts` returns
    (its first ``num_keys^2`` entries; ranks that share the tokens all-reduce them first), ``token_mask`` (bool, one for each token,
    False for padding) leaves tokens out of the mean: their logits are not read and their gradient is zero.  The loss is 0 where
    there is no token or no selection.  In the sums with the counts each probability is held to 2^-23 of itself, or to 2^-40 where it is
    below 2^-17."""
    dev = _lib.require_cuda(router_logits, counts)
    if router_logits.dim() != 3 or router_logits.shape[0] != 2 or not 0 < router_logits.shape[2] <= MAX_KEYS:
        raise _lib.FmoeError(f"expected router_logits[2,T,num_keys] with 1 to {MAX_KEYS} keys")
    nk = router_logits.shape[2]
    _lib.dtype_code(router_logits)
    if counts.dim() != 1 or counts.dtype != torch.int64 or counts.numel() < nk * nk:
        raise _lib.FmoeError("counts must be int64 with an entry for each of the num_keys^2 experts")
    mask = _token_mask(token_mask, router_logits.shape[1], dev)
    counts = contiguous(counts)
    if plain_call():
        return _loss_forward(router_logits, counts, mask)[0]
    return BalanceLossFunc.apply(router_logits, counts, mask)
