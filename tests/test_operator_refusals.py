"""What the entry points of the norm, the counts, the balance loss and the gradient clipping refuse before any CUDA call, and the
routes of their Python ops on the CPU with the library calls replaced."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from flash_moe_b200 import FmoeError, add_rms_norm, add_rms_norm_fp8, balance_loss, clip_grad_norm_, expert_counts, grad_norm

OK, BAD_ARG, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    from flash_moe_b200 import _lib, build

    build.build()
    return _lib.lib()


def p(n=1):
    """An address that is never read: the calls below end before a launch."""
    return ctypes.c_void_p(4096 * n)


def test_norm(lib):
    assert lib.fmoe_add_rms_norm(None, None, None, None, None, 1, 0, 64, 1e-6, None) == OK  # no rows
    assert lib.fmoe_add_rms_norm(p(), None, None, None, None, 1, 4, 64, 1e-6, None) == BAD_ARG  # nowhere to write
    assert lib.fmoe_add_rms_norm(p(), p(2), None, None, p(3), 1, 4, 64, 1e-6, None) == BAD_ARG  # residual without a sum
    assert lib.fmoe_add_rms_norm(p(), None, None, p(2), p(3), 1, 4, 64, 1e-6, None) == BAD_ARG  # a sum without a residual
    assert lib.fmoe_add_rms_norm(p(), None, None, None, p(2), 7, 4, 64, 1e-6, None) == BAD_ARG
    assert lib.fmoe_add_rms_norm(p(), None, None, None, p(2), 1, -1, 64, 1e-6, None) == BAD_ARG
    assert lib.fmoe_add_rms_norm(p(), None, None, None, p(2), 1, 4, 0, 1e-6, None) == BAD_ARG
    assert lib.fmoe_add_rms_norm(p(), None, None, None, p(2), 1, 4, 64, -1.0, None) == BAD_ARG
    assert lib.fmoe_add_rms_norm(p(), None, None, None, p(2), 1, 4, 64, float("nan"), None) == BAD_ARG
    assert lib.fmoe_add_rms_norm(p(), None, None, None, p(2), 1, 4, 16385, 1e-6, None) == UNSUPPORTED
    assert lib.fmoe_add_rms_norm_fp8(p(), None, None, None, p(2), None, 1, 4, 64, 0, 1e-6, None) == BAD_ARG
    assert lib.fmoe_add_rms_norm_fp8(p(), None, None, None, p(2), p(3), 1, 4, 64, 48, 1e-6, None) == BAD_ARG
    size = lib.fmoe_add_rms_norm_backward_workspace_bytes(4, 64, 1)
    assert size >= 64 * 4
    args = [p(), None, p(2), None, p(3), p(4), 1, 4, 64, 1e-6]
    assert lib.fmoe_add_rms_norm_backward(*args, p(5), size - 1, None) == WORKSPACE
    assert lib.fmoe_add_rms_norm_backward(*args, None, size, None) == WORKSPACE
    assert lib.fmoe_add_rms_norm_backward(None, *args[1:], p(5), size, None) == BAD_ARG
    assert lib.fmoe_add_rms_norm_backward(*args, ctypes.c_void_p(4098), size, None) == 4
    assert lib.fmoe_add_rms_norm_backward_workspace_bytes(0, 64, 1) == 0


def test_counts(lib):
    assert lib.fmoe_expert_counts(None, None, -1, 4, 8, p(), None, None) == BAD_ARG
    assert lib.fmoe_expert_counts(None, None, 4, 4, 8, None, None, None) == BAD_ARG
    assert lib.fmoe_expert_counts(None, None, 0, 4, 0, None, None, None) == OK


def test_loss(lib):
    prepared, ws = lib.fmoe_balance_loss_prepared_bytes(8), lib.fmoe_balance_loss_workspace_bytes(4, 8)
    assert prepared > 0 and ws > 0
    assert lib.fmoe_balance_loss_prepared_bytes(0) == 0 and lib.fmoe_balance_loss_prepared_bytes(2049) == 0

    def forward(logits=p(), dtype=1, counts=p(2), T=4, nk=8, loss=p(3), stats=p(4), prep=p(5), prep_bytes=prepared, w=p(6), w_bytes=ws):
        return lib.fmoe_balance_loss_forward(logits, 16, 8, dtype, counts, None, T, nk, loss, stats, prep, prep_bytes, w, w_bytes, None, None)

    assert forward(logits=None) == BAD_ARG and forward(counts=None) == BAD_ARG and forward(loss=None) == BAD_ARG
    assert forward(stats=None) == BAD_ARG and forward(T=-1) == BAD_ARG and forward(nk=0) == BAD_ARG and forward(dtype=9) == BAD_ARG
    assert forward(nk=2049) == UNSUPPORTED
    assert forward(prep=None) == WORKSPACE and forward(prep_bytes=prepared - 1) == WORKSPACE
    assert forward(w=None) == WORKSPACE and forward(w_bytes=ws - 1) == WORKSPACE

    def backward(logits=p(), dtype=1, T=4, nk=8, stats=p(2), prep=p(3), prep_bytes=prepared, up=p(4), out=p(5)):
        return lib.fmoe_balance_loss_backward(logits, 16, 8, dtype, T, nk, stats, prep, prep_bytes, up, out, None, None)

    assert backward(T=0) == OK
    for name in ("logits", "stats", "up", "out"):
        assert backward(**{name: None}) == BAD_ARG
    assert backward(prep=None) == WORKSPACE and backward(prep_bytes=prepared - 1) == WORKSPACE
    assert backward(nk=4096) == UNSUPPORTED and backward(dtype=-1) == BAD_ARG


def test_clip(lib):
    def clip(ptrs, numels, codes, max_norm=1.0, eps=1e-6, scale=1.0, norm=p(), ws=p(2), size=None):
        n = len(ptrs)
        size = lib.fmoe_grad_norm_workspace_bytes(n) if size is None else size
        return lib.fmoe_clip_grad_norm((ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numels), (ctypes.c_int32 * n)(*codes), n,
                                       max_norm, eps, scale, None, norm, ws, size, None)

    assert clip([4096], [8], [0], max_norm=-1.0) == BAD_ARG and clip([4096], [8], [0], max_norm=float("nan")) == BAD_ARG
    assert clip([4096], [8], [0], eps=-1.0) == BAD_ARG and clip([4096], [8], [0], scale=-1.0) == BAD_ARG
    assert clip([4096], [8], [0], norm=None) == BAD_ARG and clip([None], [8], [0]) == BAD_ARG
    assert clip([4096], [-8], [0]) == BAD_ARG and clip([4096], [8], [3]) == BAD_ARG
    assert clip([4096], [8], [0], ws=None) == WORKSPACE and clip([4096], [8], [0], size=8) == WORKSPACE
    assert clip([4096], [8], [0], scale=float("inf")) == BAD_ARG and clip([4096], [8], [0], scale=float("nan")) == BAD_ARG
    assert clip([4096], [8], [0], ws=ctypes.c_void_p(4104)) == 4  # sums of 8 bytes, but the rule is 16
    assert clip([4098], [8], [0]) == 4  # a float32 between two others
    # memory that two tensors share, whatever their order
    assert clip([8192, 4096], [8, 1025], [0, 0]) == BAD_ARG and clip([4096, 4096], [8, 8], [1, 1]) == BAD_ARG
    assert lib.fmoe_grad_norm_workspace_bytes(0) == 0


def test_no_cpu_path():
    x, c = torch.zeros(2, 4, 8), torch.zeros(64, dtype=torch.int64)
    param = torch.nn.Parameter(torch.zeros(3))
    param.grad = torch.ones(3)
    for call in (lambda: add_rms_norm(x), lambda: add_rms_norm_fp8(x), lambda: expert_counts(c.view(8, 8), 4),
                 lambda: balance_loss(x, c), lambda: clip_grad_norm_(param, 1.0), lambda: grad_norm(x)):
        with pytest.raises(FmoeError, match="CUDA"):
            call()


def test_gradients_that_cannot_be_taken():
    p = torch.nn.Parameter(torch.zeros(4, 4))
    p.grad = torch.zeros(4, 4).to_sparse()
    with pytest.raises(FmoeError, match="sparse"):
        clip_grad_norm_(p, 1.0)
    p.grad = torch.zeros(1, 4).expand(4, 4)
    with pytest.raises(FmoeError, match="CUDA"):
        clip_grad_norm_(p, 1.0)
    with pytest.raises(FmoeError, match="negative"):
        clip_grad_norm_(p, -1.0)


def test_dense():
    from flash_moe_b200.ops.grad_clip import _dense

    x = torch.zeros(4, 3, 2)
    assert _dense(x) and _dense(x.permute(2, 0, 1)) and _dense(x[1:]) and _dense(x[:, :1, :][:1])
    assert not _dense(x[:, 1:]) and not _dense(x[..., :1]) and not _dense(torch.zeros(1).expand(4)) and _dense(torch.zeros(1, 1).t())


@pytest.fixture
def ops_without_a_gpu(monkeypatch):
    """The norm doubles its input, the loss sums the logits, out of autograd's sight as the library does."""
    import sys

    norm, bal = sys.modules["flash_moe_b200.ops.add_rms_norm"], sys.modules["flash_moe_b200.ops.balance"]
    monkeypatch.setattr(norm, "_forward", lambda x, r, w, eps: (torch.from_numpy(2 * x.detach().numpy()), torch.from_numpy(x.detach().numpy().copy())))
    monkeypatch.setattr(norm, "_backward", lambda dn, ds, s, w, eps, want: (2 * dn if ds is None else 2 * dn + ds, torch.ones(s.shape[-1]) if want else None))
    monkeypatch.setattr(bal._lib, "require_cuda", lambda *t: t[0].device)
    monkeypatch.setattr(bal, "_loss_forward", lambda x, c, m: (torch.tensor(float(x.detach().sum())), torch.zeros(1)))
    monkeypatch.setattr(bal, "_loss_backward", lambda x, state, up: up * torch.ones_like(x))


NORM = lambda x: add_rms_norm(x, x, None)[0]  # noqa: E731
LOSS = lambda x: balance_loss(torch.stack([x, x]), torch.zeros(9, dtype=torch.int64))  # noqa: E731


@pytest.mark.parametrize("op", [NORM, LOSS])
def test_tangents_are_refused_not_dropped(op, ops_without_a_gpu):
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(2, 3), torch.ones(2, 3))
        with pytest.raises(RuntimeError, match="jvp"):
            op(dual)


def test_gradients_reach_every_input(ops_without_a_gpu):
    """x and residual share a gradient without sharing its memory once both have accumulated it."""
    x, r, w = (torch.ones(s).requires_grad_() for s in ((2, 3), (2, 3), (3,)))
    normed, summed = add_rms_norm(x, r, w)
    (normed.sum() + summed.sum()).backward()
    assert torch.equal(x.grad, torch.full((2, 3), 3.0)) and torch.equal(r.grad, x.grad) and torch.equal(w.grad, torch.ones(3))
    x.grad.zero_()
    assert torch.equal(r.grad, torch.full((2, 3), 3.0))
    both = torch.ones(2, 3, requires_grad=True)
    add_rms_norm(both, both, None)[0].sum().backward()  # the same tensor twice
    assert torch.equal(both.grad, torch.full((2, 3), 4.0))
    loss = balance_loss(torch.zeros(2, 4, 3).requires_grad_(), torch.zeros(9, dtype=torch.int64))
    assert loss.requires_grad
    with torch.no_grad():
        assert not balance_loss(torch.zeros(2, 4, 3).requires_grad_(), torch.zeros(9, dtype=torch.int64)).requires_grad
