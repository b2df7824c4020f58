"""Contracts of the operators around the layer that need no GPU, with the library calls replaced."""

import sys

import pytest
import torch
from torch.autograd import forward_ad

from flash_moe_b200 import FmoeError, add_rms_norm_fp8, clip_grad_norm_, grad_norm


@pytest.fixture
def fp8_without_a_gpu(monkeypatch):
    """The op doubles its input, out of autograd's sight as the library does."""
    def doubled(x, residual, weight, eps, group):
        y = torch.from_numpy(2 * x.detach().numpy())
        return y, torch.ones(x.shape[0], 1), y.clone()

    norm = sys.modules["flash_moe_b200.ops.add_rms_norm"]
    monkeypatch.setattr(norm, "_forward_fp8", doubled, raising=False)
    monkeypatch.setattr(norm._lib, "require_cuda", lambda *t: t[0].device)
    monkeypatch.setattr(norm._lib, "call", lambda name, *a: 0)


@pytest.mark.parametrize("op", [lambda x: add_rms_norm_fp8(x), lambda x: add_rms_norm_fp8(x, x)])
def test_tangents_are_refused_not_dropped(op, fp8_without_a_gpu):
    with torch.no_grad(), forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="jvp"):
            op(forward_ad.make_dual(torch.ones(2, 3), torch.ones(2, 3)))
        assert torch.equal(op(torch.ones(2, 3))[0], torch.full((2, 3), 2.0))  # a level alone is no tangent


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("op", [lambda x: add_rms_norm_fp8(x)[0], lambda x: add_rms_norm_fp8(x, x)[2]])
def test_a_trace_records_the_op(op, fp8_without_a_gpu):
    with torch.no_grad():
        traced = torch.jit.trace(op, (torch.ones(2, 3),), check_trace=False)
        assert torch.equal(traced(torch.full((2, 3), 3.0)), torch.full((2, 3), 6.0))


def test_without_a_residual_the_sum_is_x_itself(fp8_without_a_gpu):
    x = torch.ones(2, 3)
    assert add_rms_norm_fp8(x)[2] is x and add_rms_norm_fp8(x, x)[2] is not x
    with forward_ad.dual_level():
        assert add_rms_norm_fp8(x)[2] is x


@pytest.fixture
def clip_without_a_gpu(monkeypatch):
    """Collects what the library would be given."""
    given = []
    clip = sys.modules["flash_moe_b200.ops.grad_clip"]
    monkeypatch.setattr(clip._lib, "require_cuda", lambda *t: t[0].device)
    monkeypatch.setattr(clip, "_call", lambda name, grads, head, scale: given.append((name, grads)) or torch.zeros(()))
    return given


def test_a_tensor_with_gaps_given_twice_counts_once(clip_without_a_gpu):
    base = torch.arange(24.0).view(4, 6)
    gaps, other, repeated = base[:, ::2], base[:, 1::2], base[:1].expand(4, 6)
    grad_norm([gaps, base, gaps, other, base[:, ::2], repeated, base, repeated.detach()])
    ((name, grads),) = clip_without_a_gpu
    assert name == "fmoe_grad_norm" and [t.flatten().tolist() for t in grads] == [
        t.flatten().tolist() for t in (gaps, base, other, repeated)]


def test_norms_refuse_tangents(clip_without_a_gpu):
    plain = torch.nn.Parameter(torch.ones(3))
    plain.grad = torch.ones(3)
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(FmoeError, match="jvp"):
            grad_norm([torch.ones(2), dual])
        p = torch.nn.Parameter(torch.ones(3))
        p.grad = dual
        with pytest.raises(FmoeError, match="jvp"):
            clip_grad_norm_([plain, p], 1.0)
        assert not clip_without_a_gpu
        grad_norm(torch.ones(2))  # a level alone is no tangent
        clip_grad_norm_(plain, 1.0)
    assert len(clip_without_a_gpu) == 2


def test_a_refused_argument_is_not_called_shared_memory(monkeypatch):
    """The library has one code for arguments that it refuses; only gradients that do share memory are said to."""
    clip = sys.modules["flash_moe_b200.ops.grad_clip"]
    monkeypatch.setattr(clip._lib, "require_cuda", lambda *t: t[0].device)
    monkeypatch.setattr(clip, "_workspace_bytes", lambda n: 8)
    monkeypatch.setattr(clip._lib, "call", lambda *a: clip._lib.ERR_BAD_ARG)
    a, b = (torch.nn.Parameter(torch.zeros(6)) for _ in range(2))
    flat = torch.ones(12)
    a.grad, b.grad = flat[:6], flat[6:]
    with pytest.raises(FmoeError, match="code 1") as e:
        clip_grad_norm_([a, b], 1.0)
    assert "share" not in str(e.value)
    b.grad = flat[5:11]
    with pytest.raises(FmoeError, match="share memory"):
        clip_grad_norm_([b, a], 1.0)


def test_workspaces_have_one_size_on_every_device():
    """Sizes are kept per shape, whatever device was current when they were asked for: those of a B200's 148 SMs, here as on a GPU."""
    from flash_moe_b200 import _lib, build

    build.build()
    lib = _lib.lib()
    assert lib.fmoe_grad_norm_workspace_bytes(96) == 2 * 148 * 8 and lib.fmoe_grad_norm_workspace_bytes(97) == 2 * 2 * 148 * 8
    # two CTAs an SM of two groups each, a float32 row of sums a group
    assert lib.fmoe_add_rms_norm_backward_workspace_bytes(1 << 20, 2048, 1) == 2 * 2 * 148 * 2048 * 4


class OwnLayer(torch.nn.Module):
    """What a caller may put in a stack's place of a layer: it takes the states and a residual, no more."""

    def forward(self, x, residual=None):
        return 2 * x if residual is None else residual + 2 * x, x.detach()


@pytest.mark.parametrize("pre_norm,fused_norm", [(False, False), (True, False), (True, True)])
def test_layers_of_a_stack_that_know_no_routing(pre_norm, fused_norm, monkeypatch):
    from flash_moe_b200 import FlashMoEConfig
    from flash_moe_b200.modules.stack import FlashMoEStack

    norm = sys.modules["flash_moe_b200.ops.add_rms_norm"]
    monkeypatch.setattr(norm, "add_rms_norm", lambda x, r, w, eps: (x * w, x) if r is None else ((x + r) * w, x + r))
    monkeypatch.setattr(torch.nn.functional, "rms_norm", lambda x, shape, w, eps: x * w)
    stack = FlashMoEStack(FlashMoEConfig(16, 16, "silu", 16, 2), 2, pre_norm=pre_norm, fused_norm=fused_norm)
    stack.layers[0], stack.layers[1] = OwnLayer(), OwnLayer()
    x = torch.ones(1, 2, 16, requires_grad=True)
    y, logits = stack(x)
    assert torch.equal(y, torch.full_like(y, 9.0)) and len(logits) == 2
    with pytest.raises(TypeError, match="return_routing"):
        stack(x, return_routing=True)


@pytest.fixture
def layer_without_a_gpu(monkeypatch):
    """A layer whose forwards select expert 1, 2, 3, ... for every token, and whose loss says what it was given."""
    from flash_moe_b200 import FlashMoE, FlashMoEConfig
    from flash_moe_b200.modules import flash_moe

    layer = FlashMoE(FlashMoEConfig(16, 16, "silu", 16, 2))
    calls = []

    def forward(x, return_routing=False):
        calls.append(return_routing)
        if return_routing:
            layer.last_indices, layer.last_gates = torch.full((x.shape[1], 2), len(calls)), torch.ones(x.shape[1], 2)
        return x, torch.zeros(x.shape[1], 2, 4, requires_grad=True).transpose(0, 1)

    balance = sys.modules["flash_moe_b200.ops.balance"]
    monkeypatch.setattr(flash_moe._lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(layer, "_forward_differentiable", forward)
    monkeypatch.setattr(balance, "expert_counts", lambda indices, n, mask: indices)
    monkeypatch.setattr(balance, "balance_loss", lambda logits, counts, mask: int(counts[0, 0]))
    return layer


def test_balance_loss_counts_the_ids_of_its_logits(layer_without_a_gpu):
    layer, x = layer_without_a_gpu, torch.ones(1, 3, 16)
    first, second = (layer(x, return_routing=True)[1] for _ in range(2))
    assert [layer.balance_loss(t) for t in (first, second, first)] == [1, 2, 1]
    assert layer.balance_loss(second.detach().double()) == 2  # of the last forward
    layer(x)
    assert layer.balance_loss(first) == 1 and torch.equal(layer.last_indices, torch.full((3, 2), 2))


def test_balance_loss_refuses_logits_without_ids(layer_without_a_gpu):
    layer, x = layer_without_a_gpu, torch.ones(1, 3, 16)
    with pytest.raises(FmoeError, match="return_routing"):
        layer.balance_loss(layer(x)[1])
    routed = layer(x, return_routing=True)[1]
    with pytest.raises(FmoeError, match="return_routing"):  # as many tokens, but the ids are another forward's
        layer.balance_loss(layer(x)[1])
    with pytest.raises(FmoeError, match="return_routing"):
        layer.balance_loss(routed.detach())
    layer(x, return_routing=True)
    with pytest.raises(FmoeError):
        layer.balance_loss(routed[:, :2])


def test_modules_pickled_without_the_newer_attributes(layer_without_a_gpu, monkeypatch):
    """nn.Module comes back with the attributes that it had."""
    from flash_moe_b200 import FlashMoEConfig
    from flash_moe_b200.modules.stack import FlashMoEStack

    monkeypatch.setattr(torch.nn.functional, "rms_norm", lambda x, shape, w, eps: x * w)
    stack = FlashMoEStack(FlashMoEConfig(16, 16, "silu", 16, 2), 1, pre_norm=True)
    stack.layers[0] = OwnLayer()
    stack.__dict__.pop("fused_norm")
    assert torch.equal(stack(torch.ones(1, 2, 16, requires_grad=True))[0], torch.full((1, 2, 16), 3.0))
    layer_without_a_gpu.__dict__.pop("_routed_last", None)
    layer_without_a_gpu(torch.ones(1, 3, 16))
