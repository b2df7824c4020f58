"""Norm, counts, balance loss and clipping together, as a training step of a stack uses them, against the same step by torch's own
functions around the layers; the serving form of the norm in front of a layer; hot experts chosen with the counts.

The two steps differ by roundings of float32 values only, which travel through sums of at most H + I = 768 terms a product
and a handful of products: gradients agree to within 10 * 768 * 2^-24 < 5e-4 of their norm."""

import pytest
import torch

pytestmark = pytest.mark.gpu

H, I, N, K = 128, 256, 256, 8


def make_stack(fused, dtype=torch.float32, layers=3):
    from flash_moe_b200 import FlashMoEConfig
    from flash_moe_b200.modules.stack import FlashMoEStack

    stack = FlashMoEStack(FlashMoEConfig(H, I, "silu", N, K, True), layers, seeds=list(range(layers)), pre_norm=True, fused_norm=fused)
    torch.manual_seed(99)
    with torch.no_grad():
        for w in stack.norms:
            w.add_(0.1 * torch.randn_like(w))
    return stack.to(dtype).cuda().train()


def plain_balance(logits, indices, mask):
    """By the whole [T, N] probabilities."""
    keep = torch.ones(logits.shape[1], dtype=torch.bool, device="cuda") if mask is None else mask.reshape(-1)
    nk = logits.shape[2]
    p = torch.softmax(logits[:, keep].double(), -1)
    probs = (p[0][:, :, None] * p[1][:, None, :]).mean(0).reshape(-1)
    f = torch.bincount(indices[keep].reshape(-1), minlength=N).double()
    return (nk * nk * (f / f.sum() * probs).sum()).float()


def step(stack, x, target, mask, ours):
    from flash_moe_b200.modules.stack import FlashMoEStack

    stack.zero_grad(set_to_none=True)
    y, logits = stack(x, return_routing=True)
    if ours:
        aux = FlashMoEStack.balance_loss(stack, logits, mask)
    else:
        aux = torch.stack([plain_balance(lg, layer.last_indices, mask) for lg, layer in zip(logits, stack.layers)]).mean()
    loss = ((y - target) * mask[..., None]).float().square().mean() + 0.5 * aux
    loss.backward()
    if ours:
        norm = stack.clip_grad_norm_(0.25)
    else:
        norm = torch.nn.utils.clip_grad_norm_(stack.parameters(), 0.25)
    return loss.detach(), norm, {n: p.grad.clone() for n, p in stack.named_parameters()}


def data(dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(5)
    x, target = (torch.randn(2, 40, H, device="cuda", generator=g).to(dtype) for _ in range(2))
    mask = torch.arange(40, device="cuda")[None, :] < torch.tensor([[40], [27]], device="cuda")  # a padded batch
    return x, target, mask


def test_training_step():
    x, target, mask = data()
    got_loss, got_norm, got = step(make_stack(True), x, target, mask, True)
    want_loss, want_norm, want = step(make_stack(False), x, target, mask, False)
    assert abs(float(got_loss) - float(want_loss)) <= 1e-5 * float(want_loss)
    assert abs(float(got_norm) - float(want_norm)) <= 5e-4 * float(want_norm) and float(want_norm) > 0.25  # it did clip
    for name, w in want.items():
        assert float((got[name] - w).norm()) <= 5e-4 * float(w.norm()) + 1e-12, name
    total = torch.stack([g.square().sum() for g in got.values()]).sum().sqrt()
    assert abs(float(total) - 0.25) < 1e-4


def test_fused_norm_changes_training_alone():
    """Without gradients the stack runs as before: the skip connection in the layers' last product."""
    x, _, _ = data()
    a, b = make_stack(True).eval(), make_stack(False).eval()
    with torch.no_grad():
        ya, la = a(x)
        yb, lb = b(x)
    assert torch.equal(ya, yb) and all(torch.equal(p, q) for p, q in zip(la, lb))


def test_fused_norm_under_autocast_and_mixed_types():
    """Torch's norm stays where the norm's weights have another type than the states and where autocast chooses the types: the same
    bits as without `fused_norm`."""
    x, _, _ = data()
    a, b = make_stack(True), make_stack(False)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        ya, yb = a(x)[0], b(x)[0]
    assert ya.dtype == yb.dtype and torch.equal(ya, yb)
    a, b = make_stack(True, torch.bfloat16), make_stack(False, torch.bfloat16)
    for stack in (a, b):
        stack.norms[1].data = stack.norms[1].data.float()
    outcomes = []
    for stack in (a, b):
        try:
            outcomes.append(stack(x.bfloat16())[0])
        except (RuntimeError, ValueError) as e:
            outcomes.append(str(e))
    assert type(outcomes[0]) is type(outcomes[1])
    assert outcomes[0] == outcomes[1] if isinstance(outcomes[0], str) else torch.equal(*outcomes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_training_step_in_16_bits_runs(dtype):
    """Every gradient is there and finite, and the norm is the one of the clipped gradients."""
    from flash_moe_b200 import check_status, grad_norm

    x, target, mask = data(dtype)
    stack = make_stack(True, dtype)
    loss, norm, grads = step(stack, x, target, mask, True)
    check_status()
    assert bool(loss.isfinite()) and float(norm) > 0
    assert len(grads) == len(list(stack.parameters())) and all(bool(g.isfinite().all()) for g in grads.values())
    after = float(grad_norm(grads.values()))
    # each value is off by half a step of its type, at random: far less than half a step of the norm
    assert abs(after - min(0.25, float(norm))) <= torch.finfo(dtype).eps / 2 * 0.25


def test_captured_training_step():
    """Forward, balance loss, backward and clipping in one CUDA graph, replayed with other inputs, while an eager step's graph of the
    same leaves is gone: the same bits as eager."""
    x, target, mask = data()
    stack = make_stack(True, layers=2)
    want = []
    for scale in (1.0, 0.5):
        _, norm, grads = step(stack, x * scale, target, mask, True)
        want.append((norm.clone(), grads))
    static = x.clone()
    stack.zero_grad(set_to_none=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(stack, static, target, mask, True)
    torch.cuda.current_stream().wait_stream(side)
    stack.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm, grads = step(stack, static, target, mask, True)
    for scale, (want_norm, want_grads) in zip((1.0, 0.5), want):
        static.copy_(x * scale)
        graph.replay()
        assert abs(float(norm) - float(want_norm)) <= 1e-5 * float(want_norm)
        for name, g in want_grads.items():
            # a captured step takes other dense products than an eager one, whose sums are in another order
            assert float((grads[name] - g).norm()) <= 5e-4 * float(g.norm()) + 1e-12, name


def test_layer_methods_refuse_what_does_not_belong_together():
    from flash_moe_b200 import FmoeError

    stack = make_stack(False, layers=2)
    x, _, _ = data()
    _, logits = stack(x)
    with pytest.raises(FmoeError, match="return_routing"):
        stack.layers[0].balance_loss(logits[0])
    _, logits = stack(x, return_routing=True)
    assert stack.layers[0].balance_loss(logits[0]).item() > 0
    with pytest.raises(FmoeError):
        stack.layers[0].balance_loss(logits[0][:, :7])
    with pytest.raises(FmoeError):
        stack.balance_loss(logits[:1])


def test_hot_experts():
    """On the GPU the counts choose them; the CPU's choice by torch.bincount is the same."""
    from flash_moe_b200 import read_status
    from flash_moe_b200.parallel import choose_hot_experts

    g = torch.Generator().manual_seed(3)
    idx = (torch.rand(500, 8, generator=g) ** 3 * 300).long()
    idx[::7, 3] = -1
    idx[::11, 2] = 5000  # ids that are no expert's count for nobody, and are not reported here
    read_status()
    assert torch.equal(choose_hot_experts(idx.cuda(), 300, 12).cpu().sort().values, choose_hot_experts(idx, 300, 12).sort().values)
    assert read_status() == 0


def test_serving_norm_between_layers():
    """One token at a time: the residual's addition and the norm in one call give what the addition and `rms_norm`, which the stack's
    own path takes, give one after the other.  (Only up to here: a rounding of y can make the next layer select other experts.)"""
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8
    from flash_moe_b200.ops.rms_norm import rms_norm

    stack = make_stack(False, torch.bfloat16, layers=2).eval()
    x = torch.randn(1, 1, H, device="cuda").bfloat16()
    with torch.no_grad():
        xn, s = add_rms_norm(x, None, stack.norms[0])
        y, _ = stack.layers[0](xn)
        xn, s1 = add_rms_norm(y, s, stack.norms[1])
        q, scales, s8 = add_rms_norm_fp8(y, s, stack.norms[1])
        assert torch.equal(s, x) and torch.equal(s1, s + y) and torch.equal(s8, s1)
        want = rms_norm(s1, stack.norms[1])
        # the two add the squares in another order: the float32 values differ by less than (H / 32 + 24) 2^-24 of them, which a
        # rounding to bfloat16 turns into one step at most
        assert bool(((xn.float() - want.float()).abs() <= 2.0**-7 * want.float().abs()).all())
        # half a step of 8 bits, 2^-4 of the value or 2^-10 of the scale, and half a step of bfloat16 that only xn has
        off = (q.float() * scales - xn.float()).abs()
        assert bool((off <= torch.maximum(xn.float().abs() * (2.0**-4 + 2.0**-7), scales * 2.0**-10 + 2.0**-8 * xn.float().abs())).all())
        out, _ = stack.layers[1](xn)
        assert out.shape == x.shape


def tiled(tile, rows):
    """`rows` rows that repeat those of `tile`."""
    out = tile.new_empty((rows, *tile.shape[1:]))
    whole = rows // len(tile) * len(tile)
    out[:whole].view(-1, *tile.shape).copy_(tile)
    out[whole:].copy_(tile[: rows - whole])
    return out


def test_norm_offsets_beyond_32_bits():
    """2^31 values and a few rows more: the last rows are the bits of a small call."""
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8

    H, tail = 1000, 5
    rows = 2**31 // H + 100
    g = torch.Generator(device="cuda").manual_seed(1)
    tile = torch.randn(64, H, device="cuda", generator=g).bfloat16()
    w = torch.randn(H, device="cuda", generator=g).bfloat16()
    big = tiled(tile, rows)
    last = big[-tail:].clone()
    with torch.no_grad():
        for got, want in zip(add_rms_norm(big, big, w), add_rms_norm(last, last, w)):
            assert torch.equal(got[-tail:], want)
        for got, want in zip(add_rms_norm_fp8(big, None, w, group_size=64), add_rms_norm_fp8(last, None, w, group_size=64)):
            assert torch.equal(got[-tail:].float(), want.float())
    del got
    big.requires_grad_(True)
    (dx,) = torch.autograd.grad(add_rms_norm(big, None, w)[0], big, big.detach())
    small = last.requires_grad_(True)
    (want,) = torch.autograd.grad(add_rms_norm(small, None, w)[0], small, small.detach())
    assert torch.equal(dx[-tail:], want)


def test_clip_offsets_beyond_32_bits():
    from flash_moe_b200 import clip_grad_norm_

    param = torch.nn.Parameter(torch.empty(2**31 + 1000, device="cuda", dtype=torch.bfloat16))
    param.grad = torch.full_like(param, 2.0**-16)
    param.grad[-1] = 1.0
    norm = clip_grad_norm_(param, 0.5)
    expected = (1.0 + (2**31 + 999) * 2.0**-32) ** 0.5
    assert abs(float(norm) - expected) <= 2.0**-20 * expected  # 11 u are derived for any gradients: 2^-20.5
    assert abs(float(param.grad[-1]) - 0.5 / expected) <= 2.0**-8 and bool((param.grad[-3:-1] == param.grad[0]).all())
    assert abs(float(param.grad[0]) * 2.0**16 - 0.5 / expected) <= 2.0**-8


def test_two_streams_at_once():
    """Calls of every operator on two streams, not ordered against each other: each has the bits of a call alone."""
    from flash_moe_b200 import add_rms_norm, balance_loss, clip_grad_norm_, expert_counts

    def work(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x, r = (torch.randn(700, 512, device="cuda", generator=g) for _ in range(2))
        logits = torch.randn(2, 900, 64, device="cuda", generator=g)
        idx = torch.randint(0, 4096, (900, 8), device="cuda", generator=g)
        return x, r, logits, idx

    def run(x, r, logits, idx):
        x, logits = x.clone().requires_grad_(True), logits.clone().requires_grad_(True)
        n, s = add_rms_norm(x, r)
        loss = balance_loss(logits, expert_counts(idx, 4096))
        ((n * s).sum() + loss).backward()
        return [n.detach(), s.detach(), loss.detach(), clip_grad_norm_([x, logits], 0.1), x.grad, logits.grad]

    inputs = [work(s) for s in (1, 2)]
    want = [run(*i) for i in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[j].append(run(*inputs[j]))
    torch.cuda.synchronize()
    for j in range(2):
        for outputs in got[j]:
            assert all(torch.equal(a, b) for a, b in zip(outputs, want[j]))
