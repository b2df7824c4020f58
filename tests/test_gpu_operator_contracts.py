"""What the headers and docstrings of the norm, the clipping and the balance loss promise at the ends of their ranges: 8-bit
quotients, rows shorter than a 16-byte piece, weights that start anywhere, tensors given twice, the widest rows of keys."""

import pytest
import torch
from test_gpu_add_rms_norm import DTYPES, EPS, U, inputs, near, randn, row_u, sum_and_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [None, 32, 64, 128])
@pytest.mark.parametrize("H", [256, 512, 333, 2048, 8200])
def test_fp8_quotients(H, group, dtype):
    """scale = max |y| / 448 by a product with the rounded 1 / 448: 2^-24 for each of the two roundings, 2^-23 in all.  q = e4m3(y / scale)
    by an approximate reciprocal of that scale, 2 ulp = 2^-22 of it, and a product, 2^-24: less than 2^-21 of the quotient, so q is
    what one of the ends of that interval rounds to.

    A row of +-1 has a mean square of 1 and is its own norm, so y is the weight, exactly.  The weights of a block are multiples of 1/448
    of its largest, many of them in the middle between two values of 8 bits."""
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8

    g = torch.Generator().manual_seed(H)
    size = group or H
    # odd multiples of 16: 5 bits, of which e4m3 keeps 4; the factor has what the type's bits leave
    middles = torch.tensor([17.0, 19, 21, 23, 25, 27, 29, 31])[torch.randint(0, 8, (H,), generator=g)] * 2.0 ** torch.randint(-3, 4, (H,), generator=g)
    middles[::size] = 448.0
    bases = torch.randint(1, {torch.bfloat16: 4, torch.float16: 16}.get(dtype, 64), (-(-H // size),), generator=g) * 2.0 + 1
    w = middles * bases.repeat_interleave(size)[:H] * 2.0**-9
    assert torch.equal(w.to(dtype).float(), w)
    if H % 2 == 0 and dtype is torch.float32:
        w[1::2] = torch.randn(w[1::2].shape, generator=g)  # any bits at all
    signs = torch.randint(0, 2, (6, H), generator=g) * 2.0 - 1
    x, r, wd = ((signs * 0.25).to(dtype).cuda(), (signs * 0.75).to(dtype).cuda(), w.to(dtype).cuda())
    with torch.no_grad():
        normed, summed = add_rms_norm(x, r, None, 0.0)
        assert torch.equal(summed.cpu().float(), signs) and torch.equal(normed, summed)
        q, scales, _ = add_rms_norm_fp8(x, r, wd, 0.0, group)
    y = (signs * w).double()
    want = torch.nn.functional.pad(y.abs(), (0, -H % size)).view(6, -1, size).amax(-1) / 448
    assert bool(((scales.cpu().double() - want).abs() <= want * 2.0**-23).all())
    quotient = y / scales.cpu().double().repeat_interleave(size, 1)[:, :H]
    # a float32 in between would round twice: the ends' last bits are set away from the quotient by more than they are rounded
    ends = [(quotient * (1 + sign * 2.0**-21)).float().to(torch.float8_e4m3fn).float() for sign in (-1, 1)]
    q = q.cpu().float()
    assert bool(((q == ends[0]) | (q == ends[1])).all())


def check_norm(x, r, w, dn, ds):
    """Forward, gradients and 8 bits against the formulas in 64 bits, within the bounds that test_gpu_add_rms_norm.py derives."""
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8

    T, H = x.shape
    x, r, w = (t.requires_grad_() for t in (x, r, w))
    normed, summed = add_rms_norm(x, r, w, EPS)
    dx, dr, dw = torch.autograd.grad((normed, summed), (x, r, w), (dn, ds))
    normed, summed, x, r, w = (t.detach() for t in (normed, summed, x, r, w))
    want, y = sum_and_norm(x, r, w)
    assert torch.equal(summed, want) and torch.equal(dx, dr)
    near(normed, y, y.abs() * row_u(H))
    s, wd, dnd, dsd = summed.double(), w.double(), dn.double(), ds.double()
    rstd = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS)
    g = dnd * wd
    k, kabs = (rstd**2 * v.mean(-1, keepdim=True) for v in (g * s, (g * s).abs()))
    near(dx, dsd + rstd * (g - s * k), 3 * row_u(H) * (dsd.abs() + rstd * (g.abs() + s.abs() * kabs)))
    terms = dnd * s * rstd
    near(dw, terms.sum(0), (row_u(H) + (T + 32) * U) * terms.abs().sum(0))
    for group in (None, 32, 64):
        size = group or H
        blocks = -(-H // size)
        q, scales, again = add_rms_norm_fp8(x, r, w, EPS, group)
        assert torch.equal(again, summed) and scales.shape == (T, blocks)
        top = torch.nn.functional.pad(y.abs(), (0, blocks * size - H)).view(T, blocks, size).amax(-1)
        scale = (top / 448).clamp(min=2.0**-126)  # a row of one value may well be zero
        assert bool(((scales.double() - scale).abs() <= scale * (row_u(H) + 2 * U)).all())
        wide = scales.double().repeat_interleave(size, 1)[:, :H]
        bound = torch.maximum(y.abs() * 2.0**-4, wide * 2.0**-10) + y.abs() * (row_u(H) + 8 * U)
        assert bool(((q.double() * wide - y).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", [80, 512, 8192, 16384, 16380])
def test_weights_that_start_anywhere(H, dtype):
    """Rows of whole aligned pieces beside a weight that starts between two of them."""
    x, r, w = inputs(3, H, dtype, seed=H)
    odd = torch.empty(H + 1, device="cuda", dtype=dtype)[1:].copy_(w)
    assert odd.data_ptr() % 16 != 0 and x.data_ptr() % 16 == 0
    check_norm(x, r, odd, randn(3, H, seed=1, dtype=dtype), randn(3, H, seed=2, dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", range(1, 12))
def test_rows_shorter_than_a_piece(H, dtype):
    """Several of them in one 16-byte piece, from two rows to more than a CTA takes at once; what stands behind the arrays is left alone."""
    for T in (2, 3, 9, 40, 2500):
        whole = [torch.full((T * H + 8,), float("nan"), device="cuda", dtype=dtype) for _ in range(2)]
        x, r = (t[: T * H].view(T, H).copy_(randn(T, H, seed=T + i, dtype=dtype, scale=1.0 + i)) for i, t in enumerate(whole))
        w = randn(H, seed=5, dtype=dtype, scale=0.2) + 1
        check_norm(x.detach(), r.detach(), w, randn(T, H, seed=1, dtype=dtype), randn(T, H, seed=2, dtype=dtype))
        assert all(bool(t[T * H :].isnan().all()) for t in whole)


def test_norm_of_a_tensor_with_gaps_given_twice():
    from flash_moe_b200 import grad_norm

    gaps = randn(40, 30, seed=1, dtype=torch.float32)[:, ::2]
    once = grad_norm(gaps)
    assert torch.equal(grad_norm([gaps, gaps]), once)
    assert abs(float(once) - float(gaps.double().norm())) <= 11 * U * float(once)


def test_norm_of_tensors_that_overlap():
    """Nothing is written, so nothing is refused: each counts whole.  No graph goes through the norm."""
    from flash_moe_b200 import grad_norm

    flat = randn(100, seed=2, dtype=torch.float32).requires_grad_()
    parts = [flat[:60], flat[40:], flat.detach()[30:70]]
    got = grad_norm(parts)
    want = sum(float(p.detach().double().square().sum()) for p in parts) ** 0.5
    assert not got.requires_grad and abs(float(got) - want) <= 11 * U * want


def test_two_forwards_before_their_losses():
    """Two micro-batches of one size, one of them without a graph: each loss has the ids of its own forward."""
    from flash_moe_b200 import FlashMoE, FlashMoEConfig, FmoeError, balance_loss, expert_counts

    torch.manual_seed(0)
    layer = FlashMoE(FlashMoEConfig(64, 64, "silu", 256, 4)).cuda().train()
    a, b = (torch.randn(1, 50, 64, device="cuda") for _ in range(2))
    logits_a = layer(a, return_routing=True)[1]
    ids_a = layer.last_indices.clone()
    with torch.no_grad():
        logits_b = layer(b, return_routing=True)[1]
    ids_b = layer.last_indices.clone()
    assert not torch.equal(ids_a, ids_b)
    for logits, ids in ((logits_a, ids_a), (logits_b, ids_b)):
        assert torch.equal(layer.balance_loss(logits), balance_loss(logits, expert_counts(ids, 256)))
    (grad,) = torch.autograd.grad(layer.balance_loss(logits_a), layer.router_gate.weight)
    assert bool((grad != 0).any())
    with pytest.raises(FmoeError, match="return_routing"):
        layer.balance_loss(layer(a)[1])


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_hot_experts_of_ids_of_any_integers(dtype):
    """Ids that are no expert's count for nobody and are not reported: unsigned bytes have no -1 to put in their place."""
    from flash_moe_b200 import read_status
    from flash_moe_b200.parallel import choose_hot_experts

    ids = (torch.arange(300) % 7).view(60, 5).to(dtype)
    ids[::3, 1] = 120
    read_status()
    got = choose_hot_experts(ids.cuda(), 100, 3)
    assert read_status() == 0
    # experts with equal counts may take each other's place, so what has to agree is how often the chosen ones were selected
    seen = torch.bincount(ids.long().reshape(-1), minlength=100)[:100]
    assert torch.equal(seen[got.cpu()].sort().values, seen[choose_hot_experts(ids, 100, 3)].sort().values)
