"""What the headers and docstrings of the norm, the clipping and the balance loss promise at the ends of their ranges: 8-bit
quotients, rows shorter than a 16-byte piece, weights that start anywhere, tensors given twice, the widest rows of keys."""

import pytest
import torch
from test_gpu_add_rms_norm import DTYPES, EPS, U, inputs, near, randn, row_u, sum_and_norm
from test_gpu_balance import logits_of, reference, routing

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,nk,k", [(5, 1001, 3), (3, 1024, 2), (140, 1030, 16), (20, 1537, 4), (9, 2047, 3), (2, 2048, 2), (30, 2048, 8)])
def test_loss_of_many_keys(T, nk, k, dtype):
    """Up to the largest number of keys: eight items of 256 columns side by side, sums over 32 blocks; the bounds of
    test_gpu_balance.py.  Gradients past the largest float16, as this weight of the loss gives where two tokens have 2048 keys, are
    infinite."""
    from flash_moe_b200 import balance_loss, expert_counts

    upstream = 2.0**19 if dtype == torch.float16 else 0.01
    mask = torch.arange(T, device="cuda") % 5 != 0 if T > 100 else None
    counts = expert_counts(routing(T, nk, k, T), nk * nk, mask)
    logits = logits_of(T, nk, dtype, T).detach().requires_grad_()
    loss = balance_loss(logits, counts, mask)
    (got,) = torch.autograd.grad(loss, logits, torch.tensor(upstream, device="cuda"))
    want_loss, loss_slack, want, slack = reference(logits, counts, mask, upstream)
    assert abs(loss.item() - want_loss) <= loss_slack
    fi = torch.finfo(dtype)
    over = fi.max * (1 + fi.eps / 4)  # half a step past the largest value, where rounding goes to infinity
    inf, size = got.isinf(), want.abs()
    assert bool((inf <= (size + slack >= over)).all()) and bool((~inf <= (size - slack <= over)).all())
    assert torch.equal(got[inf].sign().double(), want[inf].sign())
    off = (got.double() - want).abs()
    assert bool((off <= slack + (size + slack) * fi.eps / 2 + fi.tiny * fi.eps)[~inf].all())
    if mask is not None:
        assert bool((got[:, ~mask] == 0).all())


@pytest.mark.parametrize("nk", [16, 64, 200])
@pytest.mark.parametrize("gap", [0.0, 6.0, 11.0, 14.0, 20.0, 26.0, 30.0, 50.0])
def test_selections_of_improbable_experts_alone(gap, nk):
    """One expert (3, 5) has all selections, few enough that their mean rounds to 0, and both its keys lie `gap` below the others: no other
    term covers what is lost of their probabilities, from about 2^-4 / nk down to 0.

    In the units of test_gpu_balance.py, p being off by (nk / 32 + 16 + |t|) u of itself and its two float16 pieces by 2^-23 of it or 2^-40: G
    is off by (2 nk + 32 + |t|) u p C + 2^-40 C, the loss by p_0 times as much, a gradient by p (|G| + |s|) own units and p times what G
    and s are off.  Exponentials below 2^-126 are 0."""
    from flash_moe_b200 import balance_loss

    T = 40
    counts = torch.zeros(nk * nk, dtype=torch.int64, device="cuda")
    counts[3 * nk + 5] = 4
    logits = 0.5 * randn(2, T, nk, seed=nk, dtype=torch.float32)
    logits[0, :, 3] -= gap
    logits[1, :, 5] -= gap
    logits.requires_grad_()
    loss = balance_loss(logits, counts)
    (got,) = torch.autograd.grad(loss, logits)
    x = logits.detach().double()
    p, c = torch.softmax(x, -1), counts.double().view(nk, nk)
    G = torch.stack([p[1] @ c.t(), p[0] @ c])
    s = (p[0] * G[0]).sum(-1)
    scale = nk * nk / 4 / T
    t = x.amax(-1, keepdim=True) - x
    unit, lost = (2 * nk + 32 + 2 * (gap + 4)) * U, torch.stack([c.sum(1), c.sum(0)])[:, None] * 2.0**-40
    s_off = unit * s + (p[0] * lost[0]).sum(-1)
    want = scale * p * (G - s[None, :, None])
    slack = scale * (p * (unit * G + lost + s_off[None, :, None] + t * U * (G + s[None, :, None])) + 2.0**-126 * (G + s[None, :, None] + lost))
    assert abs(loss.item() - scale * float(s.sum())) <= scale * float(s_off.sum()) + U * scale * float(s.sum())
    off, bound = (got.double() - want).abs(), slack + (want.abs() + slack) * U + 2.0**-149
    assert bool((off <= bound).all()), float((off - bound).max())
    if gap <= 6:  # here the bounds are relative ones
        assert float((off / want.abs().clamp(min=1e-30)).max()) < 1e-3


def test_clipping_by_a_norm_that_ranks_share():
    """Ranks that hold different parameters add up the squares of their norms and scale by the common factor: the gradients are those of one
    rank that holds all.  Norm and factor are off by a few float32 roundings more than that rank's."""
    from flash_moe_b200 import clip_grad_norm_, grad_norm

    def rank(seed):
        params = [torch.nn.Parameter(torch.zeros(n, device="cuda")) for n in (300, 7)]
        for i, p in enumerate(params):
            p.grad = randn(p.numel(), seed=seed + i, dtype=torch.float32)
        return params

    for max_norm in (1.0, 1e3):
        one = [*rank(1), *rank(5)]
        norm = clip_grad_norm_(one, max_norm)
        ranks = [rank(1), rank(5)]
        total = sum(grad_norm([p.grad for p in r]).square() for r in ranks).sqrt()  # the sum is the all-reduce
        assert abs(float(total) - float(norm)) <= 32 * U * float(norm)
        for r in ranks:
            clip_grad_norm_(r, float("inf"), grad_scale=(max_norm / (total + 1e-6)).clamp(max=1.0))
        for a, b in zip(one, [*ranks[0], *ranks[1]]):
            assert bool(((a.grad - b.grad).abs() <= 64 * U * b.grad.abs()).all())
