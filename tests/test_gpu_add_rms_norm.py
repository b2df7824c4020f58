"""`add_rms_norm`, its gradient and its 8-bit form against the formulas in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of float32 and h half a step of the result's type.  A float32 sum of n
terms is off by at most (n - 1) u of the sum of their absolute values; the kernels add 8 or fewer terms of a piece in a row and
then over pieces, lanes and warps, so a row of H values is off by less than (H / 32 + 16) u.  The factors behind it (division by
H, + eps, rsqrtf with 2 ulp, two or three products) add 8 u."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0**-24
EPS = 1e-6


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def row_u(H):
    return (H / 32 + 24) * U


def randn(*shape, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def inputs(T, H, dtype, seed=0):
    return (randn(T, H, seed=seed, dtype=dtype), randn(T, H, seed=seed + 1, dtype=dtype, scale=2.0),
            randn(H, seed=seed + 2, dtype=dtype, scale=0.2) + 1)


def near(got, want, slack):
    """|got - want| <= slack + half a step of got's type (relative to want, and absolute among the subnormal numbers)."""
    fi = torch.finfo(got.dtype)
    bound = slack + (want.abs() + slack) * half_step(got.dtype) + fi.tiny * fi.eps
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


def sum_and_norm(x, r, w):
    s = x if r is None else (x.float() + r.float()).to(x.dtype)
    f = s.double()
    rms = torch.sqrt(f.square().mean(-1, keepdim=True) + EPS)
    return s, f / rms * (1.0 if w is None else w.double())


SIZES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 250), (1, 1024), (33, 1000), (7, 1001), (300, 96), (9, 2048), (4, 3000), (3, 4097),
         (2, 8192), (2, 16384), (1, 16383), (700, 264)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H", SIZES)
def test_forward(T, H, dtype):
    from flash_moe_b200 import add_rms_norm

    x, r, w = inputs(T, H, dtype)
    for residual in (r, None):
        for weight in (w, None):
            with torch.no_grad():
                normed, summed = add_rms_norm(x, residual, weight, EPS)
            s, y = sum_and_norm(x, residual, weight)
            assert torch.equal(summed, s)  # one float32 addition, one rounding
            near(normed, y, y.abs() * row_u(H))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H", SIZES)
def test_gradients(T, H, dtype):
    from flash_moe_b200 import add_rms_norm

    x, r, w = (t.requires_grad_() for t in inputs(T, H, dtype, seed=10))
    dn, ds = randn(T, H, seed=20, dtype=dtype), randn(T, H, seed=21, dtype=dtype)
    normed, summed = add_rms_norm(x, r, w, EPS)
    dx, dr, dw = torch.autograd.grad((normed, summed), (x, r, w), (dn, ds))
    assert torch.equal(dx, dr)
    s, wd, dnd, dsd = summed.detach().double(), w.detach().double(), dn.double(), ds.double()
    rstd = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS)
    g = dnd * wd
    k = rstd**2 * (g * s).mean(-1, keepdim=True)
    kabs = rstd**2 * (g * s).abs().mean(-1, keepdim=True)
    near(dx, dsd + rstd * (g - s * k), 3 * row_u(H) * (dsd.abs() + rstd * (g.abs() + s.abs() * kabs)))
    terms = dnd * s * rstd
    # chains over the rows of a group, then over the groups: fewer than T + 32 additions
    near(dw, terms.sum(0), (row_u(H) + (T + 32) * U) * terms.abs().sum(0))


def test_gradients_against_differences():
    from flash_moe_b200 import add_rms_norm

    T, H = 4, 24
    x, r, w = (t.requires_grad_() for t in inputs(T, H, torch.float32, seed=30))
    dn, ds = (randn(T, H, seed=31 + i, dtype=torch.float32) for i in range(2))

    def value(x, r, w):
        s = x.detach().double() + r.detach().double()
        n = s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * w.detach().double()
        return float((n * dn.double() + s * ds.double()).sum())

    grads = torch.autograd.grad(add_rms_norm(x, r, w, EPS), (x, r, w), (dn, ds))
    for i, (t, got) in enumerate(zip((x, r, w), grads)):
        for at in (0, 5, t.numel() - 1):
            step = torch.zeros(t.numel(), dtype=torch.float64, device="cuda")
            step[at] = 1e-5
            step = step.view_as(t)
            args = [v.detach().double() for v in (x, r, w)]
            hi, lo = ([a + s * step if j == i else a for j, a in enumerate(args)] for s in (1, -1))
            want = (value(*hi) - value(*lo)) / 2e-5
            # central differences in 64 bits: third derivatives times 1e-10, 1e-16 / 1e-5 of a value near 100
            assert abs(float(got.reshape(-1)[at]) - want) < 1e-5 + 1e-5 * abs(want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("use", ["normed", "summed", "no_residual", "no_weight", "only_weight"])
def test_partly_used(use, dtype):
    """Outputs that nobody uses, arguments that are left out or need no gradient."""
    from flash_moe_b200 import add_rms_norm

    T, H = 37, 72
    x, r, w = inputs(T, H, dtype, seed=40)
    dn = randn(T, H, seed=43, dtype=dtype)
    if use == "only_weight":
        w.requires_grad_()
        normed, _ = add_rms_norm(x, r, w)
        (dw,) = torch.autograd.grad(normed, w, dn)
        leaves = [t.detach().clone().requires_grad_() for t in (x, r, w)]
        assert torch.equal(dw, torch.autograd.grad(add_rms_norm(*leaves)[0], leaves[2], dn)[0])
        return
    x.requires_grad_()
    if use == "summed":
        _, summed = add_rms_norm(x, r.requires_grad_(), w.requires_grad_())
        dx, dr, dw = torch.autograd.grad(summed, (x, r, w), dn, allow_unused=True)
        assert torch.equal(dx, dn) and torch.equal(dr, dn) and dw is None
    elif use == "normed":
        normed, summed = add_rms_norm(x, r, w)
        (dx,) = torch.autograd.grad(normed, x, dn)
        leaf = x.detach().clone().requires_grad_()
        both = add_rms_norm(leaf, r, w)
        assert torch.equal(dx, torch.autograd.grad(both, leaf, (dn, torch.zeros_like(dn)))[0])
    elif use == "no_residual":
        normed, summed = add_rms_norm(x, None, w)
        assert summed is x
        (dx,) = torch.autograd.grad((normed, summed), x, (dn, dn))
        leaf = x.detach().clone().requires_grad_()
        (want,) = torch.autograd.grad(add_rms_norm(leaf, None, w)[0], leaf, dn)
        assert torch.equal(dx, want + dn)
    else:
        normed, summed = add_rms_norm(x, r)
        leaf = x.detach().clone().requires_grad_()
        ones = add_rms_norm(leaf, r, torch.ones_like(w))
        assert torch.equal(normed, ones[0])
        assert torch.equal(torch.autograd.grad(normed, x, dn)[0], torch.autograd.grad(ones[0], leaf, dn)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [None, 32, 64, 128])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 1024), (3, 40), (5, 333), (17, 2048), (2, 8200), (600, 160), (2, 16383)])
def test_fp8(T, H, group, dtype):
    from flash_moe_b200 import add_rms_norm_fp8

    x, r, w = inputs(T, H, dtype, seed=50)
    x[0] = 0
    r[0] = 0  # a row of zeros
    q, scales, summed = add_rms_norm_fp8(x, r, w, EPS, group)
    s, y = sum_and_norm(x, r, w)
    assert torch.equal(summed, s) and q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    size = group or H
    blocks = -(-H // size)
    assert scales.shape == (T, blocks) and scales.dtype == torch.float32
    top = torch.nn.functional.pad(y.abs(), (0, blocks * size - H)).view(T, blocks, size).amax(-1)
    want = (top / 448).clamp(min=2.0**-126)
    assert bool(((scales.double() - want).abs() <= want * (row_u(H) + U)).all())
    wide = scales.double().repeat_interleave(size, 1)[:, :H]
    # half a step: 2^-4 of the value, 2^-10 of the scale among the subnormal numbers (below 2^-6 of the scale)
    bound = torch.maximum(y.abs() * 2.0**-4, wide * 2.0**-10) + y.abs() * (row_u(H) + 4 * U)
    assert bool(((q.double() * wide - y).abs() <= bound).all())
    assert bool((q[0].float() == 0).all()) and bool((scales[0] == 2.0**-126).all())
    if T > 1:
        reach = torch.nn.functional.pad(q.float().abs(), (0, blocks * size - H)).view(T, blocks, size).amax(-1)
        assert bool((reach[1:] == 448).all())


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_values_that_are_not_finite_stay_in_their_row(value):
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8

    x, r, w = inputs(6, 128, torch.bfloat16, seed=60)
    clean = add_rms_norm(x, r, w)
    clean8 = add_rms_norm_fp8(x, r, w, group_size=32)
    x[2, 5] = value
    normed, summed = add_rms_norm(x, r, w)
    q, scales, _ = add_rms_norm_fp8(x, r, w, group_size=32)
    rest = [0, 1, 3, 4, 5]
    assert torch.equal(normed[rest], clean[0][rest]) and torch.equal(scales[rest], clean8[1][rest])
    assert torch.equal(q[rest].float(), clean8[0][rest].float())
    assert not bool(torch.isfinite(normed[2, 5])) and not bool(torch.isfinite(scales[2, 0]))
    assert not bool(torch.isfinite(q[2, 5].float()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_alignment_and_leading_dimensions(dtype):
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8

    x, r, w = inputs(12, 80, dtype, seed=70)
    want = add_rms_norm(x, r, w)
    wide = torch.empty(12, 90, dtype=dtype, device="cuda")
    wide[:, 5:85] = x
    odd = torch.empty(12 * 80 + 1, dtype=dtype, device="cuda")[1:].view(12, 80)
    odd.copy_(r)
    got = add_rms_norm(wide[:, 5:85], odd, w)
    for a, b in zip(got, want):
        # rows that are not made of aligned 16-byte pieces are read value by value: another order of the same sum
        near(a, b.double(), b.double().abs() * 2 * row_u(80))
    assert torch.equal(got[1], want[1])
    for a, b in zip(add_rms_norm(x.view(3, 4, 80), r.view(3, 4, 80), w), want):
        assert torch.equal(a, b.view(3, 4, 80))
    q, scales, _ = add_rms_norm_fp8(x.view(3, 4, 80), r.view(3, 4, 80), w, group_size=32)
    assert q.shape == (3, 4, 80) and scales.shape == (3, 4, 3)
    leaf = x.clone().requires_grad_()
    dn = torch.ones(80, device="cuda", dtype=dtype).expand(12, 80)  # a gradient without memory of its own
    (a,) = torch.autograd.grad(add_rms_norm(leaf, r, w)[0], leaf, dn)
    (b,) = torch.autograd.grad(add_rms_norm(leaf, r, w)[0], leaf, dn.contiguous())
    assert torch.equal(a, b)


def test_without_a_residual_the_sum_is_x_itself():
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8

    x = torch.randn(40, 64, device="cuda").t()  # not contiguous
    with torch.no_grad():
        assert add_rms_norm(x)[1] is x
        assert add_rms_norm_fp8(x)[2] is x
    leaf = x.clone().requires_grad_(True)
    normed, summed = add_rms_norm(leaf)
    assert summed is leaf and torch.equal(normed, add_rms_norm(x)[0])


def test_x_as_its_own_residual():
    """s = x + x is exact, and so is the sum of the two equal gradients.  The other call has a residual too, of zeros: without one the
    sum is x itself, whose gradient autograd adds to the rounded one of the norm, one rounding more than the fused gradient has."""
    from flash_moe_b200 import add_rms_norm

    x = torch.randn(9, 72, device="cuda").bfloat16().requires_grad_(True)
    normed, summed = add_rms_norm(x, x)
    doubled = (2 * x.detach()).requires_grad_(True)
    normed_of, summed_of = add_rms_norm(doubled, torch.zeros_like(doubled))
    assert torch.equal(summed, doubled) and torch.equal(normed, normed_of)
    up = torch.randn_like(normed)
    (got,), (half,) = torch.autograd.grad((normed, summed), x, (up, up)), torch.autograd.grad((normed_of, summed_of), doubled, (up, up))
    assert torch.equal(got, 2 * half)


def test_no_rows():
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8

    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    normed, summed = add_rms_norm(x, x, w)
    assert normed.shape == summed.shape == (0, 64)
    (dw,) = torch.autograd.grad(normed, w, torch.empty_like(normed))
    assert torch.equal(dw, torch.zeros_like(w))
    with torch.no_grad():
        q, scales, _ = add_rms_norm_fp8(x, x, w, group_size=32)
    assert q.shape == (0, 64) and scales.shape == (0, 2)


def test_refusals():
    from flash_moe_b200 import FmoeError, add_rms_norm, add_rms_norm_fp8

    x, r, w = inputs(4, 64, torch.bfloat16)
    for args in [(x, r[:2], w), (x, r.float(), w), (x, r, w[:32]), (x, r, w.float()), (x, r.cpu(), w), (x.double(), None, None),
                 (x, r, w, -1.0), (x, r, w, float("nan")), (torch.empty(2, 16385, device="cuda"), None, None),
                 (torch.empty(3, 0, device="cuda"), None, None)]:
        with pytest.raises(FmoeError):
            add_rms_norm(*args)
    for group in (0, 16, 100, 256):
        with pytest.raises(FmoeError):
            add_rms_norm_fp8(x, r, w, EPS, group)
    with pytest.raises(FmoeError, match="no gradient"):
        add_rms_norm_fp8(x, r, w.clone().requires_grad_())


def test_second_derivative_is_refused():
    from flash_moe_b200 import add_rms_norm

    x = randn(3, 16, seed=1, dtype=torch.float32).requires_grad_()
    (g,) = torch.autograd.grad(add_rms_norm(x)[0].square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_other_stream_and_graph():
    """A call on a side stream, and forward and backward captured and replayed with other inputs."""
    from flash_moe_b200 import add_rms_norm

    x, r, w = inputs(50, 264, torch.bfloat16, seed=80)
    dn = randn(50, 264, seed=83, dtype=torch.bfloat16)

    def step(x, r, w):
        x, r, w = (t.detach().requires_grad_() for t in (x, r, w))
        out = add_rms_norm(x, r, w)
        return (*out, *torch.autograd.grad(out, (x, r, w), (dn, dn)))

    want = [t.clone() for t in step(x, r, w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, r, w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = [t.clone() for t in (x, r, w)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for seed in (90, 91):
        fresh = inputs(50, 264, torch.bfloat16, seed=seed)
        for a, b in zip(static, fresh):
            a.copy_(b)
        graph.replay()
        for a, b in zip(out, step(*fresh)):
            assert torch.equal(a, b)
