"""`grad_norm` and `clip_grad_norm_` against the formulas in 64 bits.

u = 2^-24 is half a step of float32.  A piece of 32 KiB is summed in float32 by 256 threads: a thread has at most 64 squares of
16-bit values (32 of float32) in four chains of 16, and one value of a ragged end more; each is one fused step with one rounding,
all terms are positive, two additions join the chains: 16 + 1 + 2 = 19 u on the sum, all further sums are in float64.  The root
halves that and is rounded once to float32: 10.5 u, so 11 u on the norm.  The factor adds a sum, a quotient and a product (14 u in
all), its product with a gradient one more (15 u), and then comes the rounding to the gradient's type."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0**-24


def gradients(shapes, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    params = []
    for i, shape in enumerate(shapes):
        dt = dtype[i % len(dtype)] if isinstance(dtype, list) else dtype
        p = torch.nn.Parameter(torch.zeros(shape, device="cuda", dtype=dt))
        p.grad = (torch.randn(shape, device="cuda", generator=g) * scale).to(dt)
        params.append(p)
    return params


def expected(params, max_norm, scale=1.0, eps=1e-6):
    grads = [p.grad.double() for p in params if p.grad is not None]
    norm = scale * math.sqrt(sum(float(g.square().sum()) for g in grads))
    factor = scale * min(1.0, max_norm / (norm + eps))
    return norm, [g * factor for g in grads]


def check(params, max_norm, scale=1.0, **more):
    from flash_moe_b200 import clip_grad_norm_

    norm, grads = expected(params, max_norm, scale)
    got = clip_grad_norm_(params, max_norm, **more)
    assert got.shape == () and got.dtype == torch.float32
    assert abs(float(got) - norm) <= 11 * U * norm
    for p, want in zip(params, grads):
        fi = torch.finfo(p.dtype)
        bound = want.abs() * (fi.eps / 2 * (1 + 15 * U) + 15 * U) + fi.tiny * fi.eps
        assert bool(((p.grad.double() - want).abs() <= bound).all())
    return float(got)


SHAPES = [(1,), (7,), (8,), (1000,), (8191,), (8192,), (8193,), (3, 5, 7), (129, 257), (1024, 40)]


@pytest.mark.parametrize("dtype", [*DTYPES, DTYPES])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_many_shapes(max_norm, dtype):
    check(gradients(SHAPES, dtype), max_norm)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_value(dtype):
    check(gradients([(1,)], dtype, scale=5.0), 0.25)


def test_more_tensors_than_one_launch_takes():
    check(gradients([(1 + 37 * i,) for i in range(250)], DTYPES, seed=3), 1.0)


def test_large_tensors():
    check(gradients([(2_000_003,), (4096, 1030)], torch.bfloat16, seed=4, scale=1e-3), 0.1)


def test_scales():
    check(gradients(SHAPES, torch.bfloat16, seed=5), 1e6, scale=0.125, grad_scale=0.125)
    check(gradients(SHAPES, torch.bfloat16, seed=5), 1.0, scale=8.0, grad_scale=8.0)
    check(gradients(SHAPES, torch.float32, seed=5), 1.0, scale=2.0**-10, grad_scale=torch.full((), 2.0**-10, device="cuda"))


def test_nothing_is_written_below_the_limit():
    from flash_moe_b200 import clip_grad_norm_

    params = gradients(SHAPES, torch.float16, seed=6)
    before = [p.grad.clone() for p in params]
    clip_grad_norm_(params, 1e6)
    assert all(torch.equal(p.grad, b) for p, b in zip(params, before))


def test_limit_of_zero_and_empty_calls():
    from flash_moe_b200 import clip_grad_norm_, grad_norm

    params = gradients(SHAPES, torch.float32, seed=7)
    clip_grad_norm_(params, 0.0)
    assert all(bool((p.grad == 0).all()) for p in params)
    assert float(clip_grad_norm_(params, 1.0)) == 0.0
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(grad_norm([])) == 0.0
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    norm = clip_grad_norm_(p, 1.0)  # without a gradient
    assert float(norm) == 0.0 and norm.is_cuda
    p.grad = torch.zeros(3, device="cuda")
    empty = torch.nn.Parameter(torch.zeros(0, device="cuda"))
    empty.grad = torch.zeros(0, device="cuda")
    assert float(clip_grad_norm_([empty], 1.0)) == 0.0 and float(clip_grad_norm_([p, empty], 1.0)) == 0.0


def test_gradients_given_twice_count_once():
    from flash_moe_b200 import clip_grad_norm_

    params = gradients([(100,), (50,)], torch.float32, seed=8)
    norm, grads = expected(params, 1.0)
    twin = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    twin.grad = params[0].grad
    got = clip_grad_norm_([*params, params[0], twin], 1.0)
    assert abs(float(got) - norm) <= 11 * U * norm
    assert torch.allclose(params[0].grad.double(), grads[0], rtol=16 * U, atol=0)


def test_alignment_and_orders():
    """Gradients that start at any value of a buffer, and dense ones whose dimensions are not in order."""
    base = torch.randn(50_000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    for dtype in DTYPES:
        flat = base.to(dtype)
        params, at = [], 1
        for n in (5, 8200, 16385, 100):
            p = torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=dtype))
            p.grad = flat[at : at + n]
            params.append(p)
            at += n
        rest = flat.clone()
        check(params, 1.0)
        assert torch.equal(flat[0], rest[0]) and torch.equal(flat[at:], rest[at:])  # the neighbours are left alone
        p = torch.nn.Parameter(torch.zeros(60, 40, device="cuda", dtype=dtype).t())
        p.grad = torch.randn(60, 40, device="cuda").to(dtype).t()
        assert not p.grad.is_contiguous()
        check([p], 1.0)


@pytest.mark.parametrize("value,norm", [(float("inf"), float("inf")), (float("nan"), float("nan"))])
def test_values_that_are_not_finite(value, norm):
    """As the formula says: an infinite norm makes the factor zero, a NaN makes every gradient one."""
    from flash_moe_b200 import clip_grad_norm_

    params = gradients([(9000,), (70,)], torch.bfloat16, seed=11)
    params[0].grad[4321] = value
    got = float(clip_grad_norm_(params, 1.0))
    assert got == norm or (math.isnan(got) and math.isnan(norm))
    if math.isnan(norm):
        assert all(bool(p.grad.isnan().all()) for p in params)
    else:
        assert bool((params[1].grad == 0).all()) and bool(params[0].grad[4321].isnan()) and int(params[0].grad.isnan().sum()) == 1


def test_norm_alone():
    from flash_moe_b200 import grad_norm

    params = gradients(SHAPES, DTYPES, seed=12)
    norm, _ = expected(params, 1.0)
    before = [p.grad.clone() for p in params]
    assert abs(float(grad_norm([p.grad for p in params])) - norm) <= 11 * U * norm
    assert abs(float(grad_norm([p.grad for p in params], 0.5)) - norm / 2) <= 11 * U * norm
    assert all(torch.equal(p.grad, b) for p, b in zip(params, before))
    gaps = params[-1].grad[:, ::2]
    want = math.sqrt(float(gaps.double().square().sum()))
    assert abs(float(grad_norm(gaps)) - want) <= 11 * U * want


def test_refusals():
    from flash_moe_b200 import FmoeError, clip_grad_norm_, grad_norm

    (p,) = gradients([(8, 8)], torch.float32)
    for max_norm, more in [(-1.0, {}), (float("nan"), {}), (1.0, dict(grad_scale=-1.0)), (1.0, dict(grad_scale=float("inf"))),
                           (1.0, dict(grad_scale=1e39)),  # infinite as a float32
                           (1.0, dict(eps=-1.0)), (1.0, dict(grad_scale=torch.ones((), device="cuda", dtype=torch.float64))),
                           (1.0, dict(grad_scale=torch.ones(2, device="cuda"))), (1.0, dict(grad_scale=torch.ones(())))]:
        before = p.grad.clone()
        with pytest.raises(FmoeError):
            clip_grad_norm_(p, max_norm, **more)
        assert torch.equal(p.grad, before)
    flat = torch.zeros(100, device="cuda")
    a, b = (torch.nn.Parameter(torch.zeros(60, device="cuda")) for _ in range(2))
    a.grad, b.grad = flat[:60], flat[40:]
    with pytest.raises(FmoeError, match="share memory"):
        clip_grad_norm_([a, b], 1.0)
    c = torch.nn.Parameter(torch.zeros(8, 4, device="cuda"))
    c.grad = torch.ones(8, 8, device="cuda")[:, ::2]
    with pytest.raises(FmoeError, match="gaps"):
        clip_grad_norm_(c, 1.0)
    c.grad = torch.ones(1, 4, device="cuda").expand(8, 4)
    with pytest.raises(FmoeError, match="gaps"):
        clip_grad_norm_(c, 1.0)
    with pytest.raises(FmoeError):
        grad_norm(torch.ones(3, device="cuda", dtype=torch.float64))
    with pytest.raises(FmoeError):
        grad_norm([torch.ones(3, device="cuda"), torch.ones(3)])


def test_autograd_sees_the_change():
    from flash_moe_b200 import clip_grad_norm_

    (p,) = gradients([(64,)], torch.float32)
    version = p.grad._version
    clip_grad_norm_(p, 1e-3)
    assert p.grad._version > version


def test_other_stream_and_graph():
    from flash_moe_b200 import clip_grad_norm_

    params = gradients([(3000,), (77, 9)], torch.bfloat16, seed=13)
    fresh = [p.grad.clone() for p in params]
    want = float(clip_grad_norm_(params, 1.0))
    clipped = [p.grad.clone() for p in params]

    def reset():
        for p, g in zip(params, fresh):
            p.grad.copy_(g)

    reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm = clip_grad_norm_(params, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert float(norm) == want and all(torch.equal(p.grad, c) for p, c in zip(params, clipped))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 1.0)
    for _ in range(2):
        reset()
        graph.replay()
        assert float(norm) == want and all(torch.equal(p.grad, c) for p, c in zip(params, clipped))
