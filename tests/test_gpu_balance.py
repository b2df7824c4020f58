"""`expert_counts` and `balance_loss` against the formulas in 64 bits, the latter over the whole [T, num_experts] probabilities.

u = 2^-24 is half a step of float32.  A probability e^t / sum, t = x - max, comes from a few float32 operations, a sum over nk
values and the exponential of base 2 at t log2 e.  That product is rounded, by at most |t| log2 e u, which is |t| u of the
exponential: nothing for the keys that matter, more than its other errors together where the probability is below e^-16.  So p is
off by less than (nk / 32 + 16 + |t|) u of itself.  The products with the centred counts are sums of nk terms: off by nk u of the
sum of their absolute values, plus what the probabilities are off, where the |t| weigh in with sum p |t| <= sum p ln(1 / p) <= ln nk,
less than 8.  So G_h is off by (2 nk + 32) u of p |C - mean|, which bounds what the differences G_h - s and the loss are off; a
gradient, p (G - s), is off by |t| u of p (|G| + |s|) more; half a step of its type comes on top.  The exponential is 0 where it
would be below 2^-126, the smallest normal float32: that much of |G| + |s| a gradient may be off as well."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0**-24


def routing(T, nk, k, seed, skew=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = torch.arange(1, nk * nk + 1, dtype=torch.float64, device="cuda") ** -skew
    at = torch.multinomial(p, T * k, replacement=True, generator=g).view(T, k) if T * k else torch.zeros(T, k, dtype=torch.int64, device="cuda")
    return torch.randperm(nk * nk, device="cuda", generator=g)[at]


def logits_of(T, nk, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, 2, nk, device="cuda", generator=g).to(dtype).transpose(0, 1)


def counts_by_hand(indices, N, mask=None):
    rows = indices if mask is None else indices[mask]
    rows = rows.reshape(-1).cpu()
    return torch.bincount(rows[(rows >= 0) & (rows < N)], minlength=N)


@pytest.mark.parametrize("T,N,k", [(1, 1, 1), (1, 64, 8), (64, 65536, 32), (1000, 100, 7), (4096, 16384, 64), (3, 5, 3),
                                   (777, 1 << 20, 5), (20000, 16, 4), (5000, 60, 64), (70000, 9001, 8), (300000, 16384, 40),
                                   (9000, 102401, 50)])
def test_counts(T, N, k):
    from flash_moe_b200 import check_status, expert_counts

    g = torch.Generator(device="cuda").manual_seed(T + N)
    idx = torch.randint(0, N, (T, k), device="cuda", generator=g)
    mask = torch.rand(T, device="cuda", generator=g) < 0.6
    got = expert_counts(idx, N)
    assert got.dtype == torch.int64 and torch.equal(got.cpu(), counts_by_hand(idx, N))
    assert torch.equal(expert_counts(idx, N, mask).cpu(), counts_by_hand(idx, N, mask))
    idx[torch.rand(T, k, device="cuda", generator=g) < 0.3] = -1
    assert torch.equal(expert_counts(idx, N, mask).cpu(), counts_by_hand(idx, N, mask))
    check_status()  # empty slots raise nothing
    assert torch.equal(expert_counts(idx.to(torch.int32), N, mask).cpu(), counts_by_hand(idx, N, mask))


def test_counts_of_one_expert():
    """Every selection is the same expert: as many additions to one place as there are."""
    from flash_moe_b200 import expert_counts

    for T, k in ((5000, 64), (300, 8), (200000, 64)):
        for N in (16384, 200000):
            got = expert_counts(torch.full((T, k), 77, device="cuda"), N)
            assert int(got[77]) == T * k and int(got.sum()) == T * k


def test_counts_leave_bad_ids_out_and_say_so():
    from flash_moe_b200 import expert_counts, read_status
    from flash_moe_b200._lib import STATUS_BAD_EXPERT_ID

    read_status()
    idx = torch.tensor([[0, 5, -2], [16, 3, 1 << 40]], device="cuda")
    got = expert_counts(idx, 16)
    assert got.tolist() == [1, 0, 0, 1, 0, 1] + [0] * 10
    assert read_status() & STATUS_BAD_EXPERT_ID
    expert_counts(idx, 16, torch.tensor([False, False], device="cuda"))
    assert read_status() == 0  # what a masked token holds is not looked at


def test_counts_without_tokens_slots_or_experts():
    from flash_moe_b200 import expert_counts

    for shape in ((0, 4), (4, 0)):
        assert torch.equal(expert_counts(torch.zeros(shape, dtype=torch.int64, device="cuda"), 8), torch.zeros(8, dtype=torch.int64, device="cuda"))
    assert expert_counts(torch.full((2, 2), -1, device="cuda"), 0).numel() == 0


def test_counts_of_views():
    from flash_moe_b200 import expert_counts

    idx = routing(100, 16, 8, seed=1)
    assert torch.equal(expert_counts(idx[::2, ::3], 256).cpu(), counts_by_hand(idx[::2, ::3], 256))
    mask = torch.zeros(10, 10, dtype=torch.bool, device="cuda")
    mask[:, :4] = True  # sequences and positions, as an attention mask has them
    assert torch.equal(expert_counts(idx, 256, mask).cpu(), counts_by_hand(idx, 256, mask.view(-1)))


def reference(logits, counts, mask, upstream):
    """(loss, its slack, dlogits, its slack) in 64 bits."""
    _, T, nk = logits.shape
    c = counts[: nk * nk].double().view(nk, nk)
    keep = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask.view(-1)
    rows = logits.detach().double()[:, keep].requires_grad_()
    total, tokens = float(c.sum()), int(keep.sum())
    dlogits = torch.zeros(2, T, nk, dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(dlogits)
    if not total or not tokens:
        return 0.0, 0.0, dlogits, slack
    p = torch.softmax(rows, -1)
    loss = 0.0
    for part in p.split(max(1, (1 << 27) // (nk * nk)), 1):  # [tokens, nk, nk] at a time
        loss = loss + nk * nk * ((c / total) * (part[0][:, :, None] * part[1][:, None, :]).sum(0)).sum() / tokens
    (grad,) = torch.autograd.grad(loss, rows, torch.tensor(upstream, dtype=torch.float64, device="cuda"))
    dlogits[:, keep] = grad
    p = p.detach()
    d = (c - total / (nk * nk)).abs() + 1
    bound = torch.stack([p[1] @ d.t(), p[0] @ d])
    s = (p[0] * bound[0]).sum(-1)
    unit = (2 * nk + 32) * U * nk * nk / total
    t = (rows.detach().amax(-1, keepdim=True) - rows.detach()).clamp(max=750.0)  # e^-750 is 0 in 64 bits too
    own = (2 * nk + 32 + t) * U * nk * nk / total
    slack[:, keep] = abs(upstream) / tokens * (own * p + 2.0**-126 * nk * nk / total) * (bound + s[None, :, None])
    return loss.item(), unit * float(s.mean()) + U * loss.item(), dlogits, slack


def check(T, nk, k, dtype, masked=0.0, seed=0, upstream=1.0, counts=None, logits=None):
    from flash_moe_b200 import balance_loss, expert_counts

    g = torch.Generator(device="cuda").manual_seed(seed + 5)
    mask = torch.rand(T, device="cuda", generator=g) >= masked if masked else None
    if counts is None:
        counts = expert_counts(routing(T, nk, k, seed), nk * nk, mask)
    if logits is None:
        logits = logits_of(T, nk, dtype, seed)
    logits = logits.detach().requires_grad_()
    loss = balance_loss(logits, counts, mask)
    assert loss.shape == () and loss.dtype == torch.float32
    (got,) = torch.autograd.grad(loss, logits, torch.tensor(upstream, device="cuda"))
    want_loss, loss_slack, want, slack = reference(logits, counts, mask, upstream)
    assert abs(loss.item() - want_loss) <= loss_slack
    fi = torch.finfo(logits.dtype)
    bound = slack + (want.abs() + slack) * fi.eps / 2 + fi.tiny * fi.eps
    off = (got.double() - want).abs()
    assert got.dtype == logits.dtype and bool((off <= bound).all()), float((off - bound).max())
    if mask is not None:
        assert bool((got[:, ~mask] == 0).all())
    with torch.no_grad():
        assert torch.equal(balance_loss(logits, counts, mask), loss)


SIZES = [(1, 1, 1), (1, 8, 4), (2, 3, 2), (5, 16, 4), (130, 32, 8), (500, 64, 16), (129, 100, 7), (64, 127, 3), (300, 128, 64),
         (257, 130, 9), (128, 256, 32), (17, 257, 5), (40, 512, 8), (6, 640, 3), (3, 1000, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,nk,k", SIZES)
def test_loss_and_gradient(T, nk, k, dtype):
    # float16: a loss scale keeps the gradients, about 1 / (T nk), out of the subnormal numbers
    check(T, nk, k, dtype, seed=T, upstream=float(2 ** round(math.log2(T * nk))) if dtype == torch.float16 else 0.01)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,nk,k", [(60001, 16, 4), (40000, 64, 8), (38017, 100, 5), (45000, 192, 3)])
def test_many_tokens(T, nk, k, dtype):
    """Several items for every SM, masked tokens among them, and a last item with few or no tokens."""
    check(T, nk, k, dtype, masked=0.1, seed=T, upstream=float(2 ** round(math.log2(T * nk))) if dtype == torch.float16 else 1.0)


def test_offsets_beyond_32_bits():
    """2^31 logits and a few rows more.  With the number of rows as the upstream gradient a row's gradient is that of any batch with
    its own number; it is compared by the bounds of the formula, not with another call, whose sums of 64 columns are others: where
    G - s cancels, two right results differ by more than a step of their type."""
    from flash_moe_b200 import balance_loss, expert_counts

    nk, rows, tail = 512, 2**31 // 1024 + 200, 200
    g = torch.Generator(device="cuda").manual_seed(2)
    counts = expert_counts(torch.randint(0, nk * nk // 7, (4096, 32), device="cuda", generator=g), nk * nk)
    tile = torch.randn(128, 2, nk, device="cuda", generator=g).bfloat16()
    flat = tile.new_empty(rows, 2, nk)
    flat[: rows // 128 * 128].view(-1, 128, 2, nk).copy_(tile)
    flat[rows // 128 * 128 :].copy_(tile[: rows % 128])
    logits = flat.transpose(0, 1).requires_grad_(True)
    (got,) = torch.autograd.grad(balance_loss(logits, counts), logits, torch.tensor(float(rows), device="cuda"))
    for part in (slice(0, tail), slice(rows - tail, rows)):
        _, _, want, slack = reference(logits.detach()[:, part], counts, None, float(tail))
        bound = slack + (want.abs() + slack) * 2.0**-8 + torch.finfo(torch.bfloat16).tiny
        assert bool(((got[:, part].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,nk,k", [(1, 8, 4), (100, 33, 5), (700, 64, 16)])
def test_masked_tokens(T, nk, k, dtype):
    check(T, nk, k, dtype, masked=0.4, seed=3, upstream=512.0 if dtype == torch.float16 else 1.0)


def test_masked_tokens_are_not_read():
    from flash_moe_b200 import balance_loss, expert_counts

    T, nk = 200, 40
    idx, mask = routing(T, nk, 4, seed=1), torch.arange(T, device="cuda") % 3 != 0
    counts = expert_counts(idx, nk * nk, mask)
    clean = logits_of(T, nk, torch.bfloat16, 2)
    dirty = clean.clone()
    dirty[:, ~mask] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38] * (nk // 4), device="cuda").bfloat16()
    out = []
    for x in (clean, dirty):
        x = x.detach().requires_grad_()
        loss = balance_loss(x, counts, mask)
        out.append((loss, torch.autograd.grad(loss, x)[0]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


def test_keys_without_probability():
    """-inf takes keys out of the softmax: their gradient is zero, the others' is that of the rest."""
    logits = logits_of(50, 24, torch.float32, 4).clone()
    logits[0, :, 3:7] = -float("inf")
    logits[1, ::2, 20:] = -float("inf")
    check(50, 24, 4, torch.float32, seed=5, logits=logits)


def test_large_and_lowest_logits():
    """Differences that overflow an exponential without the row's maximum taken off, and values at the ends of the type."""
    for dtype in DTYPES:
        logits = logits_of(40, 16, dtype, 6).clone()
        logits[0, :10] *= 100
        logits[1, 10:20, 0] = torch.finfo(dtype).max
        logits[1, 20:30, 5:] = torch.finfo(dtype).min
        check(40, 16, 4, dtype, seed=7, logits=logits, upstream=64.0)


def test_a_row_that_is_not_finite_spoils_the_loss_and_its_own_gradient():
    from flash_moe_b200 import balance_loss

    logits = logits_of(30, 16, torch.float32, 8).clone()
    logits[0, 4] = -float("inf")  # no key is left: 0 / 0, as torch.softmax gives
    logits.requires_grad_()
    loss = balance_loss(logits, torch.ones(256, dtype=torch.int64, device="cuda").cumsum(0))
    (g,) = torch.autograd.grad(loss, logits)
    assert bool(loss.isnan()) and bool(g[:, 4].isnan().any())
    rest = [i for i in range(30) if i != 4]
    assert bool(g[:, rest].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["even", "one", "row", "column", "huge", "nearly_even"])
def test_counts_of_every_kind(kind, dtype):
    T, nk = 150, 48
    n = nk * nk
    g = torch.Generator(device="cuda").manual_seed(9)
    counts = {
        "even": torch.full((n,), 7),
        "one": torch.zeros(n).index_fill_(0, torch.tensor([100]), 60000),
        "row": (torch.arange(n) // nk == 3).long() * 500,
        "column": (torch.arange(n) % nk == 5).long() * 500,
        "huge": torch.randint(0, 1 << 40, (n,)),  # summed over ranks and steps
        "nearly_even": torch.randint(5000, 5003, (n,)),
    }[kind].to("cuda", torch.int64)
    del g
    check(T, nk, 4, dtype, seed=10, counts=counts, upstream=4096.0 if dtype == torch.float16 else 1.0)


def test_even_counts_give_one_and_no_gradient():
    from flash_moe_b200 import balance_loss

    x = logits_of(100, 32, torch.float32, 1).requires_grad_()
    loss = balance_loss(x, torch.full((1024,), 3, dtype=torch.int64, device="cuda"))
    assert float(loss) == 1.0 and bool((torch.autograd.grad(loss, x)[0] == 0).all())


def test_nothing_selected_or_no_token():
    from flash_moe_b200 import balance_loss

    x = logits_of(10, 8, torch.bfloat16, 1).requires_grad_()
    ones = torch.ones(64, dtype=torch.int64, device="cuda")
    for counts, mask in [(0 * ones, None), (ones, torch.zeros(10, dtype=torch.bool, device="cuda"))]:
        loss = balance_loss(x, counts, mask)
        assert float(loss) == 0.0 and bool((torch.autograd.grad(loss, x)[0] == 0).all())
    empty = torch.zeros(2, 0, 8, device="cuda", requires_grad=True)
    loss = balance_loss(empty, ones)
    assert float(loss) == 0.0 and torch.autograd.grad(loss, empty)[0].shape == (2, 0, 8)


def test_more_experts_than_keys_squared():
    """A table of 70 experts has 8 x 8 keys; the six behind them are never selected and are not part of the loss."""
    from flash_moe_b200 import balance_loss

    counts = torch.arange(70, device="cuda")
    x = logits_of(20, 8, torch.float32, 1)
    assert torch.equal(balance_loss(x, counts), balance_loss(x, counts[:64].clone()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """The same logits as [2, T, nk], as the layer's view, as a slice of wider rows and in reversed order of dimensions."""
    from flash_moe_b200 import balance_loss, expert_counts

    T, nk = 77, 24
    counts = expert_counts(routing(T, nk, 4, 1), nk * nk)
    base = logits_of(T, nk, dtype, 2)
    wide = torch.empty(T, 2, nk + 9, dtype=dtype, device="cuda")
    wide[:, :, 5 : 5 + nk] = base.transpose(0, 1)
    shapes = [base, base.contiguous(), wide[:, :, 5 : 5 + nk].transpose(0, 1), base.permute(2, 1, 0).contiguous().permute(2, 1, 0)]
    got = []
    for x in shapes:
        x = x.detach().requires_grad_()
        loss = balance_loss(x, counts)
        got.append((loss, torch.autograd.grad(loss, x, torch.full((), 8.0, device="cuda"))[0]))
    for loss, grad in got[1:]:
        assert torch.equal(loss, got[0][0]) and torch.equal(grad, got[0][1])


def test_gradient_against_differences():
    from flash_moe_b200 import balance_loss, expert_counts

    T, nk = 5, 7
    counts = expert_counts(routing(T, nk, 6, 3), nk * nk)
    x = logits_of(T, nk, torch.float32, 4).requires_grad_()
    (got,) = torch.autograd.grad(balance_loss(x, counts), x)
    f = counts.double().view(nk, nk) / counts.sum()

    def value(v):
        a, b = torch.softmax(v, -1)
        return float(nk * nk * torch.einsum("ti,ij,tj->", a, f, b) / T)

    for h, t, i in [(0, 0, 0), (1, 4, 6), (0, 2, 3), (1, 1, 1)]:
        d = torch.zeros(2, T, nk, dtype=torch.float64, device="cuda")
        d[h, t, i] = 1e-5
        want = (value(x.detach().double() + d) - value(x.detach().double() - d)) / 2e-5
        assert abs(float(got[h, t, i]) - want) < 1e-6


def test_refusals():
    from flash_moe_b200 import FmoeError, balance_loss, expert_counts

    x, c = logits_of(10, 8, torch.float32, 1), torch.ones(64, dtype=torch.int64, device="cuda")
    mask = torch.ones(10, dtype=torch.bool, device="cuda")
    for args in [(x[0], c), (x[:1], c), (x.double(), c), (x, c[:63]), (x, c.float()), (x, c.to(torch.int32)), (x, c, mask[:9]),
                 (x, c, mask.int()), (x, c, mask.cpu()), (x, c.cpu()), (torch.zeros(2, 3, 2049, device="cuda"), c),
                 (torch.zeros(2, 3, 0, device="cuda"), c)]:
        with pytest.raises(FmoeError):
            balance_loss(*args)
    idx = routing(10, 8, 2, 1)
    for args in [(idx[0], 64), (idx, -1), (idx.float(), 64), (idx, 64, mask[:3]), (idx, 64, mask.float()), (idx.cpu(), 64)]:
        with pytest.raises(FmoeError):
            expert_counts(*args)


def test_other_stream_and_graphs():
    """A call on a side stream; two captured steps that are replayed in turn with other inputs."""
    from flash_moe_b200 import balance_loss, expert_counts

    T, nk, k = 140, 40, 6

    def data(seed):
        return routing(T, nk, k, seed), logits_of(T, nk, torch.bfloat16, seed)

    def step(idx, x):
        x = x.detach().requires_grad_()
        counts = expert_counts(idx, nk * nk)
        loss = balance_loss(x, counts)
        return counts, loss, torch.autograd.grad(loss, x)[0]

    want = step(*data(1))
    side = torch.cuda.Stream()
    args = data(1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        static = [t.clone() for t in data(2)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out))
    for seed in (3, 4):
        for i, (graph, static, _) in enumerate(graphs):
            for a, b in zip(static, data(seed + 10 * i)):
                a.copy_(b)
            graph.replay()
        for i, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, step(*data(seed + 10 * i))))
