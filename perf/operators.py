"""Performance cases of the operators around the layer: what a training step of a stack of FlashMoE layers, and its serving, call
next to the layers themselves.

  norm      `add_rms_norm`: the residual's addition and the RMS pre-norm of the next block, without a graph (serving)
  train     the same with its gradients
  fp8       `add_rms_norm_fp8`: the same with an output in 8 bits, one scale for each row or for each `group` columns
  counts    `expert_counts`: how often each expert was selected
  balance   counts, then `balance_loss` on the router's logits and its gradient
  clip      `clip_grad_norm_`: the global norm of the gradients of a stack, and clipping

Sizes are those of the benchmark configurations, the tests and generic ones around them.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-6
CLIP_EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # one token of one sequence being generated, default width: latency
        dict(kind="norm", dtype="bfloat16", tokens=1, hidden=1024, name="norm_1"),
        # a batch of 64 sequences being generated, decoder width, one scale a token for a product in 8 bits
        dict(kind="fp8", dtype="bfloat16", tokens=64, hidden=2048, group=0, name="fp8_64"),
        # prefill of 8 x 2048 tokens, decoder width, one scale for each 128 columns
        dict(kind="fp8", dtype="bfloat16", tokens=16384, hidden=2048, group=128, name="fp8_16384"),
        # a short ragged batch of training in float16: 3 x 259 tokens, a width that no tile divides
        dict(kind="train", dtype="float16", tokens=777, hidden=1000, name="train_777_f16"),
        # a training batch of 16 x 2048 tokens, decoder width
        dict(kind="train", dtype="bfloat16", tokens=32768, hidden=2048, name="train_32768"),
        # what a server watches after one step of 64 sequences: the load of 65536 experts
        dict(kind="counts", tokens=64, experts=65536, top_k=32, zipf=0.7, masked=0.0, name="counts_64"),
        # a calibration batch for a million experts whose popularity follows Zipf's law
        dict(kind="counts", tokens=32768, experts=1 << 20, top_k=16, zipf=1.1, masked=0.0, name="counts_32768"),
        # a small float32 training step, 4 x 125 tokens of which some are padding
        dict(kind="balance", dtype="float32", tokens=500, experts=4096, top_k=16, zipf=0.7, masked=0.1, name="balance_500_f32"),
        # a training step of the default layer
        dict(kind="balance", dtype="bfloat16", tokens=4096, experts=16384, top_k=64, zipf=0.7, masked=0.0, name="balance_4096"),
        # one layer of the decoder configuration over its full global batch, padded sequences
        dict(kind="balance", dtype="bfloat16", tokens=131072, experts=65536, top_k=32, zipf=0.7, masked=0.05, name="balance_131072"),
        # gradients of the small float32 layer, whose norm is below the limit
        dict(kind="clip", dtype="float32", layers=1, hidden=256, intermediate=1024, experts=1024, clipped=False, name="clip_1_f32"),
        # gradients of four blocks of the default layer, clipped; averaged over 8 ranks where the sum is wanted
        dict(kind="clip", dtype="bfloat16", layers=4, hidden=1024, intermediate=4096, experts=16384, clipped=True, name="clip_4"),
    ]


def log_int(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "fp8", "train", "train", "counts", "balance", "balance", "balance", "clip"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind in ("norm", "fp8", "train"):
        hidden = log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            hidden = max(8, hidden // 8 * 8)
        case = dict(kind=kind, dtype=dtype, tokens=log_int(rng, 1, min(32768, (1 << 25) // hidden)), hidden=hidden)
        if kind == "fp8":
            case["group"] = rng.choice([0, 64, 128])
        return case
    if kind == "clip":
        return dict(kind=kind, dtype=dtype, layers=rng.randint(1, 4), hidden=log_int(rng, 64, 1024), intermediate=log_int(rng, 64, 2048),
                    experts=log_int(rng, 64, 16384), clipped=rng.random() < 0.5)
    keys = log_int(rng, 8, 1024 if kind == "counts" else 512)
    tokens = log_int(rng, 1, min(131072, (1 << 25) // keys if kind == "counts" else (1 << 33) // (keys * keys)))
    case = dict(kind=kind, tokens=tokens, experts=keys * keys + rng.choice([0, 0, rng.randrange(2 * keys)]),
                top_k=log_int(rng, 1, min(64, keys)), zipf=rng.choice([0.0, 0.7, 1.1]), masked=rng.choice([0.0, 0.1, 0.5]))
    if kind == "balance":
        case["dtype"] = dtype
    return case


def gradient_shapes(case):
    """Parameters of a pre-norm stack: norm weight, gate, up, down, router, the two expert tables."""
    H, I, N = case["hidden"], case["intermediate"], case["experts"]
    return [(H,), (I, H), (I, H), (H, I), (2 * math.isqrt(N), H), (N, H), (N, H)] * case["layers"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    state = dict(kind=kind)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", dtype=DTYPES[case["dtype"]], generator=gen).mul_(std)

    if kind in ("norm", "fp8", "train"):
        T, H = case["tokens"], case["hidden"]
        state["x"], state["residual"] = normal(T, H), normal(T, H, std=2.0)
        state["weight"] = normal(H, std=0.1).add_(1.0)
        if kind == "fp8":
            state["group"] = case["group"]
        if kind == "train":
            for name in ("x", "residual", "weight"):
                state[name].requires_grad_()
            state["dnormed"], state["dsummed"] = normal(T, H, std=0.1), normal(T, H, std=0.1)
    elif kind == "clip":
        # half of the experts were selected by nobody: their rows are zero
        state["parameters"] = []
        for shape in gradient_shapes(case):
            p = torch.nn.Parameter(torch.empty(shape, device="cuda", dtype=DTYPES[case["dtype"]]))
            p.grad = normal(*shape, std=1e-2)
            if shape[0] == case["experts"]:
                p.grad[torch.rand(shape[0], device="cuda", generator=gen) < 0.5] = 0
            state["parameters"].append(p)
        state["scale"] = 8.0 if case["clipped"] else 1.0
        state["max_norm"] = 1.0 if case["clipped"] else 1e4
    else:
        T, N, k = case["tokens"], case["experts"], case["top_k"]
        nk = math.isqrt(N)
        rank = np.arange(1, nk * nk + 1, dtype=np.float64) ** -case["zipf"]
        cdf = torch.from_numpy(np.cumsum(rank / rank.sum())).cuda()
        at = torch.searchsorted(cdf, torch.rand(T, k, device="cuda", dtype=torch.float64, generator=gen)).clamp_(max=nk * nk - 1)
        state["indices"] = torch.randperm(nk * nk, device="cuda", generator=gen)[at]  # popular experts lie anywhere
        state["experts"], state["keys"] = N, nk
        state["mask"] = torch.rand(T, device="cuda", generator=gen) >= case["masked"] if case["masked"] else None
        if kind == "balance":
            # as the layer returns them: a view [2, T, nk] of rows [T, 2 nk]
            state["logits"] = normal(T, 2, nk).transpose(0, 1).requires_grad_()
            # the loss's weight; in float16 times the loss scale that keeps gradients of 1 / (T nk) out of the subnormal numbers
            loss_scale = 2.0 ** round(math.log2(T * nk)) if case["dtype"] == "float16" else 1.0
            state["upstream"] = torch.full((), 0.01 * loss_scale, device="cuda")
    return state


def plain_norm(state):
    s = (state["x"].float() + state["residual"].float()).to(state["x"].dtype)
    f = s.float()
    rstd = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    return s, f, rstd


def plain_counts(state):
    idx, N = state["indices"], state["experts"]
    live = (idx >= 0) & (idx < N)
    if state["mask"] is not None:
        live &= state["mask"][:, None]
    bins = torch.where(live, idx, N).reshape(-1)
    return torch.zeros(N + 1, dtype=torch.int64, device=idx.device).scatter_add_(0, bins, torch.ones_like(bins))[:N]


def plain_balance(state):
    counts = plain_counts(state)
    nk, logits = state["keys"], state["logits"].detach()
    c = counts[: nk * nk].view(nk, nk)
    p = torch.exp(logits.float() - logits.float().amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    tokens = torch.full((), logits.shape[1], device=logits.device)
    if state["mask"] is not None:
        p = p * state["mask"][None, :, None]
        tokens = state["mask"].sum()
    # without its mean the matrix gives the same gradient, and keeps the bits that the differences below are made of
    total = c.sum()
    mean = total / (nk * nk)
    f = c.float() - mean
    g = torch.stack([p[1] @ f.t(), p[0] @ f])
    s = (p[0] * g[0]).sum(-1, keepdim=True)
    scale = nk * nk / (total.double() * tokens).clamp(min=1)
    loss = (scale * s.sum(dtype=torch.float64) + ((total > 0) & (tokens > 0))).float()
    grad = (p * (g - s) * (scale * state["upstream"]).float()).to(logits.dtype)
    return dict(counts=counts, loss=loss, dlogits=grad)


def plain_clip(state):
    grads = [p.grad for p in state["parameters"]]
    norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt() * state["scale"]
    factor = (state["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0) * state["scale"]
    return dict(norm=norm, grads=[g.copy_((g.float() * factor).to(g.dtype)) for g in grads])


def plain(state):
    kind = state["kind"]
    if kind == "counts":
        return dict(counts=plain_counts(state))
    if kind == "balance":
        return plain_balance(state)
    if kind == "clip":
        return plain_clip(state)
    with torch.no_grad():
        s, f, rstd = plain_norm(state)
        w = state["weight"].float()
        y = f * rstd * w
        if kind == "fp8":
            T, H = s.shape
            group = state["group"] or H
            blocks = torch.nn.functional.pad(y, (0, -H % group)).view(T, -1, group)
            scales = (blocks.abs().amax(-1) / E4M3_MAX).clamp(min=2.0**-126)
            q = (blocks / scales[..., None]).view(T, -1)[:, :H].to(torch.float8_e4m3fn)
            return dict(q=q, scales=scales, summed=s)
        out = dict(normed=y.to(s.dtype), summed=s)
        if kind == "train":
            dn = state["dnormed"].float()
            g = dn * w
            dot = (g * f).mean(-1, keepdim=True)
            dx = (state["dsummed"].float() + rstd * (g - f * (rstd * rstd * dot))).to(s.dtype)
            out.update(dx=dx, dresidual=dx, dweight=(dn * f * rstd).sum(0).to(s.dtype))
        return out


def run(state):
    if not own:
        return plain(state)
    from flash_moe_b200 import add_rms_norm, add_rms_norm_fp8, balance_loss, clip_grad_norm_, expert_counts

    kind = state["kind"]
    if kind == "norm":
        with torch.no_grad():
            normed, summed = add_rms_norm(state["x"], state["residual"], state["weight"], EPS)
        return dict(normed=normed, summed=summed)
    if kind == "fp8":
        with torch.no_grad():
            q, scales, summed = add_rms_norm_fp8(state["x"], state["residual"], state["weight"], EPS, state["group"] or None)
        return dict(q=q, scales=scales, summed=summed)
    if kind == "train":
        normed, summed = add_rms_norm(state["x"], state["residual"], state["weight"], EPS)
        dx, dr, dw = torch.autograd.grad((normed, summed), (state["x"], state["residual"], state["weight"]),
                                         (state["dnormed"], state["dsummed"]))
        return dict(normed=normed, summed=summed, dx=dx, dresidual=dr, dweight=dw)
    if kind == "clip":
        norm = clip_grad_norm_(state["parameters"], state["max_norm"], grad_scale=state["scale"])
        return dict(norm=norm, grads=[p.grad for p in state["parameters"]])
    counts = expert_counts(state["indices"], state["experts"], state["mask"])
    if kind == "counts":
        return dict(counts=counts)
    loss = balance_loss(state["logits"], counts, state["mask"])
    (grad,) = torch.autograd.grad(loss, state["logits"], state["upstream"])
    return dict(counts=counts, loss=loss, dlogits=grad)


def work(case):
    kind = case["kind"]
    size = 4 if case.get("dtype") == "float32" else 2
    if kind in ("norm", "fp8", "train"):
        n = case["tokens"] * case["hidden"]
        if kind == "norm":
            return dict(bytes=4 * n * size + case["hidden"] * size, flops=6 * n)
        if kind == "fp8":
            groups = -(-case["hidden"] // (case["group"] or case["hidden"]))
            return dict(bytes=n * (3 * size + 1) + case["hidden"] * size + case["tokens"] * groups * 4, flops=8 * n)
        # x, residual, both gradients; normed, summed, dx
        return dict(bytes=7 * n * size + 2 * case["hidden"] * size, flops=18 * n)
    if kind == "clip":
        n = sum(math.prod(s) for s in gradient_shapes(case))
        return dict(bytes=n * size * (2 if case["clipped"] else 1), flops=2 * n + (n if case["clipped"] else 0))
    T, N, k = case["tokens"], case["experts"], case["top_k"]
    nk = math.isqrt(N)
    moved = T * k * 8 + N * 8 + (T if case["masked"] else 0)
    if kind == "counts":
        return dict(bytes=moved, flops=T * k)
    # the logits and their gradient; the two products with the counts, and about ten operations a logit around them
    return dict(bytes=moved + 4 * T * nk * size, flops=4 * T * nk * nk + 20 * T * nk)


def exact(case, seed):
    state = prepare(case, seed)
    kind = state["kind"]
    if kind == "clip":
        grads = [p.grad.double() for p in state["parameters"]]
        norm = state["scale"] * math.sqrt(sum(float(torch.dot(g.view(-1), g.view(-1))) for g in grads))
        factor = state["scale"] * min(1.0, state["max_norm"] / (norm + CLIP_EPS))
        return dict(norm=norm, grads=[g * factor for g in grads])
    if kind in ("norm", "fp8", "train"):
        x, r, w = (state[n].detach().double() for n in ("x", "residual", "weight"))
        summed = x + r
        s = summed.to(state["x"].dtype).double()  # what is normalised is the sum as it is stored
        H = s.shape[1]
        rms = torch.sqrt(torch.einsum("th,th->t", s, s) / H + EPS)[:, None]
        y = s / rms * w
        if kind == "norm":
            return dict(normed=y, summed=summed)
        if kind == "fp8":
            group = case["group"] or H
            starts = range(0, H, group)
            scales = torch.stack([y[:, a : a + group].abs().max(1).values / E4M3_MAX for a in starts], 1)
            q = torch.cat([y[:, a : a + group] / scales[:, i : i + 1] for i, a in enumerate(starts)], 1)
            return dict(q=q, scales=scales, summed=summed)
        # y_h = s_h w_h / rms with d rms / d s_h = s_h / (H rms)
        dn, ds = state["dnormed"].double(), state["dsummed"].double()
        drms = -torch.einsum("th,th,h->t", dn, s, w)[:, None] / rms**2
        dx = dn * w / rms + drms * s / (H * rms) + ds
        return dict(normed=y, summed=summed, dx=dx, dresidual=dx, dweight=torch.einsum("th,th->h", dn, s / rms))
    idx = state["indices"] if state["mask"] is None else state["indices"][state["mask"]]
    counts = torch.bincount(idx.reshape(-1), minlength=state["experts"])
    if kind == "counts":
        return dict(counts=counts)
    nk, T = state["keys"], state["logits"].shape[1]
    f = counts[: nk * nk].double().view(nk, nk) / max(1, int(counts[: nk * nk].sum()))
    keep = torch.ones(T, dtype=torch.bool, device="cuda") if state["mask"] is None else state["mask"]
    tokens = max(1, int(keep.sum()))
    loss, dlogits = 0.0, torch.zeros(2, T, nk, dtype=torch.float64, device="cuda")
    for at in range(0, T, 8192):  # pieces: 64 bits of every token at once would not fit beside three states
        rows = keep[at : at + 8192, None]
        a, b = torch.softmax(state["logits"].detach()[:, at : at + 8192].double(), -1) * rows
        da, db = torch.einsum("ij,tj->ti", f, b), torch.einsum("ij,ti->tj", f, a)
        s = torch.einsum("ti,ti->t", a, da)[:, None]
        loss += float(s.sum())
        dlogits[0, at : at + 8192], dlogits[1, at : at + 8192] = a * (da - s), b * (db - s)
    scale = nk * nk / tokens
    return dict(counts=counts, loss=scale * loss, dlogits=dlogits * (scale * float(state["upstream"])))
