"""Cases that measure three operators with which a training step keeps less between its forward and its backward
pass, through the entry points that a user calls: the cross-entropy of a language model's head without its logits
(hidden states and the head's weight in, loss and their gradients out), and SwiGLU and RMSNorm (alone, and with the
residual add before it) that keep their inputs for the backward in 8 bits.

``own`` false: the operators in plain torch operations, in 32 bits, rounded once.  ``own`` true: the framework's
calls.  ``listed()`` holds one case per kind of use, ``draw(rng)`` gives another of the same ranges, ``exact`` the
results in 64 bits.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
IGNORED = -100
LOSS_SCALE = 65536.0
EPS = 1e-5
BLOCK = 128  # elements that share a scale
LARGEST = 6 * 8192 * 4096 * 128256  # operations of the largest listed head


def listed() -> list[dict]:
    return [
        # the log-probability of one token at a large vocabulary, as a serving loop scores a candidate
        dict(name="head_token", kind="head", use="score", batch=1, seq=2, hidden=4096, vocab=128256, dtype="bf16"),
        # the quickstart decoder's training step (smallest)
        dict(name="head_quickstart_fp32", kind="head", use="mean", batch=2, seq=16, hidden=32, vocab=64, dtype="fp32"),
        # the notebook demo's head: a narrow model under an odd vocabulary, fp16 with a loss scale
        dict(name="head_demo_fp16", kind="head", use="mean", batch=32, seq=256, hidden=20, vocab=50257, dtype="fp16"),
        # answers behind prompts, every token's loss weighted by its own factor
        dict(name="head_answers_bf16", kind="head", use="weighted", batch=8, seq=1024, hidden=2048, vocab=32000, dtype="bf16"),
        # a small decoder whose width is no multiple of a tile, in full precision
        dict(name="head_odd_fp32", kind="head", use="mean", batch=1, seq=2047, hidden=1090, vocab=32001, dtype="fp32"),
        # pretraining of a large-vocabulary model (largest)
        dict(name="head_bf16", kind="head", use="mean", batch=4, seq=2049, hidden=4096, vocab=128256, dtype="bf16"),
        # the quickstart decoder's feed-forward activation
        dict(name="swiglu_quickstart_fp32", kind="swiglu", rows=32, cols=64, dtype="fp32"),
        # an odd width: blocks of 128 end anywhere in a row, and the last one is short
        dict(name="swiglu_odd_fp16", kind="swiglu", rows=4095, cols=2907, dtype="fp16"),
        # the feed-forward activation of a large decoder's training step
        dict(name="swiglu_bf16", kind="swiglu", rows=16384, cols=14336, dtype="bf16"),
        # the quickstart decoder's norm
        dict(name="norm_quickstart_fp32", kind="norm", residual=False, rows=32, cols=32, dtype="fp32"),
        # an odd width in full precision
        dict(name="norm_odd_fp32", kind="norm", residual=False, rows=8191, cols=1090, dtype="fp32"),
        # the residual add and the norm behind it, a large decoder's training step
        dict(name="norm_residual_bf16", kind="norm", residual=True, rows=16384, cols=4096, dtype="bf16"),
    ]


# ---------------------------------------------------------------------- drawn cases


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["head", "head", "head", "swiglu", "norm", "norm"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if kind == "head":
        hidden = rng.choice([64, 1024, 2048, 4096, _log(rng, 16, 4096), _log(rng, 16, 4096)])
        vocab = rng.choice([260, 32000, 50257, 128256, _log(rng, 64, 128256), _log(rng, 64, 128256)])
        # an fp32 product takes about sixteen times a bf16 one; and logits of 32 bits have to fit beside each other
        most = min(LARGEST // (16 if dtype == "fp32" else 1) // (6 * hidden * vocab), 2**30 // vocab, 16384)
        seq = _log(rng, 2, max(2, min(4097, most)))
        return dict(kind=kind, use=rng.choice(["mean", "mean", "weighted", "score"]), batch=_log(rng, 1, max(1, min(32, most // seq))),
                    seq=seq, hidden=hidden, vocab=vocab, dtype=dtype)
    if kind == "swiglu":
        cols = rng.choice([4096, 14336, _log(rng, 16, 16384), _log(rng, 16, 16384)])
        return dict(kind=kind, rows=_log(rng, 1, 2 * 10**8 // cols // (2 if dtype == "fp32" else 1)), cols=cols, dtype=dtype)
    cols = rng.choice([1024, 4096, 8192, _log(rng, 16, 16384), _log(rng, 16, 16384)])
    return dict(kind=kind, residual=rng.random() < 0.6, rows=_log(rng, 1, min(1 << 17, 6 * 10**7 // cols // (2 if dtype == "fp32" else 1))),
                cols=cols, dtype=dtype)


# ---------------------------------------------------------------------- inputs


def _randn(shape, dtype: torch.dtype, gen: torch.Generator, scale: float = 1.0) -> Tensor:
    """Normal values made in slices, so that a large 16-bit tensor needs no fp32 copy of itself."""

    out = torch.empty(shape, dtype=dtype, device="cuda")
    for part in out.view(-1).split(1 << 28):
        part.copy_(torch.randn(part.numel(), generator=gen, device="cuda").mul_(scale))
    return out


def prepare(case: dict, seed: int) -> dict:
    dtype = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "head":
        b, n, h, v = case["batch"], case["seq"], case["hidden"], case["vocab"]
        train = case["use"] != "score"
        labels = torch.randint(0, v, (b, n), generator=gen, device="cuda")
        weight = _randn((v, h), dtype, gen, 2.0 / math.sqrt(h))
        # hidden states that point to the next token's row: a loss as late in pretraining
        hidden = torch.randn((b, n, h), generator=gen, device="cuda")
        hidden[:, :-1] += 1.5 * weight[labels[:, 1:]].float()
        if case["use"] == "weighted":
            at = torch.arange(n, device="cuda")
            prompt = torch.randint(0, max(1, n // 2), (b, 1), generator=gen, device="cuda")
            end = n - torch.randint(0, max(1, n // 4), (b, 1), generator=gen, device="cuda")
            labels = labels.masked_fill((at < prompt) | (at >= end), IGNORED)  # the prompt, and padding behind the answer
            s.update(factors=torch.randn((b, n - 1), generator=gen, device="cuda") / (b * n))
        s.update(labels=labels, weight=weight.requires_grad_(train), states=hidden.to(dtype).requires_grad_(train))
        return s
    shape = (case["rows"], case["cols"])
    if case["kind"] == "swiglu":
        s.update(gate=_randn(shape, dtype, gen, 1.5).requires_grad_(), up=_randn(shape, dtype, gen, 1.0).requires_grad_(),
                 grad=_randn(shape, dtype, gen, 0.1))
        return s
    s.update(x=_randn(shape, dtype, gen, 1.0).requires_grad_(), grad=_randn(shape, dtype, gen, 0.1),
             weight=(1 + _randn((case["cols"],), torch.float32, gen, 0.1)).to(dtype).requires_grad_())
    if case["residual"]:
        s.update(stream=_randn(shape, dtype, gen, 3.0).requires_grad_(), grad_sum=_randn(shape, dtype, gen, 0.1))
    return s


# ---------------------------------------------------------------------- one pass


def run(s: dict):
    kind = s["kind"]
    if not own:
        with torch.no_grad():
            return {"head": _plain_head, "swiglu": _plain_swiglu, "norm": _plain_norm}[kind](s)
    from picotron_amd.nn.triton_kernels import triton_linear_cross_entropy, triton_residual_rms_norm, triton_rms_norm, triton_swiglu

    if kind == "head":
        if s["use"] == "score":
            with torch.no_grad():
                return [triton_linear_cross_entropy(s["states"], s["weight"], s["labels"], shift=True, reduction="none")]
        if s["use"] == "weighted":
            losses = triton_linear_cross_entropy(s["states"], s["weight"], s["labels"], shift=True, reduction="none")
            return [losses.detach(), *torch.autograd.grad([losses], [s["states"], s["weight"]], [s["factors"]])]
        loss = triton_linear_cross_entropy(s["states"], s["weight"], s["labels"], shift=True)
        scaled = loss * LOSS_SCALE if s["dtype"] == "fp16" else loss
        return [loss.detach(), *torch.autograd.grad(scaled, [s["states"], s["weight"]])]
    if kind == "swiglu":
        y = triton_swiglu(s["gate"], s["up"], checkpoint_8bit=True)
        return [y.detach(), *torch.autograd.grad([y], [s["gate"], s["up"]], [s["grad"]])]
    if s["residual"]:
        h, y = triton_residual_rms_norm(s["x"], s["stream"], s["weight"], EPS, checkpoint_8bit=True)
        d = torch.autograd.grad([h, y], [s["x"], s["weight"]], [s["grad_sum"], s["grad"]])
        return [h.detach(), y.detach(), *d]
    y = triton_rms_norm(s["x"], s["weight"], EPS, checkpoint_8bit=True)
    return [y.detach(), *torch.autograd.grad([y], [s["x"], s["weight"]], [s["grad"]])]


# ---------------------------------------------------------------------- plain forms


def _plain_head(s: dict) -> list[Tensor]:
    h = s["hidden"]
    x, labels = s["states"][:, :-1].reshape(-1, h).float(), s["labels"][:, 1:].reshape(-1, 1)
    w = s["weight"].float()
    kept = labels != IGNORED
    logits = x @ w.t()
    top = logits.amax(-1, keepdim=True)
    lse = top + (logits - top).exp().sum(-1, keepdim=True).log()
    token = torch.where(kept, lse - logits.gather(-1, labels.clamp_min(0)), 0.0)
    if s["use"] == "mean":
        count = kept.sum()
        loss = (token.double().sum() / count).float()
        slope = kept / count * (LOSS_SCALE if s["dtype"] == "fp16" else 1.0)
    else:
        loss = token.view(s["batch"], s["seq"] - 1)
        if s["use"] == "score":
            return [loss]
        slope = torch.where(kept, s["factors"].reshape(-1, 1), 0.0)
    grad = logits.sub_(lse).exp_().mul_(slope)  # softmax times the weight of the row
    grad.scatter_add_(-1, labels.clamp_min(0), -slope)
    states = torch.zeros_like(s["states"])
    states[:, :-1] = (grad @ w).view(s["batch"], -1, h)
    return [loss, states, (grad.t() @ x).to(s["weight"].dtype)]


def _kept_in_8_bits(x: Tensor) -> Tensor:
    """What the backward pass reads of blocks (..., 128): a code between -127 and 127 for each element and a step for
    the block, both formed in 32 bits.  A block that holds an infinity or a NaN comes back as NaN, one below 2^-100 as 0."""

    top = x.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, 127)  # a tensor: by a number, torch multiplies with a rounded reciprocal
    step = torch.where(top < 2.0**-100, 0.0, torch.where(top.isfinite(), top / most, math.nan))
    codes = torch.where(step > 0, (x * (most / top)).round(), 0.0)
    return codes * step


def _blocks(x: Tensor) -> Tensor:
    """The last dimension in blocks, the last of them filled up with zeros."""

    return torch.nn.functional.pad(x, (0, -x.size(-1) % BLOCK)).unflatten(-1, (-1, BLOCK))


def _plain_swiglu(s: dict) -> list[Tensor]:
    dtype, shape = s["gate"].dtype, s["gate"].shape
    sigmoid = lambda y: 1 / (1 + (-y).exp())  # noqa: E731
    g, u, d = s["gate"].float(), s["up"].float(), s["grad"].float()
    y = (g * sigmoid(g) * u).to(dtype)
    read = lambda x: _kept_in_8_bits(_blocks(x.reshape(-1))).view(-1)[: x.numel()].view(shape)  # noqa: E731
    g, u = read(g), read(u)
    part = sigmoid(g)
    return [y, (d * u * (part * (1 + g * (1 - part)))).to(dtype), (d * (g * part)).to(dtype)]


def _plain_norm(s: dict) -> list[Tensor]:
    dtype, cols = s["x"].dtype, s["cols"]
    x, w, d = s["x"].float(), s["weight"].float(), s["grad"].float()
    out = []
    if s["residual"]:
        h = (x + s["stream"].float()).to(dtype)
        out.append(h)
        x = h.float()
    rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    out.append((x * rstd * w).to(dtype))
    hat = _kept_in_8_bits(_blocks(x)).flatten(-2)[:, :cols] * rstd
    dw = (d * hat).double().sum(0)
    d = d * w
    dx = rstd * (d - hat * (d * hat).mean(-1, keepdim=True))
    if s["residual"]:
        dx = dx + s["grad_sum"].float()
    return [*out, dx.to(dtype), dw.to(dtype)]


# ---------------------------------------------------------------------- what a pass needs


def work(case: dict) -> dict:
    e = SIZES[case["dtype"]]
    if case["kind"] == "head":
        b, n, h, v = case["batch"], case["seq"], case["hidden"], case["vocab"]
        kept = b * (n - 1)
        if case["use"] == "weighted":  # mean tokens of an answer (the prompt and the padding are uniform)
            kept = b * max(1, n - 1 - (max(1, n // 2) - 1) // 2 - (max(1, n // 4) - 1) // 2)
        if case["use"] == "score":
            return {"bytes": (kept + v) * h * e + 12 * kept, "flops": 2 * kept * h * v}
        return {"bytes": 2 * (b * n + v) * h * e + 12 * b * n, "flops": 6 * kept * h * v}
    n = case["rows"] * case["cols"]
    kept = n + 4 * (n // BLOCK)  # codes and steps, which the forward writes and the backward reads
    if case["kind"] == "swiglu":
        return {"bytes": 6 * n * e + 4 * kept, "flops": 40 * n}
    return {"bytes": (7 if case["residual"] else 4) * n * e + 2 * kept, "flops": 20 * n}


# ---------------------------------------------------------------------- 64-bit results


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"head": _exact_head, "swiglu": _exact_swiglu, "norm": _exact_norm}[case["kind"]](s)


def _exact_head(s: dict) -> list[Tensor]:
    b, n, h, v = s["batch"], s["seq"], s["hidden"], s["vocab"]
    w = s["weight"].detach().double()
    x, labels = s["states"].detach(), s["labels"]
    losses = torch.zeros((b, n - 1), dtype=torch.float64, device="cuda")
    dx = torch.zeros((b, n, h), dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w)
    kept = labels[:, 1:] != IGNORED
    if s["use"] == "mean":
        factors = kept.double() / kept.sum() * (LOSS_SCALE if s["dtype"] == "fp16" else 1.0)
    else:
        factors = s.get("factors", losses).double()
    step = max(1, (1 << 27) // v)  # rows of logits at a time
    for i in range(b):
        for t in range(0, n - 1, step):
            at = (torch.nonzero(kept[i, t:t + step]) + t).squeeze(1)
            if at.numel() == 0:
                continue
            rows = x[i, at].double()
            log_softmax = torch.log_softmax(rows @ w.t(), -1)
            label = labels[i, at + 1]
            losses[i, at] = -log_softmax.gather(1, label[:, None])[:, 0]
            if s["use"] == "score":
                continue
            grad = log_softmax.exp_()
            grad[torch.arange(at.numel(), device="cuda"), label] -= 1
            grad *= factors[i, at, None]
            dx[i, at] = grad @ w
            dw += grad.t() @ rows
    if s["use"] == "score":
        return [losses]
    return [losses.sum() / kept.sum() if s["use"] == "mean" else losses, dx, dw]


def _stored(x: Tensor) -> Tensor:
    """Elements of blocks (..., 128) as the 8-bit checkpoint holds them: the code is the whole number nearest to the
    element times the 32-bit quotient of 127 and the block's largest magnitude (that product held in 32 bits too)."""

    top = x.abs().max(-1, keepdim=True).values.float()
    factor = (127 / top.double()).float().double()
    code = (x.double() * factor).float().double().round()
    return torch.nan_to_num(code) * (top.double() / 127)


def _exact_swiglu(s: dict) -> list[Tensor]:
    n, out = s["gate"].numel(), [torch.empty(s["gate"].shape, dtype=torch.float64, device="cuda") for _ in range(3)]
    flat = [t.detach().reshape(-1) for t in (s["gate"], s["up"], s["grad"])]
    for o in range(0, n, 1 << 25):  # whole blocks
        g, u, d = (t[o:o + (1 << 25)].double() for t in flat)
        m = g.numel()
        out[0].view(-1)[o:o + m] = torch.nn.functional.silu(g) * u
        g, u = (_stored(torch.cat((t, t.new_zeros(-m % BLOCK))).view(-1, BLOCK)).view(-1)[:m] for t in (g, u))
        part = torch.sigmoid(g)
        out[1].view(-1)[o:o + m] = d * u * (part + g * part * torch.sigmoid(-g))
        out[2].view(-1)[o:o + m] = d * g * part
    return out


def _exact_norm(s: dict) -> list[Tensor]:
    rows, cols = s["rows"], s["cols"]
    dtype = s["x"].dtype
    w = s["weight"].detach().double()
    whole = lambda: torch.empty((rows, cols), dtype=torch.float64, device="cuda")  # noqa: E731
    total, y, dx, dw = whole(), whole(), whole(), torch.zeros(cols, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 25) // cols)
    for r in range(0, rows, step):
        x = s["x"].detach()[r:r + step].double()
        if s["residual"]:  # the sum is held in the inputs' type, and everything behind it starts from there
            x = x + s["stream"].detach()[r:r + step].double()
            total[r:r + step] = x
            x = x.float().to(dtype).double()
        rstd = 1 / (x.pow(2).sum(-1, keepdim=True) / cols + EPS).sqrt()
        y[r:r + step] = x * rstd * w
        blocks = torch.cat((x, x.new_zeros(x.size(0), -cols % BLOCK)), 1).view(x.size(0), -1, BLOCK)
        hat = _stored(blocks).view(x.size(0), -1)[:, :cols] * rstd
        d = s["grad"][r:r + step].double()
        dw += (d * hat).sum(0)
        d = d * w
        dx[r:r + step] = rstd * (d - hat * ((d * hat).sum(-1, keepdim=True) / cols))
        if s["residual"]:
            dx[r:r + step] += s["grad_sum"][r:r + step].double()
    return [total, y, dx, dw] if s["residual"] else [y, dx, dw]
