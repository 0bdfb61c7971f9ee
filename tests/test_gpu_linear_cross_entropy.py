"""The cross-entropy of a head without its logits against the formula in 64 bits, with tolerances counted from the roundings."""

from __future__ import annotations

import math

import pytest
import torch

from picotron_amd import ops
from picotron_amd.nn.triton_kernels import (
    LinearCrossEntropyWithFallback,
    TritonLinearCrossEntropyUnavailable,
    triton_linear_cross_entropy,
)

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(n, h, v, dtype, device, seed=0, spread=2.0, ignored=0.25):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(n, h, generator=g, device=device).to(dtype)
    w = (torch.randn(v, h, generator=g, device=device) * spread / math.sqrt(h)).to(dtype)
    t = torch.randint(0, v, (n,), generator=g, device=device)
    if ignored:
        t = t.masked_fill(torch.rand(n, generator=g, device=device) < ignored, -100)
    return x, w, t


def oracle(x, w, t, factors, ignore=-100):
    """Losses, gradients for ``factors`` in 64 bits, and what bounds the errors: for the gradients, the sums of the
    terms' magnitudes, and the largest error of a logit that fp32 sums can have."""

    x, w = x.double(), w.double()
    keep = t != ignore
    x = torch.where(keep[:, None], x, 0.0)
    logits = x @ w.t()
    log_p = torch.log_softmax(logits, -1)
    at = t.clamp_min(0)[:, None]
    losses = torch.where(keep, -log_p.gather(1, at)[:, 0], 0.0)
    c = torch.where(keep, factors.double(), 0.0)[:, None]
    p = log_p.exp()
    g = p.clone()
    g.scatter_(1, at, torch.expm1(log_p.gather(1, at)))
    g = g * c
    # a sum of h products in fp32, rounded at each addition at worst; 32-bit operands in planes leave out terms of 2^-24
    slack = (x.shape[1] + 8) * 2.0**-24 * float((x.abs() @ w.abs().t()).max()) + 2.0**-22
    return losses, g @ w, g.t() @ x, g.abs() @ w.abs(), g.abs().t() @ x.abs(), slack


def check(loss, dx, dw, x, w, t, factors, scale=1.0, reduction="none", ignore=-100):
    losses, dx64, dw64, ax, aw, slack = oracle(x, w, t, factors, ignore)
    keep = t != ignore
    if loss is not None:
        # exp, its sum and the logarithm: a few roundings each; a loss of a sum adds one rounding
        limit = 2 * slack + 2.0**-20 * (1 + losses.abs())
        if reduction == "none":
            assert torch.all((loss.double() - losses).abs() <= limit)
        else:
            want = losses.sum() / (keep.sum() if reduction == "mean" else 1)
            assert abs(float(loss) - float(want)) <= float(limit.max()) * (1 if reduction == "mean" else int(keep.sum()) + 1)
    eps = torch.finfo(x.dtype).eps
    # G's own rounding, that of exp(l - m) to 11 bits, and what the logits' errors make of the softmax; the fp32 sums
    terms = max(x.shape[0], w.shape[0])
    part = {torch.float32: 2.0**-22}.get(x.dtype, eps / 2 + 2.0**-11) + 4 * slack + 2.0**-18 + terms * 2.0**-24
    # and the result's, twice where an incoming gradient other than a power of two follows on it; the smallest step of fp16
    for got, want, total in ((dx, dx64, ax), (dw, dw64, aw)):
        if got is not None:
            floor = 2.0**-24 if x.dtype == torch.float16 else 1e-36
            limit = part * total * scale + eps * want.abs() * scale + floor + 2.0**-28 * float(total.max()) * scale
            off = (got.double() - want * scale).abs()
            assert torch.all(off <= limit), float((off / limit).max())


def check_rows(dx, x, w, t, factors, floor=1e-36):
    """The states' gradients with what check allows, each state's relative to its own."""

    _, want, _, total, _, slack = oracle(x, w, t, factors)
    eps = torch.finfo(x.dtype).eps
    part = {torch.float32: 2.0**-22}.get(x.dtype, eps / 2 + 2.0**-11) + 4 * slack + 2.0**-18 + w.shape[0] * 2.0**-24
    limit = part * total + eps * want.abs() + floor + 2.0**-28 * total.amax(1, keepdim=True)
    off = (dx.double() - want).abs()
    assert torch.all(off <= limit), float((off / limit).max())


SIZES = [(1, 1, 1), (1, 64, 260), (2, 20, 257), (33, 32, 64), (255, 64, 256), (256, 128, 255), (300, 100, 1000), (513, 200, 1027),
         (1100, 72, 3001), (700, 520, 130), (5, 192, 64), (1030, 160, 2100), (70, 129, 70000), (12, 2000, 168), (300, 1100, 90)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,v", SIZES)
def test_token_losses_and_gradients(gpu, dtype, n, h, v):
    x, w, t = make(n, h, v, dtype, gpu, seed=n + h + v, ignored=0.25 if n > 2 else 0)
    factors = torch.randn(n, generator=torch.Generator(device=gpu).manual_seed(1), device=gpu)
    x.requires_grad_()
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t, reduction="none")
    assert loss.dtype == torch.float32 and loss.shape == (n,)
    dx, dw = torch.autograd.grad([loss], [x, w], [factors])
    check(loss.detach(), dx, dw, x.detach(), w.detach(), t, factors)
    with torch.no_grad():
        assert torch.equal(triton_linear_cross_entropy(x, w, t, reduction="none"), loss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h,v", SIZES)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_reduced_loss_and_gradients(gpu, dtype, n, h, v, reduction):
    x, w, t = make(n, h, v, dtype, gpu, seed=n * 3 + v, ignored=0.25 if n > 2 else 0)
    scale = 1024.0 if dtype == torch.float16 else 1.0
    x.requires_grad_()
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t, reduction=reduction)
    dx, dw = torch.autograd.grad(loss * scale, [x, w])
    count = (t != -100).sum() if reduction == "mean" else 1
    check(loss.detach(), dx, dw, x.detach(), w.detach(), t, torch.ones(n, device=gpu) / count, scale, reduction)


@pytest.mark.parametrize("dtype", DTYPES)
def test_incoming_gradient_is_applied(gpu, dtype):
    x, w, t = make(70, 48, 300, dtype, gpu)
    x.requires_grad_()
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w], torch.full((), 0.3, device=gpu))
    check(loss.detach(), dx, dw, x.detach(), w.detach(), t, torch.ones(70, device=gpu) / (t != -100).sum(), float(torch.tensor(0.3)), "mean")


def test_gradients_by_differences(gpu):
    x, w, t = make(9, 7, 11, torch.float32, gpu, ignored=0.3)
    x.requires_grad_()
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])

    def value(x, w):
        keep = t != -100
        return torch.nn.functional.cross_entropy((x @ w.t())[keep], t[keep])

    # central differences of the 64-bit formula: its third derivative times the step's square, 1e-8, and 2^-52 / 1e-4
    for which, grad in ((0, dx), (1, dw)):
        for place in range(0, grad.numel(), 5):
            args = [x.detach().double(), w.detach().double()]
            step = torch.zeros_like(args[which]).view(-1)
            step[place] = 1e-4
            step = step.view_as(args[which])
            up, down = list(args), list(args)
            up[which], down[which] = args[which] + step, args[which] - step
            want = float(value(*up) - value(*down)) / 2e-4
            assert abs(float(grad.view(-1)[place]) - want) <= 1e-6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_shift(gpu, dtype, reduction):
    b, s, h, v = 3, 37, 40, 301
    x, w, t = make(b * s, h, v, dtype, gpu, seed=5)
    x, t = x.view(b, s, h).requires_grad_(), t.view(b, s)
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t, shift=True, reduction=reduction)
    factors = torch.randn(b, s - 1, device=gpu, generator=torch.Generator(device=gpu).manual_seed(3))
    if reduction == "mean":
        factors = torch.ones_like(factors) / (t[:, 1:] != -100).sum()
        dx, dw = torch.autograd.grad(loss * 256, [x, w])
    else:
        assert loss.shape == (b, s - 1)
        dx, dw = torch.autograd.grad([loss], [x, w], [factors * 256])
    assert dx[:, -1].count_nonzero() == 0
    flat = lambda y: y.reshape(b * (s - 1), *y.shape[2:])  # noqa: E731
    check(flat(loss.detach()) if reduction == "none" else loss.detach(), flat(dx[:, :-1]), dw, flat(x.detach()[:, :-1]), w.detach(),
          flat(t[:, 1:]), flat(factors), 256.0, reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("ignored", [0.0, 0.6])
@pytest.mark.parametrize("h", [72, 200])
def test_chunks_of_tokens(gpu, dtype, reduction, ignored, h):
    n, v = 1300, 519
    x, w, t = make(n, h, v, dtype, gpu, seed=8, ignored=ignored)
    factors = torch.randn(n, device=gpu, generator=torch.Generator(device=gpu).manual_seed(3))
    x.requires_grad_()
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t, reduction=reduction, chunk_tokens=300)
    if reduction == "mean":
        factors = torch.ones(n, device=gpu) / (t != -100).sum()
        dx, dw = torch.autograd.grad(loss * 512, [x, w])
    else:
        dx, dw = torch.autograd.grad([loss], [x, w], [factors * 512])
    check(loss.detach(), dx, dw, x.detach(), w.detach(), t, factors, 512.0, reduction)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(gpu, dtype):
    """Strided and offset states, labels, weights and gradients; a broadcast gradient."""

    b, s, h, v = 2, 45, 64, 333
    g = torch.Generator(device=gpu).manual_seed(4)
    big = torch.randn(s, b, 3, h + 5, generator=g, device=gpu).to(dtype)
    x = big[:, :, 1, 3:3 + h].transpose(0, 1)
    wide = (torch.randn(v, 2, h + 8, generator=g, device=gpu) * 0.2).to(dtype)
    w = wide[:, 1, :h]
    t = torch.randint(0, v, (s, b, 2), generator=g, device=gpu)[:, :, 1].t()
    factors = torch.randn(s, b, generator=g, device=gpu).t()
    xx, ww = x.detach().requires_grad_(), w.detach().requires_grad_()
    assert not xx.is_contiguous() and not ww.is_contiguous()
    loss = triton_linear_cross_entropy(xx, ww, t, reduction="none")
    dx, dw = torch.autograd.grad([loss], [xx, ww], [factors])
    flat = lambda y: y.reshape(b * s, *y.shape[2:])  # noqa: E731
    check(flat(loss.detach()), flat(dx), dw, flat(x), w, flat(t), flat(factors))
    plain = triton_linear_cross_entropy(x.contiguous(), w.contiguous(), t.contiguous(), reduction="none")
    assert torch.equal(plain, loss)
    loss = triton_linear_cross_entropy(xx, ww, t, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), [xx, ww])  # an expanded gradient
    check(None, flat(dx), dw, flat(x), w, flat(t), torch.ones(b * s, device=gpu))
    # states and weights whose last dimension is not the contiguous one, a weight used for two rows
    xt = x.transpose(1, 2).contiguous().transpose(1, 2)
    wt = w.t().contiguous().t()
    assert torch.equal(triton_linear_cross_entropy(xt, wt, t, reduction="none"), plain)
    same = w[:1].expand(v, h)
    got = triton_linear_cross_entropy(x, same, t, reduction="none")
    assert torch.all((got - math.log(v)).abs() <= 2.0**-18)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("h", [64, 192])
def test_nothing_kept(gpu, dtype, reduction, h):
    x, w, _ = make(40, h, 300, dtype, gpu)
    t = torch.full((40,), 7, device=gpu)
    x.requires_grad_()
    w.requires_grad_()
    for chunk in (None, 10):
        loss = triton_linear_cross_entropy(x, w, t, ignore_index=7, reduction=reduction, chunk_tokens=chunk)
        dx, dw = torch.autograd.grad(loss.sum(), [x, w])
        assert torch.isnan(loss) if reduction == "mean" else not loss.any()
        assert not dx.any() and not dw.any()


@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 64), (0, 5, 64), (3, 1, 64)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_no_tokens(gpu, shape, reduction):
    x = torch.randn(shape, device=gpu, requires_grad=True)
    w = torch.randn(50, 64, device=gpu, requires_grad=True)
    t = torch.zeros(shape[:-1], dtype=torch.long, device=gpu)
    shift = len(shape) == 3 and shape[1] < 2
    loss = triton_linear_cross_entropy(x, w, t, shift=shift, reduction=reduction)
    dx, dw = torch.autograd.grad(loss.sum(), [x, w])
    assert dx.shape == shape and not dx.any() and not dw.any()
    assert torch.isnan(loss) if reduction == "mean" else loss.numel() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [64, 192])
def test_ignored_rows_may_hold_anything(gpu, dtype, h):
    x, w, t = make(300, h, 500, dtype, gpu, ignored=0.5)
    dirty = torch.where((t == -100)[:, None], math.nan, x)
    dirty[(t == -100).nonzero()[0]] = math.inf
    out = []
    for y in (x, dirty):
        y = y.clone().requires_grad_()
        v = w.clone().requires_grad_()
        loss = triton_linear_cross_entropy(y, v, t)
        out.append((loss, *torch.autograd.grad(loss, [y, v])))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert not out[0][1][t == -100].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [64, 192])
def test_not_finite(gpu, dtype, h):
    x, w, t = make(300, h, 500, dtype, gpu, ignored=0)
    for bad in (math.nan, math.inf):
        y = x.clone()
        y[5, 3] = bad
        loss = triton_linear_cross_entropy(y, w, t, reduction="none")
        assert torch.isnan(loss[5]) and loss.isnan().sum() == 1
    for label in (500, -1, 2**40):
        s = t.clone()
        s[7] = label
        y, v = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = triton_linear_cross_entropy(y, v, s, reduction="none")
        assert torch.isnan(loss[7]) and loss.isnan().sum() == 1
        dx, dw = torch.autograd.grad(loss.nansum(), [y, v])  # its own gradient is zero there
        assert dx[7].isnan().all() and dx.isnan().any(1).sum() == 1 and dw.isnan().all()
        assert torch.isnan(triton_linear_cross_entropy(y, v, s))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [64, 128, 192])
def test_far_logits(gpu, dtype, h):
    """Rows far apart in level (the tiles' largest differ by hundreds), and labels of nearly all the weight."""

    x, w, t = make(64, h, 1000, dtype, gpu, ignored=0, spread=1.0)
    w[:, 0] = torch.linspace(-30, 30, 1000, device=gpu).to(dtype)
    x[:, 0] = torch.linspace(-16, 16, 64, device=gpu).to(dtype)
    t[::2] = (x.double() @ w.double().t()).argmax(1)[::2]
    factors = torch.ones(64, device=gpu)
    x.requires_grad_()
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad([loss], [x, w], [factors])
    check(loss.detach(), dx, dw, x.detach(), w.detach(), t, factors)


@pytest.mark.parametrize("power", [-90, -60, -20, 20, 60, 100])
def test_magnitudes_of_32_bits(gpu, power):
    """States and weights far from one in opposite directions; rows of one tensor 2^20 apart."""

    x, w, t = make(200, 64, 500, torch.float32, gpu)
    factors = torch.ones(200, device=gpu)
    spread = torch.where(torch.arange(200, device=gpu) % 2 == 0, 1.0, 2.0**-20)[:, None]
    x = (x * spread * 2.0**power).requires_grad_()
    w = (w * 2.0**-power).requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad([loss], [x, w], [factors])
    unit = 2.0**power
    check(loss.detach(), dx * unit, dw / unit, (x / unit).detach(), (w * unit).detach(), t, factors)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [64, 192])
def test_one_side_alone(gpu, dtype, h):
    x, w, t = make(90, h, 300, dtype, gpu)
    both = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    dx, dw = torch.autograd.grad(triton_linear_cross_entropy(*both, t), both)
    a = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(triton_linear_cross_entropy(a, w, t), a)[0], dx)
    b = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(triton_linear_cross_entropy(x, b, t), b)[0], dw)


def test_gradients_are_handed_out_once(gpu):
    x, w, t = make(90, 64, 300, torch.bfloat16, gpu)
    x.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="handed out"):
        loss.backward()
    losses = triton_linear_cross_entropy(x, w, t, reduction="none")
    first = torch.autograd.grad(losses.sum(), x, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(losses.sum(), x)[0], first)


@pytest.mark.parametrize("h", [64, 192])
def test_runs_repeat_to_the_bit(gpu, h):
    x, w, t = make(600, h, 3000, torch.bfloat16, gpu)
    x.requires_grad_()
    w.requires_grad_()
    runs = []
    for _ in range(3):
        loss = triton_linear_cross_entropy(x, w, t)
        runs.append((loss, *torch.autograd.grad(loss, [x, w])))
    for run in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(run, runs[0]))


def test_autocast(gpu):
    x, w, t = make(90, 64, 300, torch.float32, gpu)
    x.requires_grad_()
    w.requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = triton_linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert dx.dtype == dw.dtype == torch.float32
    a, b = x.detach().bfloat16().requires_grad_(), w.detach().bfloat16().requires_grad_()
    other = triton_linear_cross_entropy(a, b, t)
    assert torch.equal(other, loss)
    assert all(torch.equal(p, q.float()) for p, q in zip((dx, dw), torch.autograd.grad(other, [a, b])))


def test_tied_weights_add_up(gpu):
    """The head's weight is the embedding's too."""

    t = make(64, 64, 300, torch.float32, gpu, ignored=0)[2].view(2, 32)
    w = torch.randn(300, 64, device=gpu, generator=torch.Generator(device=gpu).manual_seed(2)).requires_grad_()
    loss = triton_linear_cross_entropy(torch.nn.functional.embedding(t, w), w, t, shift=True)
    got = torch.autograd.grad(loss, w)[0]
    v = w.detach().double().requires_grad_()
    logits = torch.nn.functional.embedding(t, v)[:, :-1] @ v.t()
    want = torch.autograd.grad(torch.nn.functional.cross_entropy(logits.flatten(0, 1), t[:, 1:].flatten()), v)[0]
    # both products' sums of at most 300 terms in fp32 and the softmax of logits of up to 100, as above
    assert torch.all((got.double() - want).abs() <= (4 * 72 * 2.0**-24 * 150 + 2.0**-18) * want.abs().max())


@pytest.mark.parametrize("dtype,h", [(torch.float32, 64), (torch.bfloat16, 64), (torch.bfloat16, 192)])
def test_captured(gpu, dtype, h):
    x, w, t = make(300, h, 700, dtype, gpu)
    x.requires_grad_()
    w.requires_grad_()

    def step():
        loss = triton_linear_cross_entropy(x, w, t, chunk_tokens=256)
        return (loss, *torch.autograd.grad(loss, [x, w]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        y, v, s = make(300, h, 700, dtype, gpu, seed=seed + 20, ignored=0.2 * seed)
        with torch.no_grad():
            x.copy_(y)
            w.copy_(v)
            t.copy_(s)
        graph.replay()
        got = [o.detach().clone() for o in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_on_another_stream(gpu):
    x, w, t = make(300, 64, 700, torch.bfloat16, gpu)
    want = triton_linear_cross_entropy(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = triton_linear_cross_entropy(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_large(gpu):
    """The second chunk and a tail of tiles at sizes of training: over 2^31 bytes of exponentials in all."""

    n, h, v = 9000, 256, 128257
    x, w, t = make(n, h, v, torch.bfloat16, gpu, ignored=0)
    x.requires_grad_()
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])
    total, dw64, rows = 0.0, torch.zeros(v, h, dtype=torch.float64, device=gpu), []
    a, b = x.detach().double(), w.detach().double()
    for i in range(0, n, 1000):
        p = torch.log_softmax(a[i:i + 1000] @ b.t(), -1)
        total -= float(p.gather(1, t[i:i + 1000, None]).sum())
        p = p.exp_()
        p[torch.arange(p.size(0), device=gpu), t[i:i + 1000]] -= 1
        p /= n
        rows.append(p @ b)
        dw64 += p.t() @ a[i:i + 1000]
    assert abs(float(loss) - total / n) <= 2.0**-18 * total / n
    for got, want in ((dx, torch.cat(rows)), (dw, dw64)):
        # roundings of the result and of G, independent of each other: half a step of bf16 each, at most, in the norm
        assert float((got.double() - want).norm() / want.norm()) <= 2 * 2.0**-9


def test_fallback_class_runs_the_kernels(gpu):
    x, w, t = make(90, 64, 300, torch.bfloat16, gpu)
    head = LinearCrossEntropyWithFallback(use_triton=True)
    assert torch.equal(head(x, w, t), triton_linear_cross_entropy(x, w, t)) and not head._fallback_warned
    # the PyTorch form rounds the logits, of up to 10, to bf16
    assert abs(float(LinearCrossEntropyWithFallback()(x, w, t)) - float(head(x, w, t))) <= 10 * 2.0**-8


def test_refusals(gpu):
    x, w, t = make(8, 64, 30, torch.float32, gpu)
    for args in ((x.half(), w, t), (x.double(), w.double(), t), (x, w[:, :32], t), (x, w, t[:4]), (x, w, t.int()), (x, w[0], t),
                 (x[0], w, t[0]), (x, w, t.cpu()), (x[:, :0], w[:, :0], t), (x.half()[:, :0], w.half()[:, :0], t), (x, w[:0], t)):
        with pytest.raises(TritonLinearCrossEntropyUnavailable):
            triton_linear_cross_entropy(*args)
    with pytest.raises(TritonLinearCrossEntropyUnavailable):
        triton_linear_cross_entropy(x, w, t, shift=True)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(x, w, t, reduction="none", want_dx=True, grad_losses=torch.ones(9, device=gpu))


def test_between_the_graphs_of_a_compiled_model(gpu):
    x, w, t = make(90, 64, 300, torch.float32, gpu)
    layer = torch.nn.Linear(64, 64, bias=False).to(gpu)

    def loss_of():
        return triton_linear_cross_entropy(layer(x).relu(), w, t)

    outs = []
    torch._dynamo.reset()
    for f in (loss_of, torch.compile(loss_of, backend="aot_eager")):
        layer.zero_grad()
        loss = f()
        loss.backward()
        outs.append((loss.detach(), layer.weight.grad.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_many_tokens_without_gradients(gpu):
    """More tokens than a chunk of sums takes, at a vocabulary whose tiles make that few."""

    n, h, v = 700, 160, 300000
    x, w, t = make(n, h, v, torch.bfloat16, gpu, ignored=0.2)
    whole = triton_linear_cross_entropy(x, w, t, reduction="none")
    parts = triton_linear_cross_entropy(x, w, t, reduction="none", chunk_tokens=256)
    assert torch.equal(whole, parts)
    want = torch.nn.functional.cross_entropy(x.double() @ w.double().t(), t, reduction="none")
    slack = (h + 8) * 2.0**-24 * float((x.double().abs() @ w.double().abs().t()).max()) + 2.0**-22
    assert torch.all((whole.double() - want).abs() <= 2 * slack + 2.0**-20 * (1 + want.abs()))


def test_more_tokens_than_a_chunk_of_a_small_vocabulary(gpu):
    """A million rows: a chunk's exponentials would fit, its grids would not."""

    n, h, v = 1_100_000, 136, 10
    x, w, t = make(n, h, v, torch.bfloat16, gpu)
    x.requires_grad_()
    w.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t, reduction="none")
    factors = torch.rand(n, device=gpu)
    dx, dw = torch.autograd.grad(loss, [x, w], factors)
    part = slice(n - 3000, n)
    check(loss.detach()[part], dx[part], None, x.detach()[part], w.detach(), t[part], factors[part])
    with torch.no_grad():
        assert torch.equal(triton_linear_cross_entropy(x, w, t, reduction="none"), loss)
    want = torch.zeros(v, h, dtype=torch.float64, device=gpu)
    size = torch.zeros_like(want)
    slack = 0.0
    for i in range(0, n, 100_000):
        p = slice(i, i + 100_000)
        _, _, dw64, _, aw, more = oracle(x.detach()[p], w.detach(), t[p], factors[p])
        want, size, slack = want + dw64, size + aw, max(slack, more)
    # as in check, with the fp32 sums' errors over the kept rows: at worst one rounding of the running sum for each, of which the
    # signs of a million do not agree: sqrt(n) of them
    limit = (2.0**-9 + 2.0**-11 + 4 * slack + 2.0**-18 + math.sqrt(n) * 2.0**-24) * size + 2.0**-8 * want.abs()
    assert torch.all((dw.double() - want).abs() <= limit)


def test_calls_of_two_threads(gpu):
    """Each on a stream of its own: the same bits as one after the other."""

    import threading

    cases = [make(*size, dtype, gpu, seed) for seed, (size, dtype) in enumerate(
        [((300, 72, 1000), torch.float32), ((300, 192, 2000), torch.bfloat16), ((20, 64, 500), torch.float16), ((700, 40, 900), torch.bfloat16)])]

    def run(x, w, t):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = triton_linear_cross_entropy(x, w, t, reduction="sum")
        return [loss.detach(), *torch.autograd.grad(loss, [x, w])]

    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(order):
        try:
            stream = torch.cuda.Stream(gpu)
            with torch.cuda.stream(stream):
                for _ in range(5):
                    for i in order:
                        got = run(*cases[i])
                        stream.synchronize()
                        if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                            wrong.append(i)
        except Exception as error:  # noqa: BLE001
            wrong.append(error)

    threads = [threading.Thread(target=work, args=(order,)) for order in ((0, 1, 2, 3), (3, 2, 1, 0))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong


@pytest.mark.parametrize("dtype,h", [(torch.float32, 64), (torch.float32, 200), (torch.float16, 64), (torch.float16, 192), (torch.bfloat16, 64),
                                     (torch.bfloat16, 192)])
@pytest.mark.parametrize("n,v,chunk", [(300, 1000, 0), (40, 1000, 0), (300, 20000, 0), (600, 1000, 256)])
def test_token_weights_far_apart(gpu, dtype, h, n, v, chunk):
    """Weights from 1 down to 2^-60: every state's gradient is right relative to its own size, whatever the others weigh."""

    x, w, t = make(n, h, v, dtype, gpu, seed=n + v)
    power = torch.linspace(0, -60, n, device=gpu)[torch.randperm(n, generator=torch.Generator().manual_seed(2)).to(gpu)]
    factors = power.exp2() * torch.where(torch.arange(n, device=gpu) % 3 == 0, -1.0, 1.0)
    _, dx, dw = ops.linear_cross_entropy(x, w, t, reduction="none", want_loss=False, want_dx=True, want_dw=True, grad_losses=factors,
                                         grad_dtype=torch.float32, chunk_tokens=chunk)
    check(None, None, dw, x, w, t, factors)
    check_rows(dx, x, w, t, factors)
    # one gradient alone: the same
    alone = ops.linear_cross_entropy(x, w, t, reduction="none", want_loss=False, want_dx=True, grad_losses=factors, grad_dtype=torch.float32,
                                     chunk_tokens=chunk)[1]
    assert torch.equal(alone, dx)
    alone = ops.linear_cross_entropy(x, w, t, reduction="none", want_loss=False, want_dw=True, grad_losses=factors, grad_dtype=torch.float32,
                                     chunk_tokens=chunk)[2]
    check(None, None, alone, x, w, t, factors)


@pytest.mark.parametrize("h", [192, 72])
def test_token_weights_far_apart_in_16_bits(gpu, h):
    """Gradients in fp16, through whole lines (192) and in parts (72): from 2^14 down to 2^-10."""

    x, w, t = make(300, h, 1000, torch.float16, gpu, spread=4.0)
    factors = torch.linspace(14, -10, 300, device=gpu).exp2() * 0.75
    x.requires_grad_()
    loss = triton_linear_cross_entropy(x, w, t, reduction="none")
    dx = torch.autograd.grad([loss], [x], [factors])[0]
    check_rows(dx, x.detach(), w, t, factors, floor=2.0**-25)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [64, 192])
def test_token_weights_of_any_kind(gpu, dtype, h):
    """Zeros, the largest and smallest of fp32, all of them small, and infinities, which stay with their state."""

    x, w, t = make(64, h, 300, dtype, gpu, ignored=0)

    def dx_of(factors):
        return ops.linear_cross_entropy(x, w, t, reduction="none", want_loss=False, want_dx=True, want_dw=True, grad_losses=factors,
                                        grad_dtype=torch.float32)[1:]

    ones = torch.ones(64, device=gpu)
    one, dw_one = dx_of(ones)
    for power in (-80, -20, 20, 80):  # a power of two of all changes nothing else
        dx, dw = dx_of(ones * 2.0**power)
        assert torch.equal(dx * 2.0**-power, one) and torch.equal(dw * 2.0**-power, dw_one)
    factors = ones.clone()
    factors[3], factors[5], factors[7] = 0.0, 2.0**-126, 2.0**-140
    dx, dw = dx_of(factors)
    assert not dx[3].any()
    keep = torch.arange(64, device=gpu) > 7
    assert torch.equal(dx[keep], one[keep])
    check(None, None, dw, x, w, t, factors)
    assert not dx_of(ones * 0)[0].any() and not dx_of(ones * 0)[1].any()
    factors[3], factors[5] = torch.inf, -torch.inf
    dx = dx_of(factors)[0]
    assert not dx[3].isfinite().all() and not dx[5].isfinite().all() and torch.equal(dx[keep], one[keep])


def minus_infinity(dtype, h, n, v, gpu):
    """An infinite entry of the weight takes its word out of the softmax, and leaves everything else as it was."""

    x, w, t = make(n, h, v, dtype, gpu, ignored=0)
    t = t.masked_fill((t == 7) | (t == v - 1), 9)
    x[:, 3] = x[:, 3].abs() + 0.5
    out = w.clone()
    out[7, 3] = out[v - 1, 3] = -math.inf
    a, b = x.clone().requires_grad_(), out.clone().requires_grad_()
    loss = triton_linear_cross_entropy(a, b, t, reduction="none")
    assert loss.isfinite().all()
    dx, dw = torch.autograd.grad([loss], [a, b], [torch.ones(n, device=gpu)])
    # as if the words were not there; in the entry's column dx is 0 * -inf
    words = (torch.arange(v, device=gpu) != 7) & (torch.arange(v, device=gpu) != v - 1)
    place = torch.cumsum(words, 0) - 1
    others = torch.arange(h, device=gpu) != 3
    check(loss.detach(), None, dw[words], x, w[words], place[t], torch.ones(n, device=gpu))
    assert not dw[~words].any()
    losses, dx64, _, ax, _, slack = oracle(x, w[words], place[t], torch.ones(n, device=gpu))
    part = {torch.float32: 2.0**-22}.get(dtype, torch.finfo(dtype).eps / 2 + 2.0**-11) + 4 * slack + 2.0**-18 + v * 2.0**-24
    limit = (part + torch.finfo(dtype).eps) * ax + 2.0**-24
    assert torch.all(((dx.double() - dx64).abs() <= limit)[:, others])
    t[0] = 7
    loss = triton_linear_cross_entropy(x, out, t, reduction="none")
    assert loss[0] == math.inf and loss[1:].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h", [20, 64, 128, 192])
@pytest.mark.parametrize("n,v", [(40, 500), (300, 500), (300, 9000), (512, 512)])
def test_words_whose_logits_are_minus_infinity(gpu, dtype, h, n, v):
    minus_infinity(dtype, h, n, v, gpu)


@pytest.mark.parametrize("h", [20, 64, 192])
@pytest.mark.parametrize("n,v", [(1, 12), (40, 500), (300, 500), (300, 9000)])
def test_words_whose_logits_are_minus_infinity_in_32_bits(gpu, h, n, v):
    minus_infinity(torch.float32, h, n, v, gpu)


@pytest.mark.parametrize("n,v", [(40, 500), (300, 9000)])
def test_infinities_in_32_bits_are_those_of_the_product(gpu, n, v):
    """Of either sign, in states and words: each loss is what the formula gives, and tokens without one are as they were."""

    x, w, t = make(n, 64, v, torch.float32, gpu, ignored=0)
    clean = triton_linear_cross_entropy(x, w, t, reduction="none")
    for bad in (math.inf, -math.inf, math.nan):
        y = x.clone()
        y[5, 3] = bad
        loss = triton_linear_cross_entropy(y, w, t, reduction="none")
        assert loss[5].isnan() and torch.equal(loss[torch.arange(n, device=gpu) != 5], clean[torch.arange(n, device=gpu) != 5])
    u = w.clone()
    u[7, 3] = math.inf  # a logit of +inf or -inf, by the state's sign
    t = t.masked_fill(t == 7, 9)
    loss = triton_linear_cross_entropy(x, u, t, reduction="none")
    assert torch.equal(loss.isnan(), x[:, 3] > 0) and loss[x[:, 3] < 0].isfinite().all()


def gradients_of(run, x, w):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = run(x, w)
    return (loss.detach(), *torch.autograd.grad(loss.sum(), [x, w]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_saved_tensors_hooks(gpu, dtype, reduction):
    """What a deferred loss saves goes through them; a mean's or sum's gradients, which are no saved tensors, do not."""

    x, w, t = make(600, 64, 300, dtype, gpu)
    packed = []

    def pack(tensor):
        packed.append(tensor.shape)
        return tensor.cpu()

    def hooked(a, b):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda tensor: tensor.to(gpu)):
            return triton_linear_cross_entropy(a, b, t, reduction=reduction)

    got = gradients_of(hooked, x, w)
    want = gradients_of(lambda a, b: triton_linear_cross_entropy(a, b, t, reduction=reduction), x, w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert sorted(map(tuple, packed)) == ([] if reduction == "mean" else [(300, 64), (600,), (600, 64)])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("use_reentrant", [False, True])
def test_under_activation_checkpointing(gpu, dtype, reduction, use_reentrant):
    from torch.utils.checkpoint import checkpoint

    x, w, t = make(90, 64, 300, dtype, gpu)

    def head(a, b):
        return triton_linear_cross_entropy(a.tanh(), b, t, reduction=reduction)

    want = gradients_of(lambda a, b: head(a.sin(), b), x, w)
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = checkpoint(head, a.sin(), b, use_reentrant=use_reentrant)
    loss.sum().backward()
    assert all(torch.equal(p, q) for p, q in zip((loss.detach(), a.grad, b.grad), want))


def test_transforms_are_refused_and_fall_back(gpu):
    """Forward-mode and functorch's transforms see no derivative of the kernels: an error, or the PyTorch form's."""

    x, w, t = make(20, 64, 30, torch.float32, gpu)
    head = LinearCrossEntropyWithFallback(use_triton=True)
    plain = LinearCrossEntropyWithFallback()
    along = torch.randn(20, 64, device=gpu)
    for transform in (lambda f: torch.func.grad(lambda a: f(a, w, t))(x), lambda f: torch.func.jvp(lambda a: f(a, w, t), (x,), (along,))[1],
                      lambda f: torch.func.vmap(lambda a: f(a[None], w, t[:1]))(x)):
        with pytest.raises(RuntimeError):
            transform(triton_linear_cross_entropy)
        head._fallback_warned = False
        with pytest.warns(RuntimeWarning, match="linear cross-entropy unavailable"):
            got = transform(head)
        assert torch.equal(got, transform(plain))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        triton_linear_cross_entropy(torch.autograd.forward_ad.make_dual(x, along), w, t)


def confident(n, h, v, dtype, gpu, level):
    """Labels ahead of all other words by 0 to 24, every logit near ``level``."""

    x, w, t = make(n, h, v, dtype, gpu, ignored=0, spread=0.5)
    x = x * 0.25
    x[:, 0], w[:, 0] = 8.0, level / 8  # exact in each type
    direction = w[t, 1:].double()
    gap = torch.linspace(0, 24, n, device=gpu, dtype=torch.float64)[:, None]
    x[:, 1:] = (x[:, 1:].double() + gap * direction / direction.square().sum(1, keepdim=True)).to(dtype)
    return x, w, t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [20, 64, 192])
@pytest.mark.parametrize("n,v", [(50, 300), (300, 1000), (300, 9000)])
@pytest.mark.parametrize("level", [0, 40, -90])
def test_confident_labels(gpu, dtype, h, n, v, level):
    """A softmax close to 1 at the label: the loss and its gradient are right to a few roundings of 1, not of the logits' level."""

    x, w, t = confident(n, h, v, dtype, gpu, level)
    one = torch.ones(n, device=gpu)
    loss, dx, dw = ops.linear_cross_entropy(x, w, t, reduction="none", want_loss=True, want_dx=True, want_dw=True, grad_losses=one,
                                            grad_dtype=torch.float32)
    losses, dx64, dw64, ax, aw, slack = oracle(x, w, t, one)
    rest = -torch.expm1(-losses)  # of the softmax, beside the label's
    # logits that are off by the slack move the loss by twice that times the rest; the sum of exponentials near 1, its logarithm
    # and exp - 1 round a few times to 24 bits; a narrow model's sum grows by 8 words of every 32 at a time, each time rounded by half
    # a step of 2^-23 while it lies below 2
    few = 2.0**-21 + v / 32 * 2.0**-24
    assert torch.all((loss.double() - losses).abs() <= 2 * slack * rest + few * (1 + losses))
    part = {torch.float32: 2.0**-22}.get(dtype, torch.finfo(dtype).eps / 2 + 2.0**-11) + 4 * slack + 2.0**-18 + max(n, v) * 2.0**-24
    at_label = torch.zeros_like(dw64).index_add_(0, t, x.double().abs())
    floor = 2.0**-28 * float(ax.max())
    assert torch.all((dx.double() - dx64).abs() <= part * ax + few * w[t].double().abs() + floor)
    assert torch.all((dw.double() - dw64).abs() <= part * aw + few * at_label + 2.0**-28 * float(aw.max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [64, 192])
def test_a_vocabulary_of_one_word(gpu, dtype, h):
    x, w, t = make(300, h, 1, dtype, gpu, ignored=0, spread=30.0)
    loss, dx, dw = ops.linear_cross_entropy(x, w, t, reduction="none", want_loss=True, want_dx=True, want_dw=True,
                                            grad_losses=torch.ones(300, device=gpu))
    assert not loss.any() and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("h", [20, 64, 128, 192, 1030])
@pytest.mark.parametrize("n,v", [(1, 300), (3, 40), (50, 1000), (256, 3000), (250, 200)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_few_tokens_are_exact_at_their_labels(gpu, dtype, h, n, v, reduction):
    """The softmax's entries at the labels, most of each gradient, are not those of the matrix cores' 16 bits."""

    x, w, t = make(n, h, v, dtype, gpu, spread=0.5, ignored=0.25 if n > 3 else 0, seed=n)
    t[n // 2:] = t[: n - n // 2].clone()  # words that are several tokens' label
    factors = torch.randn(n, device=gpu, generator=torch.Generator(device=gpu).manual_seed(5))
    if reduction == "mean":
        factors = torch.ones(n, device=gpu) / (t != -100).sum()
    _, dx, dw = ops.linear_cross_entropy(x, w, t, reduction=reduction, want_loss=False, want_dx=True, want_dw=True, grad_dtype=torch.float32,
                                         grad_losses=factors if reduction == "none" else None)
    losses, dx64, dw64, ax, aw, slack = oracle(x, w, t, factors)
    keep = t != -100
    label = torch.where(keep, -torch.expm1(-losses) * factors.abs(), 0.0)[:, None]  # what G holds there
    at = t.clamp_min(0)
    own_x = label * w[at].double().abs()
    own_w = torch.zeros_like(dw64).index_add_(0, at, label * torch.where(keep[:, None], x, 0).double().abs())
    exact = 4 * slack + 2.0**-18 + max(n, v) * 2.0**-24
    part = exact + torch.finfo(dtype).eps / 2 + 2.0**-11
    for got, want, total, own in ((dx, dx64, ax, own_x), (dw, dw64, aw, own_w)):
        limit = exact * own + part * (total - own) + 2.0**-28 * float(total.max())
        off = (got.double() - want).abs()
        assert torch.all(off <= limit), float((off / limit).max())


@pytest.mark.parametrize("dtype,n,h", [(torch.float32, 300, 64), (torch.float16, 300, 192), (torch.float16, 100, 192), (torch.float16, 100, 64),
                                       (torch.bfloat16, 100, 192), (torch.bfloat16, 100, 64)])
def test_captured_with_weights(gpu, dtype, n, h):
    """Tokens with weights of their own, far apart in some replays and alike in others; calls of few tokens."""

    x, w, t = make(n, h, 700, dtype, gpu)
    factors = torch.ones(n, device=gpu)
    x.requires_grad_()
    w.requires_grad_()

    def step():
        loss = triton_linear_cross_entropy(x, w, t, reduction="none")
        return (loss, *torch.autograd.grad([loss], [x, w], [factors]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        y, v, s = make(n, h, 700, dtype, gpu, seed=seed + 20, ignored=0.3 * seed)
        with torch.no_grad():
            x.copy_(y)
            w.copy_(v)
            t.copy_(s)
            factors.copy_(torch.linspace(0, -10 * seed, n, device=gpu).exp2())
        graph.replay()
        got = [o.detach().clone() for o in out]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        check(got[0], got[1], got[2], x.detach(), w.detach(), t, factors)
