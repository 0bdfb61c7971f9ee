"""Sequence log-probabilities and the preference loss on the GPU against their definition in 64 bits: vocabularies around the
kernels' sizes, labels that leave rows and sequences empty, special values, strides, types, gradients, streams and graphs."""

from __future__ import annotations

import pytest
import torch

from gpu_util import randn
from picotron_amd import _lib, ops
from picotron_amd.nn import RotaryEmbedding
from picotron_amd.nn.triton_kernels import (
    PreferenceLossWithFallback,
    TritonPreferenceUnavailable,
    preference_loss_with_pytorch,
    triton_adamw_step,
    triton_preference_loss,
    triton_sequence_log_probs,
)
from picotron_amd.optim import AdamW8bit

pytestmark = pytest.mark.gpu

# An exp's argument is rounded to 2^-24 of |x - max| (below 40 here, twice the largest logit) by the shift and the product
# with log2(e), the exp itself to 2^-23; a sum has at most 64 additions in a row in a batch, one a batch, and twelve of the
# joins.  Relative to the sum: (2 * 40 + 2 + 64 + 16 + 12) * 2^-24, and as much for what is divided or subtracted again.
REL = 2.0 * (80 + 2 + 64 + 16 + 12) * 2.0**-24


def inputs(batch, seq, vocab, dtype, device, seed, scale=2.0):
    logits = randn((batch, seq, vocab), dtype, device, seed, scale)
    g = torch.Generator(device=device).manual_seed(seed + 1)
    labels = torch.randint(0, vocab, (batch, seq), generator=g, device=device)
    at = torch.arange(seq, device=device)
    prompt = torch.randint(0, max(1, seq // 2), (batch, 1), generator=g, device=device)
    end = seq - torch.randint(0, max(1, seq // 4), (batch, 1), generator=g, device=device)
    labels = labels.masked_fill((at < prompt) | (at >= end), -100)
    if batch > 2:
        labels[1] = -100  # a sequence that keeps nothing
    return logits, labels, torch.randn(batch, generator=g, device=device) * 3


def token_log_probs(logits, labels, shift):
    """(log-probability and mask of each position, the log-softmax) in 64 bits."""

    y = torch.log_softmax(logits.detach().double(), -1)
    want = torch.full_like(labels, -100)
    if shift:
        want[:, :-1] = labels[:, 1:]
    else:
        want.copy_(labels)
    keep = want != -100
    return torch.where(keep, y.gather(-1, want.clamp_min(0)[..., None])[..., 0], 0.0), keep, y, want


def check_log_probs(got, logits, labels, shift=True, average=False):
    token, keep, _, _ = token_log_probs(logits, labels, shift)
    n = keep.sum(1).clamp_min(1) if average else torch.ones_like(keep.sum(1))
    exact = token.sum(1) / n
    bound = (keep.sum(1) * REL + 2.0**-23 * token.abs().sum(1)) / n + 2.0**-24 * exact.abs()
    assert ((got.double() - exact).abs() <= bound).all(), float(((got.double() - exact).abs() / bound).nan_to_num(0).max())


def check_grad(got, logits, labels, slope, shift=True, slope_rel=2.0**-22):
    """``slope`` [batch] in 64 bits, known to ``slope_rel`` of itself: p is right to REL of itself, 1 - p to REL * p more."""

    _, keep, y, want = token_log_probs(logits, labels, shift)
    p = y.exp()
    one = torch.zeros_like(p).scatter_(-1, want.clamp_min(0)[..., None], 1.0)
    g = (slope[:, None] * keep)[..., None]
    exact = g * (one - p)
    half = torch.finfo(logits.dtype).eps / 2
    bound = half * exact.abs() + g.abs() * (REL * p + 2.0**-23 * one) + slope_rel * exact.abs() + torch.finfo(logits.dtype).tiny * half
    off = (got.double() - exact).abs()
    assert (off <= bound).all(), float((off / bound).nan_to_num(0).max())
    assert not got[~keep].any()


def slope_of(rewards, beta, loss, smooth):
    """d loss / d log_prob [2 pairs] from the rewards in 64 bits."""

    c, r = rewards.chunk(2)
    h = c - r
    dh = {"sigmoid": smooth * torch.sigmoid(h) - (1 - smooth) * torch.sigmoid(-h), "hinge": -(h < 1).double(),
          "ipo": 2 * (h / beta - 0.5 / beta) / beta}[loss]
    return torch.cat((dh, -dh)) * beta / c.numel()


VOCABS = [1, 2, 7, 8, 63, 64, 127, 260, 511, 1000, 2047, 2048, 4097, 8192, 16384, 32001, 50257]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", VOCABS)
def test_vocabularies(gpu, dtype, vocab):
    logits, labels, _ = inputs(3, 9, vocab, dtype, gpu, vocab)
    logits.requires_grad_()
    out = triton_sequence_log_probs(logits, labels)
    check_log_probs(out.detach(), logits, labels)
    up = torch.tensor([0.7, -1.3, 2.1], device=gpu)
    (grad,) = torch.autograd.grad(out, logits, up)
    assert grad.dtype == dtype
    check_grad(grad, logits, labels, up.double())


@pytest.mark.parametrize("vocab,dtype", [(128256, torch.bfloat16), (200_001, torch.float32), (128256, torch.float16)])
@pytest.mark.parametrize("batch,seq", [(1, 2), (2, 40)])
def test_large_vocabularies(gpu, vocab, dtype, batch, seq):
    logits, labels, _ = inputs(batch, seq, vocab, dtype, gpu, 3)
    logits.requires_grad_()
    out = triton_sequence_log_probs(logits, labels)
    check_log_probs(out.detach(), logits, labels)
    (grad,) = torch.autograd.grad(out, logits, torch.ones_like(out))
    check_grad(grad, logits, labels, torch.ones(batch, dtype=torch.float64, device=gpu))


@pytest.mark.parametrize("batch,seq", [(1, 1), (1, 2), (5, 1), (2, 1025), (1, 5000), (300, 3)])
@pytest.mark.parametrize("shift", [True, False])
@pytest.mark.parametrize("average", [True, False])
def test_lengths(gpu, batch, seq, shift, average):
    logits, labels, _ = inputs(batch, seq, 65, torch.float32, gpu, 5)
    logits.requires_grad_()
    out = triton_sequence_log_probs(logits, labels, shift=shift, average=average)
    check_log_probs(out.detach(), logits, labels, shift, average)
    up = torch.linspace(-1, 2, batch, device=gpu)
    (grad,) = torch.autograd.grad(out, logits, up)
    keep = token_log_probs(logits, labels, shift)[1]
    slope = up.double() / (keep.sum(1).clamp_min(1) if average else 1)
    check_grad(grad, logits, labels, slope, shift)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("loss,smooth", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("average", [True, False])
def test_preference_loss(gpu, dtype, loss, smooth, average):
    beta, pairs = 0.25, 3
    logits, labels, reference = inputs(2 * pairs, 13, 1003, dtype, gpu, 7)
    logits.requires_grad_()
    out = triton_preference_loss(logits, labels, reference, beta=beta, label_smoothing=smooth, loss=loss, average=average)
    token, keep, _, _ = token_log_probs(logits, labels, True)
    n = keep.sum(1).clamp_min(1) if average else torch.ones(2 * pairs, device=gpu)
    y = token.sum(1) / n
    check_log_probs(out.log_probs, logits, labels, average=average)
    rewards = beta * (y - reference.double())
    off = beta * (12 * REL + 2.0**-23 * 12 * 25)  # of a sequence's log-probability, 12 tokens of at most 25
    assert (torch.cat((out.chosen_rewards, out.rejected_rewards)).double() - rewards).abs().max() <= off + 2.0**-23 * rewards.abs().max()
    want = preference_loss_with_pytorch(logits.detach().double(), labels, reference.double(), beta=beta, label_smoothing=smooth,
                                        loss=loss, average=average)
    # |dL/dh| is at most 1 (sigmoid, hinge) or 2 |h/beta - 1/(2 beta)| / beta
    h = (rewards[:pairs] - rewards[pairs:]).abs().max()
    steep = 1.0 if loss != "ipo" else 2 * (h / beta + 0.5 / beta) / beta
    assert abs(float(out.loss.detach()) - float(want.loss)) <= 2 * off * steep + 2.0**-21 * abs(float(want.loss)) + 2.0**-22
    scale = 1024.0 if dtype == torch.float16 else 1.0
    (grad,) = torch.autograd.grad(out.loss * scale, logits)
    slope = slope_of(rewards, beta, loss, smooth) / n
    # ln of each slope moves by at most |dh| (sigmoid); ipo's by its own relative change
    rel = 2 * off * (1.5 if loss != "ipo" else 1 / (beta * float(slope[:pairs].abs().min() * n.min()) * pairs / 2)) + 2.0**-20
    check_grad(grad, logits, labels, slope * scale, slope_rel=rel)


def test_gradient_by_differences(gpu):
    logits, labels, reference = inputs(4, 6, 33, torch.float32, gpu, 9)
    logits.requires_grad_()
    loss = lambda x: triton_preference_loss(x, labels, reference, beta=0.3, label_smoothing=0.1).loss  # noqa: E731
    (grad,) = torch.autograd.grad(loss(logits), logits)
    v = torch.randn_like(logits)
    v /= v.norm()
    with torch.no_grad():
        slope = (loss(logits + 0.05 * v) - loss(logits - 0.05 * v)).double() / 0.1
    # third derivatives are below 1 along a unit direction (0.05^2 / 6), the loss is right to 1e-6 (by 0.1)
    assert abs(float(slope) - float((grad.double() * v.double()).sum())) < 5e-4 + 2e-5


@pytest.mark.parametrize("h", [0.0, 50.0, -50.0, 1e4, -1e4, float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("loss,smooth", [("sigmoid", 0.0), ("sigmoid", 0.1), ("sigmoid", 1.0), ("hinge", 0.0), ("ipo", 0.0)])
def test_margins_of_any_size(gpu, h, loss, smooth):
    """A reference that makes the margin what it is, on one-entry vocabularies (log-probability 0)."""

    logits = torch.zeros(2, 3, 1, device=gpu, requires_grad=True)
    labels = torch.zeros(2, 3, dtype=torch.int64, device=gpu)
    reference = torch.tensor([-h, 0.0], device=gpu)
    options = dict(beta=1.0, label_smoothing=smooth, loss=loss)
    out = triton_preference_loss(logits, labels, reference, **options)
    want = preference_loss_with_pytorch(logits.detach().double(), labels, reference.double(), **options)
    torch.testing.assert_close(out.loss.detach().double(), want.loss, rtol=2.0**-20, atol=2.0**-22, equal_nan=True)
    (grad,) = torch.autograd.grad(out.loss, logits)
    if abs(h) < 1e30:
        assert not grad.any()  # softmax of one entry is 1


def test_masked_vocabulary_and_special_rows(gpu):
    logits, labels, _ = inputs(4, 5, 300, torch.float32, gpu, 11)
    labels[:] = torch.randint(0, 100, (4, 5), device=gpu)
    lowest = torch.finfo(torch.float32).min
    logits[0, :, 100:] = -float("inf")      # a masked vocabulary
    logits[1, :, 100:] = lowest             # one masked by the type's lowest value
    logits[2, 1] = -float("inf")            # a row with nothing
    logits[3, 2, 7] = float("nan")
    logits.requires_grad_()
    out = triton_sequence_log_probs(logits, labels)
    check_log_probs(out.detach()[:2], logits[:2], labels[:2])
    assert out[2].isnan() and out[3].isnan()
    (grad,) = torch.autograd.grad(out, logits, torch.ones(4, device=gpu))
    check_grad(grad[:2], logits[:2], labels[:2], torch.ones(2, dtype=torch.float64, device=gpu))
    assert not grad[:2, :, 100:].any()
    assert grad[2, 1].isnan().all() and grad[2, 0].isfinite().all() and grad[3, 2].isnan().all() and grad[3, 3].isfinite().all()
    # special values where no label asks for them are never read
    labels[2, 2] = labels[3, 3] = -100
    out = triton_sequence_log_probs(logits, labels)
    check_log_probs(out.detach()[:2], logits[:2], labels[:2])
    (grad,) = torch.autograd.grad(out, logits, torch.ones(4, device=gpu))
    assert out.isfinite().all() and grad.isfinite().all() and not grad[2, 1].any() and not grad[3, 2].any()


def test_a_label_at_minus_infinity(gpu):
    logits = torch.zeros(2, 2, 8, device=gpu)
    logits[0, 0, 3] = -float("inf")
    labels = torch.full((2, 2), 3, device=gpu)
    assert triton_sequence_log_probs(logits, labels)[0] == -float("inf")
    out = triton_preference_loss(logits.requires_grad_(), labels)
    assert out.loss.isinf() and out.chosen_rewards[0] == -float("inf")
    (grad,) = torch.autograd.grad(out.loss, logits)
    # the loss rises with slope beta: d/dy = -beta, softmax 1/7 on the others
    torch.testing.assert_close(grad[0, 0, :3], torch.full((3,), 0.1 / 7, device=gpu), rtol=1e-5, atol=0)


@pytest.mark.parametrize("label", [-1, 8, 2**40, -(2**40)])
def test_labels_outside_the_vocabulary_give_nan(gpu, label):
    logits = torch.randn(2, 3, 8, device=gpu, requires_grad=True)
    labels = torch.ones(2, 3, dtype=torch.int64, device=gpu)
    labels[0, 2] = label
    out = triton_sequence_log_probs(logits, labels)
    assert out[0].isnan() and out[1].isfinite()
    (grad,) = torch.autograd.grad(out, logits, torch.ones(2, device=gpu))
    assert grad[1].isfinite().all()
    assert triton_preference_loss(logits, labels).loss.isnan()


def test_another_ignored_label(gpu):
    logits, labels, _ = inputs(2, 9, 50, torch.float32, gpu, 13)
    other = labels.masked_fill(labels == -100, 7)
    assert torch.equal(triton_sequence_log_probs(logits, labels.masked_fill(labels == 7, -100)),
                       triton_sequence_log_probs(logits, other, ignore_index=7))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(gpu, dtype):
    """Rows with gaps, off every alignment, in another order, read twice, and labels of a larger tensor."""

    vocab = 4099
    base, labels, _ = inputs(3, 8, vocab, dtype, gpu, 17)
    forms = {
        "gaps": torch.zeros(3, 8, vocab + 5, dtype=dtype, device=gpu)[..., 3:3 + vocab],
        "time first": torch.zeros(8, 3, vocab, dtype=dtype, device=gpu).transpose(0, 1),
        "every second": torch.zeros(3, 16, vocab, dtype=dtype, device=gpu)[:, ::2],
    }
    for name, x in forms.items():
        x.copy_(base)
        x = x.detach().requires_grad_()
        wide = torch.full((3, 20), 5, dtype=torch.int64, device=gpu)
        wide[:, 1:17:2] = labels
        out = triton_sequence_log_probs(x, wide[:, 1:17:2])
        check_log_probs(out.detach(), base, labels)
        (grad,) = torch.autograd.grad(out, x, torch.ones(3, device=gpu))
        check_grad(grad, base, labels, torch.ones(3, dtype=torch.float64, device=gpu)), name
    one = base[:1].detach().requires_grad_()
    out = triton_sequence_log_probs(one.expand(3, -1, -1), labels)
    (grad,) = torch.autograd.grad(out, one, torch.ones(3, device=gpu))
    parts = []
    for b in range(3):
        y = triton_sequence_log_probs(one, labels[b:b + 1])
        parts.append(torch.autograd.grad(y, one, torch.ones(1, device=gpu))[0].double())
    # three rounded gradients added, in an order of torch's: two more roundings of the sums
    total = sum(parts)
    assert ((grad.double() - total).abs() <= 3 * torch.finfo(dtype).eps * sum(p.abs() for p in parts) + 1e-30).all()


def test_empty_batches(gpu):
    empty = torch.zeros(0, 3, 8, device=gpu, requires_grad=True)
    out = triton_sequence_log_probs(empty, torch.zeros(0, 3, dtype=torch.int64, device=gpu))
    assert out.shape == (0,) and torch.autograd.grad(out.sum(), empty)[0].shape == empty.shape
    none = torch.zeros(2, 0, 8, device=gpu, requires_grad=True)
    out = triton_sequence_log_probs(none, torch.zeros(2, 0, dtype=torch.int64, device=gpu))
    assert not out.any() and torch.autograd.grad(out.sum(), none)[0].shape == none.shape
    ignored = torch.randn(2, 3, 8, device=gpu, requires_grad=True)
    out = triton_preference_loss(ignored, torch.full((2, 3), -100, device=gpu), beta=0.5)
    torch.testing.assert_close(float(out.loss.detach()), 0.6931471805599453, rtol=1e-6, atol=0)
    assert not torch.autograd.grad(out.loss, ignored)[0].any()


def test_graph_of_autograd(gpu):
    logits, labels, reference = inputs(4, 7, 130, torch.float32, gpu, 19)
    logits.requires_grad_()
    out = triton_preference_loss(logits, labels, reference)
    first = torch.autograd.grad(out.loss, logits, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(out.loss, logits)[0], first)  # a second backward reads the same logits
    out = triton_preference_loss(logits, labels, reference)
    with torch.no_grad():
        logits += 1.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.loss.backward()
    with torch.no_grad():
        assert not triton_preference_loss(logits, labels, reference).loss.requires_grad
    # a loss divided in place, as gradient accumulation does
    loss = triton_preference_loss(logits, labels, reference).loss
    loss /= 4
    torch.testing.assert_close(torch.autograd.grad(loss, logits)[0], torch.autograd.grad(triton_preference_loss(logits, labels, reference).loss, logits)[0] / 4,
                               rtol=2.0**-22, atol=0)


def test_results_do_not_depend_on_the_run(gpu):
    logits, labels, reference = inputs(8, 300, 5003, torch.bfloat16, gpu, 23)
    logits.requires_grad_()
    runs = []
    for _ in range(3):
        out = triton_preference_loss(logits, labels, reference)
        runs.append([*(t.detach() for t in out), torch.autograd.grad(out.loss, logits)[0]])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_another_stream_and_replays(gpu):
    logits, labels, reference = inputs(4, 9, 1000, torch.bfloat16, gpu, 29)
    static, ids, ref = logits.clone().requires_grad_(), labels.clone(), reference.clone()

    def call():
        out = triton_preference_loss(static, ids, ref)
        return out.loss, torch.autograd.grad(out.loss, static)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        loss, grad = (t.detach().clone() for t in call())
    torch.cuda.current_stream().wait_stream(stream)
    want = call()
    assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])
    del want  # no eager graph of the same leaf lives through the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        loss, grad = call()
    for step in range(4):
        x, y, r = inputs(4, 9, 1000, torch.bfloat16, gpu, 31 + step)
        with torch.no_grad():
            static.copy_(x)
        ids.copy_(y)
        ref.copy_(r)
        graph.replay()
        torch.cuda.synchronize()
        out = triton_preference_loss(x.requires_grad_(), y, r)
        assert torch.equal(loss.detach(), out.loss.detach()) and torch.equal(grad, torch.autograd.grad(out.loss, x)[0]), step


def test_offsets_beyond_32_bits(gpu):
    """Logits of more than 2^31 elements: the last sequences' rows lie behind them."""

    batch, seq, vocab = 4, 4200, 128256  # 2.15e9 elements, 4.3 GB
    logits = torch.zeros(batch, seq, vocab, dtype=torch.bfloat16, device=gpu)
    labels = torch.full((batch, seq), -100, dtype=torch.int64, device=gpu)
    tail = randn((5, vocab), torch.bfloat16, gpu, 41, 2.0)
    logits[3, -6:-1] = tail
    labels[3, -5:] = torch.randint(0, vocab, (5,), device=gpu)
    logits.requires_grad_()
    out = triton_sequence_log_probs(logits, labels)
    check_log_probs(out.detach()[3:], logits[3:, -6:], labels[3:, -6:])
    (grad,) = torch.autograd.grad(out, logits, torch.ones(4, device=gpu))
    check_grad(grad[3:, -6:], logits[3:, -6:], labels[3:, -6:], torch.ones(1, dtype=torch.float64, device=gpu))
    assert not grad[:3].any() and not grad[3, :-6].any()


@pytest.mark.parametrize("case", ["dtype", "rank", "labels", "label type", "class stride", "devices", "reference device"])
def test_refusals(gpu, case):
    logits, labels, reference = torch.randn(2, 3, 8, device=gpu), torch.zeros(2, 3, dtype=torch.int64, device=gpu), torch.zeros(2, device=gpu)
    if case == "dtype":
        logits = logits.double()
    elif case == "rank":
        logits = logits[None]
    elif case == "labels":
        labels = labels[:, :2]
    elif case == "label type":
        labels = labels.int()
    elif case == "class stride":
        logits = torch.randn(2, 8, 3, device=gpu).transpose(1, 2)
    elif case == "devices":
        labels = labels.cpu()
    else:
        reference = reference.cpu()
    with pytest.raises((TritonPreferenceUnavailable, ValueError)):
        triton_preference_loss(logits, labels, reference)
    if case != "reference device":
        with pytest.raises(TritonPreferenceUnavailable):
            triton_sequence_log_probs(logits, labels)


def test_workspace_of_another_call_is_refused(gpu):
    logits, labels, _ = inputs(2, 5, 9, torch.float32, gpu, 1)
    _, ws = ops.sequence_log_probs(logits[:, :1].contiguous(), labels[:, :1].contiguous())
    with pytest.raises(ValueError, match="workspace"):
        ops.sequence_log_probs_bwd(logits.repeat(1, 9, 1), labels.repeat(1, 9), ws, grad_log_probs=torch.ones(2, device=gpu))


def test_one_step_of_preference_tuning(gpu):
    """The three together as a trainer uses them: a decoder-like layer rotates at packed positions, its logits give the loss
    against a reference model, and the 8-bit optimizer steps."""

    torch.manual_seed(5)
    vocab, dim, heads = 301, 64, 4
    rope = RotaryEmbedding(dim // heads, 1e4, use_triton_rope=True, layout="rotate_half", rotary_dim=8,
                           scaling=dict(type="linear", factor=2.0))
    embed = torch.nn.Parameter(torch.randn(vocab, dim, device=gpu) * 0.1)
    mix = torch.nn.Parameter(torch.randn(dim, dim, device=gpu) * 0.1)
    ids = torch.randint(0, vocab, (4, 12), device=gpu)
    labels = ids.masked_fill(torch.arange(12, device=gpu) < 4, -100)
    positions = torch.cat((torch.arange(5), torch.arange(7))).to(gpu).repeat(4, 1)

    def logits(rotate):
        h = embed[ids] @ mix
        q = h.view(4, 12, heads, dim // heads).transpose(1, 2)
        q, k = rotate(q, q, positions)
        mixed = (q + k.cumsum(2) * 0.1).transpose(1, 2).reshape(4, 12, dim)
        return mixed @ embed.t()

    loss = PreferenceLossWithFallback(use_triton=True, beta=0.5, label_smoothing=0.05)
    with torch.no_grad():
        reference = loss.log_probs(logits(rope), labels) + torch.tensor([0.3, -0.2, 0.1, 0.4], device=gpu)
    out = loss(logits(rope), labels, reference)
    out.loss.backward()
    grads = [embed.grad.clone(), mix.grad.clone()]
    embed.grad = mix.grad = None
    plain = PreferenceLossWithFallback(beta=0.5, label_smoothing=0.05)
    slow = RotaryEmbedding(dim // heads, 1e4, layout="rotate_half", rotary_dim=8, scaling=dict(type="linear", factor=2.0))
    want = plain(logits(slow), labels, reference)
    want.loss.backward()
    torch.testing.assert_close(out.loss, want.loss, rtol=1e-5, atol=1e-6)
    for g, p in zip(grads, (embed, mix)):  # sums of a few hundred fp32 products in another order
        assert (g - p.grad).norm() <= 1e-5 * p.grad.norm()
    optimizer = AdamW8bit([embed, mix], lr=1e-2)
    before = [embed.detach().clone(), mix.detach().clone()]
    triton_adamw_step(optimizer)
    for p, b in zip((embed, mix), before):
        assert p.isfinite().all() and (p != b).any()
    assert not loss._fallback_warned and not rope._triton_fallback_warned


@pytest.mark.parametrize("use", ["loss", "log_probs"])
def test_under_the_compiler(gpu, use):
    logits, labels, reference = inputs(4, 9, 300, torch.bfloat16, gpu, 5)
    logits.requires_grad_()

    def step(x):
        if use == "loss":
            return triton_preference_loss(x * 2, labels, reference, beta=0.2).loss * 3
        return (triton_sequence_log_probs(x * 2, labels) * reference).sum()

    want = step(logits)
    (grad,) = torch.autograd.grad(want, logits)
    got = torch.compile(step, backend="aot_eager")(logits)
    (compiled,) = torch.autograd.grad(got, logits)
    assert torch.equal(got, want) and torch.equal(compiled, grad)
    with torch.no_grad():
        assert torch.equal(torch.compile(step, backend="aot_eager")(logits), want)


@pytest.mark.parametrize("batch,seq", [(16384, 1), (5462, 3), (2048, 8), (1022, 16)])
def test_many_short_sequences(gpu, batch, seq):
    logits, labels, reference = inputs(batch, seq, 40, torch.float32, gpu, 7)
    out = triton_preference_loss(logits, labels, reference, beta=0.5, shift=False)
    check_log_probs(out.log_probs, logits, labels, shift=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vecs", [257, 511, 513, 767, 1023, 1024, 1025])
@pytest.mark.parametrize("rows", [1023, 1024])
def test_rows_a_wave_or_a_workgroup_takes(gpu, dtype, vecs, rows):
    per = 128 // torch.finfo(dtype).bits
    logits, labels, _ = inputs(1, rows, vecs * per - 3, dtype, gpu, 11)
    got = triton_sequence_log_probs(logits, labels, shift=False)
    check_log_probs(got, logits, labels, shift=False)


@pytest.mark.parametrize("vocab,dtype", [(33_000, torch.bfloat16), (50257, torch.float16), (128256, torch.bfloat16), (70_001, torch.float32)])
@pytest.mark.parametrize("rows", [64, 65, 128, 129])
def test_parts_of_rows(gpu, vocab, dtype, rows):
    logits, labels, _ = inputs(1, rows, vocab, dtype, gpu, 12)
    logits.requires_grad_()
    out = triton_sequence_log_probs(logits, labels)
    check_log_probs(out.detach(), logits.detach(), labels)
    (grad,) = torch.autograd.grad(out, logits, torch.full((1,), -1.5, device=gpu))
    check_grad(grad, logits.detach(), labels, torch.full((1,), -1.5, dtype=torch.float64, device=gpu))


# What follows the rows, by route: one launch for few tokens (one wave a sequence, several waves a sequence); sums and loss in
# launches of their own (many sequences, more than 256 pairs; few long sequences of more than 16384 tokens); rows in parts joined in
# the one launch (up to 64 rows) and in one of their own (up to 128).
ROUTES = [
    *[(6, 13, 1003, torch.float32), (4, 600, 130, torch.float32), (2, 1025, 65, torch.float16), (4, 3000, 130, torch.bfloat16)],
    *[(16384, 1, 40, torch.float32), (5462, 3, 40, torch.float32), (1022, 16, 77, torch.bfloat16), (514, 40, 260, torch.float16)],
    *[(2, 9000, 65, torch.float32), (4, 8200, 33, torch.bfloat16)],
    *[(2, 32, 33_000, torch.bfloat16), (4, 16, 70_001, torch.float32), (2, 31, 128256, torch.float16)],
    *[(2, 33, 128256, torch.bfloat16), (4, 32, 200_001, torch.float32), (2, 64, 128257, torch.float16), (6, 30, 128256, torch.bfloat16)],
]


@pytest.mark.parametrize("batch,seq,vocab,dtype", ROUTES)
@pytest.mark.parametrize("loss,average", [("sigmoid", False), ("sigmoid", True), ("ipo", True), ("hinge", False)])
def test_losses_on_every_route(gpu, batch, seq, vocab, dtype, loss, average):
    """Each step against the one before it: log-probabilities against 64 bits, rewards against them, and loss, slopes and gradient
    against the rewards."""

    beta, pairs, shift = 0.25, batch // 2, seq > 1
    logits, labels, reference = inputs(batch, seq, vocab, dtype, gpu, batch + seq)
    token, keep, _, _ = token_log_probs(logits, labels, shift)
    n = keep.sum(1).clamp_min(1).double() if average else torch.ones(batch, dtype=torch.float64, device=gpu)
    reference = (token.sum(1) / n + reference.double()).float()  # margins of a few, however long the sequences
    logits.requires_grad_()
    out = triton_preference_loss(logits, labels, reference, beta=beta, loss=loss, average=average, shift=shift)
    check_log_probs(out.log_probs, logits, labels, shift, average)
    rewards = torch.cat((out.chosen_rewards, out.rejected_rewards)).double()
    # the log-probability's one rounding, the reward's own
    off = beta * 2.0**-24 * out.log_probs.double().abs() + 2.0**-24 * rewards.abs()
    assert ((rewards - beta * (out.log_probs.double() - reference.double())).abs() <= off * (1 + 2.0**-20) + 1e-30).all()
    c, r = rewards.chunk(2)
    h = c - r
    dh = 2.0**-23 * (c.abs() + r.abs())  # one rounding of each reward, and h's
    u = h / beta - 0.5 / beta
    each = {"sigmoid": -torch.nn.functional.logsigmoid(h), "hinge": torch.relu(1 - h), "ipo": u.square()}[loss]
    # a few roundings of an fp32 function (2^-21), the margin's error by a slope of 1, or of 2 u / beta
    du = dh / beta + 2.0**-22 * (h.abs() + 0.5) / beta
    error = dh + 2.0**-21 * each if loss != "ipo" else 2 * u.abs() * du + du.square() + 2.0**-21 * each
    assert abs(float(out.loss.detach()) - float(each.mean())) <= float(error.mean()) + 2.0**-23 * float(each.mean()) + 1e-30
    (grad,) = torch.autograd.grad(out.loss, logits)
    # sigmoid: ln of the slope moves by the margin's error; ipo's by that of u; hinge's not at all (no margin lies that near 1)
    rel = {"sigmoid": dh, "hinge": torch.zeros_like(h), "ipo": du / u.abs()}[loss] + 2.0**-20
    assert loss != "hinge" or ((h - 1).abs() > dh).all()
    slope = slope_of(rewards, beta, loss, 0.0) / n
    rel = rel.repeat(2)
    for at in range(0, batch, max(1, 8_000_000 // (seq * vocab))):
        part = slice(at, at + max(1, 8_000_000 // (seq * vocab)))
        check_grad(grad[part], logits.detach()[part], labels[part], slope[part], shift, slope_rel=rel[part][:, None, None])


@pytest.mark.parametrize("dtype,batch,seq,vocab", [(torch.bfloat16, 7, 1201, 65_537), (torch.float32, 3, 700, 128_256),
                                                   (torch.float16, 2, 11_003, 25_000)])
def test_every_row_of_a_large_gradient(gpu, dtype, batch, seq, vocab):
    """1 GB and more, whose rows are dealt to the XCDs in ranges: every element is written, the items behind the last
    whole range among them, into a buffer of NaN."""

    logits, labels, _ = inputs(batch, seq, vocab, dtype, gpu, 43)
    assert logits.nbytes >= 1 << 30
    up = torch.linspace(0.5, 2.0, batch, device=gpu)
    _, ws = ops.sequence_log_probs(logits, labels)
    grad = torch.full_like(logits, float("nan"))
    _lib.raw_call("pt_sequence_log_probs_bwd", logits.data_ptr(), batch, *ops._sequence_rows(logits, labels, True), -100,
                  up.data_ptr(), None, grad.data_ptr(), grad.stride(0), grad.stride(1), ws.data_ptr(), ws.numel(),
                  ops.dtype_code(dtype), ops._stream(logits.device))
    assert torch.equal(grad, ops.sequence_log_probs_bwd(logits, labels, ws, grad_log_probs=up))
    for b in range(batch):
        # 64 bits of a few hundred rows at a time; a slice's last label is the next one's first
        for at in range(0, seq - 1, 500):
            rows = slice(at, min(at + 501, seq))
            g = grad[b:b + 1, rows].clone()
            x, y = logits[b:b + 1, rows], labels[b:b + 1, rows]
            if rows.stop < seq:
                g[:, -1] = 0.0  # has its label in the next slice
            check_grad(g, x, y, up[b:b + 1].double())
    assert not grad[:, -1].any()
