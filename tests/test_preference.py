"""Preference loss and sequence log-probabilities on the CPU: the PyTorch forms against the definition in 64 bits and
against differences, the fallback, and refusals."""

from __future__ import annotations

import math
import warnings

import pytest
import torch

from picotron_amd import _lib, ops
from picotron_amd.nn.triton_kernels import (
    PreferenceLossWithFallback,
    TritonPreferenceUnavailable,
    preference_loss_with_pytorch,
    sequence_log_probs_with_pytorch,
    triton_preference_loss,
    triton_sequence_log_probs,
)


def inputs(batch=4, seq=6, vocab=11, dtype=torch.float64):
    torch.manual_seed(0)
    logits = torch.randn(batch, seq, vocab, dtype=dtype) * 2
    labels = torch.randint(0, vocab, (batch, seq))
    labels[:, :2] = -100
    labels[1, 4:] = -100
    labels[3] = -100  # nothing kept
    return logits, labels, torch.randn(batch, dtype=dtype)


@pytest.mark.parametrize("shift", [True, False])
@pytest.mark.parametrize("average", [True, False])
def test_log_probs_by_hand(shift, average):
    logits, labels, _ = inputs()
    got = sequence_log_probs_with_pytorch(logits, labels, shift=shift, average=average)
    for b in range(4):
        terms = []
        for t in range(6 - shift):
            y = int(labels[b, t + shift])
            if y != -100:
                row = logits[b, t].tolist()
                terms.append(row[y] - math.log(sum(math.exp(x) for x in row)))
        want = sum(terms) / (len(terms) if average and terms else 1)
        assert math.isclose(float(got[b]), want, rel_tol=1e-12, abs_tol=1e-12)


@pytest.mark.parametrize("loss,smooth", [("sigmoid", 0.0), ("sigmoid", 0.1), ("sigmoid", 1.0), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("with_reference", [True, False])
def test_loss_by_hand_and_by_differences(loss, smooth, with_reference):
    logits, labels, reference = inputs()
    reference = reference if with_reference else None
    beta = 0.3
    options = dict(beta=beta, label_smoothing=smooth, loss=loss)
    y = sequence_log_probs_with_pytorch(logits, labels)
    r = torch.zeros(4) if reference is None else reference
    out = preference_loss_with_pytorch(logits.requires_grad_(), labels, reference, **options)
    total = 0.0
    for i in range(2):
        h = beta * float((y[i] - r[i]) - (y[i + 2] - r[i + 2]))
        s = 1 / (1 + math.exp(-h))
        total += {"sigmoid": -(1 - smooth) * math.log(s) - smooth * math.log(1 - s), "hinge": max(0.0, 1 - h),
                  "ipo": (h / beta - 1 / (2 * beta)) ** 2}[loss]
    assert math.isclose(float(out.loss.detach()), total / 2, rel_tol=1e-6)
    torch.testing.assert_close(out.chosen_rewards, beta * (y - r)[:2])
    torch.testing.assert_close(out.rejected_rewards, beta * (y - r)[2:])
    torch.testing.assert_close(out.log_probs, y)
    assert not out.chosen_rewards.requires_grad and not out.log_probs.requires_grad
    assert torch.autograd.gradcheck(lambda x: preference_loss_with_pytorch(x, labels, reference, **options).loss, (logits,))


def test_stepper_warns_once_and_falls_back():
    logits, labels, reference = inputs(dtype=torch.float32)
    fused = PreferenceLossWithFallback(use_triton=True, beta=0.2, label_smoothing=0.1)
    with pytest.warns(RuntimeWarning, match="Triton preference loss unavailable"):
        out = fused(logits, labels, reference)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        log_probs = fused.log_probs(logits, labels)
        off = PreferenceLossWithFallback()(logits, labels, reference)
    want = preference_loss_with_pytorch(logits, labels, reference, beta=0.2, label_smoothing=0.1)
    assert torch.equal(out.loss, want.loss) and torch.equal(log_probs, want.log_probs)
    assert torch.equal(off.loss, preference_loss_with_pytorch(logits, labels, reference).loss)


@pytest.mark.parametrize("options", [dict(loss="other"), dict(beta=0.0), dict(beta=-1.0), dict(beta=float("inf")), dict(label_smoothing=-0.1),
                                     dict(label_smoothing=1.5), dict(loss="hinge", label_smoothing=0.1)])
def test_options_are_refused(options):
    logits, labels, reference = inputs()
    for fn in (triton_preference_loss, preference_loss_with_pytorch):
        with pytest.raises(ValueError):
            fn(logits, labels, reference, **options)
    with pytest.raises(ValueError):
        PreferenceLossWithFallback(**options)


def test_pairs_and_references_are_refused():
    logits, labels, reference = inputs()
    for fn in (triton_preference_loss, preference_loss_with_pytorch):
        for bad in ((logits[:3], labels[:3], reference[:3]), (logits[:0], labels[:0], None), (logits[0], labels[0], None),
                    (logits, labels, reference[:2]), (logits, labels, labels[:, 0]), (logits, labels, reference.clone().requires_grad_())):
            with pytest.raises(ValueError):
                fn(*bad)


def test_fast_paths_refuse_the_cpu():
    logits, labels, reference = inputs(dtype=torch.float32)
    with pytest.raises(TritonPreferenceUnavailable):
        triton_sequence_log_probs(logits, labels)
    with pytest.raises(TritonPreferenceUnavailable):
        triton_preference_loss(logits, labels, reference)


@pytest.mark.parametrize("logits,labels", [
    (torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int64)), (torch.zeros(2, 3, 0), torch.zeros(2, 3, dtype=torch.int64)),
    (torch.zeros(2, 5, 3).transpose(1, 2), torch.zeros(2, 3, dtype=torch.int64)), (torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int32)),
    (torch.zeros(2, 3, 5), torch.zeros(2, 2, dtype=torch.int64)),
])
def test_shapes_are_refused(logits, labels):
    with pytest.raises(ValueError):
        ops._sequence_rows(logits, labels, True)


def _logp(**change):
    a = dict(logits=4096, batch=2, seq=3, bs=24, ss=8, vocab=8, labels=4096, lbs=3, lss=1, shift=1, ignore=-100, average=0, out=4096,
             ws=4096, size=1 << 20, dtype=0, stream=None)
    return "pt_sequence_log_probs", {**a, **change}


def _loss(**change):
    a = dict(logits=4096, pairs=1, seq=3, bs=24, ss=8, vocab=8, labels=4096, lbs=3, lss=1, shift=1, ignore=-100, average=0, reference=None,
             beta=0.1, smooth=0.0, kind=0, loss=4096, rewards=4096, log_probs=4096, ws=4096, size=1 << 20, dtype=0, stream=None)
    return "pt_preference_loss", {**a, **change}


def _bwd(**change):
    a = dict(logits=4096, batch=2, seq=3, bs=24, ss=8, vocab=8, labels=4096, lbs=3, lss=1, shift=1, ignore=-100, grad_log_probs=4096,
             grad_loss=None, grad=8192, gbs=24, gss=8, ws=4096, size=1 << 20, dtype=0, stream=None)
    return "pt_sequence_log_probs_bwd", {**a, **change}


# Addresses that are never read: the checks come before any launch.
@pytest.mark.parametrize("call,code", [
    *[(make(**change), _lib.PT_EINVAL) for make in (_logp, _loss, _bwd) for change in (
        dict(dtype=5), dict(seq=-1), dict(vocab=0), dict(shift=2), dict(logits=None), dict(labels=None), dict(ws=None), dict(ws=4100), dict(size=16))],
    *[(make(**change), _lib.PT_EUNSUPPORTED) for make in (_logp, _loss, _bwd) for change in (
        dict(vocab=1 << 29), dict(seq=1 << 24), dict(seq=1 << 40))],
    (_logp(batch=-1), _lib.PT_EINVAL), (_logp(out=None), _lib.PT_EINVAL), (_logp(batch=1 << 22), _lib.PT_EUNSUPPORTED),
    (_loss(pairs=0), _lib.PT_EINVAL), (_loss(pairs=1 << 40), _lib.PT_EINVAL), (_loss(kind=3), _lib.PT_EINVAL), (_loss(beta=0.0), _lib.PT_EINVAL),
    (_loss(beta=float("nan")), _lib.PT_EINVAL), (_loss(smooth=1.5), _lib.PT_EINVAL), (_loss(loss=None), _lib.PT_EINVAL),
    (_loss(rewards=None), _lib.PT_EINVAL), (_loss(log_probs=None), _lib.PT_EINVAL),
    (_bwd(grad=None), _lib.PT_EINVAL), (_bwd(grad=4096), _lib.PT_EINVAL), (_bwd(grad=8196), _lib.PT_EINVAL), (_bwd(gss=9), _lib.PT_EINVAL),
    (_bwd(gbs=25), _lib.PT_EINVAL), (_bwd(grad_loss=4096), _lib.PT_EINVAL), (_bwd(grad_log_probs=None), _lib.PT_EINVAL),
])
def test_entry_points_refuse(call, code):
    fn, arguments = call
    assert getattr(_lib.lib(), fn)(*arguments.values()) == code
    assert _lib.lib().pt_last_error().decode().startswith(fn + ":")


def test_nothing_to_do():
    for make in (_logp, _bwd):
        fn, arguments = make(batch=0, logits=None, labels=None, ws=None)
        assert getattr(_lib.lib(), fn)(*arguments.values()) == _lib.PT_OK
    assert _lib.lib().pt_sequence_log_probs_workspace_bytes(-1, 3, 8, 0) == 0
    assert _lib.lib().pt_sequence_log_probs_workspace_bytes(2, 1 << 40, 8, 0) == 0


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_left_out_rows_may_hold_anything(value):
    logits, labels, reference = inputs()
    want = preference_loss_with_pytorch(logits.requires_grad_(), labels, reference)
    (grad,) = torch.autograd.grad(want.loss, logits)
    other = logits.detach().clone()
    keep = torch.zeros(4, 6, dtype=torch.bool)
    keep[:, :-1] = labels[:, 1:] != -100
    other[~keep] = value
    out = preference_loss_with_pytorch(other.requires_grad_(), labels, reference)
    assert torch.equal(out.loss, want.loss) and torch.equal(torch.autograd.grad(out.loss, other)[0], grad)
    assert not grad[~keep].any()


@pytest.mark.parametrize("label", [-1, 11, 2**40, -(2**40)])
def test_labels_outside_the_vocabulary_give_nan(label):
    logits, labels, reference = inputs()
    want = sequence_log_probs_with_pytorch(logits, labels)
    labels[0, 3] = label
    got = sequence_log_probs_with_pytorch(logits.requires_grad_(), labels)
    assert got[0].isnan() and torch.equal(got[1:], want[1:])
    (grad,) = torch.autograd.grad(got.sum(), logits)
    assert grad[1:].isfinite().all()
    assert preference_loss_with_pytorch(logits, labels, reference).loss.isnan()
    # the label that leaves positions out may be one of the vocabulary, or far from it
    for ignored in (3, 2**40):
        other = labels.clamp(0, 10)
        assert torch.equal(sequence_log_probs_with_pytorch(logits, other.masked_fill(other == 3, ignored), ignore_index=ignored),
                           sequence_log_probs_with_pytorch(logits, other.masked_fill(other == 3, -100)))


@pytest.mark.parametrize("vocab", [1 << 31, 1 << 33, 1 << 61, 1 << 62, (1 << 63) - 1])
@pytest.mark.parametrize("dtype", [0, 1])
def test_vocabularies_beyond_any_row_are_refused(vocab, dtype):
    """Also where their bytes pass 64 bits."""

    for make in (_logp, _loss, _bwd):
        fn, arguments = make(vocab=vocab, dtype=dtype)
        assert getattr(_lib.lib(), fn)(*arguments.values()) == _lib.PT_EUNSUPPORTED
    assert _lib.lib().pt_sequence_log_probs_workspace_bytes(2, 3, vocab, dtype) == 0
