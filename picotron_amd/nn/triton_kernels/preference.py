"""Preference loss on a model's logits, forward and backward, on gfx950.

The reference's DPO trainer forms whole log-softmax tensors of the policy's and the reference model's logits
and gathers the labels' entries (src/picotron_dpo/dpo_trainer.py:297).  Here ``triton_sequence_log_probs`` reads the logits
once and returns one log-probability a sequence -- all that the reference model is asked for -- and
``triton_preference_loss`` is the loss on the policy's logits themselves: no fp32 copy of them, no softmax kept, and
a backward that reads them a second time and writes their gradient (the weight of a sequence's tokens depends on every
token of its pair, so no single pass can write it).

Logits are (batch, seq, vocab), labels (batch, seq) int64 with ``ignore_index`` at the prompt and the padding.  With ``shift``
(the default) the logits of position t are scored against label t + 1; without it against label t.  The logits are left
alone and only read; the gradient is a new tensor of their layout, computed in fp32 and rounded once, with what arrives from
above (an fp16 loss scale) applied before the rounding.  A label outside the vocabulary gives NaN.
"""

from __future__ import annotations

import math
import warnings
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from picotron_amd import ops
from picotron_amd.nn.triton_kernels._gate import no_graph, require_hip

IGNORE_INDEX = -100


class TritonPreferenceUnavailable(RuntimeError):
    """Raised when the fused (HIP) preference loss cannot safely run."""


class PreferenceLoss(NamedTuple):
    """The loss (fp32 scalar, differentiable in the logits), and for logging, without gradients: the pairs' rewards
    ``beta * (log_prob - reference)`` and every sequence's log-probability."""

    loss: Tensor
    chosen_rewards: Tensor
    rejected_rewards: Tensor
    log_probs: Tensor


class _SequenceLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, labels: Tensor, shift: bool, ignore_index: int, average: bool):  # type: ignore[override]
        out, ws = ops.sequence_log_probs(logits, labels, shift=shift, ignore_index=ignore_index, average=average)
        ctx.save_for_backward(logits, labels, ws)
        ctx.how = (shift, ignore_index)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):  # type: ignore[override]
        logits, labels, ws = ctx.saved_tensors
        shift, ignore_index = ctx.how
        d = ops.sequence_log_probs_bwd(logits, labels, ws, grad_log_probs=grad, shift=shift, ignore_index=ignore_index)
        return d, None, None, None, None


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, labels: Tensor, reference: Tensor | None, how: dict):  # type: ignore[override]
        loss, rewards, log_probs, ws = ops.preference_loss(logits, labels, reference, **how)
        ctx.save_for_backward(logits, labels, ws)
        ctx.how = how
        ctx.mark_non_differentiable(rewards, log_probs)
        ctx.set_materialize_grads(False)  # no zeros for them
        return loss, rewards, log_probs

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor | None, *_):  # type: ignore[override]
        if grad is None:
            return None, None, None, None
        logits, labels, ws = ctx.saved_tensors
        d = ops.sequence_log_probs_bwd(logits, labels, ws, grad_loss=grad, shift=ctx.how["shift"],
                                       ignore_index=ctx.how["ignore_index"])
        return d, None, None, None


def _validate(logits: Tensor, labels: Tensor, shift: bool) -> None:
    require_hip(TritonPreferenceUnavailable, "preference loss", logits, labels)
    if logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TritonPreferenceUnavailable("HIP preference loss supports float logits only.")
    if labels.device != logits.device:
        raise TritonPreferenceUnavailable("HIP preference loss needs logits and labels on one device.")
    try:
        ops._sequence_rows(logits, labels, shift)
    except ValueError as error:
        raise TritonPreferenceUnavailable(f"HIP preference loss: {error}.") from error


def _check_options(loss: str, beta: float, label_smoothing: float) -> None:
    if loss not in ops.PREFERENCE_LOSSES:
        raise ValueError(f"loss must be one of {sorted(ops.PREFERENCE_LOSSES)}.")
    if not (beta > 0 and math.isfinite(beta)):
        raise ValueError("beta must be positive.")
    if not 0 <= label_smoothing <= 1:
        raise ValueError("label_smoothing must be between 0 and 1.")
    if label_smoothing and loss != "sigmoid":
        raise ValueError("label_smoothing belongs to the sigmoid loss.")


def _check_pairs(logits: Tensor, reference: Tensor | None) -> None:
    if logits.dim() != 3 or logits.size(0) < 2 or logits.size(0) % 2 != 0:
        raise ValueError("A preference loss takes pairs: an even number of sequences, the chosen ones first.")
    if reference is not None:
        if tuple(reference.shape) != (logits.size(0),) or not reference.is_floating_point():
            raise ValueError("Reference log-probabilities must be one float a sequence.")
        if reference.requires_grad:
            raise ValueError("Reference log-probabilities must not require gradients (detach them).")


def triton_sequence_log_probs(
    logits: Tensor, labels: Tensor, *, shift: bool = True, ignore_index: int = IGNORE_INDEX, average: bool = False
) -> Tensor:
    """Each sequence's log-probability of its kept labels (their mean with ``average``), fp32 of (batch,); 0 for a
    sequence that keeps none.  Differentiable in the logits."""

    plain = no_graph(logits)
    if plain:  # what the native launcher takes needs no check here
        require_hip(TritonPreferenceUnavailable, "preference loss", logits, labels)
        out = ops._launch_here("pt_sequence_log_probs", logits, labels, bool(shift), ignore_index, bool(average))
        if out is not None:
            return out[0]
    _validate(logits, labels, shift)
    if plain:
        return ops.sequence_log_probs(logits, labels, shift=shift, ignore_index=ignore_index, average=average)[0]
    return _SequenceLogProbs.apply(logits, labels, bool(shift), int(ignore_index), bool(average))


def triton_preference_loss(
    logits: Tensor, labels: Tensor, reference_log_probs: Tensor | None = None, *, beta: float = 0.1,
    label_smoothing: float = 0.0, loss: str = "sigmoid", shift: bool = True, ignore_index: int = IGNORE_INDEX,
    average: bool = False,
) -> PreferenceLoss:
    """The mean preference loss over pairs of sequences: sequence i of the batch is the chosen one of pair i, sequence
    i + batch / 2 the rejected one.  With y the sequences' log-probabilities (:func:`triton_sequence_log_probs`),
    r the reference model's (zeros when absent) and ``h = beta * ((y_c - r_c) - (y_r - r_r))``, a pair's loss is

    - ``"sigmoid"``: ``-(1 - e) ln s(h) - e ln s(-h)``, e the ``label_smoothing`` (direct preference optimization);
    - ``"hinge"``: ``max(0, 1 - h)``;
    - ``"ipo"``: ``(h / beta - 1 / (2 beta))^2`` (usually with ``average``).
    """

    _check_options(loss, beta, label_smoothing)
    _check_pairs(logits, reference_log_probs)
    _validate(logits, labels, shift)
    reference = reference_log_probs
    if reference is not None:
        if reference.device != logits.device:
            raise TritonPreferenceUnavailable("HIP preference loss needs the reference log-probabilities on the logits' device.")
        reference = reference.float().contiguous()
    how = dict(beta=float(beta), label_smoothing=float(label_smoothing), kind=loss, shift=bool(shift),
               ignore_index=int(ignore_index), average=bool(average))
    if no_graph(logits):
        value, rewards, log_probs, _ = ops.preference_loss(logits, labels, reference, **how)
    else:
        value, rewards, log_probs = _PreferenceLoss.apply(logits, labels, reference, how)
    pairs = logits.size(0) // 2
    return PreferenceLoss(value, rewards[:pairs], rewards[pairs:], log_probs)


def sequence_log_probs_with_pytorch(
    logits: Tensor, labels: Tensor, *, shift: bool = True, ignore_index: int = IGNORE_INDEX, average: bool = False
) -> Tensor:
    """:func:`triton_sequence_log_probs` in PyTorch, NaN for a label outside the vocabulary among the rest (a gather there
    is an error, on a GPU one that ends the process)."""

    if shift:
        logits, labels = logits[:, :-1], labels[:, 1:]
    keep = labels != ignore_index
    logits = logits.masked_fill(~keep.unsqueeze(-1), 0.0)  # what is left out may be no numbers, and asks for no gradient
    logits = logits.to(torch.promote_types(logits.dtype, torch.float32))
    inside = (labels >= 0) & (labels < logits.size(-1))
    token = F.log_softmax(logits, dim=-1).gather(-1, labels.masked_fill(~(keep & inside), 0).unsqueeze(-1)).squeeze(-1)
    total = torch.where(keep, token.masked_fill(~inside, math.nan), 0.0).sum(-1)
    return total / keep.sum(-1).clamp_min(1) if average else total


def preference_loss_with_pytorch(
    logits: Tensor, labels: Tensor, reference_log_probs: Tensor | None = None, *, beta: float = 0.1,
    label_smoothing: float = 0.0, loss: str = "sigmoid", shift: bool = True, ignore_index: int = IGNORE_INDEX,
    average: bool = False,
) -> PreferenceLoss:
    """:func:`triton_preference_loss` in PyTorch."""

    _check_options(loss, beta, label_smoothing)
    _check_pairs(logits, reference_log_probs)
    log_probs = sequence_log_probs_with_pytorch(logits, labels, shift=shift, ignore_index=ignore_index, average=average)
    rewards = beta * (log_probs if reference_log_probs is None else log_probs - reference_log_probs.to(log_probs.dtype))
    chosen, rejected = rewards.chunk(2)
    h = chosen - rejected
    if loss == "sigmoid":
        # a weight of 0 keeps an infinite margin's other term out
        value = -(1 - label_smoothing) * F.logsigmoid(h) if label_smoothing < 1 else torch.zeros_like(h)
        if label_smoothing:
            value = value - label_smoothing * F.logsigmoid(-h)
    elif loss == "hinge":
        value = torch.relu(1 - h)
    else:
        value = (h / beta - 1 / (2 * beta)).square()
    return PreferenceLoss(value.mean(), chosen.detach(), rejected.detach(), log_probs.detach())


class PreferenceLossWithFallback:
    """Run the fused loss when enabled, else (or on failure) the PyTorch form, warning once."""

    def __init__(self, *, use_triton: bool = False, beta: float = 0.1, label_smoothing: float = 0.0, loss: str = "sigmoid",
                 average: bool = False) -> None:
        _check_options(loss, beta, label_smoothing)
        self.use_triton = use_triton
        self.options = dict(beta=beta, label_smoothing=label_smoothing, loss=loss, average=average)
        self._fallback_warned = False

    def _run(self, fused, plain, *args, **options):
        if self.use_triton:
            try:
                return fused(*args, **options)
            except Exception as error:
                if not self._fallback_warned:
                    warnings.warn(
                        f"Triton preference loss unavailable; using PyTorch fallback: {error}",
                        RuntimeWarning,
                        stacklevel=3,
                    )
                    self._fallback_warned = True
        return plain(*args, **options)

    def __call__(self, logits: Tensor, labels: Tensor, reference_log_probs: Tensor | None = None, *,
                 shift: bool = True) -> PreferenceLoss:
        return self._run(triton_preference_loss, preference_loss_with_pytorch, logits, labels, reference_log_probs,
                         shift=shift, **self.options)

    def log_probs(self, logits: Tensor, labels: Tensor, *, shift: bool = True) -> Tensor:
        """The sequences' log-probabilities (the reference model's, for the loss)."""

        return self._run(triton_sequence_log_probs, sequence_log_probs_with_pytorch, logits, labels, shift=shift,
                         average=self.options["average"])
