"""Cross-entropy of a language model's head without its logits, forward and backward, on gfx950.

The reference's train loop forms the whole logits, ``output_projection(hidden)`` of (batch, seq, vocab), and
``F.cross_entropy`` of them (src/picotron/training/train_loop.py:136-145); at 8192 tokens of a 128256-word vocabulary
they are 2.1 GB in bf16, their gradient as much again, and autograd keeps them from the loss to the backward.
``triton_linear_cross_entropy`` takes the hidden states and the head's weight instead.  It returns ``F.cross_entropy`` of
``F.linear(hidden, weight)`` in fp32, and computes the gradients of both with the loss; what is kept for the
backward is those gradients alone (of the inputs' type; of fp16 inputs in fp32, as a loss scale arrives only with the
backward).  The backward multiplies them by what arrives from above, on the device, and not even that where it is 1.
They are handed out once: a second backward through the same graph raises.  16-bit gradients are so rounded twice where what
arrives is no power of two, but for fp16.  As those of ``triton_cross_entropy`` they are no saved tensors: saved-tensor hooks (CPU
offload) do not see them, and activation checkpointing that does not re-enter holds those of the first forward.

With ``reduction="none"`` each token's loss comes back and takes a gradient of its own; the forward then keeps its inputs,
and the backward forms the softmax again.  So does the loss of up to 512 fp16 states.  A state's gradient is as accurate relative
to its own weight as to any other's.

Ignored tokens cost nothing: their rows take no part in any product, may hold anything, and get zeros as their gradient.
A label outside the vocabulary gives NaN, in the loss and the gradients it enters (PICOTRON_HIP_CE_CHECK=1 raises
instead, at the cost of a host sync).  Under autocast the inputs are cast as ``F.linear`` would cast them.
"""

from __future__ import annotations

import os
import warnings

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from picotron_amd import ops
from picotron_amd.nn.triton_kernels._gate import native_graph, no_graph, require_hip
from picotron_amd.nn.triton_kernels.cross_entropy import _CHECK_ENV, IGNORE_INDEX, TritonCrossEntropyUnavailable, _check_targets


class TritonLinearCrossEntropyUnavailable(RuntimeError):
    """Raised when the fused (HIP) cross-entropy of a head cannot safely run."""


_REPEATED_BACKWARD = (
    "the gradients of the fused head's cross-entropy were handed out by an earlier backward through this graph "
    "(retain_graph=True); backpropagate through the loss once, or use reduction='none'"
)


class _ReducedLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden: Tensor, weight: Tensor, labels: Tensor, how: dict):  # type: ignore[override]
        want_dx, want_dw = ctx.needs_input_grad[:2]
        dtype = torch.float32 if hidden.dtype == torch.float16 else hidden.dtype
        loss, dx, dw = ops.linear_cross_entropy(hidden, weight, labels, want_dx=want_dx, want_dw=want_dw, grad_dtype=dtype, **how)
        ctx.gradients = (dx, dw)
        ctx.dtype = hidden.dtype
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):  # type: ignore[override]
        if ctx.gradients is None:
            raise RuntimeError(_REPEATED_BACKWARD)
        gradients, ctx.gradients = ctx.gradients, None
        dx, dw = ops.scale_gradients(gradients, grad, ctx.dtype)
        return dx, dw, None, None


class _DeferredLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden: Tensor, weight: Tensor, labels: Tensor, how: dict):  # type: ignore[override]
        ctx.save_for_backward(hidden, weight, labels)
        ctx.how = how
        return ops.linear_cross_entropy(hidden, weight, labels, **how)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):  # type: ignore[override]
        hidden, weight, labels = ctx.saved_tensors
        want_dx, want_dw = ctx.needs_input_grad[:2]
        _, dx, dw = ops.linear_cross_entropy(hidden, weight, labels, want_loss=False, want_dx=want_dx, want_dw=want_dw,
                                             grad_losses=grad, **ctx.how)
        return dx, dw, None, None


def _check_options(reduction: str, chunk_tokens: int | None) -> None:
    if reduction not in ops.REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(ops.REDUCTIONS)}.")
    if chunk_tokens is not None and (isinstance(chunk_tokens, bool) or not isinstance(chunk_tokens, int) or chunk_tokens < 1):
        raise ValueError("chunk_tokens must be a positive integer or None.")


def _checks_targets() -> bool:
    return os.environ.get(_CHECK_ENV, "") not in ("", "0")


def _autocast(*tensors: Tensor) -> tuple[Tensor, ...]:
    """As F.linear under autocast casts its inputs."""

    if not torch.is_autocast_enabled("cuda"):
        return tensors
    dtype = torch.get_autocast_dtype("cuda")
    return tuple(t.to(dtype) if t.is_floating_point() and t.is_cuda and t.dtype != torch.float64 else t for t in tensors)


def triton_linear_cross_entropy(
    hidden: Tensor, weight: Tensor, labels: Tensor, *, shift: bool = False, ignore_index: int = IGNORE_INDEX,
    reduction: str = "mean", chunk_tokens: int | None = None,
) -> Tensor:
    """``F.cross_entropy(F.linear(hidden, weight).float(), labels)`` without the logits, fp32.

    ``hidden`` is (batch, seq, hidden) or (tokens, hidden), ``weight`` (vocab, hidden) of the same type, ``labels`` int64 of
    the leading shape; with ``shift`` the state at t is scored against label t + 1 (the last position of each
    sequence against none).  ``reduction``: ``"mean"`` over the labels != ``ignore_index`` (NaN of none), ``"sum"``, or
    ``"none"`` for every token's loss, 0 at ignored ones.  Differentiable once in ``hidden`` and ``weight``.

    With gradients the call holds exponentials of about ``2 * vocab`` bytes a token in 16 bits, ``4 * vocab`` in fp32, of at most 2 GiB.
    ``chunk_tokens`` bounds how many tokens are worked on at a time, in multiples of 256, and so these bytes alone.  Beside
    them lie the gathered states, up to 256 MB of a product's parts, a copy of the weight where it is fp32 or its rows are no
    whole 64 elements (fp32: as two 16-bit planes), and with more than one chunk the sum of the weight's gradient in fp32
    (2.1 GB at 128256 x 4096): less than all tokens a chunk may take more memory.  16-bit models of up to 128 hold no exponentials and
    take no notice of it.

    A few fp32 tokens at a large vocabulary take longer than ``F.linear`` and ``F.cross_entropy``, as the weight's planes are
    formed first (one token of 4096 at 128256 words: 1.83 ms, those 0.39; 256 tokens: 2.0 and 1.9)."""

    if torch.compiler.is_compiling():  # runs between a compiled model's graphs
        return _outside_graphs(hidden, weight, labels, shift, ignore_index, reduction, chunk_tokens)
    return _linear_cross_entropy(hidden, weight, labels, shift, ignore_index, reduction, chunk_tokens)


def _linear_cross_entropy(
    hidden: Tensor, weight: Tensor, labels: Tensor, shift: bool, ignore_index: int, reduction: str, chunk_tokens: int | None
) -> Tensor:
    _check_options(reduction, chunk_tokens)
    require_hip(TritonLinearCrossEntropyUnavailable, "linear cross-entropy", hidden, weight, labels)
    hidden, weight = _autocast(hidden, weight)
    plain = no_graph(hidden, weight)
    if (plain or native_graph()) and not _checks_targets():  # what the native code takes needs no check here
        loss = ops._launch_here("pt_linear_cross_entropy", hidden, weight, labels, bool(shift), ignore_index,
                                ops.REDUCTIONS[reduction], chunk_tokens or 0, not plain)
        if loss is not None:
            return loss
    if weight.device != hidden.device or labels.device != hidden.device:
        raise TritonLinearCrossEntropyUnavailable("HIP linear cross-entropy needs its inputs on one device.")
    try:
        ops.head_rows(hidden, weight, labels, shift)
    except ValueError as error:
        raise TritonLinearCrossEntropyUnavailable(f"HIP linear cross-entropy: {error}.") from error
    try:
        _check_targets(labels[:, 1:] if shift else labels, weight.size(0), ignore_index)
    except TritonCrossEntropyUnavailable as error:
        raise TritonLinearCrossEntropyUnavailable(str(error)) from error
    how = dict(shift=bool(shift), ignore_index=int(ignore_index), reduction=reduction, chunk_tokens=chunk_tokens or 0)
    if plain:
        return ops.linear_cross_entropy(hidden, weight, labels, **how)[0]
    return (_DeferredLoss if ops.head_defers(hidden, reduction) else _ReducedLoss).apply(hidden, weight, labels, how)


_outside_graphs = torch.compiler.disable(_linear_cross_entropy)


def linear_cross_entropy_with_pytorch(
    hidden: Tensor, weight: Tensor, labels: Tensor, *, shift: bool = False, ignore_index: int = IGNORE_INDEX,
    reduction: str = "mean",
) -> Tensor:
    """:func:`triton_linear_cross_entropy` in PyTorch, logits and all."""

    _check_options(reduction, None)
    if shift:
        hidden, labels = hidden[:, :-1], labels[:, 1:]
    logits = F.linear(hidden, weight)
    logits = logits.to(torch.promote_types(logits.dtype, torch.float32))
    loss = F.cross_entropy(logits.reshape(-1, logits.size(-1)), labels.reshape(-1), ignore_index=ignore_index, reduction=reduction)
    return loss.view(labels.shape) if reduction == "none" else loss


class LinearCrossEntropyWithFallback:
    """Run the fused head and loss when enabled, else (or on failure) the PyTorch form, warning once."""

    def __init__(self, *, use_triton: bool = False, ignore_index: int = IGNORE_INDEX, reduction: str = "mean",
                 chunk_tokens: int | None = None) -> None:
        _check_options(reduction, chunk_tokens)
        self.use_triton = use_triton
        self.ignore_index = ignore_index
        self.reduction = reduction
        self.chunk_tokens = chunk_tokens
        self._fallback_warned = False

    def __call__(self, hidden: Tensor, weight: Tensor, labels: Tensor, *, shift: bool = False) -> Tensor:
        how = dict(shift=shift, ignore_index=self.ignore_index, reduction=self.reduction)
        if self.use_triton:
            try:
                return triton_linear_cross_entropy(hidden, weight, labels, chunk_tokens=self.chunk_tokens, **how)
            except Exception as error:
                if not self._fallback_warned:
                    warnings.warn(
                        f"Triton linear cross-entropy unavailable; using PyTorch fallback: {error}",
                        RuntimeWarning,
                        stacklevel=2,
                    )
                    self._fallback_warned = True
        return linear_cross_entropy_with_pytorch(hidden, weight, labels, **how)
