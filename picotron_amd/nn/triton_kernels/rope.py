"""Fused rotary embedding (forward and backward) on gfx950 behind picotron's Triton-RoPE
surface.

Drop-in for ``picotron.nn.triton_kernels.rope`` (reference
src/picotron/nn/triton_kernels/rope.py).  The reference kernel is forward-only: it raises
when autograd is recording and needs contiguous ``(batch, heads, seq, head_dim)`` input
with interleaved pairs.  Here the rotation is an autograd Function whose backward is the
inverse rotation (``pt_rope(..., inverse=1)``); it accepts strided views (such as the
``(B, S, H, D)``-memory transpose that attention produces), both the interleaved and the
rotate-half layouts, and query + key in one launch.  Angle tables are fp32.
"""

from __future__ import annotations

import torch
from torch import Tensor

from picotron_amd import ops
from picotron_amd.nn.triton_kernels._gate import no_graph, require_hip


class TritonRoPEUnavailable(RuntimeError):
    """Raised when the fused (HIP) RoPE path cannot safely run."""


class _RoPEFunction(torch.autograd.Function):
    """Rotate one or two (B, H, S, D) views by fp32 angle tables (by minus the angles when
    ``inverse``); the backward is the rotation the other way.  (Two named states, the second one
    None or not: torch.compile calls a forward with variable arguments without its ctx where no
    input asks for a gradient.)"""

    @staticmethod
    def forward(ctx, layout: str, inverse: bool, cosine: Tensor, sine: Tensor, x0: Tensor, x1: Tensor | None):  # type: ignore[override]
        ctx.layout = layout
        ctx.inverse = inverse
        ctx.save_for_backward(cosine, sine)
        out0, out1 = ops.rope(x0, cosine, sine, layout=layout, inverse=inverse, x1=x1)
        return out0 if out1 is None else (out0, out1)

    @staticmethod
    def backward(ctx, *grads: Tensor):  # type: ignore[override]
        cosine, sine = ctx.saved_tensors
        present = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[4 + i]]
        results: list[Tensor | None] = [None, None]
        if present:
            g = [_last_dim_contiguous(grads[i]) for i in present]
            g0, g1 = g[0], g[1] if len(g) > 1 else None
            if torch.is_grad_enabled() and not ops._compiling():
                # create_graph=True: the backward rotation as this Function again, so that
                # autograd can differentiate it to any order
                d = _RoPEFunction.apply(ctx.layout, not ctx.inverse, cosine, sine, g0, g1)
                d = (d, None) if g1 is None else d
            else:
                d = ops.rope(g0, cosine, sine, layout=ctx.layout, inverse=not ctx.inverse, x1=g1)
            for i, x in zip(present, d):
                results[i] = x
        return (None, None, None, None, *results)


def _last_dim_contiguous(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _validate(states: list[Tensor], cosine: Tensor, sine: Tensor) -> None:
    require_hip(TritonRoPEUnavailable, "RoPE", *states, cosine, sine)
    head_dim = states[0].size(-1)
    for s in states:
        if (
            s.ndim != 4
            or s.size(-1) != head_dim
            or s.stride(-1) != 1
            or s.dtype not in (torch.float32, torch.float16, torch.bfloat16)
            or s.dtype != states[0].dtype
        ):
            raise TritonRoPEUnavailable(
                "HIP RoPE requires 4-D (batch, heads, seq, head_dim) float states with a "
                "contiguous head_dim."
            )
    if (
        cosine.ndim != 2
        or cosine.shape != sine.shape
        or cosine.size(-1) * 2 != head_dim
        or cosine.size(0) < states[0].size(-2)
    ):
        raise TritonRoPEUnavailable("HIP RoPE requires [seq, head_dim/2] cosine/sine tables.")
    if len(states) == 2 and (
        states[1].size(0) != states[0].size(0) or states[1].size(-2) != states[0].size(-2)
    ):
        raise TritonRoPEUnavailable("RoPE query and key must share batch and sequence sizes.")


def triton_apply_rotary_embedding(
    states: Tensor, cosine: Tensor, sine: Tensor, *, layout: str = "interleaved"
) -> Tensor:
    """Rotate ``(batch, heads, sequence, head_dim)`` states (reference rope.py:52-91).

    Unlike the reference kernel this works with autograd enabled and on strided views.
    Tables of any float dtype are used in fp32.
    """

    _validate([states], cosine, sine)
    if no_graph(states, cosine, sine):
        return ops.rope(states, cosine.float(), sine.float(), layout=layout)[0]
    return _RoPEFunction.apply(layout, False, cosine.float(), sine.float(), states, None)


def triton_apply_rotary_embedding_pair(
    query: Tensor, key: Tensor, cosine: Tensor, sine: Tensor, *, layout: str = "interleaved"
) -> tuple[Tensor, Tensor]:
    """Rotate query and key (GQA: head counts may differ) in one kernel launch."""

    _validate([query, key], cosine, sine)
    if no_graph(query, key, cosine, sine):
        return ops.rope(query, cosine.float(), sine.float(), layout=layout, x1=key)
    out_q, out_k = _RoPEFunction.apply(layout, False, cosine.float(), sine.float(), query, key)
    return out_q, out_k


class _RoPEAtFunction(torch.autograd.Function):
    """Rotate one or two (B, H, S, D) views at their positions; the backward is the rotation the other way.  (Two named
    states, the second one None or not: torch.compile calls a forward with variable arguments without its ctx where no input asks for
    a gradient.)"""

    @staticmethod
    def forward(ctx, how: tuple, turns: Tensor, positions: Tensor | None, x0: Tensor, x1: Tensor | None):  # type: ignore[override]
        ctx.set_materialize_grads(False)
        ctx.how = how  # (offset, scale, layout, inverse)
        ctx.save_for_backward(turns, *((positions,) if positions is not None else ()))
        out0, out1 = _rotate_at(how, turns, positions, x0, x1)
        return out0 if out1 is None else (out0, out1)

    @staticmethod
    def backward(ctx, *grads: Tensor):  # type: ignore[override]
        turns, positions = (*ctx.saved_tensors, None)[:2]
        offset, scale, layout, inverse = ctx.how
        how = (offset, scale, layout, not inverse)
        present = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[3 + i]]
        results: list[Tensor | None] = [None, None]
        if present:
            g = [_last_dim_contiguous(grads[i]) for i in present]
            g0, g1 = g[0], g[1] if len(g) > 1 else None
            if torch.is_grad_enabled() and not ops._compiling():
                d = _RoPEAtFunction.apply(how, turns, positions, g0, g1)  # create_graph=True
                d = (d, None) if g1 is None else d
            else:
                d = _rotate_at(how, turns, positions, g0, g1)
            for i, x in zip(present, d):
                results[i] = x
        return (None, None, None, *results)


def _rotate_at(
    how: tuple, turns: Tensor, positions: Tensor | None, x0: Tensor, x1: Tensor | None
) -> tuple[Tensor, Tensor | None]:
    offset, scale, layout, inverse = how
    return ops.rope_at(x0, turns, positions=positions, offset=offset, scale=scale, layout=layout, inverse=inverse, x1=x1)


def triton_apply_rotary_at(
    query: Tensor, key: Tensor | None, positions: Tensor | int | None, frequencies, *, layout: str = "interleaved"
) -> tuple[Tensor, Tensor | None]:
    """Rotate query and key (or a single tensor, with ``key`` None) at given positions in one kernel launch.

    ``query`` and ``key`` are (batch, heads, seq, head_dim) views with a contiguous head_dim (head counts may differ).
    ``positions`` is an int32 or int64 tensor of (seq,), (1, seq) or (batch, seq) -- any values: packed documents,
    one decoded token per sequence, far into a context -- or an integer, the position of the first token, or None (0).
    ``frequencies`` is a :class:`picotron_amd.nn.RotaryFrequencies`, whose rotary_dim may be less than head_dim: the rest of a
    head is copied.  Outputs are new tensors; the backward turns the other way.  Angles carry no rounding of
    position times frequency (the reference's tables do: rope.py:13-32), so they are as exact at position 10^6 as at 1.
    """

    states = [query] if key is None else [query, key]
    offset = 0
    if isinstance(positions, Tensor):
        require_hip(TritonRoPEUnavailable, "RoPE", *states, positions)
    else:
        offset, positions = ops._first_position(positions), None
        require_hip(TritonRoPEUnavailable, "RoPE", *states)
    if layout not in ops.LAYOUTS:
        raise TritonRoPEUnavailable(f"RoPE layout must be one of {sorted(ops.LAYOUTS)}.")
    plain = no_graph(*states)
    if plain:  # decoding: what the native launcher takes needs no check here (14 us of host time, 11 this way)
        out = ops._launch_here("pt_rope_at", query, key, frequencies.turns(query.device), positions, offset,
                               frequencies.attention_factor, ops.LAYOUTS[layout], False)
        if out is not None:
            return out
    for s in states:
        if (s.ndim != 4 or s.size(-1) != query.size(-1) or s.stride(-1) != 1 or s.size(-1) % 2 != 0
                or s.dtype not in (torch.float32, torch.float16, torch.bfloat16) or s.dtype != query.dtype
                or s.device != query.device):
            raise TritonRoPEUnavailable(
                "HIP RoPE requires 4-D (batch, heads, seq, head_dim) float states of one dtype and device with an even, "
                "contiguous head_dim.")
        if s.size(0) != query.size(0) or s.size(2) != query.size(2):
            raise TritonRoPEUnavailable("RoPE query and key must share batch and sequence sizes.")
    if frequencies.rotary_dim > query.size(-1):
        raise TritonRoPEUnavailable("HIP RoPE requires frequencies of at most head_dim elements.")
    if positions is not None:
        if positions.device != query.device:
            raise TritonRoPEUnavailable("RoPE positions must be on the states' device.")
        try:
            ops._position_strides(positions, query.size(0), query.size(2))
        except ValueError as error:
            raise TritonRoPEUnavailable(f"{error}.") from error
    turns, scale = frequencies.turns(query.device), frequencies.attention_factor
    how = (offset, scale, layout, False)
    if plain:
        return _rotate_at(how, turns, positions, query, key)
    out = _RoPEAtFunction.apply(how, turns, positions, query, key)
    return (out, None) if key is None else out
