"""Rotary position embeddings with the reference's call surface (src/picotron/nn/rope.py).

``rotary_cos_sin`` and ``apply_rotary_embedding`` restate the reference functions
(interleaved pairs on a ``(batch, heads, seq, head_dim)`` view).  ``RotaryEmbedding``
keeps the reference constructor and ``forward(query, key)``; with ``use_triton_rope`` it
rotates query and key with one fused HIP launch (autograd included) using fp32 angle
tables cached per device (grown to the longest sequence seen), and warns once and falls
back otherwise.

The reference implements only the interleaved layout.  ``layout="rotate_half"`` (pairs
``(i, i + head_dim/2)``, the Llama/HF convention) is an addition; both layouts share the
same angle table.

So are rotations of a part of the head (``rotary_dim``), of frequencies scaled to longer contexts
(``scaling``) and at given positions (``forward(query, key, positions)``): any of them takes the
kernel that forms its angles from the positions (``triton_apply_rotary_at``) in place of the
tables, or :func:`apply_rotary_at` where it cannot run.  :class:`RotaryFrequencies` holds
the frequencies for both.
"""

from __future__ import annotations

import math
import warnings
from collections.abc import Mapping
from fractions import Fraction

import torch
from torch import Tensor, nn

from picotron_amd import ops
from picotron_amd.nn.triton_kernels.rope import (
    TritonRoPEUnavailable,
    triton_apply_rotary_at,
    triton_apply_rotary_embedding_pair,
)

LAYOUTS = ("interleaved", "rotate_half")


def rotary_cos_sin(
    sequence_length: int,
    head_dim: int,
    theta: float,
    *,
    device: torch.device,
    dtype: torch.dtype,
) -> tuple[Tensor, Tensor]:
    """Cosine and sine tables ``[sequence_length, head_dim/2]`` (reference rope.py:13-32)."""

    if head_dim % 2 != 0:
        raise ValueError("RoPE requires an even attention head dimension.")
    if theta <= 0:
        raise ValueError("rope_theta must be positive.")
    inverse_frequencies = 1.0 / (
        theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim)
    )
    positions = torch.arange(sequence_length, device=device, dtype=torch.float32)
    angles = torch.outer(positions, inverse_frequencies)
    return angles.cos().to(dtype=dtype), angles.sin().to(dtype=dtype)


def apply_rotary_embedding(states: Tensor, cosine: Tensor, sine: Tensor) -> Tensor:
    """Interleaved-pair rotation of ``(batch, heads, seq, head_dim)`` states
    (reference rope.py:35-51)."""

    if states.size(-1) != cosine.size(-1) * 2:
        raise ValueError("RoPE table dimension does not match the attention head dimension.")
    cosine = cosine.unsqueeze(0).unsqueeze(0)
    sine = sine.unsqueeze(0).unsqueeze(0)
    even_states = states[..., 0::2]
    odd_states = states[..., 1::2]
    rotated = torch.stack(
        (
            even_states * cosine - odd_states * sine,
            even_states * sine + odd_states * cosine,
        ),
        dim=-1,
    )
    return rotated.flatten(start_dim=-2)


def apply_rotary_embedding_rotate_half(states: Tensor, cosine: Tensor, sine: Tensor) -> Tensor:
    """Rotate-half rotation: pairs (i, i + head_dim/2) with the same angle table."""

    if states.size(-1) != cosine.size(-1) * 2:
        raise ValueError("RoPE table dimension does not match the attention head dimension.")
    half = states.size(-1) // 2
    cosine = cosine.unsqueeze(0).unsqueeze(0)
    sine = sine.unsqueeze(0).unsqueeze(0)
    first, second = states[..., :half], states[..., half:]
    return torch.cat((first * cosine - second * sine, first * sine + second * cosine), dim=-1)


# scaling type -> (required keys, optional keys with their defaults)
_SCALINGS = {
    "linear": (("factor",), {}),
    "ntk": (("factor",), {}),
    "yarn": (("factor", "original_max_positions"), {"beta_fast": 32.0, "beta_slow": 1.0, "attention_factor": None}),
    "llama3": (("factor", "original_max_positions"), {"low_freq_factor": 1.0, "high_freq_factor": 4.0}),
}


def _checked_scaling(scaling: Mapping) -> dict:
    kind = scaling.get("type")
    if kind not in _SCALINGS:
        raise ValueError(f"rotary scaling type must be one of {sorted(_SCALINGS)}; got {kind!r}.")
    required, optional = _SCALINGS[kind]
    missing = [key for key in required if key not in scaling]
    unknown = sorted(set(scaling) - {"type", *required, *optional})
    if missing or unknown:
        raise ValueError(f"rotary scaling {kind!r}: missing {missing}, unknown {unknown}.")
    values = {**optional, **scaling}
    for key, value in values.items():
        if key != "type" and value is not None and not (math.isfinite(value) and value > 0):
            raise ValueError(f"rotary scaling {key} must be a positive number; got {value!r}.")
    return {key: value if key == "type" or value is None else float(value) for key, value in values.items()}


# pi to 50 digits: a frequency is a binary fraction, and its turns per position are rounded once
_PI_DIGITS = 31415926535897932384626433832795028841971693993751
_PI_SCALE = 10**49


def _turn_bits(frequency: float) -> int:
    """``frequency / (2 pi)`` turns as a 64-bit fraction of a turn, right to half its last bit (formed in 64 bits it would
    be right to 2^-56 of a turn, 1e-4 rad at position 2^40)."""

    numerator, denominator = frequency.as_integer_ratio()
    return round(Fraction((numerator * _PI_SCALE) << 63, denominator * _PI_DIGITS)) % 2**64


def _bits_of(frequencies: list[float]) -> Tensor:
    bits = [_turn_bits(f) for f in frequencies]
    return torch.tensor([b - 2**64 if b >= 2**63 else b for b in bits], dtype=torch.int64, device="cpu")


def _elsewhere(t: Tensor, device: torch.device) -> bool:
    """True for what was kept for ``device`` and is on another: a module that was loaded with a map_location."""

    return t.device != device and (t.device.type != device.type or device.index is not None)


class RotaryFrequencies:
    """Radians per position of each rotated pair (``frequencies``, fp64 on the CPU) and the factor on cosine and sine
    (``attention_factor``): ``theta^(-2i/rotary_dim)``, scaled to contexts longer than those of training by ``scaling``:

    - ``{"type": "linear", "factor": F}``: every frequency / F (positions interpolated);
    - ``{"type": "ntk", "factor": F}``: theta * F^(rotary_dim / (rotary_dim - 2));
    - ``{"type": "yarn", "factor": F, "original_max_positions": L}``: / F for pairs that turn less than ``beta_slow``
      (1) times over L positions, kept for those above ``beta_fast`` (32), a linear ramp over the pairs between, and an
      ``attention_factor`` of 0.1 ln F + 1 unless given;
    - ``{"type": "llama3", "factor": F, "original_max_positions": L}``: / F below ``low_freq_factor`` (1) turns over L
      positions, kept above ``high_freq_factor`` (4), interpolated linearly in the number of turns between.

    It is a plan that a model keeps: :meth:`turns` is copied to a device once (before a graph capture
    that uses it there)."""

    @torch.inference_mode(False)  # (a model may be built, or first used, where tensors are another's)
    def __init__(self, rotary_dim: int, theta: float = 10_000.0, *, scaling: Mapping | None = None) -> None:
        if rotary_dim <= 0 or rotary_dim % 2 != 0:
            raise ValueError("RoPE requires an even, positive rotary dimension.")
        if not (math.isfinite(theta) and theta > 0):
            raise ValueError("rope_theta must be positive.")
        theta = float(theta)
        self.rotary_dim = rotary_dim
        self.attention_factor = 1.0
        # Python numbers, whatever device or mode torch makes tensors in here; the bits before any tracing of turns()
        values = self._scaled(_checked_scaling(scaling), theta) if scaling is not None else self._base(theta)
        self.frequencies = torch.tensor(values, dtype=torch.float64, device="cpu")
        self._bits = _bits_of(values)
        self._turns: dict[torch.device, Tensor] = {}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        if "_bits" not in state:  # stored when they were formed on first use
            self._bits = _bits_of(self.frequencies.tolist())

    def _base(self, theta: float) -> list[float]:
        return [theta ** (-2.0 * i / self.rotary_dim) for i in range(self.rotary_dim // 2)]

    def _scaled(self, s: dict, theta: float) -> list[float]:
        dim, factor = self.rotary_dim, s["factor"]
        if s["type"] == "ntk":
            theta = theta * factor ** (dim / max(dim - 2, 1))
        base = self._base(theta)
        if s["type"] == "linear":
            return [f / factor for f in base]
        if s["type"] == "yarn":
            length = s["original_max_positions"]
            if theta == 1.0:
                raise ValueError("rotary scaling 'yarn' needs a theta other than 1.")

            def pair_with(turns: float) -> float:  # the pair that turns so often over the original positions
                return dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))

            low = max(math.floor(pair_with(s["beta_fast"])), 0)
            high = min(math.ceil(pair_with(s["beta_slow"])), dim - 1)
            given = s["attention_factor"]
            self.attention_factor = given if given is not None else (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
            ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(len(base))]
            return [f * (1 - t) + f / factor * t for f, t in zip(base, ramp)]
        if s["type"] == "llama3":
            low, high = s["low_freq_factor"], s["high_freq_factor"]
            if high <= low:
                raise ValueError("rotary scaling 'llama3' needs high_freq_factor above low_freq_factor.")
            turns = [s["original_max_positions"] * f / (2 * math.pi) for f in base]
            keep = [min(max((t - low) / (high - low), 0.0), 1.0) for t in turns]
            return [f / factor * (1 - k) + f * k for f, k in zip(base, keep)]
        return base

    def turns(self, device: torch.device) -> Tensor:
        """int64 on ``device``: the bits of each frequency as a fraction of a turn per position, times 2^64."""

        found = self._turns.get(device)
        if found is None or _elsewhere(found, device):
            if device.type == "cuda" and not torch.compiler.is_compiling() and torch.cuda.is_current_stream_capturing():
                raise TritonRoPEUnavailable(
                    "HIP RoPE: the frequencies are first used on this device during graph capture; run the same call "
                    "once before capturing it.")
            with torch.inference_mode(False):  # a later pass may keep them for its backward
                found = self._bits.to(device)
            if type(found) is Tensor:  # not a dry run's
                self._turns[device] = found
        return found


def apply_rotary_at(
    states: Tensor, positions: Tensor | int | None, frequencies: RotaryFrequencies, *, layout: str = "interleaved"
) -> Tensor:
    """The rotation of ``triton_apply_rotary_at`` in PyTorch: angles as the kernel forms them, position times turns modulo 2^64
    (a product in fp64 is off by 1e-4 rad at position 2^40), then fp64; the rotation in fp32 (fp64 for fp64 states), one
    rounding to the states' type."""

    if layout not in LAYOUTS:
        raise ValueError(f"RoPE layout must be one of {LAYOUTS}.")
    seq, dim = states.size(-2), frequencies.rotary_dim
    if dim > states.size(-1):
        raise ValueError("RoPE frequencies cover more than the attention head dimension.")
    if not isinstance(positions, Tensor):
        positions = torch.arange(seq, device=states.device) + ops._first_position(positions)
    ops._position_strides(positions, states.size(0), seq)
    positions = positions if positions.dim() == 2 else positions[None]
    angles = (positions[:, None, :, None].long() * frequencies.turns(states.device)).double() * (math.pi * 2.0**-63)
    compute = torch.promote_types(states.dtype, torch.float32)
    cosine, sine = ((f(angles) * frequencies.attention_factor).to(compute) for f in (torch.cos, torch.sin))
    part = states[..., :dim].to(compute)
    if layout == "interleaved":
        first, second = part[..., 0::2], part[..., 1::2]
    else:
        first, second = part[..., : dim // 2], part[..., dim // 2 :]
    rotated = (first * cosine - second * sine, first * sine + second * cosine)
    part = torch.stack(rotated, dim=-1).flatten(-2) if layout == "interleaved" else torch.cat(rotated, dim=-1)
    return torch.cat((part.to(states.dtype), states[..., dim:]), dim=-1)


class RotaryEmbedding(nn.Module):
    """Apply RoPE to attention query and key tensors.

    ``rotary_dim`` (default: the whole head) rotates the first elements of each head; ``scaling`` is
    :class:`RotaryFrequencies`'s.  With either, or with positions given to :meth:`forward`, the angles come from the
    positions themselves; without them from fp32 tables, as in the reference."""

    # Of a module whose arguments only the tables take (a theta that is infinite), or that was stored before it had them.
    frequencies: RotaryFrequencies | None = None
    _plain = True

    def __init__(
        self,
        head_dim: int,
        theta: float = 10_000.0,
        *,
        use_triton_rope: bool = False,
        layout: str = "interleaved",
        rotary_dim: int | None = None,
        scaling: Mapping | None = None,
    ) -> None:
        super().__init__()
        if head_dim % 2 != 0:
            raise ValueError("RoPE requires an even attention head dimension.")
        if theta <= 0:
            raise ValueError("rope_theta must be positive.")
        if layout not in LAYOUTS:
            raise ValueError(f"RoPE layout must be one of {LAYOUTS}.")
        self.head_dim = head_dim
        self.theta = theta
        self.layout = layout
        self.use_triton_rope = use_triton_rope
        self._triton_fallback_warned = False
        if rotary_dim is not None and not 0 < rotary_dim <= head_dim:
            raise ValueError("rotary_dim must be positive and at most head_dim.")
        try:
            self.frequencies = RotaryFrequencies(head_dim if rotary_dim is None else rotary_dim, theta, scaling=scaling)
        except (ValueError, OverflowError):
            if rotary_dim is not None or scaling is not None:
                raise
        else:
            self._plain = scaling is None and self.frequencies.rotary_dim == head_dim
        # One fp32 table pair per device, as long as the longest sequence seen: position p's
        # angles do not depend on the table length, and the kernel reads rows 0..seq-1 of a
        # longer table, so variable sequence lengths share one pair instead of one each.
        self._fp32_tables: dict[torch.device, tuple[Tensor, Tensor]] = {}

    def _tables_fp32(self, sequence_length: int, device: torch.device) -> tuple[Tensor, Tensor]:
        tables = self._fp32_tables.get(device)
        if tables is None or tables[0].size(0) < sequence_length or _elsewhere(tables[0], device):
            tables = rotary_cos_sin(
                sequence_length, self.head_dim, self.theta, device=device, dtype=torch.float32
            )
            self._fp32_tables[device] = tables
        return tables

    def _at(self, query: Tensor, key: Tensor, positions: Tensor | int | None) -> tuple[Tensor, Tensor]:
        if self.frequencies is None:
            self.frequencies = RotaryFrequencies(self.head_dim, self.theta)  # or refused
        if self.use_triton_rope:
            try:
                return triton_apply_rotary_at(query, key, positions, self.frequencies, layout=self.layout)
            except Exception as error:
                self._warn(error)
        return (apply_rotary_at(query, positions, self.frequencies, layout=self.layout),
                apply_rotary_at(key, positions, self.frequencies, layout=self.layout))

    def _warn(self, error: Exception) -> None:
        if not self._triton_fallback_warned:
            warnings.warn(
                f"Triton RoPE unavailable; using PyTorch fallback: {error}",
                RuntimeWarning,
                stacklevel=2,
            )
            self._triton_fallback_warned = True

    def forward(
        self, query: Tensor, key: Tensor, positions: Tensor | int | None = None
    ) -> tuple[Tensor, Tensor]:
        """Rotate query and key using their shared sequence positions: 0 to seq - 1, or ``positions`` (those of
        ``triton_apply_rotary_at``)."""

        if (
            query.size(0) != key.size(0)
            or query.size(-2) != key.size(-2)
            or query.size(-1) != key.size(-1)
        ):
            raise ValueError("RoPE query and key must share batch, sequence, and head dimensions.")
        if positions is not None or not self._plain:
            return self._at(query, key, positions)
        if self.use_triton_rope:
            try:
                cosine, sine = self._tables_fp32(query.size(-2), query.device)
                return triton_apply_rotary_embedding_pair(
                    query, key, cosine, sine, layout=self.layout
                )
            except Exception as error:
                if not self._triton_fallback_warned:
                    warnings.warn(
                        f"Triton RoPE unavailable; using PyTorch fallback: {error}",
                        RuntimeWarning,
                        stacklevel=2,
                    )
                    self._triton_fallback_warned = True
        cosine, sine = rotary_cos_sin(
            query.size(-2), self.head_dim, self.theta, device=query.device, dtype=query.dtype
        )
        apply = apply_rotary_embedding if self.layout == "interleaved" else apply_rotary_embedding_rotate_half
        return apply(query, cosine, sine), apply(key, cosine, sine)
