"""AdamW with 8-bit moments.

``AdamW8bit`` is a ``torch.optim.Optimizer`` whose two moments take a byte an element each (and two bytes per 256
elements) in place of torch AdamW's eight: 1.2e9 parameters keep 2.4 GB of state instead of 9.6.
``triton_adamw_step`` (and ``AdamWStepWithFallback``) update every parameter of it in one HIP launch; ``step()`` is
the same update in PyTorch, on any device, with the same codes.

State of a parameter with n elements, in ceil(n / 256) blocks: ``exp_avg`` and ``exp_avg_sq``, uint8
[blocks, 256]; ``exp_avg_scale`` and ``exp_avg_sq_scale``, uint8 [blocks]; ``step``.  A scale byte is the exponent field
of the block's largest magnitude as fp32 (16 at least; 255 for an infinity or NaN: the block then reads as NaN), a code
the bits of magnitude * 2^(14 - scale) from the 20th up with the sign above them (first moment), or of
magnitude * 2^(30 - scale) (second moment, which is never negative).

Rounding to codes is stochastic: unbiased, where the nearest code would hold a slow average still (beta2 = 0.999
moves it by 0.1 % a step, codes lie 6 to 12 % apart).  bf16 parameters are rounded stochastically too unless
``stochastic_rounding`` is False, since most updates are below half their last place.  The random bits come from
the ``seed``, the step and an element's place among the parameters that step together: a run repeats bit for bit.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.optim import Optimizer

from picotron_amd import ops

BLOCK = 256   # elements that share a scale
UNIT = 1024   # every tensor's elements start at a multiple of it in the order of the random bits
TOP_M, TOP_V = 14, 30
_MIN_SCALE = 16
_MASK = 0xFFFFFFFF
_CODES = ("exp_avg", "exp_avg_sq")
_SCALES = ("exp_avg_scale", "exp_avg_sq_scale")
_OPTIONS = ("seed", "stochastic_rounding", "capturable")


def _signed(x: int) -> int:
    x &= _MASK
    return x - (1 << 32) if x >> 31 else x


def _down(x: Tensor, n: int) -> Tensor:
    """Shift right of int32 that brings in zeros."""

    return (x >> n) & ((1 << (32 - n)) - 1)


def _shift(x: Tensor, e: Tensor) -> Tensor:
    """x * 2^e (e int32), in two steps of which only the last may round: 2^e itself may be no fp32 number."""

    half = e >> 1
    return x * ((half + 127) << 23).view(torch.float32) * ((e - half + 127) << 23).view(torch.float32)


def encode(values: Tensor, random: Tensor, top: int) -> tuple[Tensor, Tensor]:
    """(codes uint8 [blocks, 256], scales uint8 [blocks]) of fp32 ``values`` [blocks, 256], rounded by 20
    random bits an element (``random`` int32, 2^19 everywhere for the nearest code)."""

    size = values.abs()
    scale = (size.view(torch.int32).amax(1, keepdim=True) >> 23).clamp_min(_MIN_SCALE)
    code = (_shift(size, top - scale).view(torch.int32) + random) >> 20
    if top == TOP_M:
        code = code | ((values.view(torch.int32) >> 24) & 128)
    else:
        code = torch.maximum(code, (values > 0).int())
    code = torch.where(scale == 255, 0, code)
    return code.to(torch.uint8), scale.to(torch.uint8).squeeze(1)


def decode(codes: Tensor, scales: Tensor, top: int) -> Tensor:
    """fp32 [blocks, 256] values of :func:`encode`'s codes and scales."""

    code, scale = codes.int(), scales.int()[:, None]
    value = _shift(((code & (127 if top == TOP_M else 255)) << 20).view(torch.float32), scale - top)
    if top == TOP_M:
        value = torch.where(code > 127, -value, value)
    return torch.where(scale == 255, math.nan, value)


def mixed_seed(seed: int, step: int) -> int:
    x = (seed ^ step * 0x9E3779B9) & _MASK
    x = (x ^ x >> 16) * 0x7FEB352D & _MASK
    x = (x ^ x >> 15) * 0x846CA68B & _MASK
    return x ^ x >> 16


def random_bits(first_unit: int, count: int, mixed: int, device: torch.device) -> Tensor:
    """int32 [count] (a multiple of 4) random bits of the elements from unit ``first_unit`` on: four in a row are
    successive states of Marsaglia's 32-bit xorshift generator, started from a hash of their place."""

    start = first_unit * (UNIT // 4)
    place = (torch.arange(start, start + count // 4, device=device) & _MASK).to(torch.int64)
    place = torch.where(place > 0x7FFFFFFF, place - (1 << 32), place).to(torch.int32)
    x = place * _signed(0x9E3779B1) + _signed(mixed)
    x = (x ^ _down(x, 16)) * 0x7FEB352D
    x = x ^ _down(x, 15)
    states = []
    for _ in range(4):
        x = x ^ (x << 13)
        x = x ^ _down(x, 17)
        x = x ^ (x << 5)
        states.append(x)
    return torch.stack(states, -1).view(-1)


def _blocks(p: Tensor) -> int:
    return (p.numel() + BLOCK - 1) // BLOCK


def _units(p: Tensor) -> int:
    return (p.numel() + UNIT - 1) // UNIT


class AdamW8bit(Optimizer):
    """AdamW whose moments are kept in 8 bits (see the module).  ``capturable``: the step counts are fp32 scalars on
    the parameters' device, so that a fused step can be captured in a HIP graph (after one eager step)."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, seed: int = 0, stochastic_rounding: bool = True,
                 capturable: bool = False) -> None:
        if isinstance(lr, Tensor) or not lr >= 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not eps >= 0.0:
            raise ValueError(f"Invalid epsilon value: {eps}")
        for i, beta in enumerate(betas):
            if not 0.0 <= beta < 1.0:
                raise ValueError(f"Invalid beta parameter at index {i}: {beta}")
        if not weight_decay >= 0.0:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, seed=int(seed),
                                      stochastic_rounding=bool(stochastic_rounding), capturable=bool(capturable)))

    def _new_state(self, p: Tensor, capturable: bool) -> dict:
        state = self.state[p]
        state["step"] = torch.zeros((), dtype=torch.float32, device=p.device if capturable else "cpu")
        for codes, scales in zip(_CODES, _SCALES):
            state[codes] = torch.zeros((_blocks(p), BLOCK), dtype=torch.uint8, device=p.device)
            state[scales] = torch.zeros(_blocks(p), dtype=torch.uint8, device=p.device)
        return state

    def buckets(self, groups: list[tuple[dict, list[Tensor]]]) -> list[tuple]:
        """The launches of one step over ``groups`` (param_group, its parameters that step): (param_group, params, states, their
        common step before it -- a number, or for a capturable group the device tensor -- and seed).  Creates
        what state is missing.  Parameters of a bucket share a group, a dtype and a step count; a device count belongs to one bucket,
        whose launch advances it."""

        found = []
        counted: set[int] = set()
        for group, params in groups:
            shared: dict[tuple, tuple[list, list]] = {}
            fresh: dict[tuple, Tensor] = {}
            for p in params:
                if p.numel() == 0:
                    continue
                state = self.state[p]
                if len(state) == 0:
                    state = self._new_state(p, group["capturable"])
                    if group["capturable"]:  # the parameters that start together count together
                        state["step"] = fresh.setdefault((p.dtype, p.device), state["step"])
                step = state["step"]
                key = (p.dtype, p.device, id(step) if group["capturable"] else float(step))
                ps, states = shared.setdefault(key, ([], []))
                ps.append(p)
                states.append(state)
            for (_, _, step), (ps, states) in shared.items():
                value = step
                if group["capturable"]:
                    value = states[0]["step"]
                    if id(value) in counted:  # shared with another bucket: a count of its own from here on
                        if value.is_cuda and torch.cuda.is_current_stream_capturing():
                            raise RuntimeError("AdamW8bit: parameters that step in several launches share a step count; take one "
                                               "step before capturing it")
                        value = value.clone()
                        for state in states:
                            state["step"] = value
                    counted.add(id(value))
                found.append((group, ps, states, value, self.bucket_seed(group, len(found))))
        return found

    @staticmethod
    def bucket_seed(group: dict, index: int) -> int:
        """The seed of a step's launch number ``index``: its places start at 0 again."""

        return (group["seed"] + 0x632BE5AB * index) & _MASK

    def _with_gradients(self) -> list[tuple[dict, list[Tensor]]]:
        return [(group, [p for p in group["params"] if p.grad is not None]) for group in self.param_groups]

    @torch.no_grad()
    def step(self, closure=None):
        """The update in PyTorch."""

        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = self._with_gradients()
        for _, params in groups:
            for p in params:
                if p.grad.is_sparse or not p.is_floating_point() or p.dtype == torch.float64:
                    raise RuntimeError("AdamW8bit takes dense fp32, fp16 and bf16 gradients")
        advanced: set[int] = set()
        for group, params, states, step, seed in self.buckets(groups):
            for state in states:
                if id(state["step"]) not in advanced:
                    advanced.add(id(state["step"]))
                    state["step"] += 1
            t = float(states[0]["step"])
            unit = 0
            for p, state in zip(params, states):
                self._update(group, p, state, t, unit, mixed_seed(seed, int(t)))
                unit += _units(p)
        return loss

    def _update(self, group: dict, p: Tensor, state: dict, t: float, unit: int, mixed: int) -> None:
        n, blocks = p.numel(), _blocks(p)
        (beta1, beta2), lr = group["betas"], group["lr"]
        r = random_bits(unit, blocks * BLOCK, mixed, p.device).view(blocks, BLOCK)

        def padded(x: Tensor) -> Tensor:
            y = torch.zeros(blocks * BLOCK, dtype=torch.float32, device=p.device)
            y[:n] = x.reshape(-1)
            return y.view(blocks, BLOCK)

        g = padded(p.grad)
        m = decode(state["exp_avg"], state["exp_avg_scale"], TOP_M) * beta1 + g * (1 - beta1)
        v = decode(state["exp_avg_sq"], state["exp_avg_sq_scale"], TOP_V) * beta2 + (g * (1 - beta2)) * g
        denom = v.sqrt() / math.sqrt(1 - beta2**t) + group["eps"]
        x = padded(p) * (1 - lr * group["weight_decay"]) - m / denom * (lr / (1 - beta1**t))
        if p.dtype == torch.bfloat16 and group["stochastic_rounding"]:
            bits = x.view(torch.int32)
            up = ((bits + (_down(r, 8) & 0xFFFF)) & -65536).view(torch.float32)
            x = torch.where(x.isfinite(), up, x)
        p.copy_(x.view(-1)[:n].view(p.shape))
        codes, scales = encode(m, _down(r, 12), TOP_M)
        state["exp_avg"].copy_(codes)
        state["exp_avg_scale"].copy_(scales)
        codes, scales = encode(v, (r & 0xFFFF) << 4 | _down(r, 28), TOP_V)
        state["exp_avg_sq"].copy_(codes)
        state["exp_avg_sq_scale"].copy_(scales)

    @torch.no_grad()
    def moments(self, dtype: torch.dtype = torch.float32) -> tuple[Tensor, Tensor, list[tuple[Tensor, int]]]:
        """(exp_avg, exp_avg_sq, places): the moments' values as two flat tensors, and for each parameter with
        state its first element's place in them (multiples of 1024; zeros fill the gaps).  The values are exact in fp32
        and, scales from 2^-100 on, in bf16.  One launch on a gfx950 device."""

        held = [(p, self.state[p]) for group in self.param_groups for p in group["params"] if p.numel() and len(self.state[p])]
        if not held:
            return torch.zeros(0, dtype=dtype), torch.zeros(0, dtype=dtype), []
        if any(p.device != held[0][0].device for p, _ in held):
            raise ValueError("AdamW8bit.moments takes parameters on one device")
        found = ops.adamw8_moments([p for p, _ in held], [state for _, state in held], dtype)
        if found is not None:
            return found
        total, places = 0, []
        for p, _ in held:
            places.append((p, total))
            total += _units(p) * UNIT
        out = []
        for codes, scales, top in zip(_CODES, _SCALES, (TOP_M, TOP_V)):
            flat = torch.zeros(total, dtype=dtype, device=held[0][0].device)
            for (p, state), (_, at) in zip(held, places):
                flat[at:at + p.numel()] = decode(state[codes], state[scales], top).view(-1)[:p.numel()]
            out.append(flat)
        return out[0], out[1], places

    def load_state_dict(self, state_dict: dict) -> None:
        """Restores a state of this optimizer, or of a ``torch.optim.AdamW`` over the same parameters (its fp32 moments are
        rounded to the nearest codes).  Options that its groups lack (seed and rounding, from a torch AdamW) stay as they are."""

        for group in state_dict["param_groups"]:
            for flag in ("amsgrad", "maximize"):
                if group.get(flag, False):
                    raise ValueError(f"AdamW8bit does not take a state of {flag}=True")
        # a torch AdamW's groups have no options of this optimizer's own: it keeps the ones it has
        groups = [{**{key: own[key] for key in _OPTIONS}, **group}
                  for own, group in zip(self.param_groups, state_dict["param_groups"])]
        groups += state_dict["param_groups"][len(groups):]  # more of them than here: refused by torch
        super().load_state_dict({**state_dict, "state": self._in_codes(state_dict), "param_groups": groups})
        shared: dict[tuple, Tensor] = {}
        group_of = {id(p): i for i, group in enumerate(self.param_groups) for p in group["params"]}
        for p, state in self.state.items():
            for key in (*_CODES, *_SCALES):
                if key in state:  # torch has cast the bytes to the parameter's dtype, which holds them exactly
                    state[key] = state[key].to(torch.uint8).contiguous()
            if "step" not in state or id(p) not in group_of:
                continue
            # torch hands a count over as it is, or on the device (of a fused AdamW): it becomes this optimizer's own, on the host
            # or, where it is to be captured, one for each launch again, as before
            step = float(state["step"])
            if self.param_groups[group_of[id(p)]]["capturable"]:
                key = (group_of[id(p)], p.dtype, p.device, step)
                if key not in shared:
                    shared[key] = torch.tensor(step, dtype=torch.float32, device=p.device)
                state["step"] = shared[key]
            else:
                state["step"] = torch.tensor(step, dtype=torch.float32, device="cpu")

    def _in_codes(self, state_dict: dict) -> dict:
        """The parameters' states of ``state_dict``, a torch AdamW's moments as codes.  They are rounded from the values given:
        torch's loading casts them to the parameter's dtype first, and fp16 has no second moment below 3e-8."""

        loaded = dict(state_dict["state"])
        names = [name for group in state_dict["param_groups"] for name in group["params"]]
        for name, p in zip(names, [p for group in self.param_groups for p in group["params"]]):
            if not all(key in loaded.get(name, ()) for key in _CODES) or _SCALES[0] in loaded[name]:
                continue
            state = loaded[name] = dict(loaded[name])
            for codes, scales, top in zip(_CODES, _SCALES, (TOP_M, TOP_V)):
                if state[codes].numel() != p.numel():
                    raise ValueError(f"AdamW8bit cannot take a state whose {codes} has {state[codes].numel()} elements for a "
                                     f"parameter of {p.numel()}")
                values = torch.zeros(_blocks(p) * BLOCK, dtype=torch.float32, device=p.device)
                values[:p.numel()] = state[codes].to(p.device, torch.float32).reshape(-1)
                nearest = torch.full((_blocks(p), BLOCK), 1 << 19, dtype=torch.int32, device=p.device)
                state[codes], state[scales] = encode(values.view(-1, BLOCK), nearest, top)
        return loaded

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        for group in self.param_groups:  # a torch AdamW's, from a hook of the loading, have none of these
            group.setdefault("seed", 0)
            group.setdefault("stochastic_rounding", True)
            group.setdefault("capturable", False)

