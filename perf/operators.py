"""Cases that measure three operators of preference tuning on long contexts, through the entry points
that a user calls: the rotary embedding at given positions, the preference loss on a model's logits with
the sequence log-probabilities it is made of, and the AdamW step with 8-bit states.

``own`` false: the operators in plain torch operations, in 32 bits (angles in 64), rounded once.  ``own``
true: the framework's calls.  ``listed()`` holds one case per kind of use, ``draw(rng)`` gives another of
the same ranges, ``exact`` the results in 64 bits.
"""

from __future__ import annotations

import functools
import math

import torch
from torch import Tensor

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
IGNORED = -100
LOSS_SCALE = 65536.0
THETA = 500_000.0
LR, BETAS, EPS, DECAY, STEP, SEED = 1e-4, (0.9, 0.95), 1e-8, 0.1, 101, 17
BLOCK, UNIT = 256, 1024  # elements that share a scale; every tensor starts on a unit
SCALINGS = {
    "none": None,
    "linear": dict(type="linear", factor=4.0),
    "ntk": dict(type="ntk", factor=8.0),
    "yarn": dict(type="yarn", factor=16.0, original_max_positions=8192, beta_fast=32.0, beta_slow=1.0),
    "llama3": dict(type="llama3", factor=8.0, original_max_positions=8192, low_freq_factor=1.0, high_freq_factor=4.0),
}


def listed() -> list[dict]:
    return [
        # one decoded token of 16 sequences, each at its own place in a long context (smallest calls)
        dict(name="rope_decode", kind="rope", batch=16, seq=1, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             layout="rotate_half", scaling="llama3", positions="each", dtype="bf16", train=False),
        # grouped-query attention's rotation in long-context training, several documents to a row of the batch
        dict(name="rope_packed_bf16", kind="rope", batch=2, seq=8192, heads=32, kv_heads=8, head_dim=128,
             rotary_dim=128, layout="rotate_half", scaling="yarn", positions="each", dtype="bf16", train=True),
        # a quarter of an 80-element head rotated, an odd number of tokens far into a document, fp16 training
        dict(name="rope_part_fp16", kind="rope", batch=1, seq=32769, heads=16, kv_heads=4, head_dim=80, rotary_dim=20,
             layout="interleaved", scaling="linear", positions="offset", dtype="fp16", train=True),
        # prefill of four prompts in full precision, the same positions for all, half of the head rotated
        dict(name="rope_prefill_fp32", kind="rope", batch=4, seq=4095, heads=16, kv_heads=16, head_dim=64,
             rotary_dim=32, layout="rotate_half", scaling="ntk", positions="shared", dtype="fp32", train=False),
        # the log-probability of one token at a large vocabulary, as a serving loop scores a candidate
        dict(name="score_token", kind="score", batch=1, seq=2, vocab=128256, dtype="bf16"),
        # the reference model's sequence log-probabilities over a batch of answers
        dict(name="score_bf16", kind="score", batch=8, seq=2048, vocab=32000, dtype="bf16"),
        # one pair of a byte-level model (256 bytes and 4 special tokens)
        dict(name="preference_bytes", kind="preference", batch=2, seq=24, vocab=260, dtype="fp32"),
        # the notebook demo's vocabulary (rows start anywhere in a line), fp16 under a loss scale
        dict(name="preference_demo_fp16", kind="preference", batch=16, seq=256, vocab=50257, dtype="fp16"),
        # preference tuning of a large-vocabulary model, two pairs of 2049 tokens
        dict(name="preference_bf16", kind="preference", batch=4, seq=2049, vocab=128256, dtype="bf16"),
        # the quickstart decoder's parameters: a few short tensors
        dict(name="adamw8_quickstart", kind="adamw8", layers=2, hidden=32, intermediate=64, kv=32, vocab=64, dtype="fp32"),
        # a small decoder whose widths are no multiples of a block, fp32 parameters
        dict(name="adamw8_odd_fp32", kind="adamw8", layers=8, hidden=1090, intermediate=2907, kv=545, vocab=32001,
             dtype="fp32"),
        # the update of a 1.04e9-parameter decoder held in bf16 (largest)
        dict(name="adamw8_bf16", kind="adamw8", layers=16, hidden=2048, intermediate=8192, kv=512, vocab=32000,
             dtype="bf16"),
    ]


# ---------------------------------------------------------------------- drawn cases


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["rope", "rope", "score", "preference", "preference", "adamw8"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if kind == "rope":
        head_dim = rng.choice([16, 64, 64, 80, 96, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        seq = _log(rng, 1, 16384)
        most = max(1, 10**8 // (seq * kv_heads * 4 * head_dim))
        return dict(kind=kind, batch=_log(rng, 1, min(64, most)), seq=seq, heads=kv_heads * rng.choice([1, 2, 4]),
                    kv_heads=kv_heads, head_dim=head_dim, rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4]),
                    layout=rng.choice(["interleaved", "rotate_half"]), scaling=rng.choice(sorted(SCALINGS)),
                    positions=rng.choice(["offset", "shared", "each"]), dtype=dtype, train=rng.random() < 0.6)
    if kind in ("score", "preference"):
        vocab = rng.choice([260, 32000, 50257, 128256, _log(rng, 64, 128256), _log(rng, 64, 128256)])
        most = 6 * 10**8 // (2 if dtype == "fp32" else 1) // vocab  # rows
        seq = _log(rng, 2, min(4097, max(2, most // 2)))
        return dict(kind=kind, batch=2 * _log(rng, 1, max(1, min(32, most // seq // 2))), seq=seq, vocab=vocab, dtype=dtype)
    hidden = _log(rng, 32, 1600)
    return dict(kind=kind, layers=_log(rng, 1, 16), hidden=hidden, intermediate=hidden * rng.choice([2, 3, 4]) + rng.choice([0, 0, 1]),
                kv=max(1, hidden // rng.choice([1, 2, 4])), vocab=_log(rng, 64, 50257), dtype=dtype)


# ---------------------------------------------------------------------- inputs


def _randn(shape, dtype: torch.dtype, gen: torch.Generator, scale: float = 1.0) -> Tensor:
    """Normal values made in slices, so that a large 16-bit tensor needs no fp32 copy of itself."""

    out = torch.empty(shape, dtype=dtype, device="cuda")
    for part in out.view(-1).split(1 << 28):
        part.copy_(torch.randn(part.numel(), generator=gen, device="cuda").mul_(scale))
    return out


@functools.lru_cache(maxsize=None)
def _plan(rotary_dim: int, scaling: str):
    """The framework's handle of a model's rotary frequencies, which lives as long as the model."""

    from picotron_amd.nn import RotaryFrequencies

    return RotaryFrequencies(rotary_dim, THETA, scaling=SCALINGS[scaling])


def _adamw8_places(case: dict) -> tuple[list[tuple[int, tuple[int, ...]]], int]:
    """A decoder's parameters (tied embeddings) and their places in flat buffers, each on a unit."""

    h, i, kv = case["hidden"], case["intermediate"], case["kv"]
    layer = [(h,), (h, h), (kv, h), (kv, h), (h, h), (h,), (i, h), (i, h), (h, i)]
    places, total = [], 0
    for shape in [(case["vocab"], h), *layer * case["layers"], (h,)]:
        places.append((total, shape))
        total += (math.prod(shape) + UNIT - 1) // UNIT * UNIT
    return places, total


def prepare(case: dict, seed: int) -> dict:
    kind = case["kind"]
    dtype = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if kind == "rope":
        b, n, d = case["batch"], case["seq"], case["head_dim"]
        make = lambda heads, scale: _randn((b, n, heads, d), dtype, gen, scale).transpose(1, 2)  # noqa: E731
        s.update(q=make(case["heads"], 1.0).requires_grad_(case["train"]), k=make(case["kv_heads"], 1.0).requires_grad_(case["train"]))
        start = torch.randint(0, 1 << 20, (b, 1), generator=gen, device="cuda")
        if case["positions"] == "offset":  # a chunk of a long document
            s.update(positions=1_000_000 + seed % 1000)
        elif case["positions"] == "shared":
            s.update(positions=torch.arange(n, device="cuda") + start[0])
        elif n == 1:  # every sequence at its own length
            s.update(positions=start)
        else:  # documents packed one behind the other: positions start again at each
            at = torch.arange(n, device="cuda")
            s.update(positions=(at + start) % torch.randint(min(64, n), n + 1, (b, 1), generator=gen, device="cuda"))
        if case["train"]:
            s.update(dq=make(case["heads"], 0.1), dk=make(case["kv_heads"], 0.1))
    elif kind in ("score", "preference"):
        b, n, v = case["batch"], case["seq"], case["vocab"]
        labels = torch.randint(0, v, (b, n), generator=gen, device="cuda")
        at = torch.arange(n, device="cuda")
        prompt = torch.randint(0, max(1, n // 3), (b, 1), generator=gen, device="cuda")
        end = n - torch.randint(0, max(1, n // 8), (b, 1), generator=gen, device="cuda")
        labels = labels.masked_fill((at < prompt) | (at >= end), IGNORED)  # the prompt, and padding behind the answer
        s.update(labels=labels, logits=_randn((b, n, v), dtype, gen, 2.0).requires_grad_(kind == "preference"))
        if kind == "preference":  # the reference model's log-probabilities, near the policy's
            s.update(reference=-(math.log(v) + 2.0) * (end - prompt - 1).clamp_min(0).squeeze(1).float()
                     + torch.randn(b, generator=gen, device="cuda"))
    else:
        places, total = _adamw8_places(case)
        flat = {"p": torch.zeros(total, dtype=dtype, device="cuda"), "g": torch.zeros(total, dtype=dtype, device="cuda")}
        m, v = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
        for o, shape in places:
            n = math.prod(shape)
            size = torch.rand(n, generator=gen, device="cuda").mul_(6.0).sub_(13.0).exp_()  # 2e-6 to 1e-3
            flat["p"][o:o + n] = _randn((n,), dtype, gen, 0.02)
            flat["g"][o:o + n] = (size * torch.randn(n, generator=gen, device="cuda")).to(dtype)
            m[o:o + n] = size * torch.randn(n, generator=gen, device="cuda") * 0.3
            v[o:o + n] = size.square() * (0.5 + torch.rand(n, generator=gen, device="cuda"))
        half = torch.full((total,), 1 << 19, dtype=torch.int32, device="cuda")
        flat["mc"], flat["ms"] = _encode(m, half, 14)
        flat["vc"], flat["vs"] = _encode(v, half, 30)
        s.update(flat=flat, total=total)
        if own:
            s.update(optimizer=_optimizer(flat, places))
    return s


def _optimizer(flat: dict, places: list):
    """A run under way: the optimizer over the parameters, its state as a checkpoint restores it."""

    from picotron_amd.optim import AdamW8bit

    params = []
    for o, shape in places:
        p = torch.nn.Parameter(flat["p"][o:o + math.prod(shape)].view(shape))
        p.grad = flat["g"][o:o + math.prod(shape)].view(shape)
        params.append(p)
    optimizer = AdamW8bit(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=SEED)
    for p, (o, _) in zip(params, places):
        blocks = (p.numel() + BLOCK - 1) // BLOCK
        part = lambda t: t[o:o + blocks * BLOCK].view(blocks, BLOCK)  # noqa: B023, E731
        scale = lambda t: t[o // BLOCK:o // BLOCK + blocks]  # noqa: B023, E731
        optimizer.state[p] = {"step": torch.tensor(float(STEP - 1)), "exp_avg": part(flat["mc"]), "exp_avg_scale": scale(flat["ms"]),
                              "exp_avg_sq": part(flat["vc"]), "exp_avg_sq_scale": scale(flat["vs"])}
    return optimizer


# ---------------------------------------------------------------------- one pass


def run(s: dict):
    kind = s["kind"]
    if not own:
        with torch.no_grad():
            return {"rope": _plain_rope, "score": _plain_score, "preference": _plain_preference, "adamw8": _plain_adamw8}[kind](s)
    from picotron_amd.nn.triton_kernels import triton_adamw_step, triton_apply_rotary_at, triton_preference_loss, triton_sequence_log_probs

    if kind == "rope":
        rotate = functools.partial(triton_apply_rotary_at, s["q"], s["k"], s["positions"], _plan(s["rotary_dim"], s["scaling"]), layout=s["layout"])
        if not s["train"]:
            with torch.no_grad():
                return list(rotate())
        q, k = rotate()
        return [q.detach(), k.detach(), *torch.autograd.grad([q, k], [s["q"], s["k"]], [s["dq"], s["dk"]])]
    if kind == "score":
        with torch.no_grad():
            return [triton_sequence_log_probs(s["logits"], s["labels"])]
    if kind == "preference":
        out = triton_preference_loss(s["logits"], s["labels"], s["reference"], beta=0.1, label_smoothing=0.05)
        scaled = out.loss * LOSS_SCALE if s["dtype"] == "fp16" else out.loss
        return [out.loss.detach(), out.chosen_rewards, out.rejected_rewards, *torch.autograd.grad(scaled, [s["logits"]])]
    triton_adamw_step(s["optimizer"])
    m, v, _ = s["optimizer"].moments(torch.bfloat16)
    return [s["flat"]["p"], m, v]


# ---------------------------------------------------------------------- plain forms


def _frequencies(rotary_dim: int, scaling: str) -> tuple[Tensor, float]:
    """Radians per position of each pair (64 bits), and the factor on cosine and sine."""

    c = SCALINGS[scaling]
    i = torch.arange(rotary_dim // 2, device="cuda", dtype=torch.float64)
    theta = THETA * c["factor"] ** (rotary_dim / max(rotary_dim - 2, 1)) if scaling == "ntk" else THETA
    f = theta ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        return f / c["factor"], 1.0
    if scaling == "yarn":
        length = c["original_max_positions"]
        at = lambda turns: rotary_dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(THETA))  # noqa: E731
        low, high = max(math.floor(at(c["beta_fast"])), 0), min(math.ceil(at(c["beta_slow"])), rotary_dim - 1)
        t = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - t) + f / c["factor"] * t, 0.1 * math.log(c["factor"]) + 1.0
    if scaling == "llama3":
        t = c["original_max_positions"] * f / (2 * math.pi)
        t = ((t - c["low_freq_factor"]) / (c["high_freq_factor"] - c["low_freq_factor"])).clamp(0, 1)
        return f / c["factor"] * (1 - t) + f * t, 1.0
    return f, 1.0


def _positions(s: dict) -> Tensor:
    p = s["positions"]
    if isinstance(p, int):
        p = p + torch.arange(s["seq"], device="cuda")
    return p if p.dim() == 2 else p[None]


def _plain_rope(s: dict) -> list[Tensor]:
    f, factor = _frequencies(s["rotary_dim"], s["scaling"])
    angle = (_positions(s).double()[..., None] * f)[:, None]  # (batch or 1, 1, seq, pairs)
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    r = s["rotary_dim"]

    def rotate(x: Tensor, sin: Tensor) -> Tensor:
        y = x[..., :r].float()
        a, b = (y[..., 0::2], y[..., 1::2]) if s["layout"] == "interleaved" else (y[..., : r // 2], y[..., r // 2 :])
        a, b = a * cos - b * sin, a * sin + b * cos
        y = torch.stack((a, b), -1).flatten(-2) if s["layout"] == "interleaved" else torch.cat((a, b), -1)
        return torch.cat((y.to(x.dtype), x[..., r:]), -1)

    out = [rotate(s["q"], sin), rotate(s["k"], sin)]
    return out + [rotate(s["dq"], -sin), rotate(s["dk"], -sin)] if s["train"] else out


def _log_probs(s: dict) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Per sequence, the sum over its kept tokens (in 64 bits: the loss takes its difference from another such
    sum); and the logits in 32 bits, each row's log-sum-exp, and its label."""

    x, labels = s["logits"][:, :-1].float(), s["labels"][:, 1:, None]
    top = x.amax(-1, keepdim=True)
    lse = top + (x - top).exp().sum(-1, keepdim=True).log()
    token = torch.where(labels != IGNORED, x.gather(-1, labels.clamp_min(0)) - lse, 0.0)
    return token.double().sum((1, 2)), x, lse, labels


def _plain_score(s: dict) -> list[Tensor]:
    return [_log_probs(s)[0].float()]


def _plain_preference(s: dict) -> list[Tensor]:
    beta, smooth, pairs = 0.1, 0.05, s["batch"] // 2
    log_probs, x, lse, labels = _log_probs(s)
    rewards = beta * (log_probs - s["reference"])
    h = (rewards[:pairs] - rewards[pairs:]).float()
    rewards = rewards.float()
    soft = lambda y: y.clamp_min(0) + (1 + (-y.abs()).exp()).log()  # noqa: E731 (ln(1 + e^y))
    loss = ((1 - smooth) * soft(-h) + smooth * soft(h)).mean()
    slope = (smooth / (1 + (-h).exp()) - (1 - smooth) / (1 + h.exp())) * (beta / pairs)
    scale = LOSS_SCALE if s["dtype"] == "fp16" else 1.0
    slope = torch.where(labels != IGNORED, torch.cat((slope, -slope))[:, None, None] * scale, 0.0)
    grad = (x - lse).exp() * -slope
    grad.scatter_add_(-1, labels.clamp_min(0), slope)
    whole = torch.zeros_like(s["logits"])
    whole[:, :-1] = grad
    return [loss, rewards[:pairs], rewards[pairs:], whole]


# The 8-bit states.  A block of 256 elements has one scale byte E: the exponent field (of the 32-bit float)
# of its largest magnitude, 16 at least.  An element is its magnitude times 2^(top - E), whose bits are
# then a short float with 3 bits behind the point and so many exponent bits as are left: a sign and 4 for
# the first moment (top 14), 5 for the second (top 30).  Rounding adds 20 random bits below the last kept
# one and drops them; a positive second moment stays above zero.


def _shift(x: Tensor, e: Tensor) -> Tensor:
    """x * 2^e in two exact steps, as 2^e itself may be no 32-bit float."""

    half = e >> 1
    return x * ((half + 127) << 23).view(torch.float32) * ((e - half + 127) << 23).view(torch.float32)


def _encode(y: Tensor, bits: Tensor, top: int) -> tuple[Tensor, Tensor]:
    y = y.view(-1, BLOCK)
    scale = (y.abs().amax(1, keepdim=True).view(torch.int32) >> 23).clamp_min(16)
    code = (_shift(y.abs(), top - scale).view(torch.int32) + bits.view(-1, BLOCK)) >> 20
    if top == 14:
        code = code | (y.view(torch.int32) >> 24) & 128
    else:
        code = torch.maximum(code, (y > 0).int())
    return code.to(torch.uint8).view(-1), scale.to(torch.uint8).view(-1)


def _decode(code: Tensor, scale: Tensor, top: int) -> Tensor:
    code = code.view(-1, BLOCK).int()
    y = _shift(((code & (127 if top == 14 else 255)) << 20).view(torch.float32), scale.int()[:, None] - top)
    return (torch.where(code > 127, -y, y) if top == 14 else y).view(-1)


def _mixed(seed: int, step: int) -> int:
    x = (seed ^ step * 0x9E3779B9) & 0xFFFFFFFF
    x = (x ^ x >> 16) * 0x7FEB352D & 0xFFFFFFFF
    x = (x ^ x >> 15) * 0x846CA68B & 0xFFFFFFFF
    return x ^ x >> 16


def _signed(x: int) -> int:
    return x - (1 << 32) if x >> 31 else x


def _down(x: Tensor, n: int) -> Tensor:
    """32-bit shift right that brings in zeros."""

    return (x >> n) & ((1 << (32 - n)) - 1)


def _random_bits(count: int, step: int) -> Tensor:
    """32 random bits an element: four elements in a row take successive states of a xorshift generator that
    starts from a hash of their place and the step."""

    x = torch.arange(count // 4, dtype=torch.int32, device="cuda") * _signed(0x9E3779B1) + _signed(_mixed(SEED, step))
    x = (x ^ _down(x, 16)) * 0x7FEB352D
    x = x ^ _down(x, 15)

    def after(x: Tensor) -> Tensor:
        x = x ^ x << 13
        x = x ^ _down(x, 17)
        return x ^ x << 5

    a = after(x)
    b = after(a)
    c = after(b)
    return torch.stack((a, b, c, after(c)), -1).view(-1)


def _plain_adamw8(s: dict) -> list[Tensor]:
    flat, (b1, b2) = s["flat"], BETAS
    step = s["step"] = s.get("step", STEP - 1) + 1
    r = _random_bits(s["total"], step)
    g = flat["g"].float()
    m = _decode(flat["mc"], flat["ms"], 14) * b1 + g * (1 - b1)
    v = _decode(flat["vc"], flat["vs"], 30) * b2 + (g * (1 - b2)) * g
    p = flat["p"].float() * (1 - LR * DECAY) - m / (v.sqrt() / math.sqrt(1 - b2**step) + EPS) * (LR / (1 - b1**step))
    if flat["p"].dtype == torch.bfloat16:
        p = ((p.view(torch.int32) + (_down(r, 8) & 0xFFFF)) & -65536).view(torch.float32)
    flat["p"].copy_(p)
    flat["mc"], flat["ms"] = _encode(m, _down(r, 12), 14)
    flat["vc"], flat["vs"] = _encode(v, (r & 0xFFFF) << 4 | _down(r, 28), 30)
    return [flat["p"], _decode(flat["mc"], flat["ms"], 14).bfloat16(), _decode(flat["vc"], flat["vs"], 30).bfloat16()]


# ---------------------------------------------------------------------- what a pass needs


def work(case: dict) -> dict:
    kind, e = case["kind"], SIZES[case["dtype"]]
    if kind == "rope":
        tokens = case["batch"] * case["seq"]
        n = tokens * (case["heads"] + case["kv_heads"])
        twice = 2 if case["train"] else 1
        places = {"offset": 0, "shared": case["seq"], "each": tokens}[case["positions"]]
        return {"bytes": twice * (2 * n * case["head_dim"] * e + 8 * places), "flops": twice * 3 * n * case["rotary_dim"]}
    if kind in ("score", "preference"):
        b, n, v = case["batch"], case["seq"], case["vocab"]
        # mean tokens of a prompt and of the padding (uniform)
        kept = b * v * max(1, n - 1 - max(0, max(1, n // 3) - 1) // 2 - (max(1, n // 8) - 1) // 2)
        if kind == "score":
            return {"bytes": kept * e + 8 * b * n, "flops": 4 * kept}
        return {"bytes": kept * e + b * n * v * e + 16 * b * n, "flops": 8 * kept}
    n = sum(math.prod(shape) for _, shape in _adamw8_places(case)[0])
    # parameter read and written, gradient read, two 8-bit states read and written with their scales, and
    # the states' values in 16 bits
    return {"bytes": n * (3 * e + 4 + 4) + 4 * n // BLOCK, "flops": 40 * n}


# ---------------------------------------------------------------------- 64-bit results


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rope": _exact_rope, "score": _exact_pairs, "preference": _exact_pairs, "adamw8": _exact_adamw8}[case["kind"]](s)


def _exact_rope(s: dict) -> list[Tensor]:
    """Rotation as multiplication by a complex number."""

    f, factor = _frequencies(s["rotary_dim"], s["scaling"])
    turn = torch.polar(torch.full((), factor, dtype=torch.float64, device="cuda"), _positions(s)[:, None, :, None].double() * f)
    r, h = s["rotary_dim"], s["rotary_dim"] // 2

    def rotate(x: Tensor, turn: Tensor) -> Tensor:
        y = x.double()
        if s["layout"] == "interleaved":
            y[..., :r] = torch.view_as_real(torch.view_as_complex(y[..., :r].unflatten(-1, (h, 2)).contiguous()) * turn).flatten(-2)
        else:
            z = torch.complex(y[..., :h], y[..., h:r]) * turn
            y[..., :h], y[..., h:r] = z.real, z.imag
        return y

    out = [rotate(s["q"], turn), rotate(s["k"], turn)]
    return out + [rotate(s["dq"], turn.conj()), rotate(s["dk"], turn.conj())] if s["train"] else out


def _exact_pairs(s: dict) -> list[Tensor]:
    logits, labels, v = s["logits"].detach(), s["labels"], s["vocab"]
    b, n = labels.shape
    kept = labels[:, 1:] != IGNORED
    at = labels[:, 1:].clamp_min(0)
    step = max(1, (1 << 27) // v)
    total = torch.zeros(b, dtype=torch.float64, device="cuda")
    for i in range(b):
        for t in range(0, n - 1, step):
            y = torch.log_softmax(logits[i, :-1][t:t + step].double(), -1).gather(1, at[i, t:t + step, None])[:, 0]
            total[i] += y[kept[i, t:t + step]].sum()
    if s["kind"] == "score":
        return [total]
    beta, smooth = 0.1, 0.05
    rewards = beta * (total - s["reference"].double())
    h = (rewards[: b // 2] - rewards[b // 2 :]).requires_grad_()
    with torch.enable_grad():
        loss = -((1 - smooth) * torch.nn.functional.logsigmoid(h) + smooth * torch.nn.functional.logsigmoid(-h)).mean()
        (slope,) = torch.autograd.grad(loss, h)
    slope = torch.cat((slope, -slope)) * (beta * (LOSS_SCALE if s["dtype"] == "fp16" else 1.0))
    grad = torch.zeros(logits.shape, dtype=torch.float64, device="cuda")
    for i in range(b):
        for t in range(0, n - 1, step):
            y = torch.softmax(logits[i, :-1][t:t + step].double(), -1).neg_()
            y[torch.arange(y.size(0), device="cuda"), at[i, t:t + step]] += 1
            grad[i, :-1][t:t + step] = y * (slope[i] * kept[i, t:t + step, None])
    return [loss.detach(), rewards[: b // 2], rewards[b // 2 :], grad]


def _exact_adamw8(s: dict) -> list[Tensor]:
    """The grid of a short float as steps: 2^(exponent - 3), no finer than the lowest exponent's."""

    flat, (b1, b2) = s["flat"], BETAS
    r = _random_bits(s["total"], STEP).long() & 0xFFFFFFFF

    def value(code: Tensor, scale: Tensor, low: int, signed: bool) -> Tensor:
        c = code.view(-1, BLOCK).double()
        size = c % 128 if signed else c
        e, f = torch.div(size, 8, rounding_mode="floor"), size % 8
        y = torch.where(e > 0, (1 + f / 8) * e.exp2(), f / 4) * (scale.double()[:, None] - 127 + low).exp2()
        return torch.where(c > 127, -y, y) if signed else y

    def grid(y: Tensor, low: int, bits: Tensor) -> Tensor:
        size = y.abs()
        top = (torch.frexp(size.amax(1, keepdim=True))[1] - 1).clamp_min(16 - 127)
        e = torch.maximum(torch.frexp(size)[1] - 1, top + low + 1)
        unit = (e - 3).double().exp2()
        q = torch.floor(size / unit + bits.view(-1, BLOCK) / 2.0**20)
        if low == -30:
            q = torch.maximum(q, (size > 0).double())
        return (q * unit * y.sign()).view(-1)

    g = flat["g"].double().view(-1, BLOCK)
    m = value(flat["mc"], flat["ms"], -14, True).mul_(b1).add_(g, alpha=1 - b1)
    v = value(flat["vc"], flat["vs"], -30, False).mul_(b2).addcmul_(g, g, value=1 - b2)
    p = flat["p"].double().view(-1, BLOCK) * (1 - LR * DECAY)
    p = p.addcdiv_(m, (v.sqrt() / math.sqrt(1 - b2**STEP)).add_(EPS), value=-LR / (1 - b1**STEP)).view(-1)
    if flat["p"].dtype == torch.bfloat16:  # 8 significant bits, rounded by 16 random ones
        unit = (torch.frexp(p)[1] - 8).double().exp2()
        p = torch.floor(p.abs() / unit + (r >> 8 & 0xFFFF) / 65536.0) * unit * p.sign()
    return [p, grid(m, -14, r >> 12), grid(v, -30, (r & 0xFFFF) << 4 | r >> 28)]
