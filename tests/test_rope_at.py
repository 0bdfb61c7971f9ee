"""Rotary embedding at positions, on the CPU: the frequencies of every scaling, the PyTorch form against exact
rational angles, the module's choice of path, and what the entry points refuse."""

from __future__ import annotations

import ctypes
import math
from fractions import Fraction

import pytest
import torch

from picotron_amd import _lib, ops
from picotron_amd.nn import RotaryEmbedding, RotaryFrequencies, apply_rotary_at
from picotron_amd.nn.triton_kernels import TritonRoPEUnavailable, triton_apply_rotary_at

PI = Fraction(31415926535897932384626433832795028841971693993751, 10**49)
YARN = dict(type="yarn", factor=16.0, original_max_positions=8192)
LLAMA3 = dict(type="llama3", factor=8.0, original_max_positions=8192)


def exact_turns(position: int, frequency: float) -> Fraction:
    return Fraction(position) * Fraction(frequency) / (2 * PI) % 1


def test_frequencies_without_scaling_are_the_tables():
    f = RotaryFrequencies(128, 5e5)
    assert f.attention_factor == 1.0 and f.frequencies[0] == 1.0
    assert abs(float(f.frequencies[1]) - 0.8146172339) < 1e-10  # 5e5^(-2/128)


@pytest.mark.parametrize("dim", [2, 20, 64, 128])
@pytest.mark.parametrize("scaling", [None, dict(type="linear", factor=4.0), dict(type="ntk", factor=8.0), YARN, LLAMA3])
def test_turns_are_the_frequencies_as_fractions_of_a_turn(dim, scaling):
    f = RotaryFrequencies(dim, 5e5, scaling=scaling)
    turns = f.turns(torch.device("cpu"))
    assert turns.dtype == torch.int64 and turns.shape == (dim // 2,)
    for bits, freq in zip(turns.tolist(), f.frequencies.tolist()):
        off = (Fraction(bits % 2**64, 2**64) - exact_turns(1, freq)) % 1
        # one rounding of f / 2 pi to 53 bits, and pi's own (2^-53): 2^-52 of at most 1/(2 pi)
        assert min(off, 1 - off) <= Fraction(1, 2**53)
    assert f.turns(torch.device("cpu")) is turns


def test_scaled_frequencies():
    base = RotaryFrequencies(64, 1e4).frequencies
    assert torch.equal(RotaryFrequencies(64, 1e4, scaling=dict(type="linear", factor=4.0)).frequencies, base / 4)
    ntk = RotaryFrequencies(64, 1e4, scaling=dict(type="ntk", factor=8.0)).frequencies
    assert ntk[0] == 1.0
    # the slowest pair is slowed by the factor itself: F^(-(d-2)/d * d/(d-2)) = 1/F
    assert math.isclose(float(ntk[-1]), float(base[-1]) / 8, rel_tol=1e-12)
    for scaling, slow, fast in ((dict(type="yarn", factor=4.0, original_max_positions=2048), 1.0, 32.0),
                                (dict(type="llama3", factor=4.0, original_max_positions=2048), 1.0, 4.0)):
        f = RotaryFrequencies(64, 1e4, scaling=scaling).frequencies
        turns = 2048 * base / (2 * math.pi)
        # whole pairs away from the ramp's ends, which yarn rounds outwards to pairs
        assert torch.allclose(f[turns > fast * 1.4], base[turns > fast * 1.4], rtol=1e-12, atol=0)
        assert torch.allclose(f[turns < slow / 1.4], base[turns < slow / 1.4] / 4, rtol=1e-12, atol=0)
        assert ((f >= base / 4 * (1 - 1e-12)) & (f <= base * (1 + 1e-12))).all()
    assert math.isclose(RotaryFrequencies(64, 1e4, scaling=dict(type="yarn", factor=4.0, original_max_positions=2048)).attention_factor,
                        0.1 * math.log(4.0) + 1.0)
    assert RotaryFrequencies(64, 1e4, scaling={**YARN, "attention_factor": 0.5}).attention_factor == 0.5


@pytest.mark.parametrize("arguments", [
    dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, theta=0.0), dict(rotary_dim=8, theta=float("inf")),
    dict(rotary_dim=8, scaling=dict(type="other", factor=2.0)), dict(rotary_dim=8, scaling=dict(type="linear")),
    dict(rotary_dim=8, scaling=dict(type="linear", factor=0.0)), dict(rotary_dim=8, scaling=dict(type="linear", factor=2.0, more=1)),
    dict(rotary_dim=8, scaling=dict(type="yarn", factor=2.0)),
    dict(rotary_dim=8, scaling={**LLAMA3, "low_freq_factor": 4.0}),
])
def test_frequencies_refuse(arguments):
    with pytest.raises(ValueError):
        RotaryFrequencies(**arguments)


@pytest.mark.parametrize("layout", ["interleaved", "rotate_half"])
@pytest.mark.parametrize("dim", [8, 6, 2])
def test_plain_form_against_rational_angles(layout, dim):
    torch.manual_seed(1)
    f = RotaryFrequencies(dim, 1e4, scaling=dict(type="yarn", factor=4.0, original_max_positions=64))
    x = torch.randn(2, 3, 4, 8, dtype=torch.float64)
    positions = torch.tensor([[0, 1, 999_983, -5], [7, 7, 2**20, 3]])
    y = apply_rotary_at(x, positions, f, layout=layout)
    assert torch.equal(y[..., dim:], x[..., dim:])
    for b in range(2):
        for s in range(4):
            for i, freq in enumerate(f.frequencies.tolist()):
                angle = 2 * math.pi * float(exact_turns(int(positions[b, s]), freq))
                c, n = math.cos(angle) * f.attention_factor, math.sin(angle) * f.attention_factor
                at = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + dim // 2)
                u, w = x[b, :, s, at[0]], x[b, :, s, at[1]]
                # the angle in 64 bits is off by 2^-53 of at most 2^20
                torch.testing.assert_close(y[b, :, s, at[0]], u * c - w * n, rtol=0, atol=4e-9)
                torch.testing.assert_close(y[b, :, s, at[1]], u * n + w * c, rtol=0, atol=4e-9)


@pytest.mark.parametrize("layout", ["interleaved", "rotate_half"])
def test_module_takes_positions_part_and_scaling(layout):
    torch.manual_seed(2)
    q, k = torch.randn(2, 4, 5, 16), torch.randn(2, 2, 5, 16)
    plain = RotaryEmbedding(16, 1e4, layout=layout)
    whole = plain(q, k)
    for positions in (0, torch.arange(5), torch.arange(5, dtype=torch.int32)[None]):
        for a, b in zip(plain(q, k, positions), whole):
            # the tables' fp32 angles are off by up to 4 * 2^-24 rad, twice the two roundings of a term
            torch.testing.assert_close(a, b, rtol=0, atol=3e-6)
    at_seven = plain(q, k, 7)[0]
    assert torch.equal(at_seven, plain(q, k, torch.arange(7, 12))[0]) and not torch.equal(at_seven, whole[0])
    part = RotaryEmbedding(16, 1e4, layout=layout, rotary_dim=4, scaling=YARN | {"original_max_positions": 64})
    out = part(q, k)[0]
    assert torch.equal(out[..., 4:], q[..., 4:]) and not torch.equal(out[..., :4], q[..., :4])


def test_module_warns_and_falls_back_on_the_cpu():
    q = torch.randn(1, 1, 3, 8)
    rope = RotaryEmbedding(8, use_triton_rope=True, rotary_dim=4)
    with pytest.warns(RuntimeWarning, match="Triton RoPE unavailable"):
        out = rope(q, q)
    torch.testing.assert_close(out[0], apply_rotary_at(q, None, rope.frequencies))


@pytest.mark.parametrize("rotary_dim", [0, 9, 10, 7])
def test_module_refuses_a_part_that_is_none(rotary_dim):
    with pytest.raises(ValueError):
        RotaryEmbedding(8, rotary_dim=rotary_dim)


def test_fast_path_refuses_cpu_tensors():
    with pytest.raises(TritonRoPEUnavailable):
        triton_apply_rotary_at(torch.randn(1, 1, 3, 8), None, 0, RotaryFrequencies(8))


@pytest.mark.parametrize("shape", [(3,), (2, 3), (3, 4), (4, 1), (1,), (4, 4, 1), ()])
def test_positions_of_another_shape_are_refused(shape):
    with pytest.raises(ValueError, match="positions must be"):
        ops._position_strides(torch.zeros(shape, dtype=torch.int64), 2, 4)


def test_positions_strides():
    p = torch.arange(24).view(4, 6)
    assert ops._position_strides(p[:2, ::2], 2, 3) == (6, 2)
    assert ops._position_strides(p[:1, ::2], 2, 3) == (0, 2)
    assert ops._position_strides(p[1], 4, 6) == (0, 1)
    assert ops._position_strides(p[:, :1].expand(4, 6), 4, 6) == (6, 0)
    with pytest.raises(ValueError, match="int32 or int64"):
        ops._position_strides(p.float(), 4, 6)


_DESC = (ctypes.c_int64 * 9)(1, 1, 1, 8, 8, 8, 8, 8, 8)
_D = ctypes.addressof(_DESC)


# Addresses that are never read: the checks come before any launch.
@pytest.mark.parametrize("change,code", [
    (dict(dtype=7), _lib.PT_EINVAL), (dict(layout=2), _lib.PT_EINVAL), (dict(head_dim=7), _lib.PT_EINVAL),
    (dict(head_dim=0), _lib.PT_EINVAL), (dict(rotary_dim=0), _lib.PT_EINVAL), (dict(rotary_dim=3), _lib.PT_EINVAL),
    (dict(rotary_dim=10), _lib.PT_EINVAL), (dict(position_bytes=2), _lib.PT_EINVAL), (dict(positions=4100), _lib.PT_EINVAL),
    (dict(turns=None), _lib.PT_EINVAL), (dict(turns=4100), _lib.PT_EINVAL), (dict(desc0=None), _lib.PT_EINVAL),
    (dict(x0=None), _lib.PT_EINVAL), (dict(y0=4096), _lib.PT_EINVAL), (dict(x1=4096), _lib.PT_EINVAL),
    (dict(desc0=ctypes.addressof((ctypes.c_int64 * 9)(1, -1, 1, 8, 8, 8, 8, 8, 8))), _lib.PT_EINVAL),
    (dict(rows=(1 << 20, 1 << 12, 1)), _lib.PT_EUNSUPPORTED), (dict(rows=(1 << 30, 1 << 30, 1 << 30)), _lib.PT_EUNSUPPORTED),
    (dict(rows=(1 << 32, 1, 1)), _lib.PT_EINVAL),
])
def test_entry_point_refuses(change, code):
    a = dict(x0=4096, y0=8192, desc0=_D, x1=None, y1=None, desc1=None, head_dim=8, rotary_dim=8, positions=4096, position_bytes=8,
             pbs=0, pss=1, offset=0, turns=4096, scale=1.0, layout=0, inverse=0, dtype=0, stream=None)
    rows = change.pop("rows", None) if "rows" in change else None
    if rows:
        desc = (ctypes.c_int64 * 9)(*rows, 8, 8, 8, 8, 8, 8)
        change = {"desc0": ctypes.addressof(desc)}
    a.update(change)
    assert _lib.lib().pt_rope_at(*a.values()) == code
    assert _lib.lib().pt_last_error().decode().startswith("pt_rope_at")


def test_empty_tensors_are_no_ops():
    desc = (ctypes.c_int64 * 9)(2, 0, 3, 8, 8, 8, 8, 8, 8)
    assert _lib.lib().pt_rope_at(None, None, desc, None, None, None, 8, 8, None, 0, 0, 0, 0, 4096, 1.0, 0, 0, 0, None) == _lib.PT_OK


def test_frequencies_are_the_hosts_under_another_default_device():
    want = RotaryFrequencies(16, scaling=dict(type="yarn", factor=4.0, original_max_positions=128))
    with torch.device("meta"):
        f = RotaryFrequencies(16, scaling=dict(type="yarn", factor=4.0, original_max_positions=128))
        turns = f.turns(torch.device("cpu"))
    assert torch.equal(f.frequencies, want.frequencies) and torch.equal(turns, want.turns(torch.device("cpu")))


def test_turns_of_an_inference_pass_serve_training():
    with torch.inference_mode():
        f = RotaryFrequencies(16)
        turns = f.turns(torch.device("cpu"))
    assert not turns.is_inference() and not f.frequencies.is_inference()


@pytest.mark.parametrize("dim,theta", [(2, 1e4), (64, 1e4), (128, 5e5), (128, 0.5), (256, 1e9)])
@pytest.mark.parametrize("scaling", [None, dict(type="linear", factor=3.0), YARN, LLAMA3])
def test_turns_are_rounded_once(dim, theta, scaling):
    f = RotaryFrequencies(dim, theta, scaling=scaling)
    for bits, freq in zip(f.turns(torch.device("cpu")).tolist(), f.frequencies.tolist()):
        off = (Fraction(bits % 2**64, 2**64) - exact_turns(1, freq)) % 1
        assert min(off, 1 - off) <= Fraction(1, 2**65)  # PI has as many digits as the turns were formed with


@pytest.mark.parametrize("scaling", [None, YARN, LLAMA3])
def test_first_use_compiles(scaling):
    """Nothing has asked for the turns before the module is traced."""

    torch._dynamo.reset()
    q = torch.randn(1, 2, 3, 8)
    rope = RotaryEmbedding(8, rotary_dim=4, scaling=scaling)
    turns = torch.compile(lambda x: rope.frequencies.turns(x.device) + x.sum().long() * 0, backend="aot_eager", fullgraph=True)
    assert torch.equal(turns(q), RotaryFrequencies(4, scaling=scaling).turns(q.device))
    assert torch.equal(rope.frequencies.turns(q.device), RotaryFrequencies(4, scaling=scaling).turns(q.device))


def test_modules_are_built_without_data():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        RotaryEmbedding(8, rotary_dim=4, scaling=YARN)


@pytest.mark.parametrize("layout", ["interleaved", "rotate_half"])
@pytest.mark.parametrize("far", [2**20, 2**31, 2**40, 2**48])
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32])
def test_plain_form_at_far_positions(layout, far, dtype):
    f = RotaryFrequencies(16, 5e5, scaling=YARN)
    positions = [far, far - 1, far // 3, -far + 7]
    y = apply_rotary_at(torch.ones(1, 1, 4, 16, dtype=dtype), torch.tensor(positions), f, layout=layout)[0, 0].double()
    a = f.attention_factor
    for row, p in zip(y, positions):
        for i, freq in enumerate(f.frequencies.tolist()):
            angle = 2 * math.pi * float(exact_turns(p, freq))
            u, w = (row[2 * i], row[2 * i + 1]) if layout == "interleaved" else (row[i], row[i + 8])
            # for |u| + |w| = 2: the turns' rounding of 2^-65 a position, the angle's in 64 bits (2^-51), and four roundings of
            # the type: cosine, its factor, the product, the sum
            bound = 2 * a * (2 * math.pi * abs(p) * 2.0**-65 + 2.0**-51 + 4 * torch.finfo(dtype).eps / 2)
            assert abs(float(u) - a * (math.cos(angle) - math.sin(angle))) <= bound, (p, i)
            assert abs(float(w) - a * (math.cos(angle) + math.sin(angle))) <= bound, (p, i)
    whole = apply_rotary_at(torch.ones(1, 1, 2, 16), torch.tensor([2**63 - 1, -(2**63)]), f, layout=layout)
    assert whole.isfinite().all()


def test_turns_of_a_dry_run_are_not_kept(monkeypatch):
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    f = RotaryFrequencies(8)
    with FakeTensorMode(allow_non_fake_inputs=True):
        assert isinstance(f.turns(torch.device("cuda", 0)), FakeTensor)
    assert not f._turns


def test_plain_form_refuses_another_layout():
    with pytest.raises(ValueError, match="layout"):
        apply_rotary_at(torch.randn(1, 1, 3, 8), 0, RotaryFrequencies(8), layout="half")


@pytest.mark.parametrize("position", [2.7, -0.5, float("nan"), "3"])
def test_a_position_that_is_no_integer_is_refused(position):
    x, f = torch.randn(1, 1, 3, 8), RotaryFrequencies(8)
    for call in (lambda: apply_rotary_at(x, position, f), lambda: RotaryEmbedding(8)(x, x, position), lambda: ops._first_position(position)):
        with pytest.raises(ValueError):
            call()


def test_positions_that_are_integers():
    import numpy as np

    for position in (None, 0, 5, -3, 2**62, True, 4.0, np.int64(7), np.int32(-1)):
        assert ops._first_position(position) == int(position or 0)


@pytest.mark.parametrize("arguments", [(8, float("inf")), (0,), (128, 1e-320)])
def test_modules_without_positions_take_what_the_tables_take(arguments):
    q = torch.randn(1, 2, 3, arguments[0])
    rope = RotaryEmbedding(*arguments)
    assert rope(q, q)[0].shape == q.shape
    with pytest.raises((ValueError, OverflowError)):
        rope(q, q, 5)
    with pytest.raises((ValueError, OverflowError)):
        RotaryEmbedding(*arguments, scaling=dict(type="linear", factor=2.0))


def test_a_module_stored_before_it_had_frequencies():
    rope, q = RotaryEmbedding(8), torch.randn(1, 2, 3, 8)
    want = rope(q, q)[0], rope(q, q, 5)[0]
    for name in ("frequencies", "_plain"):
        rope.__dict__.pop(name, None)
    assert torch.equal(rope(q, q)[0], want[0]) and torch.equal(rope(q, q, 5)[0], want[1])


@pytest.mark.parametrize("rotary_dim", [None, 4])
def test_a_module_loaded_onto_another_device(rotary_dim):
    """What it kept for its device lies elsewhere after a load with a map_location (the meta device stands in for it)."""

    rope, q = RotaryEmbedding(8, rotary_dim=rotary_dim), torch.randn(1, 2, 3, 8)
    want = rope(q, q)[0], rope(q, q, 5)[0]
    cpu = q.device
    rope._fp32_tables[cpu] = tuple(t.to("meta") for t in rope._tables_fp32(9, cpu))
    rope.frequencies._turns[cpu] = rope.frequencies.turns(cpu).to("meta")
    assert torch.equal(rope(q, q, 5)[0], want[1]) and torch.equal(rope(q, q)[0], want[0])
    assert {t.device for t in (rope.frequencies.turns(cpu), *rope._tables_fp32(3, cpu))} == {cpu}
    kept = rope.frequencies.turns(cpu)
    assert rope.frequencies.turns(cpu) is kept


def test_frequencies_stored_before_they_had_their_bits():
    import copy

    f = RotaryFrequencies(8, scaling=YARN)
    old = copy.copy(f)
    state = {key: value for key, value in f.__dict__.items() if key != "_bits"}
    old.__dict__.clear()
    old.__setstate__({**state, "_turns": {}})
    assert torch.equal(old.turns(torch.device("cpu")), f.turns(torch.device("cpu")))


def test_numbers_of_any_kind():
    import numpy as np

    want = RotaryFrequencies(16, 5e5, scaling=dict(type="yarn", factor=4.0, original_max_positions=128, beta_fast=32.0))
    for number in (np.float64, lambda x: np.float32(x), lambda x: torch.tensor(x, dtype=torch.float64), int):
        f = RotaryFrequencies(16, number(5e5), scaling=dict(type="yarn", factor=number(4), original_max_positions=number(128),
                                                            beta_fast=number(32)))
        assert torch.equal(f.turns(torch.device("cpu")), want.turns(torch.device("cpu"))) and f.attention_factor == want.attention_factor
        q = torch.randn(1, 2, 3, 16)
        assert torch.equal(RotaryEmbedding(16, number(5e5))(q, q, 3)[0], RotaryEmbedding(16, 5e5)(q, q, 3)[0])
