"""AdamW with 8-bit moments, on the CPU: the codes, the rounding's expected value, the update against AdamW in 64
bits, checkpoints, and what is refused."""

from __future__ import annotations

import copy
import ctypes
import math

import pytest
import torch

from picotron_amd import _lib, ops
from picotron_amd.nn.triton_kernels import adamw
from picotron_amd.nn.triton_kernels import AdamWStepWithFallback, TritonAdamWUnavailable, triton_adamw_step, triton_clip_grad_norm_and_step
from picotron_amd.optim import BLOCK, TOP_M, TOP_V, AdamW8bit, decode, encode, mixed_seed, random_bits

NEAREST = 1 << 19


def nearest(blocks):
    return torch.full((blocks, BLOCK), NEAREST, dtype=torch.int32)


@pytest.mark.parametrize("top", [TOP_M, TOP_V])
@pytest.mark.parametrize("scale", [16, 17, 100, 127, 200, 254])
def test_every_code_keeps_its_value(top, scale):
    codes = torch.arange(256, dtype=torch.uint8).view(1, 256)
    values = decode(codes, torch.tensor([scale], dtype=torch.uint8), top)
    size = codes.double() % 128 if top == TOP_M else codes.double()
    e, f = (size / 8).floor(), size % 8
    exact = torch.where(e > 0, (1 + f / 8) * 2.0**e, f / 4) * 2.0 ** (scale - 127 - top)
    exact = torch.where((codes > 127) & (top == TOP_M), -exact, exact)
    # the second moment's 32nd exponent is only reached by rounding up: 2^(255 - 127) at a scale of 254 is infinite
    finite = exact.abs() < 2.0**128
    assert torch.equal(values.double()[finite], exact[finite]) and values[~finite].isinf().all()
    in_range = size < 8 * (top + 1)  # of a block whose largest magnitude has this scale
    back, scales = encode(torch.where(in_range, values, values.flatten()[8 * top]), nearest(1), top)
    assert scales.item() == scale
    zero = (top == TOP_M) & (codes == 128)
    assert torch.equal(back[in_range & ~zero], codes[in_range & ~zero])


def test_rounding_goes_to_a_neighbour_and_its_mean_is_the_value():
    torch.manual_seed(0)
    blocks = 64
    for top, values in ((TOP_M, torch.randn(BLOCK) * torch.logspace(-8, 0, BLOCK)), (TOP_V, torch.rand(BLOCK) * torch.logspace(-12, 0, BLOCK))):
        values[0] = 1.5  # one scale for every block
        v = values.expand(blocks, BLOCK).contiguous()
        total = torch.zeros(BLOCK, dtype=torch.float64)
        for seed in range(32):
            r = random_bits(seed * blocks // 4, blocks * BLOCK, mixed_seed(3, seed), v.device).view(blocks, BLOCK)
            codes, scales = encode(v, (r >> 12) & 0xFFFFF, top)
            got = decode(codes, scales, top).double()
            lowest = 2.0 ** (127 - 126 - top - 3 + 127 - 127)  # subnormal step at a scale of 127
            step = torch.maximum(2.0 ** (v.double().abs().log2().floor() - 3), torch.tensor(lowest, dtype=torch.float64))
            assert ((got - v.double()).abs() <= step).all()
            total += got.sum(0)
        n = 32 * blocks
        off = (total / n - values.double()).abs()
        # the error of one rounding has a standard deviation of at most step / 2; five of the mean's.  Below the lowest code
        # a positive second moment takes that code instead
        kept = slice(None) if top == TOP_M else values > lowest
        assert (off <= 5 * step[0] / 2 / math.sqrt(n))[kept].all()


def test_random_bits_do_not_depend_on_where_they_start():
    whole = random_bits(0, 4096, 12345, torch.device("cpu"))
    assert torch.equal(whole[1024:2048], random_bits(1, 1024, 12345, torch.device("cpu")))
    bits = torch.stack([(random_bits(0, 1 << 16, mixed_seed(7, 1), whole.device) >> i) & 1 for i in range(32)]).double()
    # each bit's mean over 2^16 draws: five standard deviations of 1/512
    assert ((bits.mean(1) - 0.5).abs() < 5 / 512).all()
    # and neighbours agree half of the time
    assert (((bits[:, 1:] == bits[:, :-1]).double().mean(1) - 0.5).abs() < 5 / 512).all()
    # places pass 32 bits without an error
    assert random_bits((1 << 24) - 1, 1024, 5, whole.device).shape == (1024,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_step_is_adamw_rounded(dtype):
    torch.manual_seed(1)
    hp = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    p = torch.nn.Parameter((torch.randn(3, 700) * 0.02).to(dtype))
    p.grad = (torch.randn(3, 700) * 1e-2).to(dtype)
    start = p.detach().clone()
    optimizer = AdamW8bit([p], **hp)
    optimizer.step()
    g = p.grad.double()
    m, v = 0.1 * g, 0.01 * g * g
    update = hp["lr"] * (m / 0.1) / ((v / 0.01).sqrt() + 1e-8)
    x = start.double() * (1 - 1e-3) - update
    # fp32 roundings of the parts, whose sizes are |x| and |update| at most together, and one step of the parameter's type
    # (rounded stochastically in bf16, to nearest else), a subnormal's at least
    step = torch.finfo(dtype).eps * (1.0 if dtype == torch.bfloat16 else 0.5)
    bound = step * (x.abs() + torch.finfo(dtype).tiny) + 2.0**-21 * (x.abs() + update.abs())
    assert ((p.double() - x).abs() <= bound).all()
    got_m, got_v, places = optimizer.moments()
    assert places == [(p, 0)] and got_m.numel() == 3 * 1024
    assert not got_m[2100:].any() and not got_v[2100:].any()
    # neighbours of the value: a step of the fraction's last bit, at least the block's subnormal one
    for got, want, top in ((got_m, m, TOP_M), (got_v, v, TOP_V)):
        want = torch.cat((want.flatten(), torch.zeros(9 * 256 - 2100, dtype=torch.float64))).view(9, 256)
        low = 2.0 ** (want.abs().amax(1, keepdim=True).log2().floor() + 1 - top - 3)
        size = torch.maximum(2.0 ** (want.abs().clamp_min(1e-300).log2().floor() - 3), low)
        assert ((got[:9 * 256].view(9, 256).double() - want).abs() <= size * 1.001).all()


def test_moments_follow_a_slow_average():
    """What rounding to nearest would not do: the second moment decays with beta2 = 0.999 once the gradient is gone."""

    p = torch.nn.Parameter(torch.zeros(4096))
    optimizer = AdamW8bit([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0)
    p.grad = torch.ones(4096)
    optimizer.step()
    first = optimizer.moments()[1].mean()
    p.grad = torch.zeros(4096)
    for _ in range(200):
        optimizer.step()
    # the mean of 4096 random walks, each of a standard deviation below 1/3 (a step of 1/8 is taken with a probability of 1/100,
    # two hundred times): five of the mean's
    assert abs(float(optimizer.moments()[1].mean() / first) - 0.999**200) < 5 / 3 / 64


def test_positive_second_moments_stay_positive():
    p = torch.nn.Parameter(torch.zeros(256))
    g = torch.full((256,), 1e-9)
    g[0] = 1e3
    p.grad = g
    optimizer = AdamW8bit([p])
    optimizer.step()
    assert (optimizer.moments()[1][:256] > 0).all()
    p.grad = torch.zeros(256)
    for _ in range(3):
        optimizer.step()
    assert p.isfinite().all() and (p.abs() <= 1e-2).all()


def test_a_gradient_that_is_no_number_stays_in_its_block():
    p = torch.nn.Parameter(torch.zeros(700))
    p.grad = torch.ones(700)
    p.grad[300] = float("nan")
    optimizer = AdamW8bit([p])
    optimizer.step()
    m, v, _ = optimizer.moments()
    for moment in (m, v):
        assert moment[256:512].isnan().all() and moment[:256].isfinite().all() and moment[512:].isfinite().all()
    assert p[300].isnan() and p.isnan().sum() == 1
    p.grad = torch.ones(700)
    optimizer.step()
    assert p[256:512].isnan().all() and p[:256].isfinite().all()


def _trained(dtype=torch.float32, **options):
    torch.manual_seed(2)
    params = [torch.nn.Parameter((torch.randn(s) * 0.02).to(dtype)) for s in ((5, 300), (7,), (0,), (1024,))]
    optimizer = AdamW8bit(params, lr=1e-3, seed=11, **options)
    for _ in range(3):
        for p in params:
            p.grad = torch.randn_like(p)
        optimizer.step()
    return params, optimizer


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("capturable", [False, True])
def test_checkpoint_round_trip(dtype, capturable):
    params, optimizer = _trained(dtype, capturable=capturable)
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW8bit(copies, lr=1.0)
    other.load_state_dict(copy.deepcopy(optimizer.state_dict()))
    assert other.param_groups[0]["seed"] == 11 and other.param_groups[0]["lr"] == 1e-3
    for p, q in zip(params, copies):
        q.grad = p.grad
        for key, value in optimizer.state[p].items():
            assert torch.equal(value, other.state[q][key]) and value.dtype == other.state[q][key].dtype, key
    optimizer.step()
    other.step()
    for p, q in zip(params, copies):
        assert torch.equal(p, q)
    if capturable:
        assert len({id(other.state[q]["step"]) for q in copies if q.numel()}) == 1


def test_state_of_torch_adamw_is_taken():
    torch.manual_seed(3)
    p = torch.nn.Parameter(torch.randn(300))
    q = torch.nn.Parameter(p.detach().clone())
    theirs = torch.optim.AdamW([p], lr=1e-3)
    p.grad = torch.randn(300)
    theirs.step()
    ours = AdamW8bit([q])
    ours.load_state_dict(theirs.state_dict())
    m, v, _ = ours.moments()
    # the nearest code: half a step of 1/8 (the top of each binade's spacing relative to its bottom), or of a subnormal
    state = theirs.state[p]
    for got, want in ((m[:300], state["exp_avg"]), (v[:300], state["exp_avg_sq"])):
        assert ((got - want).abs() <= want.abs() / 16 + want.abs().max() * 2.0**-16).all()
    q.grad = p.grad
    ours.step()
    with pytest.raises(ValueError, match="amsgrad"):
        AdamW8bit([q]).load_state_dict(torch.optim.AdamW([p], amsgrad=True).state_dict())


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(weight_decay=-1.0),
                                 dict(lr=torch.tensor(1.0))])
def test_constructor_refuses(bad):
    with pytest.raises(ValueError):
        AdamW8bit([torch.nn.Parameter(torch.zeros(3))], **bad)


def test_fused_step_refuses_the_cpu_and_the_stepper_falls_back():
    params, optimizer = _trained()
    before = [p.detach().clone() for p in params]
    with pytest.raises(TritonAdamWUnavailable):
        triton_adamw_step(optimizer)
    with pytest.raises(TritonAdamWUnavailable):
        triton_clip_grad_norm_and_step(optimizer, 1.0)
    assert all(torch.equal(p, b) for p, b in zip(params, before))
    with pytest.warns(RuntimeWarning, match="Triton AdamW unavailable"):
        AdamWStepWithFallback(use_triton=True).step(optimizer)
    assert not torch.equal(params[0], before[0]) and float(optimizer.state[params[0]]["step"]) == 4.0


def test_sizes():
    assert ops.adamw8_sizes() == (1024, BLOCK)


_TABLE = (ctypes.c_int64 * 8)()
_T = ctypes.addressof(_TABLE)


@pytest.mark.parametrize("args,code", [
    ((None, 1, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None, None, 0, 0, 0, None), _lib.PT_EINVAL),
    ((_T + 4, 1, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None, None, 0, 0, 0, None), _lib.PT_EINVAL),
    ((_T, -1, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None, None, 0, 0, 0, None), _lib.PT_EINVAL),
    ((_T, 2, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None, None, 0, 0, 0, None), _lib.PT_EINVAL),
    ((_T, 1, 1 << 25, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None, None, 0, 0, 0, None), _lib.PT_EUNSUPPORTED),
    ((_T, 1, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0.0, None, None, None, 0, 0, 0, None), _lib.PT_EINVAL),
    ((_T, 1, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, float("nan"), None, None, None, 0, 0, 0, None), _lib.PT_EINVAL),
    ((_T, 1, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None, None, 0, 0, 9, None), _lib.PT_EINVAL),
    ((_T, 1, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, 4096, None, None, 0, 0, 0, None), _lib.PT_EINVAL),
    ((_T, 1, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, 4096, 4100, None, 0, 0, 0, None), _lib.PT_EINVAL),
])
def test_step_entry_point_refuses(args, code):
    assert _lib.lib().pt_adamw8_step(*args) == code
    assert _lib.lib().pt_last_error().decode().startswith("pt_adamw8_step")


@pytest.mark.parametrize("args,code", [
    ((None, 1, 1, 4096, 4096, 0, None), _lib.PT_EINVAL), ((_T, 1, 1, None, 4096, 0, None), _lib.PT_EINVAL),
    ((_T, 1, 1, 4096, 4104, 0, None), _lib.PT_EINVAL), ((_T, 1, 1, 4096, 4096, 5, None), _lib.PT_EINVAL),
    ((_T, 1, 1 << 25, 4096, 4096, 0, None), _lib.PT_EUNSUPPORTED),
])
def test_moments_entry_point_refuses(args, code):
    assert _lib.lib().pt_adamw8_moments(*args) == code
    assert _lib.lib().pt_last_error().decode().startswith("pt_adamw8_moments")


def test_nothing_to_do():
    assert _lib.lib().pt_adamw8_step(None, 0, 0, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None, None, None, 0, 0, 0, None) == _lib.PT_OK
    assert _lib.lib().pt_adamw8_moments(None, 0, 0, None, None, 0, None) == _lib.PT_OK
    empty = AdamW8bit([torch.nn.Parameter(torch.zeros(0))])
    empty.param_groups[0]["params"][0].grad = torch.zeros(0)
    empty.step()
    assert empty.moments()[2] == []


def _mixed(**options):
    params = [torch.nn.Parameter(torch.randn(300, dtype=t)) for t in (torch.float32, torch.bfloat16, torch.float32, torch.bfloat16)]
    return params, AdamW8bit([dict(params=params[:3]), dict(params=params[3:], lr=1e-2)], capturable=True, **options)


def _one_count_a_launch(optimizer):
    buckets = optimizer.buckets(optimizer._with_gradients())
    steps = [step for _, _, _, step, _ in buckets]
    assert len({id(step) for step in steps}) == len(steps)
    for _, _, states, step, _ in buckets:
        assert all(state["step"] is step for state in states)
    return buckets


def test_launches_do_not_share_a_step_count():
    """A launch advances its device count, so that two launches of one step must not have the same one: parameters of
    two dtypes that start together, two groups that a checkpoint restores at one count, and counts that a program shares."""

    params, optimizer = _mixed()
    for p in params:
        p.grad = torch.ones_like(p)
    assert len(_one_count_a_launch(optimizer)) == 3
    optimizer.step()
    assert [float(optimizer.state[p]["step"]) for p in params] == [1.0] * 4
    again, restored = _mixed()
    restored.load_state_dict(optimizer.state_dict())
    for p in again:
        p.grad = torch.ones_like(p)
    assert len(_one_count_a_launch(restored)) == 3
    restored.step()
    assert [float(restored.state[p]["step"]) for p in again] == [2.0] * 4
    one = torch.tensor(2.0)
    for p in again:
        restored.state[p]["step"] = one
    _one_count_a_launch(restored)
    restored.step()
    assert [float(restored.state[p]["step"]) for p in again] == [3.0] * 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_small_moments_of_torch_adamw_are_taken(dtype):
    """Second moments far below fp16's smallest number: the codes come from the values given, not from a cast of them."""

    torch.manual_seed(4)
    p = torch.nn.Parameter(torch.randn(300))
    theirs = torch.optim.AdamW([p], lr=1e-4)
    p.grad = torch.randn(300) * 1e-5
    theirs.step()
    q = torch.nn.Parameter(p.detach().to(dtype))
    ours = AdamW8bit([q], lr=1e-4)
    ours.load_state_dict(theirs.state_dict())
    m, v, _ = ours.moments()
    state = theirs.state[p]
    # half a step of 1/8, or of the lowest code (2^-17 and 2^-33 of the largest); a positive second moment takes that code at least
    for got, want, low in ((m[:300], state["exp_avg"], 2.0**-17), (v[:300], state["exp_avg_sq"], 2.0**-32)):
        assert ((got - want).abs() <= want.abs() / 16 + want.abs().max() * low).all()
    assert (v[:300] > 0).all()
    before = q.detach().float()
    q.grad = torch.zeros_like(q)
    ours.step()
    # lr * m / sqrt(v) of one earlier gradient, (0.9 * 0.1 / 0.19) / sqrt(0.999 * 0.001 / 0.002) < 1 before the codes' roundings
    # (1/16 of m, 1/32 of the root, and a step of v's lowest code), the decay of 1e-6, and a step of the type
    assert ((q.float() - before).abs() <= 2e-4 + 1e-6 * before.abs() + torch.finfo(dtype).eps * before.abs()).all()


def test_moments_of_another_size_are_refused():
    p, q = torch.nn.Parameter(torch.zeros(300)), torch.nn.Parameter(torch.zeros(300))
    theirs, ours = torch.optim.AdamW([p]), AdamW8bit([q])
    p.grad = q.grad = torch.ones(300)
    theirs.step()
    ours.step()
    before = copy.deepcopy(ours.state_dict())
    for key in ("exp_avg", "exp_avg_sq"):
        bad = copy.deepcopy(theirs.state_dict())
        bad["state"][0][key] = torch.ones(1)
        with pytest.raises(ValueError, match=key):
            ours.load_state_dict(bad)
    for key, value in before["state"][0].items():
        assert torch.equal(ours.state[q][key], value)


def test_options_stay_where_a_loaded_group_has_none():
    ps = [torch.nn.Parameter(torch.zeros(3)) for _ in range(4)]
    ours = AdamW8bit([dict(params=ps[:1], seed=5), dict(params=ps[1:2], stochastic_rounding=True)], lr=1.0, seed=17,
                     stochastic_rounding=False, capturable=True)
    theirs = torch.optim.AdamW([dict(params=ps[2:3]), dict(params=ps[3:], lr=3e-3)], lr=2e-3)
    state = theirs.state_dict()
    for group in state["param_groups"]:
        group.pop("capturable", None)
    ours.load_state_dict(state)
    assert [(g["seed"], g["stochastic_rounding"], g["capturable"], g["lr"]) for g in ours.param_groups] == [
        (5, False, True, 2e-3), (17, True, True, 3e-3)]
    with pytest.raises(ValueError, match="groups"):
        ours.load_state_dict(torch.optim.AdamW(ps[2:]).state_dict())
    with pytest.raises(ValueError, match="groups"):
        ours.load_state_dict(torch.optim.AdamW([dict(params=[p]) for p in ps[1:]]).state_dict())


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("mine", [True, False])
def test_loaded_counts_are_the_optimizers_own(capturable, mine):
    """The count of the optimizer that the state came from does not move with this one's."""

    p, q = torch.nn.Parameter(torch.ones(5)), torch.nn.Parameter(torch.ones(5))
    first = AdamW8bit([p], capturable=capturable) if mine else torch.optim.AdamW([p])
    p.grad = q.grad = torch.ones(5)
    first.step()
    second = AdamW8bit([q], capturable=capturable)
    second.load_state_dict(first.state_dict())
    second.step()
    assert float(first.state[p]["step"]) == 1.0 and float(second.state[q]["step"]) == 2.0


def test_loaded_counts_are_fp32_scalars():

    p = torch.nn.Parameter(torch.ones(5))
    theirs = torch.optim.AdamW([p])
    p.grad = torch.ones(5)
    theirs.step()
    state = theirs.state_dict()
    state["param_groups"][0]["fused"] = True
    state["state"][0]["step"] = torch.tensor(1.0, dtype=torch.float64)
    ours = AdamW8bit([p])
    ours.load_state_dict(state)
    step = ours.state[p]["step"]
    assert step.device.type == "cpu" and step.dtype == torch.float32 and step.shape == () and float(step) == 1.0


@pytest.mark.parametrize("native", [True, False])
def test_a_shared_count_advances_once(monkeypatch, native):
    """A capturable group's parameters share one count, and still do when the group is no longer capturable.  (The launches
    themselves are left out.)"""

    params, optimizer = _trained(capturable=True)
    other, plain = _trained(capturable=True)
    steps = []
    monkeypatch.setattr(adamw, "_device_table", lambda table, device: table)
    monkeypatch.setattr(ops, "adamw8_step", lambda *args, step, **options: steps.append(step))
    if not native:
        monkeypatch.setattr(_lib, "native", None)
    for o, ps in ((optimizer, params), (plain, other)):
        o.param_groups[0]["capturable"] = False
        o.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(3))], lr=0.5))
        last = o.param_groups[1]["params"][0]
        last.grad = torch.ones(3)
        o._new_state(last, False)["step"] = o.state[ps[0]]["step"]  # a program may share it between groups
    adamw._run_8bit(optimizer, optimizer._with_gradients(), torch.device("cpu"))
    plain.step()
    assert steps == [4.0, 4.0] and float(optimizer.state[params[0]]["step"]) == float(plain.state[other[0]]["step"]) == 4.0


def test_clipping_writes_no_gradient_before_the_step_is_prepared(monkeypatch):
    """A step that cannot be prepared (its table is first needed during a capture, say) is left to the fallback, whose clipping
    reads the gradients as they were."""

    params, optimizer = _trained()
    done = []

    def prepare(table, device):
        done.append("table")
        raise TritonAdamWUnavailable("first built during graph capture")

    monkeypatch.setattr(adamw, "_scan_8bit", lambda optimizer: None)
    monkeypatch.setattr(adamw, "_plan_8bit", lambda optimizer: (optimizer._with_gradients(), torch.device("cpu")))
    monkeypatch.setattr(adamw, "_grads_of", lambda params: ([p.grad for p in params], torch.device("cpu")))
    monkeypatch.setattr(adamw, "_grad_table", lambda grads, device: (None, 1))
    monkeypatch.setattr(adamw, "_device_table", prepare)
    monkeypatch.setattr(ops, "clip_grad_norm", lambda *args: (torch.tensor(1.0), torch.tensor(0.5)))
    monkeypatch.setattr(ops, "grad_scale", lambda *args: done.append("written"))
    with pytest.raises(TritonAdamWUnavailable):
        triton_clip_grad_norm_and_step(optimizer, 1.0)
    assert done == ["table"] and float(optimizer.state[params[0]]["step"]) == 3.0
