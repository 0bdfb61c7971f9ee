"""The AdamW step with 8-bit moments on the GPU: its codes are the PyTorch form's bit for bit, its parameters that
form's to fp32 rounding; sizes around the blocks, alignments, groups, captures, streams, clipping and refusals."""

from __future__ import annotations

import copy

import pytest
import torch

from gpu_util import randn
from picotron_amd import _lib, ops
from picotron_amd.nn.triton_kernels import (
    AdamWStepWithFallback,
    TritonAdamWUnavailable,
    triton_adamw_step,
    triton_clip_grad_norm_and_step,
    triton_unscale_clip_and_step,
)
from picotron_amd.optim import AdamW8bit

pytestmark = pytest.mark.gpu

HP = dict(lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
KEYS = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
SHAPES = [(1000, 37), (1,), (255,), (256,), (257,), (0,), (1023,), (1024,), (1025,), (3, 5, 7), (4097,)]


def pair(shapes, dtype, device, **options):
    """(parameters, optimizer) twice, on equal values."""

    first = [torch.nn.Parameter(randn(s, dtype, device, i, 0.02)) for i, s in enumerate(shapes)]
    second = [torch.nn.Parameter(p.detach().clone()) for p in first]
    return (first, AdamW8bit(first, **{**HP, **options})), (second, AdamW8bit(second, **{**HP, **options}))


def gradients(seed, *lists, scale=1e-3):
    for i, same in enumerate(zip(*lists)):
        g = randn(same[0].shape, same[0].dtype, same[0].device, 1000 * seed + i, scale)
        for p in same:
            p.grad = g.clone()


def same_codes(a, b, optimizer_a, optimizer_b):
    for p, q in zip(a, b):
        if p.numel():
            for key in KEYS:
                assert torch.equal(optimizer_a.state[p][key], optimizer_b.state[q][key]), (tuple(p.shape), key)
            assert float(optimizer_a.state[p]["step"]) == float(optimizer_b.state[q]["step"])


def close_parameters(a, b, steps, lr=1e-3):
    """The square root and the reciprocal are off by an ulp each, the rest by an fp32 rounding a term: 2^-21 of the update a step
    (below 10 lr with these moments), 2^-22 of the parameter; in 16 bits a value beside a border may round to the next step."""

    for p, q in zip(a, b):
        step = torch.finfo(p.dtype).eps if p.dtype != torch.float32 else 0.0
        bound = steps * (2.0**-21 * 10 * lr + (2.0**-22 + step) * q.double().abs() + step * torch.finfo(p.dtype).tiny)
        off = (p.double() - q.double()).abs()
        assert (off <= bound).all()
        if step and p.numel():  # an fp32 difference of 2^-21 changes the rounding of a 16-bit step of 2^-10 now and then
            assert (off > 0).float().mean() <= 0.02 * steps + 1 / p.numel()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("stochastic", [True, False])
def test_steps_have_the_plain_forms_codes(gpu, dtype, stochastic):
    (a, fused), (b, plain) = pair(SHAPES, dtype, gpu, seed=5, stochastic_rounding=stochastic)
    for step in range(4):
        gradients(step, a, b, scale=0.1 if dtype == torch.float16 else 1e-3)
        triton_adamw_step(fused)
        plain.step()
        same_codes(a, b, fused, plain)
        close_parameters(a, b, step + 1)
    for p in a:  # the bytes behind the last element stay zero
        if p.numel():
            for key in ("exp_avg", "exp_avg_sq"):
                assert not fused.state[p][key].view(-1)[p.numel():].any()
    for x, y in zip(fused.moments(torch.float32)[:2], plain.moments()[:2]):
        assert torch.equal(x, y)


def test_range_of_magnitudes(gpu):
    """Blocks over the whole range of fp32, a tiny value beside the largest, zeros, and whole blocks of them."""

    (a, fused), (b, plain) = pair([(256 * 40,)], torch.float32, gpu, lr=0.0, weight_decay=0.0)
    g = torch.randn(40, 256, device=gpu) * torch.logspace(-40, 18, 40, device=gpu)[:, None]
    g[3:5] = 0.0
    g[10, :250] *= 1e-6
    g[20, ::2] = 0.0
    for step in range(3):
        for p in (a[0], b[0]):
            p.grad = (g * (step + 1)).view(-1)
        triton_adamw_step(fused)
        plain.step()
        same_codes(a, b, fused, plain)


def test_special_gradients(gpu):
    (a, fused), (b, plain) = pair([(1000,), (300,)], torch.float32, gpu)
    gradients(1, a, b)
    for p in (a[0], b[0]):
        p.grad[5], p.grad[600], p.grad[999] = float("inf"), float("nan"), 3e38  # whose square is infinite
    for _ in range(2):
        triton_adamw_step(fused)
        plain.step()
        same_codes(a, b, fused, plain)
        for p, q in zip(a, b):
            assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p.isinf(), q.isinf())
        for x, y in zip(fused.moments()[:2], plain.moments()[:2]):
            assert torch.equal(x.isnan(), y.isnan())
    assert a[1].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unaligned_parameters(gpu, dtype):
    flat_p, flat_g = randn((5000,), dtype, gpu, 1, 0.02), randn((5000,), dtype, gpu, 2, 1e-3)
    a = [torch.nn.Parameter(flat_p[o:o + n]) for o, n in ((1, 700), (703, 1024), (1731, 3000))]
    for p, o in zip(a, (2, 705, 1734)):
        p.grad = flat_g[o:o + p.numel()]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    around = flat_p[[0, 701, 702, 1727, 1728, 1729, 1730, 4731]].clone()
    fused, plain = AdamW8bit(a, **HP), AdamW8bit(b, **HP)
    triton_adamw_step(fused)
    plain.step()
    same_codes(a, b, fused, plain)
    close_parameters(a, b, 1)
    assert torch.equal(flat_p[[0, 701, 702, 1727, 1728, 1729, 1730, 4731]], around)


def test_groups_types_and_late_parameters(gpu):
    """Two groups with values of their own, two types in one, and a parameter whose gradient comes later."""

    def build():
        ps = [torch.nn.Parameter(randn(s, d, gpu, i, 0.02)) for i, (s, d) in enumerate(
            [((300,), torch.float32), ((64, 65), torch.bfloat16), ((700,), torch.float32), ((2000,), torch.float32)])]
        return ps, AdamW8bit([dict(params=ps[:2], lr=1e-2, weight_decay=0.0), dict(params=ps[2:])], **HP)

    (a, fused), (b, plain) = build(), build()
    for step in range(3):
        gradients(step, a, b)
        if step == 0:
            a[3].grad = b[3].grad = None
        triton_adamw_step(fused)
        plain.step()
        same_codes(a[:3] if step == 0 else a, b[:3] if step == 0 else b, fused, plain)
        close_parameters(a, b, step + 1, lr=1e-2)
    assert float(fused.state[a[3]]["step"]) == 2.0 and float(fused.state[a[0]]["step"]) == 3.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_moments(gpu, dtype):
    a, fused = pair(SHAPES, torch.float32, gpu)[0]
    gradients(0, a)
    triton_adamw_step(fused)
    m, v, places = fused.moments(dtype)
    host = AdamW8bit([torch.nn.Parameter(p.detach().cpu()) for p in a], **HP)
    host.load_state_dict(copy.deepcopy(fused.state_dict()))
    hm, hv, host_places = host.moments(torch.float32)
    assert [at for _, at in places] == [at for _, at in host_places] and m.numel() == hm.numel()
    if dtype == torch.float16:  # out of its range: rounded
        assert torch.equal(m.cpu(), hm.half()) and torch.equal(v.cpu(), hv.half())
    else:
        assert torch.equal(m.cpu().float(), hm) and torch.equal(v.cpu().float(), hv)


def test_clip_and_step(gpu):
    for write_back in (True, False):
        (a, fused), (b, plain) = pair(SHAPES, torch.float32, gpu)
        gradients(3, a, b, scale=0.1)
        raw = [p.grad.clone() for p in a]
        norm = triton_clip_grad_norm_and_step(fused, 1.0, write_back_grads=write_back)
        want = torch.nn.utils.clip_grad_norm_(b, 1.0)
        torch.testing.assert_close(norm, want, rtol=1e-5, atol=0)
        for p, q, r in zip(a, b, raw):
            # the norms differ by the order of their sums
            torch.testing.assert_close(p.grad, q.grad if write_back else r, rtol=1e-5, atol=0)
            p.grad.copy_(q.grad)
        plain.step()
        for x, y in zip(fused.moments()[:2], plain.moments()[:2]):
            # gradients 1e-5 apart: the same code but beside a border
            assert (x != y).float().mean() < 1e-3
    sixteen = pair([(300,)], torch.bfloat16, gpu)[0]
    gradients(1, sixteen[0])
    with pytest.raises(TritonAdamWUnavailable):
        triton_clip_grad_norm_and_step(sixteen[1], 1.0)


def test_stepper_runs_the_kernel(gpu):
    (a, fused), (b, plain) = pair(SHAPES, torch.bfloat16, gpu)
    gradients(0, a, b)
    stepper = AdamWStepWithFallback(use_triton=True)
    stepper.step(fused)
    assert not stepper._fallback_warned
    plain.step()
    same_codes(a, b, fused, plain)
    with pytest.warns(RuntimeWarning, match="Triton AdamW unavailable"):  # 16-bit gradients are clipped by torch
        stepper.step(fused, max_grad_norm=1.0)
    assert float(fused.state[a[0]]["step"]) == 2.0


@pytest.mark.parametrize("scale", [1.0, 0.25, float("inf"), float("nan")])
def test_scaled_step(gpu, scale):
    """What a clip coefficient does; an infinite one reaches no byte behind the end."""

    (a, fused), (b, plain) = pair([(700,), (1025,)], torch.float32, gpu)
    gradients(0, a, b)
    (_, params, states, step, seed), = fused.buckets(fused._with_gradients())
    table, blocks = ops.adamw8_table(params, [p.grad for p in params], states)
    ops.adamw8_step(table.to(gpu), blocks, torch.float32, lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1,
                    step=step + 1, seed=seed, stochastic=True, grad_scale=torch.tensor(scale, device=gpu))
    for p in b:
        p.grad *= scale
    plain.step()
    for p, q in zip(a, b):
        for key in KEYS:
            assert torch.equal(fused.state[p][key], plain.state[q][key])
        assert torch.equal(p.isnan(), q.isnan())


def test_capturable_steps_replay(gpu):
    options = dict(capturable=True, seed=9)
    (a, graphed), (b, eager) = pair(SHAPES, torch.bfloat16, gpu, **options)
    c, plain = pair(SHAPES, torch.bfloat16, gpu, **options)[0]
    for p in a:
        p.grad = torch.zeros_like(p)
    with pytest.raises(TritonAdamWUnavailable, match="captured"):  # no state yet
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            triton_adamw_step(graphed)
    assert not graphed.state
    gradients(0, a, b, c)
    held = [p.grad for p in a]
    triton_adamw_step(graphed)
    triton_adamw_step(eager)
    plain.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        triton_adamw_step(graphed)
    for step in range(1, 5):
        gradients(step, b, c)
        for g, p in zip(held, b):
            g.copy_(p.grad)
        graph.replay()
        torch.cuda.synchronize()
        triton_adamw_step(eager)
        plain.step()
        same_codes(a, b, graphed, eager)
        same_codes(a, c, graphed, plain)
        for p, q in zip(a, b):
            assert torch.equal(p, q)
    assert float(graphed.state[a[0]]["step"]) == 5.0
    host = pair([(300,)], torch.float32, gpu)[0]
    gradients(0, host[0])
    triton_adamw_step(host[1])
    with pytest.raises(TritonAdamWUnavailable, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            triton_adamw_step(host[1])
    assert float(host[1].state[host[0][0]]["step"]) == 1.0


def test_another_stream_and_a_checkpoint(gpu):
    (a, fused), (b, plain) = pair(SHAPES, torch.float32, gpu)
    gradients(0, a, b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        triton_adamw_step(fused)
    torch.cuda.current_stream().wait_stream(stream)
    plain.step()
    same_codes(a, b, fused, plain)
    resumed = AdamW8bit(a, **HP)
    resumed.load_state_dict(copy.deepcopy(fused.state_dict()))
    gradients(1, a, b)
    triton_adamw_step(resumed)
    plain.step()
    same_codes(a, b, resumed, plain)


def test_many_tensors_and_a_large_one(gpu):
    """More records than a round of the search takes, and offsets of more than 2^31 elements behind them."""

    shapes = [(n,) for n in range(1, 340)] + [((1 << 31) + 5,)]
    a = [torch.nn.Parameter(torch.zeros(s, dtype=torch.bfloat16, device=gpu)) for s in shapes]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a[:-1]]
    gradients(0, a[:-1], b)
    big = a[-1]
    big.grad = torch.zeros_like(big)
    tail = randn((2053,), torch.bfloat16, gpu, 7, 1e-3)
    big.grad[-2053:] = tail
    fused, plain = AdamW8bit(a, **HP), AdamW8bit(b, **HP)
    triton_adamw_step(fused)
    plain.step()
    same_codes(a[:-1], b, fused, plain)
    state = fused.state[big]
    assert not state["exp_avg"][:-10].any() and state["exp_avg"].view(-1)[-251 - 1024:-251].any()
    assert not big[: -2053].any() and (big[-2053:] != 0).sum() == (tail != 0).sum()


@pytest.mark.parametrize("case", ["gradient", "layout", "state", "scale", "lr", "device"])
def test_refusals_change_nothing(gpu, case):
    a, fused = pair([(300,), (40, 8)], torch.float32, gpu)[0]
    gradients(0, a)
    triton_adamw_step(fused)
    if case == "gradient":
        a[0].grad = None
        a[0].data = a[0].data.bfloat16()
        a[0].grad = torch.zeros(300, dtype=torch.bfloat16, device=gpu)
        a[0].data = a[0].data.float()
    elif case == "layout":
        a[1].grad = torch.randn(8, 40, device=gpu).t()
    elif case == "state":
        fused.state[a[0]]["exp_avg"] = fused.state[a[0]]["exp_avg"][:1]
    elif case == "scale":
        fused.state[a[0]]["exp_avg_sq_scale"] = fused.state[a[0]]["exp_avg_sq_scale"].float()
    elif case == "lr":
        fused.param_groups[0]["lr"] = torch.tensor(1e-3)
    else:
        fused.state[a[0]]["exp_avg_sq"] = fused.state[a[0]]["exp_avg_sq"].cpu()
    before = [p.detach().clone() for p in a]
    with pytest.raises(TritonAdamWUnavailable):
        triton_adamw_step(fused)
    for p, q in zip(a, before):
        assert torch.equal(p, q) and float(fused.state[p]["step"]) == 1.0


def test_capturable_launches_of_several_dtypes_and_groups(gpu):
    """Two dtypes in a group and a second group, restored from a checkpoint: each launch counts for itself."""

    def made():
        params = [torch.nn.Parameter(randn((n,), t, gpu, n, 0.1)) for n, t in
                  ((300, torch.float32), (1300, torch.bfloat16), (5000, torch.float32), (700, torch.bfloat16))]
        return params, AdamW8bit([dict(params=params[:3]), dict(params=params[3:], lr=1e-2)], **HP, capturable=True)

    (a, fused), (b, plain) = made(), made()
    for step in range(5):
        if step == 3:
            (a2, fused2), (b2, plain2) = made(), made()
            for old, new, before, after in ((a, a2, fused, fused2), (b, b2, plain, plain2)):
                for p, q in zip(old, new):
                    q.data.copy_(p.data)
                after.load_state_dict(before.state_dict())
            a, b, fused, plain = a2, b2, fused2, plain2
        gradients(step, a, b)
        triton_adamw_step(fused)
        plain.step()
        assert [float(fused.state[p]["step"]) for p in a] == [step + 1.0] * 4
        same_codes(a, b, fused, plain)
    close_parameters(a, b, 5, lr=1e-2)


def test_scaled_loops_take_the_pytorch_step(gpu):
    """There is no fused form of the GradScaler or ZeRO sequence for 8-bit moments: the first falls back, the second refuses."""

    (a, fused), (b, plain) = pair([(300,), (1025,)], torch.float32, gpu)
    gradients(1, a, b)
    scales = [torch.amp.GradScaler("cuda", init_scale=4.0) for _ in range(2)]
    for params, scaler in ((a, scales[0]), (b, scales[1])):
        scaler.scale(torch.ones((), device=gpu))  # as a loss would
        for p in params:
            p.grad.mul_(4.0)
    with pytest.warns(RuntimeWarning):
        AdamWStepWithFallback(use_triton=True).step_with_grad_scaler(scales[0], fused, 1.0)
    scales[1].unscale_(plain)
    torch.nn.utils.clip_grad_norm_(b, 1.0)
    scales[1].step(plain)
    scales[1].update()
    same_codes(a, b, fused, plain)
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    with pytest.raises(TritonAdamWUnavailable):
        triton_unscale_clip_and_step(fused, 4.0, 1.0, parameters=a)


@pytest.mark.parametrize("count", ["host", "device"])
@pytest.mark.parametrize("native", [True, False])
def test_a_shared_count_advances_once(gpu, monkeypatch, count, native):
    """Parameters of a capturable group share their count, also when the group stops being capturable, and a program may share
    one between its host counts: the fused step advances it as the plain form does."""

    if not native:
        monkeypatch.setattr(_lib, "extension", lambda: None)
        monkeypatch.setattr(_lib, "native", None)
    (a, fused), (b, plain) = pair([(300,), (1000,), (7,)], torch.float32, gpu, capturable=count == "device")
    for step in range(4):
        gradients(step, a, b)
        triton_adamw_step(fused)
        plain.step()
        if step == 0:
            for optimizer, ps in ((fused, a), (plain, b)):
                optimizer.param_groups[0]["capturable"] = False
                for p in ps:
                    optimizer.state[p]["step"] = optimizer.state[ps[0]]["step"]
        assert float(fused.state[a[0]]["step"]) == step + 1.0
        same_codes(a, b, fused, plain)
        close_parameters(a, b, step + 1)
