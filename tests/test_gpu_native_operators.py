"""The native launchers of the rotary embedding at positions, the preference loss and the 8-bit AdamW against the general
route: the same bits, the same refusals."""

from __future__ import annotations

import pytest
import torch

from gpu_util import randn
from picotron_amd import _lib, ops
from picotron_amd.nn import RotaryFrequencies
from picotron_amd.nn.triton_kernels import adamw, triton_adamw_step, triton_clip_grad_norm_and_step
from picotron_amd.optim import AdamW8bit
from test_gpu_native import DTYPES, _both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "rotate_half"])
def test_rope_at_forms(gpu, monkeypatch, dtype, layout):
    frequencies = RotaryFrequencies(12)
    turns = frequencies.turns(torch.device("cuda", torch.cuda.current_device()))
    q = randn((2, 7, 4, 16), dtype, gpu, 3).transpose(1, 2)
    keys = [randn((2, 7, 2, 16), dtype, gpu, 4).transpose(1, 2), randn((2, 2, 7, 20), dtype, gpu, 6)[..., 2:18],
            randn((1, 1, 1, 16), dtype, gpu, 7).expand(2, 2, 7, 16), randn((2, 2, 22), dtype, gpu, 8).unfold(2, 16, 1), None]
    each = torch.arange(14, device=gpu).reshape(2, 7) * 1000 - 2000
    positions = [None, each, each.int(), each[:1], each[1], each[0].int(), each[0, :1].expand(7), each[:, :1].expand(2, 7),
                 (torch.arange(28, device=gpu).reshape(2, 14) ** 3)[:, ::2]]

    def call(k=None, p=None, x=q, t=turns, scale=1.25, **options):
        return ops.rope_at(x, t, positions=p, scale=scale, layout=options.pop("layout", layout), x1=k, **options)

    for k in keys:
        for p in positions:
            _both(monkeypatch, lambda: call(k, p, offset=5, inverse=p is None), native=True)
    for offset in (-(2**63), 2**63 - 1):
        _both(monkeypatch, lambda: call(offset=offset), native=True)
    for offset in (-(2**63) - 1, 2**63):
        _both(monkeypatch, lambda: call(offset=offset), raises=ValueError)
    for k in (randn((2, 2, 16, 7), dtype, gpu, 8).transpose(2, 3), randn((2, 2, 7, 14), dtype, gpu, 9),
              randn((1, 2, 7, 16), dtype, gpu, 9), randn((2, 2, 6, 16), dtype, gpu, 9), randn((2, 2, 7, 16), torch.float64, gpu, 9)):
        _both(monkeypatch, lambda: call(k), raises=ValueError)
    for p in (each.double(), each[:, :6], each[None], each[0, 0], torch.cat((each, each))):
        _both(monkeypatch, lambda: call(p=p), raises=ValueError)
    for t in (turns.int(), turns[::2], turns.repeat(2), turns[None]):
        _both(monkeypatch, lambda: call(t=t), raises=ValueError)
    _both(monkeypatch, lambda: call(layout="other"), raises=ValueError)
    _both(monkeypatch, lambda: call(p=each[0].cpu()), raises=ValueError)
    for shape in ((0, 4, 7, 16), (2, 0, 7, 16), (2, 4, 0, 16)):
        _both(monkeypatch, lambda: call(x=torch.empty(shape, dtype=dtype, device=gpu)), native=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [True, False])
def test_preference_forms(gpu, monkeypatch, dtype, shift):
    shape = (4, 6, 301)
    dense = randn(shape, dtype, gpu, 1)
    labels = torch.randint(0, 301, (4, 6), device=gpu)
    labels[0, 2] = labels[3] = -100
    forms = [dense, randn((6, 4, 301), dtype, gpu, 2).transpose(0, 1), randn((4, 6, 320), dtype, gpu, 3)[..., 7:308],
             randn((8, 9, 301), dtype, gpu, 4)[::2, 1:7]]
    reference = randn((4,), torch.float32, gpu, 5)
    up = randn((4,), torch.float32, gpu, 6)
    loss_up = randn((), torch.float32, gpu, 7)
    for x in forms:
        for y in (labels, labels.t().contiguous().t(), labels[:1].expand(4, 6)):
            for average in (False, True):
                _both(monkeypatch, lambda: ops.sequence_log_probs(x, y, shift=shift, average=average)[0], native=True)
                for kind, r in (("sigmoid", None), ("sigmoid", reference), ("hinge", reference), ("ipo", reference)):
                    _both(monkeypatch, lambda: ops.preference_loss(x, y, r, beta=0.3, kind=kind, shift=shift,
                                                                   average=average)[:3], native=True)
            ws = ops.sequence_log_probs(x, y, shift=shift)[1]
            _both(monkeypatch, lambda: ops.sequence_log_probs_bwd(x, y, ws, grad_log_probs=up, shift=shift), native=True)
            ws = ops.preference_loss(x, y, reference, beta=0.3, shift=shift)[3]
            _both(monkeypatch, lambda: ops.sequence_log_probs_bwd(x, y, ws, grad_loss=loss_up, shift=shift), native=True)
    ws = ops.sequence_log_probs(dense, labels, shift=shift)[1]
    _both(monkeypatch, lambda: ops.sequence_log_probs_bwd(dense, labels, ws, grad_log_probs=up[:1].expand(4), shift=shift),
          native=False)
    shared = dense[:1].expand(shape)  # its gradient needs rows of its own
    ws = ops.sequence_log_probs(shared, labels, shift=shift)[1]
    _both(monkeypatch, lambda: ops.sequence_log_probs_bwd(shared, labels, ws, grad_log_probs=up, shift=shift), native=False)
    bad = [(dense, labels.int(), None), (dense, labels[:, :5], None), (dense[0], labels[0], None),
           (dense.transpose(1, 2), labels, None), (dense, labels.cpu(), None), (dense[:3], labels[:3], None),
           (dense, labels, reference.double()), (dense, labels, reference[:3]), (dense, labels, reference.cpu()),
           (dense, labels, reference.repeat_interleave(2)[::2]), (dense.double(), labels, None)]
    for x, y, r in bad:  # (a type without kernels is a TypeError, as elsewhere in ops)
        _both(monkeypatch, lambda: ops.preference_loss(x, y, r, beta=0.3),
              raises=TypeError if x.dtype == torch.float64 else ValueError)
    _both(monkeypatch, lambda: ops.preference_loss(dense, labels, None, beta=0.3, kind="other"), raises=ValueError)
    for w, u in ((ws[:8], up), (ws, up[:3]), (ws.cpu(), up)):
        _both(monkeypatch, lambda: ops.sequence_log_probs_bwd(dense, labels, w, grad_log_probs=u), raises=ValueError)


def _optimizer(gpu, dtype, groups, capturable=False):
    params = [torch.nn.Parameter(randn((n,), dtype, gpu, 7 + n, 0.1)) for n in (1, 5, 1024, 4097, 30_000, 8)]
    split = [params] if groups == 1 else [params[:2], params[5:], params[2:5]]  # the last has no gradient: an idle group
    return params, AdamW8bit([dict(params=p, lr=1e-3 * (i + 1)) for i, p in enumerate(split)], weight_decay=0.1, seed=5,
                             capturable=capturable)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups", [1, 3])
@pytest.mark.parametrize("clip", [None, 0.05])
def test_scan_takes_the_same_8bit_steps(gpu, monkeypatch, dtype, groups, clip):
    if clip is not None and dtype != torch.float32:
        pytest.skip("clipping takes fp32 gradients")
    runs = []
    for native in (True, False):
        params, opt = _optimizer(gpu, dtype, groups)
        norms, used = [], []
        with monkeypatch.context() as m:
            if not native:
                m.setattr(adamw, "_scan_8bit", lambda optimizer: None)
            for step in range(4):
                for i, p in enumerate(params[:-1]):
                    p.grad = randn(p.shape, dtype, gpu, 100 * step + i)
                if step == 3:
                    opt.state[params[2]]["step"] += 5.0
                if native:
                    used.append(adamw._scan_8bit(opt) is not None)
                if clip is None:
                    triton_adamw_step(opt)
                else:
                    norms.append(triton_clip_grad_norm_and_step(opt, clip))
        if native:
            assert used == [False, True, True, False]
            assert [float(opt.state[p]["step"]) for p in params[:-1]] == [4.0, 4.0, 9.0, 4.0, 4.0]
        runs.append((params, [opt.state[p] for p in params[:-1]], norms))
    for a, b in zip(*(r[0] for r in runs)):
        assert torch.equal(a, b)
    for a, b in zip(*(r[1] for r in runs)):
        assert all(torch.equal(a[k], b[k]) for k in a)
    for a, b in zip(*(r[2] for r in runs)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_moments_by_either_table(gpu, monkeypatch, dtype):
    params, opt = _optimizer(gpu, dtype, 3)
    for i, p in enumerate(params[:-1]):
        p.grad = randn(p.shape, dtype, gpu, i)
    triton_adamw_step(opt)
    m, v, places = opt.moments()
    with monkeypatch.context() as c:
        c.setattr(_lib, "extension", lambda: None)
        general = opt.moments()
    assert torch.equal(m, general[0]) and torch.equal(v, general[1])
    assert [(id(p), at) for p, at in places] == [(id(p), at) for p, at in general[2]]
    wide = opt.moments(torch.float64)  # a type without kernels: in PyTorch
    for p, at in places:
        assert torch.equal(m[at:at + p.numel()].double(), wide[0][at:at + p.numel()])
        assert torch.equal(v[at:at + p.numel()].double(), wide[1][at:at + p.numel()])
    state = opt.state[params[1]]
    state["exp_avg"] = torch.cat((state["exp_avg"],) * 2, 1)[:, :256]  # strided: the kernel cannot read it
    again = opt.moments()
    assert all(torch.equal(m[at:at + p.numel()], again[0][at:at + p.numel()]) for p, at in places)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"), torch.cuda.graph(graph):
        opt.moments()


def test_8bit_scan_leaves_the_unusual_to_the_plan(gpu):
    def ready(**options):
        params, opt = _optimizer(gpu, torch.float32, 1, **options)
        for p in params[:-1]:
            p.grad = torch.ones_like(p)
        triton_adamw_step(opt)
        assert (adamw._scan_8bit(opt) is None) == bool(options)
        return params, opt

    params, opt = ready()
    params[3].grad = torch.ones(2 * 4097, device=gpu)[::2]
    assert adamw._scan_8bit(opt) is None
    scales = (30_000 + 255) // 256
    for key, value in (("exp_avg", torch.zeros(3, 256, dtype=torch.uint8, device=gpu)),
                       ("exp_avg_sq", torch.zeros(scales, 256, dtype=torch.int8, device=gpu)),
                       ("exp_avg_sq", torch.zeros(scales * 256 + 1, dtype=torch.uint8, device=gpu)[1:].view(scales, 256)),
                       ("exp_avg_scale", torch.zeros(2 * scales, dtype=torch.uint8, device=gpu)[::2]),
                       ("exp_avg_sq_scale", torch.zeros(scales, dtype=torch.uint8))):
        params, opt = ready()
        opt.state[params[4]][key] = value
        before = params[4].clone()
        assert adamw._scan_8bit(opt) is None
        with pytest.raises(adamw.TritonAdamWUnavailable):
            triton_adamw_step(opt)
        assert torch.equal(params[4], before)
        del opt.state[params[4]][key]
        assert adamw._scan_8bit(opt) is None
    params, opt = ready()
    opt.state[params[2]]["step"] = torch.tensor(1.0, dtype=torch.float64)
    assert adamw._scan_8bit(opt) is None
    ready(capturable=True)
    params, opt = ready()
    opt.zero_grad()
    assert adamw._scan_8bit(opt) is None
    triton_adamw_step(opt)  # nothing to do
    params, opt = ready()
    state = opt.state[params[0]]
    version = state["step"]._version
    triton_adamw_step(opt)
    assert state["step"]._version > version
