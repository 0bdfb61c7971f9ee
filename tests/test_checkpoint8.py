"""Activations kept in 8 bits, without a GPU: their codes, the operators' PyTorch forms, the modules, and what is refused."""

from __future__ import annotations

import math

import pytest
import torch

from picotron_amd import _lib, ops
from picotron_amd.nn import RMSNorm, SwiGLU
from picotron_amd.nn.triton_kernels import (
    TritonRMSNormUnavailable,
    TritonSwiGLUUnavailable,
    _block8,
    residual_rms_norm_with_pytorch,
    rms_norm_with_pytorch_forward,
    swiglu_with_pytorch_forward,
    triton_residual_rms_norm,
    triton_rms_norm,
    triton_swiglu,
)


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


@pytest.mark.parametrize("size", [1, 7, 127, 128, 129, 300, 1024])
def test_values_are_within_half_a_step(size):
    x = randn(5, size) * torch.tensor([1e-30, 1e-5, 1.0, 1e4, 1e37])[:, None]
    codes, steps = _block8.encode(x)
    blocks = (size + 127) // 128
    assert codes.shape == (5, blocks, 128) and codes.dtype == torch.uint8 and steps.shape == (5, blocks, 1)
    assert codes.min() >= 1
    off = (_block8.decode(codes, steps, size).double() - x.double()).abs()
    # half a step, and the roundings of the quotients and products: at most 127 steps times four of 2^-24
    step = steps.double().expand(-1, -1, 128).flatten(1)[:, :size]
    assert torch.all(off <= step * (0.5 + 4 * 127 * 2.0**-24))


def test_special_blocks():
    x = randn(6, 128)
    x[0] = 0
    x[1] *= 1e-32
    x[2, 5] = math.inf
    x[3, 7] = math.nan
    x[4, 9] = -math.inf
    values = _block8.decode(*_block8.encode(x), 128)
    assert not values[:2].any() and values[2:5].isnan().all() and values[5].isfinite().all()


def test_the_largest_values_stay_finite():
    x = randn(3, 128)
    for row, dtype in enumerate((torch.float32, torch.float16, torch.bfloat16)):
        x[row, 5], x[row, 77] = torch.finfo(dtype).min, torch.finfo(dtype).max
    values = _block8.decode(*_block8.encode(x), 128)
    assert values.isfinite().all() and torch.all((values[:, 5] / x[:, 5] - 1).abs() <= 2.0**-22)


def test_swiglu_gradients_are_those_at_the_kept_values():
    g, u, d = randn(3, 100, seed=1).requires_grad_(), randn(3, 100, seed=2).requires_grad_(), randn(3, 100, seed=3)
    y = swiglu_with_pytorch_forward(g, u, checkpoint_8bit=True)
    assert torch.equal(y, torch.nn.functional.silu(g) * u)
    got = torch.autograd.grad(y, [g, u], d)
    kept = [_block8.decode(*_block8.encode(t.detach().view(-1)), 300).view(3, 100).double().requires_grad_() for t in (g, u)]
    want = torch.autograd.grad(torch.nn.functional.silu(kept[0]) * kept[1], kept, d.double())
    for a, b in zip(got, want):
        torch.testing.assert_close(a.double(), b, rtol=2e-6, atol=1e-6)


@pytest.mark.parametrize("narrow", [0, 1])
@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, 1.0), (torch.float16, 1e-9)])
def test_swiglu_gradients_of_two_types(dtype, scale, narrow):
    """gate and up of different types: each gradient in its own."""

    inputs = [randn(3, 100, seed=1), randn(3, 100, seed=2)]
    inputs[narrow] = inputs[narrow].to(dtype)
    inputs = [t.requires_grad_() for t in inputs]
    d = randn(3, 100, seed=3, scale=scale)
    got = torch.autograd.grad(swiglu_with_pytorch_forward(*inputs, checkpoint_8bit=True), inputs, d)
    kept = [_block8.decode(*_block8.encode(t.detach().view(-1)), 300).view(3, 100).double().requires_grad_() for t in inputs]
    want = torch.autograd.grad(torch.nn.functional.silu(kept[0]) * kept[1], kept, d.double())
    for a, b, t in zip(got, want, inputs):
        assert a.dtype == t.dtype
        # a dozen roundings to 24 bits of factors of up to 4, 4 and 4; and one to 16, or to half the smallest step there
        own = 0 if t.dtype == torch.float32 else torch.finfo(t.dtype).eps / 2 * b.abs() + (2.0**-25 if t.dtype == torch.float16 else 0)
        assert torch.all((a.double() - b).abs() <= 12 * 64 * 2.0**-24 * scale + own)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shapes", [((3, 5, 16), (16,)), ((16,), (3, 5, 16)), ((3, 1, 16), (5, 1))])
def test_swiglu_of_shapes_that_broadcast(shapes, dtype):
    inputs = [randn(*shape, seed=k).to(dtype).requires_grad_() for k, shape in enumerate(shapes)]
    y = swiglu_with_pytorch_forward(*inputs, checkpoint_8bit=True)
    assert torch.equal(y, swiglu_with_pytorch_forward(*inputs))
    d = randn(*y.shape, seed=3).to(dtype)
    got = torch.autograd.grad(y, inputs, d)
    kept = [_block8.decode(*_block8.encode(t.detach().reshape(-1)), t.numel()).view(t.shape).double().requires_grad_() for t in inputs]
    want = torch.autograd.grad(torch.nn.functional.silu(kept[0]) * kept[1], kept, d.double())
    for a, b, t in zip(got, want, inputs):
        # a dozen roundings to 24 bits of factors of up to 4, 4 and 4, and a sum of at most 48 of them; and one to 16
        assert a.shape == t.shape and a.dtype == dtype
        own = 0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * b.abs()
        assert torch.all((a.double() - b).abs() <= (12 + 48) * 48 * 64 * 2.0**-24 + own)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_of_a_residual_that_broadcasts(dtype):
    x, r = randn(3, 5, 16, seed=1).to(dtype).requires_grad_(), randn(16, seed=2).to(dtype).requires_grad_()
    w, d, dh = torch.ones(16), randn(3, 5, 16, seed=3).to(dtype), randn(3, 5, 16, seed=4).to(dtype)
    h, y = residual_rms_norm_with_pytorch(x, r, w, 1e-5, checkpoint_8bit=True)
    dx, dr = torch.autograd.grad([h, y], [x, r], [dh, d])
    h64 = h.detach().double()
    rstd = (h64.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    hat = _block8.decode(*_block8.encode(h.detach()), 16).double() * rstd
    want = rstd * (d.double() - hat * (d.double() * hat).mean(-1, keepdim=True)) + dh.double()
    # roundings of terms of up to 4 * 4 * 4, a sum of 15 of them, and one to the type
    for got, exact, terms in ((dx, want, 1), (dr, want.sum((0, 1)), 15)):
        own = 0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * exact.abs()
        assert got.shape == exact.shape and torch.all((got.double() - exact).abs() <= (16 + terms) * terms * 64 * 2.0**-24 + own)


@pytest.mark.parametrize("residual", [False, True])
def test_norm_gradients_are_those_at_the_kept_values(residual):
    x, r, w, d, dh = (randn(4, 200, seed=k) for k in (1, 2, 3, 4, 5))
    w = w[0].clone().requires_grad_()
    x.requires_grad_()
    r.requires_grad_()
    if residual:
        h, y = residual_rms_norm_with_pytorch(x, r, w, 1e-5, checkpoint_8bit=True)
        got = torch.autograd.grad([h, y], [x, r, w], [dh, d])
        assert torch.equal(got[0], got[1])
        got = got[1:]
    else:
        h, y = x, rms_norm_with_pytorch_forward(x, w, 1e-5, checkpoint_8bit=True)
        got = torch.autograd.grad([y], [x, w], [d])
    assert torch.equal(y, rms_norm_with_pytorch_forward(h, w, 1e-5))
    h64 = h.detach().double()
    rstd = (h64.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    hat = _block8.decode(*_block8.encode(h.detach()), 200).double() * rstd
    gw = d.double() * w.detach().double()
    dx = rstd * (gw - hat * (gw * hat).mean(-1, keepdim=True))
    if residual:
        dx = dx + dh.double()
    torch.testing.assert_close(got[0].double(), dx, rtol=2e-6, atol=2e-6)
    torch.testing.assert_close(got[1].double(), (d.double() * hat).sum(0), rtol=2e-6, atol=2e-6)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, 1.0), (torch.float16, 1e-9)])
def test_a_residual_stream_of_32_bits_keeps_its_gradient(dtype, scale, fused):
    """A 16-bit branch added to an fp32 stream, as under autocast: the sum and its gradient are fp32."""

    x, r, d, dh = randn(4, 200, seed=1).to(dtype), randn(4, 200, seed=2), randn(4, 200, seed=3, scale=scale), randn(4, 200, seed=4, scale=scale)
    norm = RMSNorm(200, 1e-5, use_triton_rmsnorm=fused, checkpoint_8bit=True)
    norm._triton_fallback_warned = True
    x.requires_grad_()
    r.requires_grad_()
    h, y = norm.add_and_norm(x, r)
    assert h.dtype == y.dtype == torch.float32
    dx, dr = torch.autograd.grad([h, y], [x, r], [dh, d])
    assert dx.dtype == dtype and dr.dtype == torch.float32
    h64 = h.detach().double()
    rstd = (h64.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    hat = _block8.decode(*_block8.encode(h.detach()), 200).double() * rstd
    want = rstd * (d.double() - hat * (d.double() * hat).mean(-1, keepdim=True)) + dh.double()
    # a few roundings to 24 bits of terms of up to 4 * 4 * 4 of the gradients' scale, and a mean of 200 of them
    assert torch.all((dr.double() - want).abs() <= 64 * 16 * 2.0**-24 * scale)
    # and one to the branch's type, or to half its smallest step
    assert torch.all((dx.double() - want).abs() <= 64 * 16 * 2.0**-24 * scale + want.abs() * torch.finfo(dtype).eps / 2
                     + (2.0**-25 if dtype == torch.float16 else 0))


def test_gradients_are_near_the_exact_ones():
    """Within what half a step of each block, 1/254 of its largest, makes of them."""

    g, u, d = (randn(64, 128, seed=k).double() for k in (1, 2, 3))
    kept = [t.float().requires_grad_() for t in (g, u)]
    y = swiglu_with_pytorch_forward(*kept, checkpoint_8bit=True)
    got = torch.autograd.grad(y, kept, d.float())
    exact = [t.clone().requires_grad_() for t in (g, u)]
    want = torch.autograd.grad(torch.nn.functional.silu(exact[0]) * exact[1], exact, d)
    step = max(float(g.abs().max()), float(u.abs().max())) / 254
    # silu' is at most 1.1 and its slope at most 1/2; silu(g) differs by at most 1.1 steps
    limit = d.abs() * step * (1.1 + 0.5 * u.abs() + step) + 1e-5
    for a, b in zip(got, want):
        assert torch.all((a.double() - b).abs() <= limit)


def test_no_second_derivative():
    x = randn(2, 128).requires_grad_()
    w = torch.ones(128, requires_grad=True)
    for y in (swiglu_with_pytorch_forward(x, x, checkpoint_8bit=True), rms_norm_with_pytorch_forward(x, w, 1e-5, checkpoint_8bit=True)):
        with pytest.raises(RuntimeError, match="checkpoint_8bit"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_what_is_kept():
    """The saved tensors of a step: a byte an element and 4 a block, none of the inputs."""

    sizes = []

    def pack(t):
        sizes.append(t.numel() * t.element_size())
        return t

    g, u = randn(8, 256).requires_grad_(), randn(8, 256).requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        swiglu_with_pytorch_forward(g, u, checkpoint_8bit=True)
    assert sum(sizes) == 2 * (2048 + 16 * 4)


def test_modules():
    torch.manual_seed(0)
    plain, kept = SwiGLU(32, 64), SwiGLU(32, 64, checkpoint_8bit=True)
    kept.load_state_dict(plain.state_dict())
    x = randn(3, 5, 32)
    assert torch.equal(plain(x), kept(x))
    kept(x).sum().backward()
    plain(x).sum().backward()
    for p, q in zip(plain.parameters(), kept.parameters()):
        assert float((p.grad - q.grad).norm() / p.grad.norm()) < 1 / 127  # of values of one scale, kept to 1/254 of the largest
    plain, kept = RMSNorm(32), RMSNorm(32, checkpoint_8bit=True)
    r = randn(3, 5, 32, seed=1)
    torch.testing.assert_close(kept(x), plain(x))
    for a, b in zip(kept.add_and_norm(x, r), plain.add_and_norm(x, r)):
        torch.testing.assert_close(a, b)
    del kept.__dict__["checkpoint_8bit"]  # one that was stored before the option
    kept(x)


def test_fused_modules_fall_back_and_still_keep_8_bits():
    x = randn(3, 32).requires_grad_()
    with pytest.warns(RuntimeWarning, match="SwiGLU unavailable"):
        SwiGLU(32, 64, use_triton_swiglu=True, checkpoint_8bit=True)(x)
    norm = RMSNorm(32, use_triton_rmsnorm=True, checkpoint_8bit=True)
    with pytest.warns(RuntimeWarning, match="RMSNorm unavailable"):
        y = norm(x)
    assert "RMSNorm8" in type(y.grad_fn).__name__


def test_cpu_tensors_are_refused():
    x, w = randn(2, 64), torch.ones(64)
    with pytest.raises(TritonSwiGLUUnavailable):
        triton_swiglu(x, x, checkpoint_8bit=True)
    with pytest.raises(TritonRMSNormUnavailable):
        triton_rms_norm(x, w, 1e-5, checkpoint_8bit=True)
    with pytest.raises(TritonRMSNormUnavailable):
        triton_residual_rms_norm(x, x, w, 1e-5, checkpoint_8bit=True)


def test_block_size_matches_the_library():
    assert _lib.lib().pt_block8_elems() == ops.BLOCK8


BAD = _lib.PT_EINVAL


@pytest.mark.parametrize("fn,args,code", [
    ("pt_swiglu8_fwd", (256, 256, 256, 256, 256, 8, 9, None), _lib.PT_EUNSUPPORTED),
    ("pt_swiglu8_fwd", (256, 256, 256, 256, 256, -1, 0, None), BAD),
    ("pt_swiglu8_fwd", (None, 256, 256, 256, 256, 8, 0, None), BAD),
    ("pt_swiglu8_fwd", (256, 256, 256, None, 256, 8, 0, None), BAD),
    ("pt_swiglu8_fwd", (256, 256, 256, 264, 256, 8, 0, None), BAD),
    ("pt_swiglu8_fwd", (256, 256, 256, 256, 260, 8, 0, None), BAD),
    ("pt_swiglu8_fwd", (258, 256, 256, 256, 256, 8, 0, None), BAD),
    ("pt_swiglu8_fwd", (256, 256, 256, 256, 256, 1 << 39, 0, None), _lib.PT_EUNSUPPORTED),
    ("pt_swiglu8_fwd", (None, None, None, None, None, 0, 0, None), _lib.PT_OK),
    ("pt_swiglu8_bwd", (None, 256, 256, 256, 256, 8, 0, None), BAD),
    ("pt_swiglu8_bwd", (256, None, 256, 256, 256, 8, 0, None), BAD),
    ("pt_swiglu8_bwd", (256, 256, 256, None, None, 8, 0, None), _lib.PT_OK),
    ("pt_rmsnorm8_fwd", (256, None, 256, None, 256, 256, 256, 256, 4, 8, 1e-5, 9, 0, None), _lib.PT_EUNSUPPORTED),
    ("pt_rmsnorm8_fwd", (256, None, 256, None, 256, 256, 256, 256, 4, 0, 1e-5, 0, 0, None), BAD),
    ("pt_rmsnorm8_fwd", (256, 256, 256, None, 256, 256, 256, 256, 4, 8, 1e-5, 0, 0, None), BAD),
    ("pt_rmsnorm8_fwd", (None, None, 256, None, 256, 256, 256, 256, 4, 8, 1e-5, 0, 0, None), BAD),
    ("pt_rmsnorm8_fwd", (256, None, 256, None, 256, 256, 260, 256, 4, 8, 1e-5, 0, 0, None), BAD),
    ("pt_rmsnorm8_fwd", (256, None, 256, None, 256, 256, 256, 256, 1 << 31, 8, 1e-5, 0, 0, None), _lib.PT_EUNSUPPORTED),
    ("pt_rmsnorm8_bwd", (256, None, 256, 256, 256, 256, 256, 256, 256, 8, 4, 8, 0, 0, None), BAD),
    ("pt_rmsnorm8_bwd", (256, None, 256, 256, 256, 256, 256, 256, None, 1 << 20, 4, 8, 0, 0, None), BAD),
    ("pt_rmsnorm8_bwd", (None, None, 256, 256, 256, 256, 256, None, None, 0, 4, 8, 0, 0, None), BAD),
    ("pt_rmsnorm8_bwd", (256, None, 256, 256, 256, 256, None, None, None, 0, 4, 8, 0, 0, None), _lib.PT_OK),
])
def test_entry_points_refuse(fn, args, code):
    assert getattr(_lib.lib(), fn)(*args) == code
