"""The cross-entropy of a head without a GPU: its PyTorch form, its fallback, and what it refuses."""

from __future__ import annotations

import ctypes
import warnings

import pytest
import torch
from torch.nn import functional as F

from picotron_amd import _lib, ops
from picotron_amd.nn.triton_kernels import (
    LinearCrossEntropyWithFallback,
    TritonLinearCrossEntropyUnavailable,
    linear_cross_entropy_with_pytorch,
    triton_linear_cross_entropy,
)


def make(dtype=torch.float64):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 5, 8, generator=g, dtype=dtype).requires_grad_()
    w = torch.randn(11, 8, generator=g, dtype=dtype).requires_grad_()
    t = torch.randint(0, 11, (2, 5), generator=g)
    t[0, 2] = -100
    return x, w, t


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("shift", [False, True])
def test_pytorch_form(reduction, shift):
    x, w, t = make()
    got = linear_cross_entropy_with_pytorch(x, w, t, shift=shift, reduction=reduction)
    logits = x @ w.t()
    labels = t
    if shift:
        logits, labels = logits[:, :-1], t[:, 1:]
    want = F.cross_entropy(logits.transpose(1, 2), labels, reduction=reduction)
    torch.testing.assert_close(got, want)
    assert torch.autograd.gradcheck(
        lambda a, b: linear_cross_entropy_with_pytorch(a, b, t, shift=shift, reduction=reduction), (x, w))


def test_pytorch_form_computes_a_loss_of_16_bit_inputs_in_32():
    x, w, t = make(torch.float32)
    got = linear_cross_entropy_with_pytorch(x.bfloat16(), w.bfloat16(), t)
    assert got.dtype == torch.float32
    torch.testing.assert_close(got, F.cross_entropy(F.linear(x.bfloat16(), w.bfloat16()).float().transpose(1, 2), t))


def test_cpu_tensors_are_refused_and_fall_back_once():
    x, w, t = make(torch.float32)
    with pytest.raises(TritonLinearCrossEntropyUnavailable):
        triton_linear_cross_entropy(x, w, t)
    head = LinearCrossEntropyWithFallback(use_triton=True)
    with pytest.warns(RuntimeWarning, match="linear cross-entropy unavailable"):
        loss = head(x, w, t, shift=True)
    torch.testing.assert_close(loss, linear_cross_entropy_with_pytorch(x, w, t, shift=True))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        head(x, w, t)
        LinearCrossEntropyWithFallback()(x, w, t)


@pytest.mark.parametrize("options", [dict(reduction="max"), dict(chunk_tokens=0), dict(chunk_tokens=2.0), dict(chunk_tokens=True)])
def test_options(options):
    x, w, t = make(torch.float32)
    with pytest.raises(ValueError):
        triton_linear_cross_entropy(x, w, t, **options)
    with pytest.raises(ValueError):
        LinearCrossEntropyWithFallback(**options)


def test_shapes():
    x, w, t = (y.detach() for y in make(torch.float32))
    assert ops.head_rows(x, w, t, False) == (2, 5, 5) and ops.head_rows(x, w, t, True) == (2, 4, 5)
    assert ops.head_rows(x[0], w, t[0], False) == (1, 5, 5)
    for args in ((x, w, t[:, 1:], False), (x, w[:, 1:], t, False), (x, w, t.int(), False), (x[0], w, t[0], True), (x.half(), w, t, False),
                 (x.double(), w.double(), t, False), (x, w[0], t, False), (x, w[:0], t, False), (x[..., :0], w[:, :0], t, False)):
        with pytest.raises(ValueError):
            ops.head_rows(*args)


@pytest.mark.parametrize("ignore_index", [2**63, 2**64 + 5, -(2**63) - 1])
def test_an_ignore_index_that_is_no_label_of_any(ignore_index):
    x, w, t = (y.detach() for y in make(torch.float32))
    with pytest.raises(ValueError, match="ignore_index"):
        ops.linear_cross_entropy(x, w, t, ignore_index=ignore_index)


def call(**change):
    """The entry point with addresses that no kernel may reach: every call here is refused before a launch."""

    a = dict(x=256, xso=0, xsi=8, outer=1, inner=4, w=256, ldw=8, vocab=11, hidden=8, t=256, tso=0, tsi=1, ignore=-100, reduction=0,
             loss=256, dloss=None, dso=0, dsi=0, dx=None, dx_inner=4, dw=None, grad_dtype=0, ws=256, ws_bytes=1 << 40, chunk=0, dtype=0,
             stream=None)
    a.update(change)
    return _lib.lib().pt_linear_cross_entropy(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=9), _lib.PT_EUNSUPPORTED),
    (dict(x=None), _lib.PT_EINVAL),
    (dict(w=None), _lib.PT_EINVAL),
    (dict(t=None), _lib.PT_EINVAL),
    (dict(ws=None), _lib.PT_EINVAL),
    (dict(ws=264), _lib.PT_EINVAL),
    (dict(ws_bytes=100), _lib.PT_EINVAL),
    (dict(loss=None), _lib.PT_EINVAL),
    (dict(ldw=7), _lib.PT_EINVAL),
    (dict(inner=-1), _lib.PT_EINVAL),
    (dict(vocab=0), _lib.PT_EINVAL),
    (dict(hidden=0, ldw=0), _lib.PT_EINVAL),
    (dict(reduction=3), _lib.PT_EINVAL),
    (dict(dx_inner=3), _lib.PT_EINVAL),
    (dict(dx=256, grad_dtype=1), _lib.PT_EINVAL),
    (dict(dx=264), _lib.PT_EINVAL),
    (dict(dx=256, reduction=2), _lib.PT_EINVAL),
    (dict(dloss=256, reduction=2), _lib.PT_EINVAL),
    (dict(x=258), _lib.PT_EINVAL),
    (dict(outer=1 << 20, inner=1 << 20, dx_inner=1 << 20), _lib.PT_EUNSUPPORTED),
    (dict(inner=(1 << 24) + 1, dx_inner=(1 << 24) + 1), _lib.PT_EUNSUPPORTED),
    (dict(vocab=(1 << 21) + 1), _lib.PT_EUNSUPPORTED),
    (dict(hidden=(1 << 20) + 1, ldw=(1 << 20) + 1), _lib.PT_EUNSUPPORTED),
    (dict(ldw=(1 << 21) + 1), _lib.PT_EUNSUPPORTED),
])
def test_entry_point_refuses(change, code):
    assert call(**change) == code
    assert _lib.lib().pt_last_error()


def test_scale_entry_point_refuses():
    def call(from_=256, to=256, n=4, from2=None, to2=None, n2=0, a=0, b=0, scale=256):
        return _lib.lib().pt_scale_gradients(from_, to, n, from2, to2, n2, a, b, scale, None)

    assert call(b=9) == _lib.PT_EUNSUPPORTED
    assert call(to=512, a=1) == _lib.PT_EUNSUPPORTED
    for bad in (dict(to=512), dict(from_=None, b=1), dict(from_=264, to=512, b=1), dict(to=512, b=1, n=-1), dict(n2=4), dict(scale=None),
                dict(from2=256, to2=512, n2=4), dict(from2=264, to2=264, n2=4)):
        assert call(**bad) == _lib.PT_EINVAL
    assert call(from_=None, to=None, n=0, scale=None) == _lib.PT_OK


def test_any_number_of_rows_a_chunk():
    """As many as an int64 holds: a limit that limits nothing."""

    size = _lib.lib().pt_linear_cross_entropy_workspace_bytes
    weight = ctypes.c_void_p(256)
    for hidden in (64, 256):
        whole = size(5000, 32000, hidden, weight, hidden, _lib.PT_BFLOAT16, 1, 1, 0)
        for chunk in (5000, 5120, 5121, 1 << 31, (1 << 63) - 257, (1 << 63) - 256, (1 << 63) - 255, (1 << 63) - 1):
            assert size(5000, 32000, hidden, weight, hidden, _lib.PT_BFLOAT16, 1, 1, chunk) == whole
    assert call(ws_bytes=100, chunk=(1 << 63) - 1) == _lib.PT_EINVAL


def test_workspace_holds_at_most_two_gib_of_exponentials():
    size = _lib.lib().pt_linear_cross_entropy_workspace_bytes
    weight = ctypes.c_void_p(256)
    # a large batch: the gathered rows, and no more than the chunk beside them
    rows, vocab, hidden = 65536, 128256, 4096
    bytes_ = size(rows, vocab, hidden, weight, hidden, _lib.PT_BFLOAT16, 1, 1, 0)
    whole = rows * vocab * 2
    sum_of_weight = 4 * (vocab + 256) * hidden  # dw in fp32 over the chunks
    assert rows * hidden * 2 < bytes_ < rows * hidden * 2 + (1 << 31) + sum_of_weight + (1 << 28) < whole
    assert size(rows, vocab, hidden, weight, hidden, _lib.PT_BFLOAT16, 1, 1, 1024) < bytes_ - (1 << 30)
    assert size(8, 64, 32, weight, 32, 9, 1, 1, 0) == 0
