"""Tensor-level launchers for the HIP kernels: shape/stride checks, output allocation,
and the library call on the caller's current HIP stream.

Dense tensors in the kernels' own layout take a native launcher (``_lib.call`` with tensors), which
does those steps in one native call; it leaves everything else to the general route below it.

These functions never fall back to PyTorch arithmetic: if the library is missing they
raise :class:`picotron_amd._lib.HipLibraryUnavailable`, and if an entry point rejects its
arguments they raise :class:`picotron_amd._lib.HipKernelError`.  The autograd Functions
in :mod:`picotron_amd.nn.triton_kernels` are built on them.
"""

from __future__ import annotations

import ctypes
import functools

import numpy as np
import torch
from torch import Tensor

from picotron_amd import _lib

_DTYPE_CODES = {
    torch.float32: _lib.PT_FLOAT32,
    torch.float16: _lib.PT_FLOAT16,
    torch.bfloat16: _lib.PT_BFLOAT16,
}

LAYOUTS = {"interleaved": 0, "rotate_half": 1}


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODES[dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16") from None


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: torch.device) -> int:
    """The device's current HIP stream as an integer handle (torch's raw-stream query when
    present: it skips building a Stream object on every launch)."""

    index = device.index if device.index is not None else torch.cuda.current_device()
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def _launch(fn: str, first: Tensor, *args):
    """The native launcher of entry point ``fn`` on the current stream of ``first``'s device: its
    outputs, or None when the call has to take the general route."""

    if not first.is_cuda:
        return None
    return _lib.call(fn, first, *args, _stream(first.device))


@functools.lru_cache(maxsize=256)
def _rmsnorm_ws_bytes(rows: int, cols: int, code: int) -> int:
    return int(_lib.lib().pt_rmsnorm_bwd_workspace_bytes(rows, cols, code))


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _compiling() -> bool:
    """True while torch.compile traces: the launchers then record themselves as the custom
    ops registered at the end of this module (opaque to the compiler, with fake
    implementations for shape propagation) instead of calling the library; at run time the
    compiled graph calls those ops, which call the launchers eagerly."""

    return torch.compiler.is_compiling()


@functools.lru_cache(maxsize=None)
def device_supported(index: int) -> bool:
    """True if CUDA/HIP device ``index`` is a gfx950 GPU the library was built for."""

    return bool(_lib.lib().pt_device_supported(index))


def _check_cuda(*tensors: Tensor) -> torch.device:
    device = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("HIP kernels need tensors on a GPU device")
        if t.device != device:
            raise ValueError("all tensors must be on the same device")
    return device


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch_here(fn: str, first: Tensor, *args):
    """:func:`_launch`, for tensors on the current device (None for others)."""

    if not first.is_cuda or first.device.index != _current_device():
        return None
    return _launch(fn, first, *args)


def _call_on(device: torch.device, fn: str, *args) -> None:
    """:func:`_lib.raw_call` with ``device`` the current one, which a launch on its stream needs."""

    if device.index is None or device.index == _current_device():
        _lib.raw_call(fn, *args, _stream(device))
    else:
        with torch.cuda.device(device):
            _lib.raw_call(fn, *args, _stream(device))


# ------------------------------------------------------------------ RMSNorm


def _as_rows(t: Tensor, cols: int) -> Tensor:
    """(rows, cols) view of ``t`` whose last dim is contiguous; copies only if needed."""

    if t.dim() == 2 and t.size(1) == cols and (t.stride(1) == 1 or cols == 1):
        return t
    flat = t.reshape(-1, cols)
    if flat.size(0) > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    return flat


def rmsnorm_fwd(x: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    """y = x * rsqrt(mean(x^2) + eps) * weight over the last dim; returns (y, rstd fp32)."""

    if _compiling():
        return torch.ops.picotron_amd.rmsnorm_fwd(x, weight, float(eps))
    out = _launch("pt_rmsnorm_fwd", x, weight, eps)
    if out is not None:
        return out
    device = _check_cuda(x, weight)
    cols = x.size(-1)
    if weight.dim() != 1 or weight.numel() != cols:
        raise ValueError("RMSNorm weight must be 1-D with hidden-size elements")
    weight = weight.contiguous()
    x2 = _as_rows(x, cols)
    rows = x2.size(0)
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    y2 = y.view(-1, cols)
    _lib.raw_call(
        "pt_rmsnorm_fwd",
        x2.data_ptr(), x2.stride(0) if rows > 1 else cols, weight.data_ptr(), y2.data_ptr(), cols,
        rstd.data_ptr(), rows, cols, float(eps), dtype_code(x.dtype), dtype_code(weight.dtype),
        _stream(device),
    )
    return y, rstd


def rmsnorm_bwd(
    dy: Tensor,
    x: Tensor,
    weight: Tensor,
    rstd: Tensor,
    need_dx: bool = True,
    need_dw: bool = True,
) -> tuple[Tensor | None, Tensor | None]:
    """Gradients of RMSNorm w.r.t. x (x's dtype) and weight (weight's dtype)."""

    if _compiling():
        dx, dw = torch.ops.picotron_amd.rmsnorm_bwd(dy, x, weight, rstd)
        return (dx if need_dx else None), (dw if need_dw else None)
    out = _launch("pt_rmsnorm_bwd", dy, x, weight, rstd, bool(need_dx), bool(need_dw))
    if out is not None:
        return out
    device = _check_cuda(dy, x, weight, rstd)
    cols = x.size(-1)
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    weight = weight.contiguous()
    rstd = rstd.contiguous()
    x2 = _as_rows(x, cols)
    dy2 = _as_rows(dy, cols)
    rows = x2.size(0)
    if rstd.numel() != rows or rstd.dtype != torch.float32:
        raise ValueError("rstd must hold one fp32 value per row")
    dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need_dx else None
    dw = torch.empty(cols, dtype=weight.dtype, device=device) if need_dw else None
    ws = None
    ws_bytes = 0
    if need_dw:
        ws_bytes = _rmsnorm_ws_bytes(rows, cols, dtype_code(x.dtype))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=device)
    if not need_dx and not need_dw:
        return None, None
    _lib.raw_call(
        "pt_rmsnorm_bwd",
        dy2.data_ptr(), dy2.stride(0) if rows > 1 else cols, x2.data_ptr(),
        x2.stride(0) if rows > 1 else cols, weight.data_ptr(), rstd.data_ptr(), _ptr(dx), cols,
        _ptr(dw), _ptr(ws), ws_bytes, rows, cols, dtype_code(x.dtype), dtype_code(weight.dtype),
        _stream(device),
    )
    return dx, dw


def residual_rmsnorm_fwd(
    x: Tensor, residual: Tensor, weight: Tensor, eps: float
) -> tuple[Tensor, Tensor, Tensor]:
    """h = x + residual (rounded to x's dtype) and y = RMSNorm(h) in one pass; returns
    (h, y, rstd fp32)."""

    if _compiling():
        return torch.ops.picotron_amd.residual_rmsnorm_fwd(x, residual, weight, float(eps))
    out = _launch("pt_residual_rmsnorm_fwd", x, residual, weight, eps)
    if out is not None:
        return out
    device = _check_cuda(x, residual, weight)
    cols = x.size(-1)
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise ValueError("residual must match x in shape and dtype")
    if weight.dim() != 1 or weight.numel() != cols:
        raise ValueError("RMSNorm weight must be 1-D with hidden-size elements")
    weight = weight.contiguous()
    x2 = _as_rows(x, cols)
    r2 = _as_rows(residual, cols)
    rows = x2.size(0)
    h = torch.empty(x.shape, dtype=x.dtype, device=device)
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    _lib.raw_call(
        "pt_residual_rmsnorm_fwd",
        x2.data_ptr(), x2.stride(0) if rows > 1 else cols, r2.data_ptr(),
        r2.stride(0) if rows > 1 else cols, weight.data_ptr(), h.data_ptr(), cols, y.data_ptr(), cols,
        rstd.data_ptr(), rows, cols, float(eps), dtype_code(x.dtype), dtype_code(weight.dtype),
        _stream(device),
    )
    return h, y, rstd


def residual_rmsnorm_bwd(
    dy: Tensor,
    dh_in: Tensor | None,
    h: Tensor,
    weight: Tensor,
    rstd: Tensor,
    need_dw: bool = True,
    out: Tensor | None = None,
) -> tuple[Tensor, Tensor | None]:
    """dh = RMSNorm-backward(dy) + dh_in (in h's dtype) and the weight gradient.  ``out``
    (may be ``dh_in`` itself) receives dh when given."""

    if _compiling() and out is None:
        dh, dw = torch.ops.picotron_amd.residual_rmsnorm_bwd(dy, dh_in, h, weight, rstd)
        return dh, (dw if need_dw else None)
    if out is None:
        grads = _launch("pt_residual_rmsnorm_bwd", dy, dh_in, h, weight, rstd, bool(need_dw))
        if grads is not None:
            return grads
    device = _check_cuda(dy, h, weight, rstd)
    cols = h.size(-1)
    if dy.dtype != h.dtype:
        dy = dy.to(h.dtype)
    weight = weight.contiguous()
    rstd = rstd.contiguous()
    h2 = _as_rows(h, cols)
    dy2 = _as_rows(dy, cols)
    rows = h2.size(0)
    if rstd.numel() != rows or rstd.dtype != torch.float32:
        raise ValueError("rstd must hold one fp32 value per row")
    d2 = None
    if dh_in is not None:
        if dh_in.shape != h.shape:
            raise ValueError("dh_in must match h")
        if dh_in.dtype != h.dtype:
            dh_in = dh_in.to(h.dtype)
        d2 = _as_rows(dh_in, cols)
    if out is None:
        out = torch.empty(h.shape, dtype=h.dtype, device=device)
    elif out.shape != h.shape or out.dtype != h.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor like h")
    dw = torch.empty(cols, dtype=weight.dtype, device=device) if need_dw else None
    ws, ws_bytes = None, 0
    if need_dw:
        ws_bytes = _rmsnorm_ws_bytes(rows, cols, dtype_code(h.dtype))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=device)
    _lib.raw_call(
        "pt_residual_rmsnorm_bwd",
        dy2.data_ptr(), dy2.stride(0) if rows > 1 else cols, _ptr(d2),
        (d2.stride(0) if rows > 1 else cols) if d2 is not None else 0, h2.data_ptr(),
        h2.stride(0) if rows > 1 else cols, weight.data_ptr(), rstd.data_ptr(), out.data_ptr(), cols,
        _ptr(dw), _ptr(ws), ws_bytes, rows, cols, dtype_code(h.dtype), dtype_code(weight.dtype),
        _stream(device),
    )
    return out, dw


# ------------------------------------------------------------------ SwiGLU


def _flat(t: Tensor) -> Tensor:
    return t if t.is_contiguous() else t.contiguous()


def swiglu_fwd(gate: Tensor, up: Tensor) -> Tensor:
    """silu(gate) * up, elementwise, in gate's dtype."""

    if _compiling():
        return torch.ops.picotron_amd.swiglu_fwd(gate, up)
    out = _launch("pt_swiglu_fwd", gate, up)
    if out is not None:
        return out
    device = _check_cuda(gate, up)
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("SwiGLU gate and up must match in shape and dtype")
    gate, up = _flat(gate), _flat(up)
    out = torch.empty_like(gate)
    _lib.raw_call(
        "pt_swiglu_fwd", gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.numel(),
        dtype_code(gate.dtype), _stream(device),
    )
    return out


def swiglu_bwd(
    dout: Tensor, gate: Tensor, up: Tensor, need_dgate: bool = True, need_dup: bool = True
) -> tuple[Tensor | None, Tensor | None]:
    if _compiling():
        dg, du = torch.ops.picotron_amd.swiglu_bwd(dout, gate, up)
        return (dg if need_dgate else None), (du if need_dup else None)
    out = _launch("pt_swiglu_bwd", dout, gate, up, bool(need_dgate), bool(need_dup))
    if out is not None:
        return out
    device = _check_cuda(dout, gate, up)
    if dout.dtype != gate.dtype:
        dout = dout.to(gate.dtype)
    dout, gate, up = _flat(dout), _flat(gate), _flat(up)
    dg = torch.empty_like(gate) if need_dgate else None
    du = torch.empty_like(up) if need_dup else None
    _lib.raw_call(
        "pt_swiglu_bwd", dout.data_ptr(), gate.data_ptr(), up.data_ptr(), _ptr(dg), _ptr(du),
        gate.numel(), dtype_code(gate.dtype), _stream(device),
    )
    return dg, du


# ------------------------------------------------------------------ activations kept in 8 bits

BLOCK8 = 128  # elements that share a step (pt_block8_elems)


def swiglu8_fwd(gate: Tensor, up: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """:func:`swiglu_fwd`, and what :func:`swiglu8_bwd` reads of ``gate`` and ``up``: (out, codes, steps), uint8
    (blocks, 16, 2, 8) and fp32 (blocks, 2) over blocks of 128 elements of the flat tensors."""

    if _compiling():
        return torch.ops.picotron_amd.swiglu8_fwd(gate, up)
    device = _check_cuda(gate, up)
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("SwiGLU gate and up must match in shape and dtype")
    gate, up = _flat(gate), _flat(up)
    out = torch.empty_like(gate)
    blocks = (gate.numel() + BLOCK8 - 1) // BLOCK8
    codes = torch.empty((blocks, 16, 2, 8), dtype=torch.uint8, device=device)
    steps = torch.empty((blocks, 2), dtype=torch.float32, device=device)
    _call_on(device, "pt_swiglu8_fwd", gate.data_ptr(), up.data_ptr(), out.data_ptr(), codes.data_ptr(), steps.data_ptr(),
             gate.numel(), dtype_code(gate.dtype))
    return out, codes, steps


def swiglu8_bwd(
    dout: Tensor, codes: Tensor, steps: Tensor, dtype: torch.dtype, need_dgate: bool = True, need_dup: bool = True
) -> tuple[Tensor | None, Tensor | None]:
    """Gradients of ``dtype`` of SwiGLU's inputs from what :func:`swiglu8_fwd` kept of them."""

    if _compiling():
        dg, du = torch.ops.picotron_amd.swiglu8_bwd(dout, codes, steps, dtype)
        return (dg if need_dgate else None), (du if need_dup else None)
    device = _check_cuda(dout, codes, steps)
    if dout.dtype != dtype:
        dout = dout.to(dtype)
    dout, codes, steps = _flat(dout), _flat(codes), _flat(steps)
    blocks = (dout.numel() + BLOCK8 - 1) // BLOCK8
    if (codes.dtype != torch.uint8 or steps.dtype != torch.float32 or codes.shape != (blocks, 16, 2, 8)
            or steps.shape != (blocks, 2)):
        raise ValueError("SwiGLU codes and steps must be those of swiglu8_fwd for this many elements")
    dg = torch.empty_like(dout) if need_dgate else None
    du = torch.empty_like(dout) if need_dup else None
    _call_on(device, "pt_swiglu8_bwd", dout.data_ptr(), codes.data_ptr(), steps.data_ptr(), _ptr(dg), _ptr(du), dout.numel(),
             dtype_code(dtype))
    return dg, du


def rmsnorm8_fwd(
    x: Tensor, weight: Tensor, eps: float, residual: Tensor | None = None
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(h, y, rstd, codes, steps): :func:`rmsnorm_fwd` of x (h is x itself), or :func:`residual_rmsnorm_fwd` of x and
    ``residual``, and what :func:`rmsnorm8_bwd` reads of h: uint8 (rows, blocks, 128) and fp32 (rows, blocks)."""

    if _compiling():
        if residual is None:
            return x, *torch.ops.picotron_amd.rmsnorm8_fwd(x, weight, float(eps))
        return torch.ops.picotron_amd.residual_rmsnorm8_fwd(x, residual, weight, float(eps))
    device = _check_cuda(x, weight) if residual is None else _check_cuda(x, weight, residual)
    cols = x.size(-1)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must match x in shape and dtype")
    if weight.dim() != 1 or weight.numel() != cols:
        raise ValueError("RMSNorm weight must be 1-D with hidden-size elements")
    weight, flat = weight.contiguous(), _flat(x)
    rows = x.numel() // cols if cols else 0
    blocks = (cols + BLOCK8 - 1) // BLOCK8
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=device)
    residual = None if residual is None else _flat(residual)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
    codes = torch.empty((rows, blocks, BLOCK8), dtype=torch.uint8, device=device)
    steps = torch.empty((rows, blocks), dtype=torch.float32, device=device)
    _call_on(
        device, "pt_rmsnorm8_fwd", flat.data_ptr(), _ptr(residual), weight.data_ptr(), _ptr(h), y.data_ptr(), rstd.data_ptr(),
        codes.data_ptr(), steps.data_ptr(), rows, cols, float(eps), dtype_code(x.dtype), dtype_code(weight.dtype),
    )
    return (x if h is None else h), y, rstd, codes, steps


def rmsnorm8_bwd(
    dy: Tensor,
    weight: Tensor,
    rstd: Tensor,
    codes: Tensor,
    steps: Tensor,
    dtype: torch.dtype,
    dh_in: Tensor | None = None,
    need_dx: bool = True,
    need_dw: bool = True,
) -> tuple[Tensor | None, Tensor | None]:
    """Gradients of the norm's input (of ``dtype``, ``dh_in`` added) and weight, from what :func:`rmsnorm8_fwd` kept."""

    if _compiling():
        dx, dw = torch.ops.picotron_amd.rmsnorm8_bwd(dy, weight, rstd, codes, steps, dtype, dh_in)
        return (dx if need_dx else None), (dw if need_dw else None)
    device = _check_cuda(dy, weight, rstd, codes, steps)
    cols = weight.numel()
    if dy.dtype != dtype:
        dy = dy.to(dtype)
    dy, weight, rstd, codes, steps = _flat(dy), weight.contiguous(), _flat(rstd), _flat(codes), _flat(steps)
    rows = dy.numel() // cols if cols else 0
    blocks = (cols + BLOCK8 - 1) // BLOCK8
    if (dy.size(-1) != cols or rstd.numel() != rows or rstd.dtype != torch.float32 or codes.dtype != torch.uint8
            or codes.shape != (rows, blocks, BLOCK8) or steps.dtype != torch.float32 or steps.shape != (rows, blocks)):
        raise ValueError("RMSNorm rstd, codes and steps must be those of rmsnorm8_fwd for these rows")
    if dh_in is not None:
        _check_cuda(dy, dh_in)
        if dh_in.shape != dy.shape:
            raise ValueError("dh_in must match dy")
        dh_in = _flat(dh_in.to(dtype))
    dx = torch.empty(dy.shape, dtype=dtype, device=device) if need_dx else None
    dw = torch.empty(cols, dtype=weight.dtype, device=device) if need_dw else None
    ws = None
    if need_dw:
        ws = torch.empty(max(int(_lib.lib().pt_rmsnorm8_bwd_workspace_bytes(rows, cols)), 16), dtype=torch.uint8, device=device)
    _call_on(
        device, "pt_rmsnorm8_bwd", dy.data_ptr(), _ptr(dh_in), weight.data_ptr(), rstd.data_ptr(), codes.data_ptr(), steps.data_ptr(),
        _ptr(dx), _ptr(dw), _ptr(ws), 0 if ws is None else ws.numel(), rows, cols, dtype_code(dtype), dtype_code(weight.dtype),
    )
    return dx, dw


# ------------------------------------------------------------------ RoPE


def _rope_desc(x: Tensor, y: Tensor) -> ctypes.Array:
    b, h, s, _ = x.shape
    return (ctypes.c_int64 * 9)(
        b, h, s, x.stride(0), x.stride(1), x.stride(2), y.stride(0), y.stride(1), y.stride(2)
    )


def _rope_out(x: Tensor) -> Tensor:
    """A new tensor like ``x`` with a contiguous head_dim: empty_like keeps a dense input's stride order, so that a
    (B, S, H, D)-memory view comes back as one, but moves head_dim outwards for windows that overlap."""

    y = torch.empty_like(x)
    return y if y.stride(-1) == 1 else torch.empty_like(x, memory_format=torch.contiguous_format)


def rope(
    x0: Tensor,
    cos: Tensor,
    sin: Tensor,
    *,
    layout: str = "interleaved",
    inverse: bool = False,
    x1: Tensor | None = None,
) -> tuple[Tensor, Tensor | None]:
    """Rotate (batch, heads, seq, head_dim) views x0 (and x1) by the angle tables.

    ``cos``/``sin`` are fp32 ``[>= seq, head_dim/2]`` tables; row ``s`` is position ``s``.
    Outputs are new tensors with the inputs' logical shape and memory layout.
    """

    if _compiling():
        if x1 is None:
            return torch.ops.picotron_amd.rope(x0, cos, sin, layout, bool(inverse)), None
        y0, y1 = torch.ops.picotron_amd.rope_pair(x0, x1, cos, sin, layout, bool(inverse))
        return y0, y1
    if layout in LAYOUTS:
        out = _launch("pt_rope", x0, x1, cos, sin, LAYOUTS[layout], bool(inverse))
        if out is not None:
            return out
    device = _check_cuda(x0, cos, sin) if x1 is None else _check_cuda(x0, x1, cos, sin)
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}")
    tensors = [x0] if x1 is None else [x0, x1]
    head_dim = x0.size(-1)
    for t in tensors:
        if t.dim() != 4 or t.size(-1) != head_dim or t.stride(-1) != 1:
            raise ValueError("RoPE states must be 4-D (batch, heads, seq, head_dim), head_dim contiguous")
        if t.dtype != x0.dtype:
            raise ValueError("query and key must share a dtype")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("RoPE tables must be fp32")
    cos = cos.contiguous()
    sin = sin.contiguous()
    if cos.dim() != 2 or cos.shape != sin.shape or cos.size(1) * 2 != head_dim:
        raise ValueError("RoPE tables must be [seq, head_dim/2]")
    outs = [_rope_out(t) for t in tensors]
    descs = [_rope_desc(t, o) for t, o in zip(tensors, outs)]
    _lib.raw_call(
        "pt_rope",
        x0.data_ptr(), outs[0].data_ptr(), descs[0],
        None if x1 is None else x1.data_ptr(), None if x1 is None else outs[1].data_ptr(),
        None if x1 is None else descs[1],
        head_dim, cos.data_ptr(), sin.data_ptr(), cos.size(0), LAYOUTS[layout], int(inverse),
        dtype_code(x0.dtype), _stream(device),
    )
    return outs[0], (outs[1] if x1 is not None else None)


def _first_position(position) -> int:
    """The position of a call's first token, from an integer or None (0)."""

    first = int(position or 0)
    if first != (position or 0):
        raise ValueError(f"a RoPE position must be an integer, got {position!r}")
    return first


def _position_strides(positions: Tensor | None, batch: int, seq: int) -> tuple[int, int]:
    """(batch stride, sequence stride) of (seq,), (1, seq) or (batch, seq) positions."""

    if positions is None:
        return 0, 0
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("RoPE positions must be int32 or int64")
    shape = tuple(positions.shape)
    if shape == (seq,):
        return 0, positions.stride(0)
    if shape in ((batch, seq), (1, seq)):
        return (positions.stride(0) if shape[0] > 1 else 0), positions.stride(1)
    raise ValueError(f"RoPE positions must be (seq,), (1, seq) or (batch, seq), here with batch {batch} and seq {seq}; "
                     f"got {shape}")


def rope_at(
    x0: Tensor,
    turns: Tensor,
    *,
    positions: Tensor | None = None,
    offset: int = 0,
    scale: float = 1.0,
    layout: str = "interleaved",
    inverse: bool = False,
    x1: Tensor | None = None,
) -> tuple[Tensor, Tensor | None]:
    """Rotate the first ``2 * turns.numel()`` elements of each head of (batch, heads, seq, head_dim) views x0
    (and x1) by their positions' angles; the others are copied.

    ``turns``: int64, the bits of each pair's fraction of a turn per position times 2^64
    (:meth:`picotron_amd.nn.RotaryFrequencies.turns`).  ``positions``: int32 or int64 of (seq,), (1, seq) or
    (batch, seq), 0 to seq - 1 when absent; ``offset`` is added to each.  Cosine and sine are multiplied by
    ``scale``.  Outputs are new tensors with the inputs' logical shape and memory layout.
    """

    if _compiling():
        if x1 is None:
            return torch.ops.picotron_amd.rope_at(x0, turns, positions, offset, scale, layout, bool(inverse)), None
        y0, y1 = torch.ops.picotron_amd.rope_at_pair(x0, x1, turns, positions, offset, scale, layout, bool(inverse))
        return y0, y1
    if layout in LAYOUTS:
        out = _launch_here("pt_rope_at", x0, x1, turns, positions, offset, scale, LAYOUTS[layout], bool(inverse))
        if out is not None:
            return out
    tensors = [x0] if x1 is None else [x0, x1]
    device = _check_cuda(*tensors, turns, *([] if positions is None else [positions]))
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}")
    for t in tensors:
        if t.dim() != 4 or t.size(-1) != x0.size(-1) or t.stride(-1) != 1:
            raise ValueError("RoPE states must be 4-D (batch, heads, seq, head_dim), head_dim contiguous")
        if t.dtype != x0.dtype:
            raise ValueError("query and key must share a dtype")
        if t.size(0) != x0.size(0) or t.size(2) != x0.size(2):
            raise ValueError("RoPE query and key must share batch and sequence sizes")
    if turns.dtype != torch.int64 or turns.dim() != 1 or not turns.is_contiguous() or turns.numel() * 2 > x0.size(-1):
        raise ValueError("RoPE turns must be contiguous int64, one for each rotated pair of a head")
    if not -(1 << 63) <= offset < 1 << 63:
        raise ValueError("the RoPE position offset must fit 64 bits")
    pbs, pss = _position_strides(positions, x0.size(0), x0.size(2))
    outs = [_rope_out(t) for t in tensors]
    descs = [_rope_desc(t, o) for t, o in zip(tensors, outs)]
    _call_on(
        device,
        "pt_rope_at",
        x0.data_ptr(), outs[0].data_ptr(), descs[0],
        None if x1 is None else x1.data_ptr(), None if x1 is None else outs[1].data_ptr(),
        None if x1 is None else descs[1],
        x0.size(-1), 2 * turns.numel(), _ptr(positions),
        0 if positions is None else positions.element_size(), pbs, pss, int(offset), turns.data_ptr(), float(scale),
        LAYOUTS[layout], int(inverse), dtype_code(x0.dtype),
    )
    return outs[0], (outs[1] if x1 is not None else None)


# ------------------------------------------------------------------ cross-entropy


def ce_rows(logits: Tensor) -> tuple[int, int, int, int, int]:
    """(outer, inner, outer_stride, inner_stride, vocab) of a (N, V) or (B, V, S) input
    whose class dimension (dim 1) is contiguous."""

    if logits.dim() == 2:
        n, v = logits.shape
        if logits.stride(1) != 1 and v > 1:
            raise ValueError("cross-entropy logits need a contiguous class dimension")
        return n, 1, logits.stride(0), 0, v
    if logits.dim() == 3:
        b, v, s = logits.shape
        if logits.stride(1) != 1 and v > 1:
            raise ValueError("cross-entropy logits need a contiguous class dimension")
        return b, s, logits.stride(0), logits.stride(2), v
    raise ValueError("cross-entropy logits must be (N, C) or (N, C, d)")


def rows_disjoint(sizes_strides: list[tuple[int, int]], row_len: int) -> bool:
    """True if rows of ``row_len`` contiguous elements, one per index of the given
    (size, stride) dimensions, never share an element (sufficient test: each stride, in
    increasing order, clears the extent spanned by the dimensions below it)."""

    extent = row_len  # elements spanned by one index of every dimension seen so far
    for stride, size in sorted((abs(st), sz) for sz, st in sizes_strides if sz > 1):
        if stride < extent:
            return False
        extent += stride * (size - 1)
    return True


def ce_target_strides(targets: Tensor, outer: int, inner: int) -> tuple[int, int]:
    if targets.dtype != torch.long:
        raise ValueError("cross-entropy targets must be int64")
    if targets.dim() == 1 and inner == 1:
        if targets.numel() != outer:
            raise ValueError("targets must have one entry per row")
        return targets.stride(0), 0
    if targets.dim() == 2 and tuple(targets.shape) == (outer, inner):
        return targets.stride(0), targets.stride(1)
    raise ValueError("targets shape does not match the logits")


def ce_grad_buffer(logits: Tensor, class_dim: int = 1) -> Tensor | None:
    """An uninitialised tensor of the logits' shape and strides whose data starts in the same
    128-byte phase as the logits', so that every gradient row starts in the phase of its
    logits row: the fused kernels require the same 16-byte phase of a separate gradient, and
    split rows at the logits' 128-byte cache lines, which are then the gradient's lines too
    (and the result bitwise the in-place call's).  ``class_dim``: the contiguous class
    dimension, 1 for (N, C) and (N, C, d) inputs, 2 for the shifted (B, S, V) form.  None when
    the logits rows overlap in memory (an expanded tensor)."""

    native = _lib.extension() if logits.is_cuda and not _compiling() and _lib.is_available() else None
    if native is not None:
        buffer = native.ce_grad_buffer(logits, class_dim)
        if buffer is not None:
            return buffer
    dims = list(zip(logits.shape, logits.stride()))
    rows = [d for i, d in enumerate(dims) if i != class_dim]
    if not rows_disjoint(rows, logits.size(class_dim)):
        return None
    if logits.numel() == 0:
        return torch.empty_like(logits)
    span = 1 + sum((n - 1) * st for n, st in dims)
    per_line = 128 // logits.element_size()
    flat = torch.empty(span + per_line, dtype=logits.dtype, device=logits.device)
    offset = ((logits.data_ptr() - flat.data_ptr()) % 128) // logits.element_size()
    return flat.as_strided(logits.shape, logits.stride(), flat.storage_offset() + offset)


def cross_entropy(
    logits: Tensor, targets: Tensor, ignore_index: int = -100, write_grad: bool = False,
    grad: Tensor | None = None,
) -> tuple[Tensor, Tensor]:
    """Mean cross-entropy (fp32 scalar tensor) over targets != ignore_index.

    With ``write_grad`` (fp32 and bf16) d(loss)/d(logits) is written in the same pass: into
    ``grad`` when given (the logits' shape, rows in the logits rows' 16-byte phase, e.g. from
    :func:`ce_grad_buffer`; the logits are only read), else over the logits in place.  fp16
    writes its gradient in :func:`cross_entropy_scale_grad`.
    Returns (loss, workspace); the workspace holds the status word (bit 0: a target out
    of range), readable with :func:`cross_entropy_status`.
    """

    out = None if _compiling() else _launch("pt_cross_entropy", logits, targets, ignore_index, bool(write_grad), grad, 0)
    if out is not None:
        return out
    device = _check_cuda(logits, targets)
    outer, inner, os_, is_, vocab = ce_rows(logits)
    tos, tis = ce_target_strides(targets, outer, inner)
    gos = gis = 0
    if grad is not None:
        if grad.shape != logits.shape or grad.dtype != logits.dtype or grad.device != logits.device:
            raise ValueError("the gradient buffer must match the logits")
        _, _, gos, gis, _ = ce_rows(grad)
        if write_grad and not rows_disjoint([(outer, gos), (inner, gis)], vocab):
            raise ValueError("cross-entropy gradient rows overlap in memory")
    elif write_grad and not rows_disjoint([(outer, os_), (inner, is_)], vocab):
        raise ValueError("cross-entropy logits rows overlap in memory; the gradient cannot be "
                         "written into them")
    rows = outer * inner
    ws_bytes = _lib.lib().pt_cross_entropy_workspace_bytes(rows)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    loss = torch.empty((), dtype=torch.float32, device=device)
    _lib.raw_call(
        "pt_cross_entropy",
        logits.data_ptr(), outer, inner, os_, is_, vocab, targets.data_ptr(), tos, tis,
        int(ignore_index), loss.data_ptr(), int(write_grad), _ptr(grad), gos, gis, ws.data_ptr(),
        ws_bytes, dtype_code(logits.dtype), _stream(device),
    )
    return loss, ws


def cross_entropy_status(ws: Tensor) -> int:
    """Status word of a cross-entropy workspace (synchronises with the device)."""

    return int(ws[8:12].view(torch.int32).item())


def cross_entropy_scale_grad(
    dlogits: Tensor, targets: Tensor, grad_output: Tensor, ignore_index: int = -100,
    workspace: Tensor | None = None, logits: Tensor | None = None,
) -> None:
    """dlogits *= grad_output in place (skipped on device when grad_output == 1).  For fp16
    the forward left the logits unchanged and this call writes the gradient,
    (softmax - onehot) * grad_output / n_valid rounded once, from the row log-sum-exps and
    n_valid in ``workspace`` (the forward's): computed from ``logits`` into ``dlogits`` (rows
    in the same 16-byte phase) when ``logits`` is given, else over ``dlogits`` in place."""

    if not _compiling() and _launch("pt_cross_entropy_scale_grad", dlogits, targets, grad_output, ignore_index, workspace, logits, 0):
        return
    device = _check_cuda(dlogits, targets, grad_output)
    outer, inner, os_, is_, vocab = ce_rows(dlogits)
    tos, tis = ce_target_strides(targets, outer, inner)
    los = lis = 0
    if logits is not None:
        if logits.shape != dlogits.shape or logits.dtype != dlogits.dtype:
            raise ValueError("logits must match the gradient buffer")
        _, _, los, lis, _ = ce_rows(logits)
    go = grad_output.detach().to(torch.float32).reshape(())
    _lib.raw_call(
        "pt_cross_entropy_scale_grad",
        dlogits.data_ptr(), outer, inner, os_, is_, vocab, targets.data_ptr(), tos, tis,
        int(ignore_index), go.data_ptr(), _ptr(logits), los, lis, _ptr(workspace),
        dtype_code(dlogits.dtype), _stream(device),
    )


def _shifted_desc(logits: Tensor, input_ids: Tensor,
                  next_targets: bool = False) -> tuple[int, int, int, int, int, int, int]:
    """(batch, seq, batch_stride, seq_stride, vocab, ids_batch_stride, ids_seq_stride).
    ``next_targets``: ``input_ids`` holds the targets themselves, (batch, seq - 1), entry
    (b, t) for position t (the train loop's ``input_ids[:, 1:]``)."""

    if logits.dim() != 3:
        raise ValueError("shifted cross-entropy logits must be (batch, seq, vocab)")
    b, s, v = logits.shape
    if logits.stride(2) != 1 and v > 1:
        raise ValueError("cross-entropy logits need a contiguous vocabulary dimension")
    if input_ids.dtype != torch.long:
        raise ValueError("cross-entropy targets must be int64")
    want = (b, s - 1) if next_targets else (b, s)
    if input_ids.dim() != 2 or tuple(input_ids.shape) != want:
        raise ValueError(f"targets must be {want} for (batch, seq, vocab) logits")
    return b, s, logits.stride(0), logits.stride(1), v, input_ids.stride(0), input_ids.stride(1)


def _ids_ptr(input_ids: Tensor, next_targets: bool) -> int:
    """The address the shifted entry points take as input_ids: they read position t's target
    at input_ids + (t + 1) * seq_stride, so targets already shifted by one (entry t for
    position t) are passed as the address one position before them (never dereferenced)."""

    if not next_targets:
        return input_ids.data_ptr()
    return input_ids.data_ptr() - input_ids.stride(1) * input_ids.element_size()


def cross_entropy_shifted(
    logits: Tensor, input_ids: Tensor, ignore_index: int = -100, write_grad: bool = False,
    grad: Tensor | None = None, next_targets: bool = False,
) -> tuple[Tensor, Tensor]:
    """Next-token mean cross-entropy of (B, S, V) logits against input_ids[:, 1:]: equal to
    :func:`cross_entropy` on ``logits[:, :-1, :].transpose(1, 2)``.  With ``write_grad`` the
    gradient covers the whole (B, S, V) buffer (last position zero): into ``grad`` when
    given (as in :func:`cross_entropy`), else over the logits.  ``next_targets``:
    ``input_ids`` is already the (B, S - 1) targets (the train loop's ``input_ids[:, 1:]``)."""

    out = None if _compiling() else _launch("pt_cross_entropy_shifted", logits, input_ids, ignore_index, bool(write_grad), grad,
                  2 if next_targets else 1)
    if out is not None:
        return out
    device = _check_cuda(logits, input_ids)
    b, s, bs, ss, v, ibs, iss = _shifted_desc(logits, input_ids, next_targets)
    gbs = gss = 0
    if grad is not None:
        if grad.shape != logits.shape or grad.dtype != logits.dtype or grad.device != logits.device:
            raise ValueError("the gradient buffer must match the logits")
        gbs, gss = grad.stride(0), grad.stride(1)
        if grad.stride(2) != 1 and v > 1:
            raise ValueError("the gradient buffer needs a contiguous vocabulary dimension")
        if write_grad and not rows_disjoint([(b, gbs), (s, gss)], v):
            raise ValueError("cross-entropy gradient rows overlap in memory")
    elif write_grad and not rows_disjoint([(b, bs), (s, ss)], v):
        raise ValueError("cross-entropy logits rows overlap in memory; the gradient cannot be "
                         "written into them")
    ws_bytes = _lib.lib().pt_cross_entropy_workspace_bytes(b * s)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    loss = torch.empty((), dtype=torch.float32, device=device)
    _lib.raw_call(
        "pt_cross_entropy_shifted",
        logits.data_ptr(), b, s, bs, ss, v, _ids_ptr(input_ids, next_targets), ibs, iss,
        int(ignore_index), loss.data_ptr(), int(write_grad), _ptr(grad), gbs, gss,
        ws.data_ptr(), ws_bytes, dtype_code(logits.dtype), _stream(device),
    )
    return loss, ws


def cross_entropy_shifted_scale_grad(
    dlogits: Tensor, input_ids: Tensor, grad_output: Tensor, ignore_index: int = -100,
    workspace: Tensor | None = None, logits: Tensor | None = None, next_targets: bool = False,
) -> None:
    """dlogits *= grad_output in place for a gradient from :func:`cross_entropy_shifted`
    (fp16: as :func:`cross_entropy_scale_grad`, with the forward's ``workspace``, from
    ``logits`` into ``dlogits`` when ``logits`` is given)."""

    if not _compiling() and _launch("pt_cross_entropy_shifted_scale_grad", dlogits, input_ids, grad_output, ignore_index,
               workspace, logits, 2 if next_targets else 1):
        return
    device = _check_cuda(dlogits, input_ids, grad_output)
    b, s, bs, ss, v, ibs, iss = _shifted_desc(dlogits, input_ids, next_targets)
    lbs = lss = 0
    if logits is not None:
        if logits.shape != dlogits.shape or logits.dtype != dlogits.dtype:
            raise ValueError("logits must match the gradient buffer")
        lbs, lss = logits.stride(0), logits.stride(1)
    go = grad_output.detach().to(torch.float32).reshape(())
    _lib.raw_call(
        "pt_cross_entropy_shifted_scale_grad",
        dlogits.data_ptr(), b, s, bs, ss, v, _ids_ptr(input_ids, next_targets), ibs, iss,
        int(ignore_index), go.data_ptr(), _ptr(logits), lbs, lss, _ptr(workspace),
        dtype_code(dlogits.dtype), _stream(device),
    )


# ------------------------------------------------------------------ cross-entropy of a head

REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


def head_rows(hidden: Tensor, weight: Tensor, labels: Tensor, shift: bool) -> tuple[int, int, int]:
    """(outer, inner, rows of an outer index) of (batch, seq, hidden) or (tokens, hidden) states with labels of their leading
    shape; with ``shift`` position t belongs to label t + 1, and the last one to none."""

    if hidden.dim() not in (2, 3) or hidden.size(-1) < 1:
        raise ValueError("hidden states must be (batch, seq, hidden) or (tokens, hidden)")
    if weight.dim() != 2 or weight.size(1) != hidden.size(-1) or weight.size(0) < 1:
        raise ValueError("the head's weight must be (vocab, hidden)")
    if hidden.dtype != weight.dtype or hidden.dtype not in _DTYPE_CODES:
        raise ValueError("hidden states and the head's weight must be float32, float16 or bfloat16, both of one type")
    if labels.dtype != torch.int64 or labels.shape != hidden.shape[:-1]:
        raise ValueError("labels must be int64, one a hidden state")
    if shift and hidden.dim() != 3:
        raise ValueError("shifted labels need (batch, seq, hidden) states")
    if hidden.dim() == 2:
        return 1, hidden.size(0), hidden.size(0)
    seq = hidden.size(1)
    return hidden.size(0), (max(seq - 1, 0) if shift else seq), seq


def head_defers(hidden: Tensor, reduction: str) -> bool:
    """Whether the gradients of a head's loss are formed in its backward: those of single tokens' losses are; and of a mean or
    sum of up to 512 fp16 states, for which, at a large weight, another product of their logits takes less time than gradients in
    fp32 and their rounding once a loss scale has arrived (128256 words of 4096, 45 states: 1.09 ms, with fp32 gradients 1.79;
    512: 2.16 and 2.58; 1024: 3.88 and 3.92; 32000 of 2048, 64: 195 us and 264; 512: 347 and 386).  Small weights, and those that are
    copied, lose by it (512 states, 2000 words of 192: 94 us and 78; 50257 of 64: 152 and 113; 32001 of 1090: 385 and 341); they
    take the rule too, as it also says which losses can be differentiated again."""

    return reduction == "none" or (hidden.dtype == torch.float16 and hidden.numel() // hidden.size(-1) <= 512)


def linear_cross_entropy(
    hidden: Tensor,
    weight: Tensor,
    labels: Tensor,
    *,
    shift: bool = False,
    ignore_index: int = -100,
    reduction: str = "mean",
    want_loss: bool = True,
    want_dx: bool = False,
    want_dw: bool = False,
    grad_losses: Tensor | None = None,
    grad_dtype: torch.dtype | None = None,
    chunk_tokens: int = 0,
) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """Cross-entropy of ``hidden @ weight.T`` against ``labels`` without those logits, and its gradients: (loss, dx, dw).

    The loss is an fp32 scalar, or with reduction ``"none"`` fp32 of the labels' shape (seq - 1 with ``shift``).  The
    gradients (of ``grad_dtype``: the inputs' type or fp32) are those for the incoming gradient ``grad_losses``, of the loss's
    shape (of a mean or sum 1 where it is absent).  At most ``chunk_tokens`` tokens are worked on at a time (0: as many as keep the
    exponentials within 2 GiB)."""

    if not -(2**63) <= ignore_index < 2**63:  # ctypes would take it modulo 2^64, which may be a label
        raise ValueError("ignore_index must fit an int64, as the labels do")
    device = _check_cuda(hidden, weight, labels)
    outer, inner, dx_inner = head_rows(hidden, weight, labels, shift)
    if hidden.stride(-1) != 1:
        hidden = hidden.contiguous()
    vocab, width = weight.shape
    if weight.stride(1) != 1 or weight.stride(0) < width:
        weight = weight.contiguous()
    xs = (hidden.stride(0), hidden.stride(1)) if hidden.dim() == 3 else (0, hidden.stride(0))
    ts = (labels.stride(0), labels.stride(1)) if labels.dim() == 2 else (0, labels.stride(0))
    shape = labels.shape[:-1] + (inner,) if shift else labels.shape
    if shift:
        labels = labels[:, 1:]
    gs = (0, 0)
    if grad_losses is not None:
        if grad_losses.shape != (shape if reduction == "none" else ()) or grad_losses.device != device:
            raise ValueError("the losses' gradients must have the losses' shape")
        grad_losses = grad_losses.to(torch.float32)
        if reduction == "none":
            gs = (grad_losses.stride(0), grad_losses.stride(1)) if grad_losses.dim() == 2 else (0, grad_losses.stride(0))
    dtype = grad_dtype or hidden.dtype
    loss = None
    if want_loss:
        loss = torch.empty(shape if reduction == "none" else (), dtype=torch.float32, device=device)
    dx = torch.empty(hidden.shape, dtype=dtype, device=device) if want_dx else None
    dw = torch.empty(weight.shape, dtype=dtype, device=device) if want_dw else None
    if outer * inner == 0:
        if loss is not None:
            loss.fill_(float("nan") if reduction == "mean" else 0.0)
        return loss, None if dx is None else dx.zero_(), None if dw is None else dw.zero_()
    code = dtype_code(hidden.dtype)
    ws_bytes = _lib.lib().pt_linear_cross_entropy_workspace_bytes(
        outer * inner, vocab, width, weight.data_ptr(), weight.stride(0), code, int(want_dx), int(want_dw), int(chunk_tokens))
    ws = torch.empty(max(int(ws_bytes), 16), dtype=torch.uint8, device=device)
    _call_on(
        device, "pt_linear_cross_entropy", hidden.data_ptr(), *xs, outer, inner, weight.data_ptr(), weight.stride(0), vocab, width,
        labels.data_ptr(), *ts, int(ignore_index), REDUCTIONS[reduction], _ptr(loss), _ptr(grad_losses), *gs, _ptr(dx), dx_inner,
        _ptr(dw), dtype_code(dtype), ws.data_ptr(), ws.numel(), int(chunk_tokens), code,
    )
    return loss, dx, dw


def scale_gradients(grads: tuple[Tensor | None, Tensor | None], scale: Tensor, dtype: torch.dtype) -> tuple[Tensor | None, Tensor | None]:
    """Up to two contiguous gradients of one type times the device scalar ``scale``: in place, left alone where the scale is 1, or
    from fp32 to new tensors of ``dtype``.  The products are rounded once, 16-bit gradients that came rounded for a second time."""

    given = [g for g in grads if g is not None]
    device = _check_cuda(scale, *given)
    scale = scale.detach().to(torch.float32).reshape(())
    to = [None if g is None else (g if g.dtype == dtype else torch.empty(g.shape, dtype=dtype, device=device)) for g in grads]
    args = [a for g, t in zip(grads, to) for a in (_ptr(g), _ptr(t), 0 if g is None else g.numel())]
    _call_on(device, "pt_scale_gradients", *args, dtype_code(given[0].dtype), dtype_code(dtype), scale.data_ptr())
    return to[0], to[1]


# ------------------------------------------------------------------ preference loss

PREFERENCE_LOSSES = {"sigmoid": 0, "hinge": 1, "ipo": 2}


def _sequence_rows(logits: Tensor, labels: Tensor, shift: bool) -> tuple:
    """(seq, batch stride, seq stride, vocab, labels, their strides, shift) of (batch, seq, vocab) logits and (batch, seq)
    labels, as the entry points take them."""

    if logits.dim() != 3 or logits.size(2) < 1:
        raise ValueError("logits must be (batch, seq, vocab)")
    if logits.stride(2) != 1 and logits.size(2) > 1:
        raise ValueError("logits need a contiguous vocabulary dimension")
    if labels.dtype != torch.int64 or tuple(labels.shape) != tuple(logits.shape[:2]):
        raise ValueError(f"labels must be int64 of shape {tuple(logits.shape[:2])}")
    return (logits.size(1), logits.stride(0), logits.stride(1), logits.size(2), labels.data_ptr(), labels.stride(0),
            labels.stride(1), int(shift))


def _sequence_workspace(logits: Tensor) -> tuple[Tensor, int]:
    size = int(_lib.lib().pt_sequence_log_probs_workspace_bytes(*logits.shape, dtype_code(logits.dtype)))
    return torch.empty(max(size, 16), dtype=torch.uint8, device=logits.device), size


def sequence_log_probs(
    logits: Tensor, labels: Tensor, *, shift: bool = True, ignore_index: int = -100, average: bool = False
) -> tuple[Tensor, Tensor]:
    """(log-probability of each sequence's kept labels, fp32; workspace for :func:`sequence_log_probs_bwd`)."""

    out = _launch_here("pt_sequence_log_probs", logits, labels, bool(shift), ignore_index, bool(average))
    if out is not None:
        return out
    device = _check_cuda(logits, labels)
    rows = _sequence_rows(logits, labels, shift)
    ws, size = _sequence_workspace(logits)
    out = torch.empty(logits.size(0), dtype=torch.float32, device=device)
    _call_on(device, "pt_sequence_log_probs", logits.data_ptr(), logits.size(0), *rows, int(ignore_index), int(average),
             out.data_ptr(), ws.data_ptr(), size, dtype_code(logits.dtype))
    return out, ws


def preference_loss(
    logits: Tensor, labels: Tensor, reference: Tensor | None, *, beta: float, label_smoothing: float = 0.0,
    kind: str = "sigmoid", shift: bool = True, ignore_index: int = -100, average: bool = False,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(loss, rewards, log-probabilities, workspace) over logits whose first half of sequences are the chosen ones of
    the pairs and whose second half the rejected ones; ``reference``: fp32 log-probabilities, or None for zeros."""

    if kind in PREFERENCE_LOSSES:
        out = _launch_here("pt_preference_loss", logits, labels, reference, beta, label_smoothing, PREFERENCE_LOSSES[kind],
                           bool(shift), ignore_index, bool(average))
        if out is not None:
            return out
    device = _check_cuda(logits, labels, *([] if reference is None else [reference]))
    rows = _sequence_rows(logits, labels, shift)
    batch = logits.size(0)
    if batch < 2 or batch % 2 != 0:
        raise ValueError("a preference loss takes pairs: an even number of sequences, the chosen ones first")
    if reference is not None and (reference.dtype != torch.float32 or tuple(reference.shape) != (batch,)
                                  or not reference.is_contiguous()):
        raise ValueError("reference log-probabilities must be contiguous fp32, one a sequence")
    if kind not in PREFERENCE_LOSSES:
        raise ValueError(f"loss must be one of {sorted(PREFERENCE_LOSSES)}")
    ws, size = _sequence_workspace(logits)
    loss = torch.empty((), dtype=torch.float32, device=device)
    rewards = torch.empty(batch, dtype=torch.float32, device=device)
    log_probs = torch.empty_like(rewards)
    _call_on(device, "pt_preference_loss", logits.data_ptr(), batch // 2, *rows, int(ignore_index), int(average),
             _ptr(reference), float(beta), float(label_smoothing), PREFERENCE_LOSSES[kind], loss.data_ptr(),
             rewards.data_ptr(), log_probs.data_ptr(), ws.data_ptr(), size, dtype_code(logits.dtype))
    return loss, rewards, log_probs, ws


def sequence_log_probs_bwd(
    logits: Tensor, labels: Tensor, workspace: Tensor, *, grad_log_probs: Tensor | None = None,
    grad_loss: Tensor | None = None, shift: bool = True, ignore_index: int = -100,
) -> Tensor:
    """The logits' gradient, from the gradient of the log-probabilities or of the preference loss (a scalar) whose
    forward left ``workspace``."""

    up = grad_log_probs if grad_log_probs is not None else grad_loss
    grad = _launch_here("pt_sequence_log_probs_bwd", logits, labels, workspace, up, grad_log_probs is None, bool(shift),
                        ignore_index)
    if grad is not None:
        return grad
    device = _check_cuda(logits, labels, workspace, up)
    grad = ce_grad_buffer(logits, 2)
    if grad is None:  # rows that overlap in memory (an expanded tensor)
        logits = logits.contiguous()
        grad = ce_grad_buffer(logits, 2)
    rows = _sequence_rows(logits, labels, shift)
    up = up.detach().to(torch.float32).contiguous()
    if up.numel() != (1 if grad_log_probs is None else logits.size(0)):
        raise ValueError("one gradient a sequence, or one of the loss")
    size = int(_lib.lib().pt_sequence_log_probs_workspace_bytes(*logits.shape, dtype_code(logits.dtype)))
    if workspace.numel() < size:
        raise ValueError("the workspace is not that of these logits")
    _call_on(device, "pt_sequence_log_probs_bwd", logits.data_ptr(), logits.size(0), *rows, int(ignore_index),
             up.data_ptr() if grad_log_probs is not None else None, up.data_ptr() if grad_log_probs is None else None,
             grad.data_ptr(), grad.stride(0), grad.stride(1), workspace.data_ptr(), size, dtype_code(logits.dtype))
    return grad


# ------------------------------------------------------------------ AdamW


def adamw_block_elems() -> int:
    return int(_lib.lib().pt_adamw_block_elems())


@functools.lru_cache(maxsize=None)
def _adamw_block_elems() -> int:
    return adamw_block_elems()


def adamw_table(
    params: list[Tensor], grads: list[Tensor], exp_avgs: list[Tensor], exp_avg_sqs: list[Tensor]
) -> tuple[Tensor, int]:
    """Host int64 [n, 6] table for :func:`adamw_step` and its total block count."""

    per = _adamw_block_elems()
    rows = []
    first = 0
    for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs):
        n = p.numel()
        if n == 0:
            continue
        rows += (p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), n, first)
        first += (n + per - 1) // per
    table = torch.from_numpy(np.array(rows, dtype=np.int64).reshape(-1, 6))
    return table, first


_MOMENT_ALIGN = 64  # elements: every moment starts 256 bytes apart from the buffer's start


def adamw_moments(params: list[Tensor]) -> list[tuple[Tensor, Tensor]]:
    """Zeroed fp32 (exp_avg, exp_avg_sq) for each of ``params`` (one device, contiguous), as
    views of one allocation: every first moment, then every second moment, each view with its
    parameter's shape and 256-byte aligned.  The two moments of a parameter then lie a fixed
    distance apart inside one allocation; as separate allocations their placement relative to
    each other varies, and the update's four concurrent streams ran up to 8 % slower on some
    placements (1.2e9 parameters: 5.70 against 5.40 ms per step on the same parameters and
    gradients)."""

    offsets = []
    total = 0
    for p in params:
        offsets.append(total)
        total += (p.numel() + _MOMENT_ALIGN - 1) // _MOMENT_ALIGN * _MOMENT_ALIGN
    if not params:
        return []
    buf = torch.zeros(2 * total, dtype=torch.float32, device=params[0].device)
    return [(buf[o:o + p.numel()].view(p.shape), buf[total + o:total + o + p.numel()].view(p.shape))
            for p, o in zip(params, offsets)]


def adamw_step(
    table_device: Tensor,
    total_blocks: int,
    *,
    lr: float,
    beta1: float,
    beta2: float,
    eps: float,
    weight_decay: float,
    step: float,
) -> None:
    """One AdamW step over the tensors in a device table built from :func:`adamw_table`."""

    device = _check_cuda(table_device)
    _lib.call(
        "pt_adamw_step",
        table_device.data_ptr(), table_device.size(0), int(total_blocks), float(lr), float(beta1),
        float(beta2), float(eps), float(weight_decay), float(step), _stream(device),
    )


def adamw_step_scaled(
    table_device: Tensor,
    total_blocks: int,
    grad_scale: Tensor,
    *,
    lr: float,
    beta1: float,
    beta2: float,
    eps: float,
    weight_decay: float,
    step: float,
    write_grad: bool,
) -> None:
    """:func:`adamw_step` with every gradient multiplied by the fp32 device scalar
    ``grad_scale`` as it is read (and stored back when ``write_grad``)."""

    device = _check_cuda(table_device, grad_scale)
    if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1:
        raise ValueError("grad_scale must be one fp32 element")
    _lib.call(
        "pt_adamw_step_scaled",
        table_device.data_ptr(), table_device.size(0), int(total_blocks), float(lr), float(beta1),
        float(beta2), float(eps), float(weight_decay), float(step), grad_scale.data_ptr(),
        int(write_grad), _stream(device),
    )


def adamw_step_table(params: list[Tensor], steps: list[Tensor]) -> Tensor:
    """Host int64 [n] addresses of the fp32 device step of each parameter, in the row order
    of :func:`adamw_table` (which skips empty parameters)."""

    addrs = [s.data_ptr() for p, s in zip(params, steps) if p.numel() > 0]
    return torch.from_numpy(np.array(addrs, dtype=np.int64))


def adamw_step_device_step(
    table_device: Tensor,
    total_blocks: int,
    step_table_device: Tensor,
    *,
    lr: float,
    beta1: float,
    beta2: float,
    eps: float,
    weight_decay: float,
    grad_scale: Tensor | None = None,
    write_grad: bool = False,
    found_inf: Tensor | None = None,
    inv_scale: Tensor | None = None,
) -> None:
    """:func:`adamw_step` (or :func:`adamw_step_scaled` with ``grad_scale``) for a capturable
    optimizer: the step counts are fp32 device scalars, already advanced, whose addresses
    ``step_table_device`` lists in table row order.  With ``found_inf`` (the int32 flag of
    :func:`grad_stats`; needs ``grad_scale`` and ``inv_scale``) the update runs only when the
    flag is 0; when it is set the gradients are only multiplied by ``inv_scale``, decided on
    the device (advance the step counts by ``1 - found_inf``)."""

    device = _check_cuda(table_device, step_table_device)
    if step_table_device.dtype != torch.int64 or step_table_device.numel() != table_device.size(0):
        raise ValueError("the step table needs one int64 address per table row")
    for name, t, dtype in (("grad_scale", grad_scale, torch.float32), ("inv_scale", inv_scale, torch.float32),
                           ("found_inf", found_inf, torch.int32)):
        if t is not None:
            _check_cuda(t)
            if t.dtype != dtype or t.numel() != 1:
                raise ValueError(f"{name} must be one {dtype} element")
    if found_inf is None:
        _lib.call(
            "pt_adamw_step_device_step",
            table_device.data_ptr(), table_device.size(0), int(total_blocks), step_table_device.data_ptr(),
            float(lr), float(beta1), float(beta2), float(eps), float(weight_decay), _ptr(grad_scale),
            int(write_grad), _stream(device),
        )
        return
    if grad_scale is None or inv_scale is None:
        raise ValueError("a guarded step needs grad_scale and inv_scale")
    _lib.call(
        "pt_adamw_step_device_step_guarded",
        table_device.data_ptr(), table_device.size(0), int(total_blocks), step_table_device.data_ptr(),
        float(lr), float(beta1), float(beta2), float(eps), float(weight_decay), grad_scale.data_ptr(),
        int(write_grad), found_inf.data_ptr(), inv_scale.data_ptr(), _stream(device),
    )


_ADAMW8_STATE = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")


@functools.lru_cache(maxsize=None)
def adamw8_sizes() -> tuple[int, int]:
    """(elements of a table block, elements that share a scale) of the AdamW step with 8-bit moments."""

    return int(_lib.lib().pt_adamw8_block_elems()), int(_lib.lib().pt_adamw8_scale_elems())


def adamw8_reason(p: Tensor, state: dict) -> str | None:
    """Why the kernel's raw pointers may not be given parameter ``p`` and its 8-bit ``state``; None if they may."""

    if not p.is_cuda or p.dtype not in _DTYPE_CODES or p.is_sparse or not p.is_contiguous():
        return "parameters that are not dense contiguous fp32, fp16 or bf16 GPU tensors"
    per = adamw8_sizes()[1]
    blocks = (p.numel() + per - 1) // per
    for key in _ADAMW8_STATE:
        t = state.get(key)
        shape = (blocks,) if key.endswith("scale") else (blocks, per)
        if (not isinstance(t, Tensor) or t.dtype != torch.uint8 or t.device != p.device or tuple(t.shape) != shape
                or not t.is_contiguous() or (len(shape) == 2 and t.data_ptr() % 4 != 0)):
            return f"8-bit states whose {key} is not {shape} contiguous uint8 on the parameter's device"
    return None


def adamw8_table(params: list[Tensor], grads: list[Tensor], states: list[dict]) -> tuple[Tensor, int]:
    """Host int64 [n, 8] table for :func:`adamw8_step` and its block count (no empty parameters)."""

    per = adamw8_sizes()[0]
    rows = []
    first = 0
    for p, g, state in zip(params, grads, states):
        n = p.numel()
        rows += (p.data_ptr(), g.data_ptr(), state["exp_avg"].data_ptr(), state["exp_avg_scale"].data_ptr(),
                 state["exp_avg_sq"].data_ptr(), state["exp_avg_sq_scale"].data_ptr(), n, first)
        first += (n + per - 1) // per
    return torch.from_numpy(np.array(rows, dtype=np.int64).reshape(-1, 8)), first


def adamw8_step(
    table_device: Tensor,
    total_blocks: int,
    dtype: torch.dtype,
    *,
    lr: float,
    beta1: float,
    beta2: float,
    eps: float,
    weight_decay: float,
    step: float | Tensor,
    seed: int,
    stochastic: bool,
    grad_scale: Tensor | None = None,
) -> None:
    """One AdamW step with 8-bit moments over the tensors (parameters of ``dtype``) in a device table built from
    :func:`adamw8_table`.  ``step``: the step's number, or the fp32 device scalar that counts them, which the call
    advances.  ``grad_scale`` (fp32 device scalar) multiplies every gradient as it is read."""

    device = _check_cuda(table_device)
    workspace = device_step = None
    if isinstance(step, Tensor):
        if step.dtype != torch.float32 or step.numel() != 1 or step.device != device:
            raise ValueError("a device step must be one fp32 element on the table's device")
        device_step, step = step, 0.0
        workspace = torch.empty(64, dtype=torch.uint8, device=device)
    if grad_scale is not None and (grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != device):
        raise ValueError("grad_scale must be one fp32 element on the table's device")
    _call_on(
        device, "pt_adamw8_step", table_device.data_ptr(), table_device.size(0), int(total_blocks), float(lr), float(beta1),
        float(beta2), float(eps), float(weight_decay), float(step), _ptr(device_step), _ptr(workspace), _ptr(grad_scale),
        int(seed) & 0xFFFFFFFF, int(stochastic), dtype_code(dtype),
    )


def adamw8_moments(
    params: list[Tensor], states: list[dict], dtype: torch.dtype = torch.float32
) -> tuple[Tensor, Tensor, list[tuple[Tensor, int]]] | None:
    """The values of the 8-bit moments of parameters on one device, flat: (exp_avg, exp_avg_sq, each parameter's place),
    zeros between them; None where the kernel cannot read or write them."""

    device = params[0].device
    if dtype not in _DTYPE_CODES or device.type != "cuda" or not _lib.is_available() or not device_supported(device.index):
        return None
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("AdamW moments: their table is copied to the device, which a graph capture cannot hold")
    per, scale = adamw8_sizes()
    native = _lib.extension()
    found = None if native is None else native.adamw8_table(params, states, per, scale)
    if found is not None:
        table, blocks = torch.frombuffer(bytearray(found[0]), dtype=torch.int64).view(-1, 8), found[1]
    elif all(adamw8_reason(p, state) is None for p, state in zip(params, states)):
        table, blocks = adamw8_table(params, params, states)
    else:
        return None
    m = torch.empty(blocks * per, dtype=dtype, device=device)
    v = torch.empty_like(m)
    places = [(p, first * per) for p, first in zip(params, table[:, 7].tolist())]
    table = table.to(device)
    _call_on(device, "pt_adamw8_moments", table.data_ptr(), len(params), blocks, m.data_ptr(), v.data_ptr(),
             dtype_code(dtype))
    return m, v, places


def clip_grad_norm(table_device: Tensor, total_blocks: int, max_norm: float) -> tuple[Tensor, Tensor]:
    """(total_norm, clip_coef) fp32 device scalars over the gradients of a table built by
    :func:`adamw_table`: torch.nn.utils.clip_grad_norm_'s norm and clamped coefficient."""

    device = _check_cuda(table_device)
    out = torch.empty(2, dtype=torch.float32, device=device)
    ws_bytes = _lib.lib().pt_clip_grad_norm_workspace_bytes(int(total_blocks))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=device)
    _lib.call(
        "pt_clip_grad_norm",
        table_device.data_ptr(), table_device.size(0), int(total_blocks), float(max_norm),
        out.data_ptr(), out.data_ptr() + 4, ws.data_ptr(), ws_bytes, _stream(device),
    )
    return out[0], out[1:2]


CLIP_CLAMP = 0         # torch.nn.utils.clip_grad_norm_: g *= min(coef, 1)
CLIP_IF_BELOW_ONE = 1  # the ZeRO optimizer: g *= coef only when coef < 1


def grad_stats(
    table_device: Tensor,
    total_blocks: int,
    inv_scale: Tensor | None = None,
    max_norm: float | None = None,
    clip_mode: int = CLIP_CLAMP,
) -> tuple[Tensor, Tensor, Tensor]:
    """(total_norm, grad_scale, found_inf) device scalars over a table's gradients: the
    norm of g * inv_scale, inv_scale times the clip coefficient (1 without ``max_norm``),
    and whether any gradient is inf or NaN (int32)."""

    device = _check_cuda(table_device)
    if inv_scale is not None:
        _check_cuda(inv_scale)
        if inv_scale.dtype != torch.float32 or inv_scale.numel() != 1:
            raise ValueError("inv_scale must be one fp32 element")
    out = torch.empty(3, dtype=torch.float32, device=device)
    ws_bytes = _lib.lib().pt_grad_stats_workspace_bytes(int(total_blocks))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=device)
    _lib.call(
        "pt_grad_stats",
        table_device.data_ptr(), table_device.size(0), int(total_blocks), _ptr(inv_scale),
        -1.0 if max_norm is None else float(max_norm), int(clip_mode), out.data_ptr(),
        out.data_ptr() + 4, out.data_ptr() + 8, ws.data_ptr(), ws_bytes, _stream(device),
    )
    return out[0], out[1:2], out[2:3].view(torch.int32)


def grad_scale(table_device: Tensor, total_blocks: int, scale: Tensor) -> None:
    """g *= scale (fp32 device scalar) in place for every gradient of a table."""

    device = _check_cuda(table_device, scale)
    _lib.call("pt_grad_scale", table_device.data_ptr(), table_device.size(0), int(total_blocks),
              scale.data_ptr(), _stream(device))


# ------------------------------------------------------------------ utility


def copy_bytes(src: Tensor, dst: Tensor) -> None:
    """128-bit streaming device copy of src into dst (same byte size)."""

    device = _check_cuda(src, dst)
    nbytes = src.numel() * src.element_size()
    if dst.numel() * dst.element_size() != nbytes or not src.is_contiguous() or not dst.is_contiguous():
        raise ValueError("copy_bytes needs contiguous tensors of equal byte size")
    _lib.call("pt_copy", src.data_ptr(), dst.data_ptr(), nbytes, _stream(device))


# ------------------------------------------------------------------ torch.compile
#
# The launchers of the ops a compiled model contains (RMSNorm, the residual add + norm, SwiGLU,
# RoPE) as custom operators: torch.compile records a call as one opaque node (no graph break
# at the ctypes call) and propagates shapes through the fake implementations; the compiled
# graph calls the launcher eagerly.  Every output is a new tensor.  The cross-entropy and the
# optimizer step run outside picotron's compiled model (train_loop.py:136-168) and keep only
# their eager path.


@torch.library.custom_op("picotron_amd::rmsnorm_fwd", mutates_args=())
def _op_rmsnorm_fwd(x: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    return rmsnorm_fwd(x, weight, eps)


@_op_rmsnorm_fwd.register_fake
def _(x, weight, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("picotron_amd::rmsnorm_bwd", mutates_args=())
def _op_rmsnorm_bwd(dy: Tensor, x: Tensor, weight: Tensor, rstd: Tensor) -> tuple[Tensor, Tensor]:
    return rmsnorm_bwd(dy, x, weight, rstd)


@_op_rmsnorm_bwd.register_fake
def _(dy, x, weight, rstd):
    return x.new_empty(x.shape), weight.new_empty((x.size(-1),))


@torch.library.custom_op("picotron_amd::residual_rmsnorm_fwd", mutates_args=())
def _op_residual_rmsnorm_fwd(
    x: Tensor, residual: Tensor, weight: Tensor, eps: float
) -> tuple[Tensor, Tensor, Tensor]:
    return residual_rmsnorm_fwd(x, residual, weight, eps)


@_op_residual_rmsnorm_fwd.register_fake
def _(x, residual, weight, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("picotron_amd::residual_rmsnorm_bwd", mutates_args=())
def _op_residual_rmsnorm_bwd(
    dy: Tensor, dh_in: Tensor | None, h: Tensor, weight: Tensor, rstd: Tensor
) -> tuple[Tensor, Tensor]:
    return residual_rmsnorm_bwd(dy, dh_in, h, weight, rstd)


@_op_residual_rmsnorm_bwd.register_fake
def _(dy, dh_in, h, weight, rstd):
    return h.new_empty(h.shape), weight.new_empty((h.size(-1),))


@torch.library.custom_op("picotron_amd::swiglu_fwd", mutates_args=())
def _op_swiglu_fwd(gate: Tensor, up: Tensor) -> Tensor:
    return swiglu_fwd(gate, up)


@_op_swiglu_fwd.register_fake
def _(gate, up):
    return gate.new_empty(gate.shape)


@torch.library.custom_op("picotron_amd::swiglu_bwd", mutates_args=())
def _op_swiglu_bwd(dout: Tensor, gate: Tensor, up: Tensor) -> tuple[Tensor, Tensor]:
    return swiglu_bwd(dout, gate, up)


@_op_swiglu_bwd.register_fake
def _(dout, gate, up):
    return gate.new_empty(gate.shape), up.new_empty(up.shape)


@torch.library.custom_op("picotron_amd::rope", mutates_args=())
def _op_rope(x: Tensor, cos: Tensor, sin: Tensor, layout: str, inverse: bool) -> Tensor:
    return rope(x, cos, sin, layout=layout, inverse=inverse)[0]


@_op_rope.register_fake
def _(x, cos, sin, layout, inverse):
    return _rope_out(x)


@torch.library.custom_op("picotron_amd::rope_pair", mutates_args=())
def _op_rope_pair(
    x0: Tensor, x1: Tensor, cos: Tensor, sin: Tensor, layout: str, inverse: bool
) -> tuple[Tensor, Tensor]:
    y0, y1 = rope(x0, cos, sin, layout=layout, inverse=inverse, x1=x1)
    return y0, y1


@_op_rope_pair.register_fake
def _(x0, x1, cos, sin, layout, inverse):
    return _rope_out(x0), _rope_out(x1)


@torch.library.custom_op("picotron_amd::rope_at", mutates_args=())
def _op_rope_at(x: Tensor, turns: Tensor, positions: Tensor | None, offset: int, scale: float, layout: str,
                inverse: bool) -> Tensor:
    return rope_at(x, turns, positions=positions, offset=offset, scale=scale, layout=layout, inverse=inverse)[0]


@_op_rope_at.register_fake
def _(x, turns, positions, offset, scale, layout, inverse):
    return _rope_out(x)


@torch.library.custom_op("picotron_amd::rope_at_pair", mutates_args=())
def _op_rope_at_pair(x0: Tensor, x1: Tensor, turns: Tensor, positions: Tensor | None, offset: int, scale: float,
                     layout: str, inverse: bool) -> tuple[Tensor, Tensor]:
    y0, y1 = rope_at(x0, turns, positions=positions, offset=offset, scale=scale, layout=layout, inverse=inverse, x1=x1)
    return y0, y1


@_op_rope_at_pair.register_fake
def _(x0, x1, turns, positions, offset, scale, layout, inverse):
    return _rope_out(x0), _rope_out(x1)


@torch.library.custom_op("picotron_amd::swiglu8_fwd", mutates_args=())
def _op_swiglu8_fwd(gate: Tensor, up: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    return swiglu8_fwd(gate, up)


@_op_swiglu8_fwd.register_fake
def _(gate, up):
    blocks = (gate.numel() + BLOCK8 - 1) // BLOCK8
    return (gate.new_empty(gate.shape), gate.new_empty((blocks, 16, 2, 8), dtype=torch.uint8),
            gate.new_empty((blocks, 2), dtype=torch.float32))


@torch.library.custom_op("picotron_amd::swiglu8_bwd", mutates_args=())
def _op_swiglu8_bwd(dout: Tensor, codes: Tensor, steps: Tensor, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    return swiglu8_bwd(dout, codes, steps, dtype)


@_op_swiglu8_bwd.register_fake
def _(dout, codes, steps, dtype):
    return dout.new_empty(dout.shape, dtype=dtype), dout.new_empty(dout.shape, dtype=dtype)


def _fake_rmsnorm8(x):
    rows, blocks = x.numel() // x.size(-1), (x.size(-1) + BLOCK8 - 1) // BLOCK8
    return (x.new_empty(x.shape), x.new_empty(x.shape[:-1], dtype=torch.float32),
            x.new_empty((rows, blocks, BLOCK8), dtype=torch.uint8), x.new_empty((rows, blocks), dtype=torch.float32))


@torch.library.custom_op("picotron_amd::rmsnorm8_fwd", mutates_args=())
def _op_rmsnorm8_fwd(x: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    return rmsnorm8_fwd(x, weight, eps)[1:]


@_op_rmsnorm8_fwd.register_fake
def _(x, weight, eps):
    return _fake_rmsnorm8(x)


@torch.library.custom_op("picotron_amd::residual_rmsnorm8_fwd", mutates_args=())
def _op_residual_rmsnorm8_fwd(
    x: Tensor, residual: Tensor, weight: Tensor, eps: float
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    return rmsnorm8_fwd(x, weight, eps, residual)


@_op_residual_rmsnorm8_fwd.register_fake
def _(x, residual, weight, eps):
    return x.new_empty(x.shape), *_fake_rmsnorm8(x)


@torch.library.custom_op("picotron_amd::rmsnorm8_bwd", mutates_args=())
def _op_rmsnorm8_bwd(
    dy: Tensor, weight: Tensor, rstd: Tensor, codes: Tensor, steps: Tensor, dtype: torch.dtype, dh_in: Tensor | None
) -> tuple[Tensor, Tensor]:
    return rmsnorm8_bwd(dy, weight, rstd, codes, steps, dtype, dh_in)


@_op_rmsnorm8_bwd.register_fake
def _(dy, weight, rstd, codes, steps, dtype, dh_in):
    return dy.new_empty(dy.shape, dtype=dtype), weight.new_empty(weight.shape)
