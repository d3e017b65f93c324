"""The root-mean-square norm that stands before a recurrent layer (with the
residual's addition) and behind it (with a silu gate, one row per head), over
the C ABI in include/cgdr_rms_norm.h.

* :func:`rms_norm` -- output in x's type; differentiable.
* :func:`rms_norm_fp8` -- output in e4m3 with fp32 scales, for an 8-bit
  projection.

Everything runs on the current stream of the tensors' device.  Nothing here
computes on the CPU: the CUDA library does the work and raises if it is
missing.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .api import _DT
from .recurrence import _new_like, _on_device, _raw_stream, _refuse_twice, _view


def _flat(t: torch.Tensor | None, name: str, shape) -> torch.Tensor | None:
    """A [..., D] tensor as its [R, D] view."""
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{name} must have x's shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dim() == 2:
        return t
    if t.dim() == 1:
        return t[None]
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError:
        raise ValueError(f"{name}'s leading dimensions cannot be merged into rows without a copy") from None


def _forward(x, weight, eps, residual, gate, group):
    """(y, z or None), or (q, scale, z or None) with a group; all in x's shape."""
    shape = x.shape
    with _on_device(x, weight, residual, gate):
        if not shape:
            raise ValueError("x needs at least one dimension")
        D = shape[-1]
        z = None if residual is None else _new_like(x)
        scale = None
        if group is None:
            y = _new_like(x)
        else:
            if group < 1 or D % group:
                raise ValueError(f"group_size {group} must divide the {D} columns")
            y = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
            scale = x.new_empty(*shape[:-1], D // group, dtype=torch.float32)
        if x.numel():
            R = x.numel() // D
            rows = (R, D), (D, 1)  # the outputs are contiguous
            dtype = _DT.get(x.dtype, 0)
            st = _lib.load().cgdrRmsNorm(
                _view(_flat(x, "x", shape)), _view(weight), _view(_flat(residual, "residual", shape)),
                _view(_flat(gate, "gate", shape)), eps, group or 0,
                _lib.view(y.data_ptr(), dtype if group is None else _lib.DT_FP8_E4M3, *rows),
                None if scale is None else _lib.view(scale.data_ptr(), _lib.DT_FLOAT32, (R, D // group), (D // group, 1)),
                None if z is None else _lib.view(z.data_ptr(), dtype, *rows), _raw_stream(x.get_device()))
            _lib.check(st, "cgdrRmsNorm")
    return (y, z) if group is None else (y, scale, z)


@functools.lru_cache(maxsize=1024)
def _backward_bytes(R: int, D: int, dtype: int, w_dtype: int) -> int:
    """Workspace of a backward pass that wants dweight."""
    size = ctypes.c_uint64(0)
    st = _lib.load().cgdrRmsNormBackwardGetWorkspaceSize(
        _lib.view(1, dtype, (R, D), (D, 1)), _lib.view(1, w_dtype, (D,), (1,)), ctypes.byref(size))
    _lib.check(st, "cgdrRmsNormBackwardGetWorkspaceSize")
    return size.value


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual, gate):
        y, z = _forward(x, weight, eps, residual, gate, None)
        ctx.save_for_backward(x if z is None else z, weight, gate)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    def backward(ctx, dy, dz):
        _refuse_twice()
        z, weight, gate = ctx.saved_tensors
        want_x, want_w, _, want_r, want_a = ctx.needs_input_grad
        if dy is None:  # z alone was used: its gradient passes through
            return (dz if want_x else None), None, None, (dz if want_r else None), None
        shape = z.shape
        # gradients arrive with any strides (expanded ones, for a sum)
        dy = dy.contiguous()
        dz = None if dz is None else dz.contiguous()
        with _on_device(z, dy, dz):
            dx = _new_like(z) if want_x or want_r else None
            dw = _new_like(weight) if want_w else None
            da = _new_like(z) if want_a else None
            if z.numel():
                D, dtype = shape[-1], _DT[z.dtype]
                R = z.numel() // D
                rows = (R, D), (D, 1)
                flat = lambda t: None if t is None else _lib.view(t.data_ptr(), dtype, *rows)  # noqa: E731
                size = _backward_bytes(R, D, dtype, _DT[weight.dtype]) if want_w else 0
                ws = dy.new_empty(size, dtype=torch.uint8) if size else None
                st = _lib.load().cgdrRmsNormBackward(
                    _view(_flat(z, "x", shape)), _view(weight), _view(_flat(gate, "gate", shape)), ctx.eps, flat(dy),
                    flat(dz), flat(dx), _view(dw), flat(da), None if ws is None else ws.data_ptr(), size,
                    _raw_stream(z.get_device()))
                _lib.check(st, "cgdrRmsNormBackward")
            elif dw is not None:
                dw.zero_()
        return (dx if want_x else None), dw, None, (dx if want_r else None), da


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``y = z / sqrt(mean(z^2) + eps) * weight * silu(gate)`` over the last
    dimension, ``z = x + residual``.  Returns y, or ``(y, z)`` with a
    residual; z is the new residual stream, rounded to x's type, and y is the
    norm of z as it is stored.

    x, residual, gate ``[..., D]`` have one type (bf16, fp16 or fp32) and
    shape; weight ``[D]`` has that type or fp32; D <= 16384.  residual and
    gate are optional.  Last dimensions are contiguous and leading ones must
    merge into rows of one stride.  Sums are held in fp32.

    Differentiable in x, weight, residual and gate (once).  To capture a
    backward pass into a CUDA graph, capture its forward pass in the same
    graph."""
    eps = float(eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual, gate)):
        y, z = _RmsNorm.apply(x, weight, eps, residual, gate)
    else:
        y, z = _forward(x, weight, eps, residual, gate, None)
    return y if residual is None else (y, z)


def rms_norm_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    group_size: int | None = None,
) -> tuple[torch.Tensor, ...]:
    """:func:`rms_norm` with y in 8 bits: returns ``(q, scale)`` or ``(q,
    scale, z)``, ``q [..., D]`` in float8_e4m3fn and ``scale [..., D /
    group_size]`` fp32 with ``y ~ q * scale`` over groups of ``group_size``
    neighbouring columns (D, the default, or 32, 64 or 128):
    ``scale = max(amax |y|, 1e-12) / 448``, rounded to the nearest value.  y
    is not rounded before.  A row that holds a NaN has NaN scales.  Not
    differentiable."""
    q, scale, z = _forward(x, weight, float(eps), residual, gate, x.shape[-1] if group_size is None else int(group_size))
    return (q, scale) if residual is None else (q, scale, z)
