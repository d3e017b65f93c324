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

import torch

from . import _lib
from .api import _stream_handle
from .recurrence import _on_device, _view


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
    with _on_device(x, weight, residual, gate):
        if x.dim() < 1:
            raise ValueError("x needs at least one dimension")
        y = torch.empty(x.shape, dtype=x.dtype if group is None else torch.float8_e4m3fn, device=x.device)
        z = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
        scale = None
        D = x.shape[-1]
        if group is not None:
            if group < 1 or D % group:
                raise ValueError(f"group_size {group} must divide the {D} columns")
            scale = torch.empty(*x.shape[:-1], D // group, dtype=torch.float32, device=x.device)
        if x.numel():
            shape = x.shape
            y2 = y if y.dim() == 2 else y.view(-1, D)
            st = _lib.load().cgdrRmsNorm(
                _view(_flat(x, "x", shape)), _view(weight), _view(_flat(residual, "residual", shape)),
                _view(_flat(gate, "gate", shape)), eps, 0 if group is None else group,
                _view(y2) if group is None else _lib.view(y.data_ptr(), _lib.DT_FP8_E4M3, y2.shape, y2.stride()),
                None if scale is None else _view(scale.view(-1, D // group)),
                None if z is None else _view(z.view(-1, D)), _stream_handle(x.device))
            _lib.check(st, "cgdrRmsNorm")
    return (y, z) if group is None else (y, scale, z)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual, gate):
        y, z = _forward(x, weight, eps, residual, gate, None)
        ctx.save_for_backward(x if z is None else z, weight, gate)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dz):
        z, weight, gate = ctx.saved_tensors
        want_x, want_w, _, want_r, want_a = ctx.needs_input_grad
        if dy is None:  # z alone was used: its gradient passes through
            return (dz if want_x else None), None, None, (dz if want_r else None), None
        shape, D = z.shape, z.shape[-1]
        # gradients arrive with any strides (expanded ones, for a sum)
        dy = dy.contiguous()
        dz = None if dz is None else dz.contiguous()
        with _on_device(z, dy, dz):
            dx = torch.empty(shape, dtype=z.dtype, device=z.device) if want_x or want_r else None
            dw = torch.empty(weight.shape, dtype=weight.dtype, device=z.device) if want_w else None
            da = torch.empty(shape, dtype=z.dtype, device=z.device) if want_a else None
            if z.numel():
                lib = _lib.load()
                flat = lambda t: _view(_flat(t, "gradient", shape))  # noqa: E731
                z_view, dw_view = flat(z), _view(dw)
                size = ctypes.c_uint64(0)
                _lib.check(lib.cgdrRmsNormBackwardGetWorkspaceSize(z_view, dw_view, ctypes.byref(size)),
                           "cgdrRmsNormBackwardGetWorkspaceSize")
                ws = torch.empty(size.value, dtype=torch.uint8, device=z.device) if size.value else None
                st = lib.cgdrRmsNormBackward(
                    z_view, _view(weight), flat(gate), ctx.eps, flat(dy), flat(dz), flat(dx), dw_view, flat(da),
                    None if ws is None else ws.data_ptr(), size.value, _stream_handle(z.device))
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
