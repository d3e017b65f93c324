"""Token-by-token recurrences of linear recurrent layers, over the C ABI in
include/cgdr_recurrence.h, next to the chunked gated delta rule in
:mod:`.gdr`.

* :func:`recurrent_gated_delta_rule` -- the gated delta rule for serving: one
  or a few tokens a sequence, on a pool of states that is updated in place.
  The states have the layout of ``chunk_gated_delta_rule``'s
  ``initial_state`` / ``final_state``, so a prefill's final state is copied
  into the pool as it is.
* :func:`gated_linear_recurrence` -- the recurrence with a diagonal state,
  ``h_t = exp(g_t) h_{t-1} + x_t``, over whole sequences; differentiable.
* :func:`gated_linear_recurrence_step` -- the same for one token a row, on a
  pool of states.

Everything runs on the current stream of the tensors' device.  Nothing here
computes on the CPU: the CUDA library does the work and raises if it is
missing.
"""

from __future__ import annotations

import contextlib

import torch

from . import _lib
from .api import _DT, _stream_handle

_NO_GUARD = contextlib.nullcontext()
_VIEWS = _lib._VIEWS


def _view(t: torch.Tensor | None) -> bytes | None:
    """`t` as a cgdrTensor (see _lib.view, inlined: these calls are a short
    kernel's latency)."""
    if t is None:
        return None
    shape = t.shape
    n = len(shape)
    if n > _lib.MAX_DIMS:
        raise ValueError(f"tensors have at most {_lib.MAX_DIMS} dimensions, got {n}")
    return _VIEWS[n](t.data_ptr(), _DT.get(t.dtype, 0), n, *shape, *t.stride())


# The current stream's handle; the public accessor builds a Stream object first.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: _stream_handle(torch.device("cuda", index)))


def _on_device(first: torch.Tensor, *others: torch.Tensor | None):
    """Checks that all tensors are on one CUDA device and returns a context in
    which that device is current."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        if all(t is None or t.is_cuda for t in (first, *others)):
            raise ValueError("all tensors must be on one device")
        raise ValueError("all tensors must be CUDA tensors (there is no CPU implementation)")
    return _NO_GUARD if index == torch.cuda.current_device() else torch.cuda.device(index)


def _new_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _refuse_twice() -> None:
    """Backward passes call it: gradients are recorded there only for a second
    derivative, which these operators do not have."""
    if torch.is_grad_enabled():
        raise RuntimeError("this operator is differentiable once only")


def _updated(state: torch.Tensor) -> None:
    """Tells autograd that the pool has changed in place."""
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)


def _raise_on(status: torch.Tensor) -> None:
    bits = int(status.item())
    if bits:
        raise RuntimeError(f"device status 0x{bits:x}: "
                           + ("inconsistent sequence lengths " if bits & _lib.DEVICE_BAD_VARLEN else "")
                           + ("state index past the pool or named twice"
                              if bits & _lib.DEVICE_BAD_STATE_INDEX else ""))


def recurrent_gated_delta_rule(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    beta: torch.Tensor,
    state: torch.Tensor,
    actual_seq_lengths: torch.Tensor | None = None,
    scale: float | None = None,
    g: torch.Tensor | None = None,
    *,
    state_indices: torch.Tensor | None = None,
    check_device_status: bool = False,
) -> torch.Tensor:
    """The gated delta rule token by token: query, key ``[T, Nk, Dk]``, value
    ``[T, Nv, Dv]`` (bf16, fp16 or fp32), beta ``[T, Nv]`` (the same type or
    fp32), g ``[T, Nv]`` fp32 per-token log gate (optional), scale (default
    ``Dk ** -0.5``).  Returns ``out [T, Nv, Dv]``.

    ``state [S, Nv, Dv, Dk]`` (fp32 or bf16) is a pool that is updated in
    place.  ``state_indices [B]`` (int32 or int64) names the state of each
    sequence; a negative index marks a padded one (zero output, no state
    touched).  Without it sequence b owns state b.  ``actual_seq_lengths
    [B]`` (int32) gives each sequence's tokens in the packed inputs, 0
    included; without it every sequence has one token (B = T).  Rows of the
    output behind the last sequence are zero.

    No two sequences of a call may share a state: the first keeps it, the
    others are treated as padding.  ``check_device_status`` synchronises and
    raises on that, on indices past the pool and on lengths that do not sum
    to T.  The call is not differentiable."""
    with _on_device(query, key, value, beta, state, actual_seq_lengths, g, state_indices):
        out = _new_like(value)
        status = torch.empty(1, dtype=torch.int32, device=value.device) if check_device_status else None
        st = _lib.load().cgdrRecurrentGatedDeltaRule(
            _view(query), _view(key), _view(value), _view(beta), _view(state), _view(actual_seq_lengths), _view(g),
            _view(state_indices), float(scale if scale is not None else 0.0), _view(out),
            None if status is None else status.data_ptr(), _raw_stream(value.get_device()))
        _lib.check(st, "cgdrRecurrentGatedDeltaRule")
    _updated(state)
    if check_device_status:
        _raise_on(status)
    return out


def gated_linear_recurrence_step(
    x: torch.Tensor,
    g: torch.Tensor,
    state: torch.Tensor,
    *,
    state_indices: torch.Tensor | None = None,
    check_device_status: bool = False,
) -> torch.Tensor:
    """One token a row of the diagonal recurrence: ``state[i_b] = exp(g_b)
    state[i_b] + x_b``; returns the new states ``[B, D]`` in x's type.  x
    ``[B, D]`` (bf16, fp16 or fp32), g ``[B, D]`` (x's type or fp32), state
    ``[S, D]`` fp32, updated in place; ``state_indices`` and
    ``check_device_status`` as in :func:`recurrent_gated_delta_rule`.  The
    call is not differentiable."""
    with _on_device(x, g, state, state_indices):
        out = _new_like(x)
        status = torch.empty(1, dtype=torch.int32, device=x.device) if check_device_status else None
        st = _lib.load().cgdrGatedLinearRecurrenceStep(
            _view(x), _view(g), _view(state), _view(state_indices), _view(out),
            None if status is None else status.data_ptr(), _raw_stream(x.get_device()))
        _lib.check(st, "cgdrGatedLinearRecurrenceStep")
    _updated(state)
    if check_device_status:
        _raise_on(status)
    return out


def _forward(x, g, initial_state, cu_seqlens, want_final, want_chunks):
    """(out, final_state or None, chunk_states or None)"""
    with _on_device(x, g, initial_state, cu_seqlens):
        out = _new_like(x)
        final = chunks = None
        if x.dim() == 3:  # any other rank is refused by the library
            B, T, D = x.shape
            if want_final:
                N = B if cu_seqlens is None else max(cu_seqlens.numel() - 1, 0)
                final = torch.empty(N, D, dtype=torch.float32, device=x.device)
            if want_chunks:
                chunks = torch.empty(B, -(-T // _lib.RECURRENCE_CHUNK), D, dtype=torch.float32, device=x.device)
            if T == 0 and g.shape == x.shape:  # no token: the states stay what they were
                if final is not None:
                    if initial_state is None:
                        final.zero_()
                    elif initial_state.shape == final.shape:
                        final.copy_(initial_state)
                    else:
                        raise ValueError(f"initial_state must have shape [N, D] = {tuple(final.shape)}")
                return out, final, chunks
        st = _lib.load().cgdrGatedLinearRecurrence(
            _view(x), _view(g), _view(initial_state), _view(cu_seqlens), _view(out), _view(final), _view(chunks),
            _raw_stream(x.get_device()))
        _lib.check(st, "cgdrGatedLinearRecurrence")
    return out, final, chunks


class _GatedLinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, initial_state, cu_seqlens, want_final):
        out, final, chunks = _forward(x, g, initial_state, cu_seqlens, want_final, True)
        ctx.save_for_backward(x, g, initial_state, cu_seqlens, chunks)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def backward(ctx, d_out, d_final):
        _refuse_twice()
        x, g, initial_state, cu_seqlens, chunks = ctx.saved_tensors
        if d_out is None and d_final is None:
            return None, None, None, None, None
        # gradients arrive with any strides (expanded ones, for a sum)
        d_out = None if d_out is None else d_out.contiguous()
        d_final = None if d_final is None else d_final.contiguous()
        want_x, want_g, want_h0 = ctx.needs_input_grad[:3]
        with _on_device(x, d_out, d_final):
            dx = _new_like(x) if want_x else None
            dg = _new_like(g) if want_g else None
            dh0 = _new_like(initial_state) if want_h0 else None
            if x.shape[1] == 0:
                if want_h0:
                    dh0.zero_() if d_final is None else dh0.copy_(d_final)
                return dx, dg, dh0, None, None
            st = _lib.load().cgdrGatedLinearRecurrenceBackward(
                _view(x), _view(g), _view(initial_state), _view(cu_seqlens), _view(chunks), _view(d_out),
                _view(d_final), _view(dx), _view(dg), _view(dh0), _raw_stream(x.get_device()))
            _lib.check(st, "cgdrGatedLinearRecurrenceBackward")
        return dx, dg, dh0, None, None


def gated_linear_recurrence(
    x: torch.Tensor,
    g: torch.Tensor,
    initial_state: torch.Tensor | None = None,
    *,
    output_final_state: bool = False,
    cu_seqlens: torch.LongTensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``h_t = exp(g_t) h_{t-1} + x_t``, channel by channel: returns ``out
    [B, T, D]`` (h in x's type) and the final state ``[N, D]`` (fp32, or None).

    x ``[B, T, D]`` is bf16, fp16 or fp32; g ``[B, T, D]``, of x's type or
    fp32, is the log of a decay (``<= 0``; ``-inf`` forgets); initial_state
    ``[N, D]`` fp32.  With ``cu_seqlens`` (int64 ``[N + 1]`` from 0,
    non-decreasing, B = 1) the sequences are packed along T; an empty one
    keeps its initial state, and rows behind the last one are zero, with zero
    gradients.  Last dimensions are contiguous.  The state is held in fp32.

    Differentiable in x, g and initial_state (once).  The gradients are those
    of the recurrence in fp32, recomputed from x, g and one saved state per
    128 tokens.  To capture a backward pass into a CUDA graph, capture its
    forward pass in the same graph."""
    if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad
                                    or (initial_state is not None and initial_state.requires_grad)):
        return _GatedLinearRecurrence.apply(x, g, initial_state, cu_seqlens, output_final_state)
    out, final, _ = _forward(x, g, initial_state, cu_seqlens, output_final_state, False)
    return out, final
