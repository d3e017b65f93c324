"""The argument checks of include/cgdr_recurrence.h and include/cgdr_rms_norm.h
on CPU: refusals come before any device work, so host tensors stand in for
device buffers.  Without a GPU an accepted call ends with CUDA_ERROR at its
launch; with one it is not made here."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cann_operator_challenge_august_b200 as cg
from cann_operator_challenge_august_b200 import _lib
from cann_operator_challenge_august_b200.recurrence import _view

BF, F16, F32, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64
E = torch.empty


def name(status):
    return _lib.STATUS_NAMES[status]


def accepted(status):
    """Accepted: only the launch can fail, for want of a device."""
    return name(status) in ("SUCCESS", "CUDA_ERROR")


no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host tensors must not reach a launch")


# ---- the gated delta rule ---------------------------------------------------------------

def delta_args(**over):
    a = dict(query=E(6, 2, 64, dtype=BF), key=E(6, 2, 64, dtype=BF), value=E(6, 4, 48, dtype=BF),
             beta=E(6, 4, dtype=BF), state=E(8, 4, 48, 64), lens=E(3, dtype=I32), g=E(6, 4), idx=E(3, dtype=I32),
             scale=0.0, out=E(6, 4, 48, dtype=BF))
    return {**a, **over}


def delta(**over):
    a = delta_args(**over)
    return _lib.load().cgdrRecurrentGatedDeltaRule(
        *[_view(a[n]) for n in ("query", "key", "value", "beta", "state", "lens", "g", "idx")], a["scale"],
        _view(a["out"]), None, None)


@no_gpu
@pytest.mark.parametrize("over", [
    {}, dict(lens=None, idx=E(6, dtype=I64)), dict(g=None), dict(beta=E(6, 4)), dict(state=E(8, 4, 48, 64, dtype=BF)),
    dict(idx=None), dict(query=E(6, 4, 128, dtype=BF)[:, ::2, :64]),
    dict(query=E(6, 2, 50, dtype=F16), key=E(6, 2, 50, dtype=F16), value=E(6, 4, 48, dtype=F16),
         beta=E(6, 4, dtype=F16), out=E(6, 4, 48, dtype=F16), state=E(8, 4, 48, 50)),
])
def test_delta_accepts(over):
    assert accepted(delta(**over)), _lib.last_error()


@pytest.mark.parametrize("over,status", [
    (dict(query=None), "NULL_ARGUMENT"), (dict(state=None), "NULL_ARGUMENT"), (dict(out=None), "NULL_ARGUMENT"),
    (dict(query=E(6, 128, dtype=BF)), "BAD_RANK"), (dict(beta=E(6, dtype=BF)), "BAD_RANK"),
    (dict(state=E(8, 48, 64)), "BAD_RANK"), (dict(lens=E(3, 1, dtype=I32)), "BAD_RANK"),
    (dict(idx=E(3, 1, dtype=I32)), "BAD_RANK"),
    (dict(query=E(6, 2, 64, dtype=I32)), "BAD_DTYPE"), (dict(key=E(6, 2, 64)), "BAD_DTYPE"),
    (dict(out=E(6, 4, 48)), "BAD_DTYPE"), (dict(beta=E(6, 4, dtype=F16)), "BAD_DTYPE"),
    (dict(state=E(8, 4, 48, 64, dtype=F16)), "BAD_DTYPE"), (dict(g=E(6, 4, dtype=BF)), "BAD_DTYPE"),
    (dict(lens=E(3, dtype=I64)), "BAD_DTYPE"), (dict(idx=E(3)), "BAD_DTYPE"),
    (dict(key=E(6, 1, 64, dtype=BF)), "BAD_SHAPE"), (dict(value=E(5, 4, 48, dtype=BF)), "BAD_SHAPE"),
    (dict(value=E(6, 3, 48, dtype=BF)), "BAD_SHAPE"), (dict(beta=E(6, 2, dtype=BF)), "BAD_SHAPE"),
    (dict(g=E(5, 4)), "BAD_SHAPE"), (dict(state=E(8, 4, 64, 48)), "BAD_SHAPE"), (dict(idx=E(4, dtype=I32)), "BAD_SHAPE"),
    (dict(out=E(6, 4, 64, dtype=BF)), "BAD_SHAPE"),
    (dict(idx=None, state=E(2, 4, 48, 64)), "BAD_SHAPE"),  # three rows, two states
    (dict(query=E(6, 2, 300, dtype=BF), key=E(6, 2, 300, dtype=BF), state=E(8, 4, 48, 300)), "UNSUPPORTED"),
    (dict(query=E(6, 2, 128, dtype=BF)[..., ::2]), "BAD_STRIDE"), (dict(idx=E(6, dtype=I32)[::2]), "BAD_STRIDE"),
    (dict(state=E(8, 4, 64, 48).transpose(2, 3)), "BAD_STRIDE"),
    (dict(state=E(1, 4, 48, 64).expand(8, 4, 48, 64)), "BAD_STRIDE"),  # updated in place
])
def test_delta_refuses(over, status):
    assert name(delta(**over)) == status, _lib.last_error()


# ---- the diagonal recurrence --------------------------------------------------------------

def scan(**over):
    a = dict(x=E(2, 130, 24, dtype=BF), g=E(2, 130, 24), h0=E(2, 24), cu=None, out=E(2, 130, 24, dtype=BF), ht=E(2, 24),
             chunks=E(2, 2, 24))
    a.update(over)
    return _lib.load().cgdrGatedLinearRecurrence(
        *[_view(a[n]) for n in ("x", "g", "h0", "cu", "out", "ht", "chunks")], None)


def packed(**over):
    a = dict(x=E(1, 130, 24, dtype=BF), g=E(1, 130, 24), h0=E(3, 24), cu=E(4, dtype=I64),
             out=E(1, 130, 24, dtype=BF), ht=E(3, 24), chunks=E(1, 2, 24))
    return scan(**{**a, **over})


@no_gpu
def test_scan_accepts():
    assert accepted(scan()), _lib.last_error()
    assert accepted(packed()), _lib.last_error()
    assert accepted(scan(h0=None, ht=None, chunks=None, g=E(2, 130, 24, dtype=BF))), _lib.last_error()
    assert accepted(scan(x=E(2, 130, 48, dtype=BF)[..., 24:])), _lib.last_error()


@pytest.mark.parametrize("call,over,status", [
    (scan, dict(x=None), "NULL_ARGUMENT"), (scan, dict(out=None), "NULL_ARGUMENT"),
    (scan, dict(x=E(130, 24, dtype=BF)), "BAD_RANK"), (scan, dict(h0=E(24)), "BAD_RANK"),
    (scan, dict(x=E(2, 130, 24, dtype=I32)), "BAD_DTYPE"), (scan, dict(g=E(2, 130, 24, dtype=F16)), "BAD_DTYPE"),
    (scan, dict(out=E(2, 130, 24)), "BAD_DTYPE"), (scan, dict(h0=E(2, 24, dtype=BF)), "BAD_DTYPE"),
    (scan, dict(ht=E(2, 24, dtype=BF)), "BAD_DTYPE"), (packed, dict(cu=E(4, dtype=I32)), "BAD_DTYPE"),
    (scan, dict(g=E(2, 130, 1)), "BAD_SHAPE"), (scan, dict(h0=E(1, 24)), "BAD_SHAPE"),
    (scan, dict(out=E(2, 129, 24, dtype=BF)), "BAD_SHAPE"), (scan, dict(chunks=E(2, 3, 24)), "BAD_SHAPE"),
    (scan, dict(x=E(2, 0, 24, dtype=BF)), "NULL_ARGUMENT"),
    (packed, dict(h0=E(4, 24)), "BAD_SHAPE"), (packed, dict(ht=E(2, 24)), "BAD_SHAPE"),
    (scan, dict(cu=E(3, dtype=I64)), "BAD_VARLEN"), (packed, dict(cu=E(1, dtype=I64)), "BAD_VARLEN"),
    (scan, dict(g=E(2, 130, 1).expand(2, 130, 24)), "BAD_STRIDE"),
    (scan, dict(x=E(2, 130, 48, dtype=BF)[..., ::2]), "BAD_STRIDE"),
    (packed, dict(cu=E(8, dtype=I64)[::2]), "BAD_STRIDE"), (scan, dict(chunks=E(2, 2, 48)[..., :24]), "BAD_STRIDE"),
])
def test_scan_refuses(call, over, status):
    assert name(call(**over)) == status, _lib.last_error()


def scan_backward(**over):
    a = dict(x=E(2, 130, 24, dtype=BF), g=E(2, 130, 24), h0=E(2, 24), cu=None, chunks=E(2, 2, 24),
             d_out=E(2, 130, 24, dtype=BF), d_ht=E(2, 24), dx=E(2, 130, 24, dtype=BF), dg=E(2, 130, 24), dh0=E(2, 24))
    a.update(over)
    return _lib.load().cgdrGatedLinearRecurrenceBackward(
        *[_view(a[n]) for n in ("x", "g", "h0", "cu", "chunks", "d_out", "d_ht", "dx", "dg", "dh0")], None)


@pytest.mark.parametrize("over,status", [
    (dict(chunks=None), "NULL_ARGUMENT"), (dict(d_out=None, d_ht=None), "NULL_ARGUMENT"),
    (dict(dx=None, dg=None, dh0=None), "NULL_ARGUMENT"), (dict(d_out=E(2, 130, 24)), "BAD_DTYPE"),
    (dict(dg=E(2, 130, 24, dtype=BF)), "BAD_DTYPE"), (dict(dx=E(2, 131, 24, dtype=BF)), "BAD_SHAPE"),
    (dict(dh0=E(3, 24)), "BAD_SHAPE"), (dict(d_out=E(2, 130, 1, dtype=BF).expand(2, 130, 24)), "BAD_STRIDE"),
])
def test_scan_backward_refuses(over, status):
    assert name(scan_backward(**over)) == status, _lib.last_error()


def step(**over):
    a = dict(x=E(5, 24, dtype=BF), g=E(5, 24), state=E(9, 24), idx=E(5, dtype=I32), out=E(5, 24, dtype=BF))
    a.update(over)
    return _lib.load().cgdrGatedLinearRecurrenceStep(
        *[_view(a[n]) for n in ("x", "g", "state", "idx", "out")], None, None)


@no_gpu
def test_step_accepts():
    assert accepted(step()) and accepted(step(idx=None)) and accepted(step(idx=E(5, dtype=I64))), _lib.last_error()


@pytest.mark.parametrize("over,status", [
    (dict(state=None), "NULL_ARGUMENT"), (dict(x=E(5, 24, 1, dtype=BF)), "BAD_RANK"),
    (dict(state=E(9, 24, dtype=BF)), "BAD_DTYPE"), (dict(idx=E(5, dtype=BF)), "BAD_DTYPE"),
    (dict(g=E(5, 1)), "BAD_SHAPE"), (dict(state=E(9, 25)), "BAD_SHAPE"), (dict(idx=E(4, dtype=I32)), "BAD_SHAPE"),
    (dict(idx=None, state=E(4, 24)), "BAD_SHAPE"), (dict(state=E(1, 24).expand(9, 24)), "BAD_STRIDE"),
    (dict(x=E(5, 48, dtype=BF)[:, ::2]), "BAD_STRIDE"),
])
def test_step_refuses(over, status):
    assert name(step(**over)) == status, _lib.last_error()


# ---- the norm ------------------------------------------------------------------------------

FP8 = torch.float8_e4m3fn


def view(t):
    return None if t is None else _lib.view(t.data_ptr(), _lib.DT_FP8_E4M3, t.shape, t.stride()) if t.dtype == FP8 else _view(t)


def norm(**over):
    a = dict(x=E(7, 256, dtype=BF), w=E(256), residual=None, gate=None, eps=1e-6, group=0, y=E(7, 256, dtype=BF),
             scale=None, z=None)
    a.update(over)
    return _lib.load().cgdrRmsNorm(view(a["x"]), view(a["w"]), view(a["residual"]), view(a["gate"]), a["eps"],
                                   a["group"], view(a["y"]), view(a["scale"]), view(a["z"]), None)


def eight(group=128, **over):
    return norm(**{**dict(y=E(7, 256, dtype=FP8), scale=E(7, 256 // max(group, 1)), group=group), **over})


@no_gpu
def test_norm_accepts():
    rows = E(7, 256, dtype=BF)
    assert accepted(norm()) and accepted(norm(residual=rows, z=rows, gate=rows)), _lib.last_error()
    assert accepted(eight()) and accepted(eight(256)) and accepted(eight(32)), _lib.last_error()
    assert accepted(norm(x=E(7, 300, dtype=BF)[:, 3:259])), _lib.last_error()


@pytest.mark.parametrize("call,over,status", [
    (norm, dict(x=None), "NULL_ARGUMENT"), (norm, dict(y=None), "NULL_ARGUMENT"),
    (norm, dict(residual=E(7, 256, dtype=BF)), "NULL_ARGUMENT"), (norm, dict(z=E(7, 256, dtype=BF)), "NULL_ARGUMENT"),
    (norm, dict(x=E(256, dtype=BF)), "BAD_RANK"), (norm, dict(w=E(1, 256)), "BAD_RANK"),
    (norm, dict(x=E(7, 256, dtype=I32)), "BAD_DTYPE"), (norm, dict(w=E(256, dtype=F16)), "BAD_DTYPE"),
    (norm, dict(gate=E(7, 256)), "BAD_DTYPE"), (norm, dict(y=E(7, 256)), "BAD_DTYPE"),
    (norm, dict(w=E(255)), "BAD_SHAPE"), (norm, dict(gate=E(6, 256, dtype=BF)), "BAD_SHAPE"),
    (norm, dict(eps=-1.0), "BAD_SHAPE"), (norm, dict(eps=float("nan")), "BAD_SHAPE"),
    (norm, dict(x=E(7, 512, dtype=BF)[:, ::2]), "BAD_STRIDE"), (norm, dict(w=E(1).expand(256)), "BAD_STRIDE"),
    (norm, dict(x=E(2, 20000, dtype=BF), w=E(20000), y=E(2, 20000, dtype=BF)), "UNSUPPORTED"),
    (eight, dict(y=E(7, 256, dtype=BF)), "BAD_DTYPE"), (eight, dict(scale=E(7, 3)), "BAD_SHAPE"),
    (eight, dict(group=16), "UNSUPPORTED"), (eight, dict(group=0, scale=E(7, 2)), "UNSUPPORTED"),
    (eight, dict(scale=E(7, 4)[:, ::2]), "BAD_STRIDE"),
    (eight, dict(x=E(7, 200, dtype=BF), w=E(200), y=E(7, 200, dtype=FP8)), "BAD_SHAPE"),
])
def test_norm_refuses(call, over, status):
    assert name(call(**over)) == status, _lib.last_error()


def norm_backward(**over):
    a = dict(z=E(7, 256, dtype=BF), w=E(256), gate=None, eps=1e-6, dy=E(7, 256, dtype=BF), dz=None,
             dx=E(7, 256, dtype=BF), dw=E(256), dgate=None, ws=E(7 * 256 * 4 + 16, dtype=torch.uint8), size=7 * 256 * 4)
    a.update(over)
    ws = None if a["ws"] is None else a["ws"].data_ptr()
    return _lib.load().cgdrRmsNormBackward(*[_view(a[n]) for n in ("z", "w", "gate")], a["eps"],
                                           *[_view(a[n]) for n in ("dy", "dz", "dx", "dw", "dgate")], ws, a["size"], None)


@pytest.mark.parametrize("over,status", [
    (dict(dy=None), "NULL_ARGUMENT"), (dict(dx=None, dw=None), "NULL_ARGUMENT"),
    (dict(dgate=E(7, 256, dtype=BF)), "NULL_ARGUMENT"), (dict(ws=None), "NULL_ARGUMENT"),
    (dict(size=7 * 256 * 4 - 1), "WORKSPACE_TOO_SMALL"), (dict(dw=E(256, dtype=BF)), "BAD_DTYPE"),
    (dict(dy=E(7, 256)), "BAD_DTYPE"), (dict(dw=E(255)), "BAD_SHAPE"), (dict(dz=E(7, 255, dtype=BF)), "BAD_SHAPE"),
    (dict(dy=E(7, 1, dtype=BF).expand(7, 256)), "BAD_STRIDE"),
])
def test_norm_backward_refuses(over, status):
    assert name(norm_backward(**over)) == status, _lib.last_error()


def test_norm_backward_workspace():
    lib, size = _lib.load(), ctypes.c_uint64(1)
    for rows, want in ((7, 7 * 256 * 4), (100000, 592 * 256 * 4)):
        z = E(rows, 256, dtype=BF)
        assert lib.cgdrRmsNormBackwardGetWorkspaceSize(_view(z), _view(E(256)), ctypes.byref(size)) == 0
        assert size.value == want
        assert lib.cgdrRmsNormBackwardGetWorkspaceSize(_view(z), None, ctypes.byref(size)) == 0
        assert size.value == 0


# ---- the Python entries ----------------------------------------------------------------------

def test_python_entries_refuse_host_tensors():
    x = E(2, 8, 16, dtype=BF)
    for call in (lambda: cg.gated_linear_recurrence(x, x), lambda: cg.gated_linear_recurrence_step(x[0], x[0], E(8, 16)),
                 lambda: cg.rms_norm(x, E(16)), lambda: cg.rms_norm_fp8(x, E(16)),
                 lambda: cg.recurrent_gated_delta_rule(x, x, x, x[..., 0], E(2, 8, 16, 16))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
