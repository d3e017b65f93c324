"""The root-mean-square norm on the GPU against its definition in float64
(oracle/recurrent.py), element by element within bounds derived there;
gradients also against differences of the float64 definition."""

from __future__ import annotations

import pytest
import torch

from oracle import recurrent as R
from test_gpu_recurrence import BF, F16, F32, dev, guarded, rand, within

pytestmark = pytest.mark.gpu

cg = pytest.importorskip("cann_operator_challenge_august_b200")
from cann_operator_challenge_august_b200 import _lib  # noqa: E402
from cann_operator_challenge_august_b200.recurrence import _view  # noqa: E402

EPS = 1e-6


def inputs(shape, x_type, w_type, form, seed=0):
    D = shape[-1]
    t = dict(x=rand(*shape, seed=seed, dtype=x_type), w=(1 + 0.2 * rand(D, seed=seed + 1)).to(w_type), residual=None,
             gate=None)
    if "residual" in form:
        t["residual"] = rand(*shape, seed=seed + 2, dtype=x_type, scale=2.0)
    if "gate" in form:
        t["gate"] = rand(*shape, seed=seed + 3, dtype=x_type)
    return t


def z_matches(z, val, x_type):
    """z is the sum rounded to its type; where the fp32 sum itself was a tie
    the neighbour is as near."""
    within(z, val["z"], 2 * R.half_step(x_type) * val["z"].abs() * (x_type != F32) + 2 * R.U * val["z"].abs(), "z")


def check(t, *, backward=True, eps=EPS, dz=True):
    x_type, form = t["x"].dtype, t
    names = [n for n in ("x", "w", "residual", "gate") if form[n] is not None]
    leaves = {n: t[n].detach().requires_grad_() for n in names}
    got = cg.rms_norm(leaves["x"], leaves["w"], eps, residual=leaves.get("residual"), gate=leaves.get("gate"))
    y, z = got if t["residual"] is not None else (got, None)
    with torch.no_grad():
        again = cg.rms_norm(t["x"], t["w"], eps, residual=t["residual"], gate=t["gate"])
    assert torch.equal(y, again[0] if z is not None else again)
    dy = rand(*y.shape, seed=77, dtype=x_type)
    up = rand(*y.shape, seed=78, dtype=x_type) if z is not None and dz else None
    # the definition takes z as it is stored
    stored = t["x"] if z is None else z.detach()
    val, err = R.rms_norm(stored, t["w"], eps, None, t["gate"], dy, up)
    within(y, val["y"], R.rounded(err["y"], val["y"], x_type), "y")
    if z is not None:
        z_matches(z, R.rms_norm(t["x"], t["w"], eps, t["residual"])[0], x_type)
    if not backward:
        return
    outs, grads = ((y,), (dy,)) if up is None else ((y, z), (dy, up))
    got = dict(zip(names, torch.autograd.grad(outs, [leaves[n] for n in names], grads)))
    within(got["x"], val["dx"], R.rounded(err["dx"], val["dx"], x_type), "dx")
    within(got["w"], val["dw"], R.rounded(err["dw"], val["dw"], t["w"].dtype), "dw")
    if z is not None:
        assert torch.equal(got["x"], got["residual"])
    if t["gate"] is not None:
        within(got["gate"], val["dgate"], R.rounded(err["dgate"], val["dgate"], x_type), "dgate")


TYPES = [(BF, BF), (BF, F32), (F16, F16), (F16, F32), (F32, F32)]
FORMS = ["", "residual", "gate", "residual gate"]
# every split of a row over lanes, its borders, and rows that are no multiple of 16 bytes
WIDTHS = [1, 7, 32, 64, 128, 136, 256, 300, 512, 1000, 1024, 2000, 2048, 2056, 4096, 4097, 8192, 16384]


@pytest.mark.parametrize("x_type,w_type", TYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_norm_widths(D, x_type, w_type):
    for form in FORMS:
        check(inputs((5, D), x_type, w_type, form, seed=D))


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 700, 9500])
@pytest.mark.parametrize("D", [128, 1024])
def test_norm_rows(rows, D):
    """Up to more rows than the backward pass has blocks for."""
    for form in FORMS:
        check(inputs((rows, D), BF, F32, form, seed=rows))


@pytest.mark.parametrize("rows", [593, 1200])
def test_norm_rows_of_a_whole_block(rows):
    check(inputs((rows, 2048), BF, F32, "residual", seed=rows))


def test_norm_head_layouts_and_strides():
    check(inputs((2, 9, 4, 128), BF, BF, "gate"))       # [B, T, H, V]
    check(inputs((128,), BF, BF, "residual"))
    t = inputs((40, 128), BF, F32, "residual gate")
    for n in ("x", "residual", "gate"):
        wide = torch.zeros(40, 300, dtype=BF, device=dev())
        wide[:, 100:228] = t[n]
        t[n] = wide[:, 100:228]                         # rows that start on 8 bytes
    check(t)
    t["x"] = t["x"].repeat_interleave(2, 0)[::2]
    check(t, dz=False)
    cols = torch.zeros(40, 2, 128, dtype=BF, device=dev())
    cols[:, 1] = t["x"]
    t["x"] = cols[:, 1]
    check(t, backward=False)


def test_norm_refuses_rows_that_do_not_merge():
    x = rand(4, 6, 128, seed=1, dtype=BF)
    with pytest.raises(ValueError, match="merged"):
        cg.rms_norm(x.transpose(0, 1), torch.ones(128, device=dev()))
    with pytest.raises(ValueError, match="shape"):
        cg.rms_norm(x, torch.ones(128, device=dev()), gate=x[:2])
    with pytest.raises(cg.CgdrValueError):
        cg.rms_norm(x, torch.ones(64, device=dev()))


def test_norm_extreme_rows():
    """Zero rows, tiny and huge values; a row with NaN or infinity leaves the others alone."""
    t = inputs((8, 256), F32, F32, "gate", seed=1)
    t["x"][0] = 0
    t["x"][1] *= 1e-18
    t["x"][2] *= 1e15
    t["gate"][3] = 60.0
    t["gate"][4] = -60.0
    t["gate"][5] = -100.0   # silu underflows
    check(t)
    clean = cg.rms_norm(t["x"], t["w"], EPS, gate=t["gate"])
    t["x"][6, 3], t["x"][7, 9] = float("nan"), float("inf")
    dirty = cg.rms_norm(t["x"], t["w"], EPS, gate=t["gate"])
    assert torch.equal(clean[:6], dirty[:6])
    assert torch.isnan(dirty[6]).all() and torch.isnan(dirty[7, 9])


def test_norm_partial_gradients():
    t = inputs((33, 192), BF, F32, "residual gate", seed=3)
    stored = cg.rms_norm(t["x"], t["w"], EPS, residual=t["residual"], gate=t["gate"])[1]
    val, err = R.rms_norm(stored, t["w"], EPS, None, t["gate"], torch.ones(33, 192))
    for n, key in (("x", "dx"), ("w", "dw"), ("residual", "dx"), ("gate", "dgate")):
        leaf = t[n].detach().requires_grad_()
        y, _ = cg.rms_norm(*[leaf if k == n else t[k] for k in ("x", "w")], EPS,
                           **{k: leaf if k == n else t[k] for k in ("residual", "gate")})
        got, = torch.autograd.grad(y.sum(), leaf)       # an expanded gradient
        within(got, val[key], R.rounded(err[key], val[key], leaf.dtype), n)
    leaf = t["x"].detach().requires_grad_()
    _, z = cg.rms_norm(leaf, t["w"], EPS, residual=t["residual"])
    got, = torch.autograd.grad(z, leaf, stored)          # z alone
    assert torch.equal(got, stored)


def test_norm_gradient_against_differences():
    t = inputs((6, 40), F32, F32, "residual gate", seed=5)
    dy, dz = rand(6, 40, seed=6), rand(6, 40, seed=7)
    names = ("x", "w", "residual", "gate")
    leaves = [t[n].detach().requires_grad_() for n in names]
    grads = torch.autograd.grad(cg.rms_norm(leaves[0], leaves[1], EPS, residual=leaves[2], gate=leaves[3]), leaves,
                                (dy, dz))

    def loss(x, w, residual, gate):
        val, _ = R.rms_norm(x, w, EPS, residual, gate)
        return float((val["y"] * R.d(dy)).sum() + (val["z"] * R.d(dz)).sum())

    for k in range(4):
        args = [R.d(t[n]) for n in names]
        way = torch.randn(args[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64)
        sides = []
        for step in (1e-4, -1e-4):
            moved = list(args)
            moved[k] = args[k] + step * way
            sides.append(loss(*moved))
        slope = (sides[0] - sides[1]) / 2e-4
        terms = R.d(grads[k]) * way
        assert abs(slope - float(terms.sum())) <= 2e-5 * float(terms.abs().sum())


# ---- 8-bit output ---------------------------------------------------------------------------

def check_fp8(t, group):
    D, x_type = t["x"].shape[-1], t["x"].dtype
    got = cg.rms_norm_fp8(t["x"], t["w"], EPS, residual=t["residual"], gate=t["gate"], group_size=group)
    q, scale = got[:2]
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == F32 and q.shape == t["x"].shape
    stored = t["x"]
    if t["residual"] is not None:
        stored = got[2]
        z_matches(stored, R.rms_norm(t["x"], t["w"], EPS, t["residual"])[0], x_type)
    val, err = R.rms_norm(stored, t["w"], EPS, None, t["gate"])
    n = group or D
    per, e = (v.reshape(*t["x"].shape[:-1], D // n, n) for v in (val["y"], err["y"]))
    want = per.abs().amax(-1).clamp(min=1e-12) / R.FP8_MAX
    off = e.amax(-1) / R.FP8_MAX + 4 * R.U * want
    within(scale, want, off, "scale")
    ideal = per / want[..., None]
    # y and the scale are off by their bounds, the quotient by two roundings; then
    # half a step of e4m3: 2^-4 of the value, 2^-10 below the normal numbers
    bound = e / want[..., None] + ideal.abs() * (off / want + 4 * R.U)[..., None]
    bound = bound + torch.maximum(2.0 ** -4 * (ideal.abs() + bound), torch.tensor(2.0 ** -10, dtype=torch.float64))
    within(q.float(), ideal.reshape(t["x"].shape), bound.reshape(t["x"].shape), "q")
    assert float(q.float().abs().max()) == R.FP8_MAX  # each group's largest value fills the range


@pytest.mark.parametrize("x_type,w_type", TYPES)
@pytest.mark.parametrize("D,group", [(128, 128), (128, None), (64, 32), (256, 64), (384, 128), (1024, 128), (2000, None),
                                     (4096, 128), (4096, None), (5120, 32), (33, None), (16384, 128), (192, 64)])
def test_fp8(D, group, x_type, w_type):
    for form in FORMS:
        check_fp8(inputs((6, D), x_type, w_type, form, seed=D), group)


def test_fp8_head_layout():
    check_fp8(inputs((2, 5, 4, 128), BF, F32, "gate"), None)
    t = inputs((9, 256), BF, F32, "gate")
    wide = torch.zeros(9, 300, dtype=BF, device=dev())
    wide[:, 1:257] = t["x"]
    t["x"] = wide[:, 1:257]                              # rows that start on 2 bytes
    check_fp8(t, 128)


def test_fp8_extreme_rows():
    t = inputs((6, 256), F32, F32, "", seed=1)
    t["x"][0] = 0
    t["x"][1] *= 1e-30
    t["x"][2, :128] = 0
    t["x"][3, 5] = float("nan")
    t["x"][4] *= 1e4
    q, scale = cg.rms_norm_fp8(t["x"], t["w"], 0.0 + EPS, group_size=128)
    q = q.float()
    floor = torch.tensor(1e-12 / 448, device=dev())
    assert not q[0].any() and torch.allclose(scale[0], floor.expand(2), rtol=1e-6, atol=0)
    assert not q[2, :128].any() and torch.allclose(scale[2, 0], floor, rtol=1e-6, atol=0)
    assert torch.isnan(q[3]).all() and torch.isnan(scale[3]).all()
    assert torch.isfinite(q[[0, 1, 2, 4, 5]]).all()
    t["x"][3, 5] = 0.0
    again, _ = cg.rms_norm_fp8(t["x"], t["w"], EPS, group_size=128)
    assert torch.equal(again.float()[[0, 1, 2, 4, 5]], q[[0, 1, 2, 4, 5]])


def test_fp8_refuses():
    x, w = rand(4, 256, seed=1, dtype=BF), torch.ones(256, device=dev())
    for group in (0, 100, -1):
        with pytest.raises(ValueError):
            cg.rms_norm_fp8(x, w, group_size=group)
    with pytest.raises(cg.CgdrError, match="group"):
        cg.rms_norm_fp8(x, w, group_size=16)


# ---- bounds of the writes, repeatability, graphs -----------------------------------------------

@pytest.mark.parametrize("R_,D", [(3, 128), (17, 64), (2, 4097), (5, 2000), (1, 9)])
def test_norm_writes_stay_inside(R_, D):
    lib = _lib.load()
    x, w = rand(R_, D, seed=1, dtype=BF), torch.ones(D, device=dev())
    (y, cy), (z, cz), (s, cs) = guarded((R_, D), BF), guarded((R_, D), BF), guarded((R_, 1), F32)
    assert lib.cgdrRmsNorm(_view(x), _view(w), _view(x), _view(x), EPS, 0, _view(y), None, _view(z), None) == 0
    q, cq = guarded((R_, D), torch.uint8)
    q8 = _lib.view(q.data_ptr(), _lib.DT_FP8_E4M3, q.shape, q.stride())
    assert lib.cgdrRmsNorm(_view(x), _view(w), None, _view(x), EPS, D, q8, _view(s), None, None) == 0
    (dx, c1), (dw, c2), (da, c3) = guarded((R_, D), BF), guarded((D,), F32), guarded((R_, D), BF)
    ws, c4 = guarded((R_, D), F32)
    assert lib.cgdrRmsNormBackward(_view(z), _view(w), _view(x), EPS, _view(x), _view(x), _view(dx), _view(dw),
                                   _view(da), ws.data_ptr(), R_ * D * 4, None) == 0
    torch.cuda.synchronize()
    for check_guard in (cy, cz, cs, cq, c1, c2, c3, c4):
        check_guard()


def test_norm_is_deterministic_and_graphs_replay():
    t = inputs((5000, 256), BF, F32, "residual gate", seed=1)
    dy = rand(5000, 256, seed=9, dtype=BF)

    def both():
        leaves = [t[n].detach().requires_grad_() for n in ("x", "w", "residual", "gate")]
        y, z = cg.rms_norm(leaves[0], leaves[1], EPS, residual=leaves[2], gate=leaves[3])
        return (y, z) + torch.autograd.grad((y, z), leaves, (dy, dy))

    ref = both()
    for a, b in zip(ref, both()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(ref, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    t["x"].mul_(0.5)
    graph.replay()
    for a, b in zip(out, both()):
        assert torch.equal(a, b)
