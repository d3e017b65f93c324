"""The token-by-token recurrences on the GPU against their definitions in
float64 (oracle/recurrent.py), element by element within bounds derived
there; gradients also against differences of the float64 definition."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import recurrent as R

pytestmark = pytest.mark.gpu

cg = pytest.importorskip("cann_operator_challenge_august_b200")
from cann_operator_challenge_august_b200 import _lib  # noqa: E402
from cann_operator_challenge_august_b200.recurrence import _view  # noqa: E402

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


def within(got, ref, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, what
    both = torch.isnan(got) & torch.isnan(ref)
    bad = ~(((got - ref).abs() <= bound) | both | (got == ref))
    assert not bad.any(), (f"{what}: {int(bad.sum())}/{bad.numel()} outside, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0]} for {ref[bad][0]} +- {torch.as_tensor(bound).expand_as(ref)[bad][0]}")


def rand(*shape, seed, dtype=F32, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=gen)).to(dtype).to(dev())


def gates(*shape, seed, dtype=F32):
    gen = torch.Generator().manual_seed(seed)
    return torch.nn.functional.logsigmoid(torch.randn(*shape, generator=gen) + 2).to(dtype).to(dev())


# ---- the diagonal recurrence --------------------------------------------------------------

def check_scan(B, T, D, x_type, g_type, *, cu=None, state=True, seed=0, x=None, g=None):
    N = B if cu is None else len(cu) - 1
    x = rand(B, T, D, seed=seed, dtype=x_type, scale=0.5) if x is None else x
    g = gates(B, T, D, seed=seed + 1, dtype=g_type) if g is None else g
    h0 = rand(N, D, seed=seed + 2) if state else None
    do, dht = rand(B, T, D, seed=seed + 3, dtype=x_type), rand(N, D, seed=seed + 4)
    cut = None if cu is None else torch.tensor(cu, dtype=torch.int64, device=x.device)
    leaves = [t.detach().requires_grad_() for t in (x, g) + ((h0,) if state else ())]
    o, ht = cg.gated_linear_recurrence(leaves[0], leaves[1], leaves[2] if state else None, output_final_state=True,
                                       cu_seqlens=cut)
    grads = torch.autograd.grad((o, ht), leaves, (do, dht))
    with torch.no_grad():  # the path without a backward pass saves no states
        o2, ht2 = cg.gated_linear_recurrence(x, g, h0, output_final_state=True, cu_seqlens=cut)
        o3, none = cg.gated_linear_recurrence(x, g, h0, cu_seqlens=cut)
    assert torch.equal(o, o2) and torch.equal(ht, ht2) and torch.equal(o, o3) and none is None
    val, err = R.linear_recurrence(x, g, h0, cu, do, dht)
    within(o, val["o"], R.rounded(err["o"], val["o"], x_type), "o")
    within(ht, val["ht"], R.rounded(err["ht"], val["ht"], F32), "final state")
    within(grads[0], val["dx"], R.rounded(err["dx"], val["dx"], x_type), "dx")
    within(grads[1], val["dg"], R.rounded(err["dg"], val["dg"], g_type), "dg")
    if state:
        within(grads[2], val["dh0"], R.rounded(err["dh0"], val["dh0"], F32), "dh0")
    return x, g, h0, o, ht, grads


TYPES = [(BF, BF), (BF, F32), (F16, F16), (F16, F32), (F32, F32)]


@pytest.mark.parametrize("x_type,g_type", TYPES)
@pytest.mark.parametrize("B,T,D", [(1, 1, 128), (2, 63, 64), (1, 64, 8), (3, 65, 100), (2, 300, 33), (1, 1030, 260)])
def test_scan_fixed_length(B, T, D, x_type, g_type):
    check_scan(B, T, D, x_type, g_type, seed=T + D)
    check_scan(B, T, D, x_type, g_type, seed=T, state=False)


@pytest.mark.parametrize("x_type,g_type", [(BF, F32), (F32, F32)])
@pytest.mark.parametrize("cu,T", [
    ([0, 1], 1), ([0, 0, 5], 9), ([0, 64, 128], 128), ([0, 1, 1, 1, 64, 129, 129, 300], 300), ([0, 0, 0], 3),
    ([0, 5, 6, 7, 8, 9, 10, 70, 71, 600, 601], 640), ([0, 513, 1100], 1100),
])
def test_scan_packed(cu, T, x_type, g_type):
    check_scan(1, T, 96, x_type, g_type, cu=cu, seed=T)
    check_scan(1, T, 37, x_type, g_type, cu=cu, seed=T, state=False)


def test_scan_many_short_sequences():
    lens = [(7 * i + 3) % 6 for i in range(400)]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    check_scan(1, cu[-1] + 11, 64, BF, BF, cu=cu)


@pytest.mark.parametrize("B,T,D", [(1, 4100, 72), (3, 2049, 300), (1, 700, 4104)])
def test_scan_long(B, T, D):
    check_scan(B, T, D, BF, BF, seed=5)


@pytest.mark.parametrize("B,T,D", [
    (4, 300, 2560),    # a CTA for each of 160 slabs, clusters of four that keep pace, three segments
    (3, 300, 3264),    # 153 slabs of an odd count a row: no neighbours to keep pace with
    (5, 150, 4096),    # more CTAs than the GPU holds at once
    (1, 1100, 3712),   # 58 slabs: clusters of eight CTAs of four warps
])
def test_scan_launch_shapes(B, T, D):
    """The ways the grid is laid out; a sample of the channels against the definition."""
    x, g = rand(B, T, D, seed=1, dtype=BF), gates(B, T, D, seed=2, dtype=BF)
    h0, do, dht = rand(B, D, seed=3), rand(B, T, D, seed=4, dtype=BF), rand(B, D, seed=5)
    leaves = [t.requires_grad_() for t in (x, g, h0)]
    o, ht = cg.gated_linear_recurrence(*leaves, output_final_state=True)
    dx, dg, dh0 = torch.autograd.grad((o, ht), leaves, (do, dht))
    at = torch.cat([torch.arange(0, D, 61), torch.arange(D - 3, D)]).to(dev())
    val, err = R.linear_recurrence(x[..., at], g[..., at], h0[..., at], None, do[..., at], dht[..., at])
    for n, t, kind in (("o", o, BF), ("ht", ht, F32), ("dx", dx, BF), ("dg", dg, BF), ("dh0", dh0, F32)):
        within(t[..., at], val[n], R.rounded(err[n], val[n], kind), n)


def test_scan_strided_views():
    wide = rand(2, 200, 3, 64, seed=1, dtype=BF)
    g = gates(200, 2, 64, seed=2).transpose(0, 1)
    check_scan(2, 200, 64, BF, F32, x=wide[:, :, 1], g=g)
    check_scan(2, 100, 60, BF, F32, x=wide[:, ::2, 2, 3:63], g=g[:, 100:, 4:])


def test_scan_expanded_gradient_and_unused_outputs():
    x, g = rand(2, 90, 40, seed=1), gates(2, 90, 40, seed=2)
    h0 = rand(2, 40, seed=3)
    leaves = [t.requires_grad_() for t in (x, g, h0)]
    o, ht = cg.gated_linear_recurrence(*leaves, output_final_state=True)
    for outs, do, dht in (((o.sum(),), torch.ones(2, 90, 40), None), ((ht.sum(),), None, torch.ones(2, 40))):
        got = torch.autograd.grad(outs, leaves, retain_graph=True)
        val, err = R.linear_recurrence(x, g, h0, None, do, dht)
        for n, t in zip(("dx", "dg", "dh0"), got):
            within(t, val[n], R.rounded(err[n], val[n], F32), n)
    for k in range(3):  # one gradient at a time
        one = torch.autograd.grad((o, ht), [leaves[k]], (torch.ones_like(o), torch.ones_like(ht)), retain_graph=True)
        val, err = R.linear_recurrence(x, g, h0, None, torch.ones(2, 90, 40), torch.ones(2, 40))
        n = ("dx", "dg", "dh0")[k]
        within(one[0], val[n], R.rounded(err[n], val[n], F32), n)


def test_scan_gradient_against_differences():
    """The derivative along random directions, by central differences of the
    float64 definition: their error is O(step^2), below 1e-6 of the terms."""
    B, T, D = 2, 75, 12
    x, g, h0 = rand(B, T, D, seed=1), gates(B, T, D, seed=2), rand(B, D, seed=3)
    do, dht = rand(B, T, D, seed=4), rand(B, D, seed=5)
    leaves = [t.detach().requires_grad_() for t in (x, g, h0)]
    grads = torch.autograd.grad(cg.gated_linear_recurrence(*leaves, output_final_state=True), leaves, (do, dht))

    def loss(*args):
        val, _ = R.linear_recurrence(*args)
        return float((val["o"] * R.d(do)).sum() + (val["ht"] * R.d(dht)).sum())

    for k in range(3):
        args = [R.d(t) for t in (x, g, h0)]
        way = torch.randn(args[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64)
        step = 1e-4
        sides = []
        for sign in (1, -1):
            moved = list(args)
            moved[k] = args[k] + sign * step * way
            sides.append(loss(*moved))
        slope = (sides[0] - sides[1]) / (2 * step)
        terms = R.d(grads[k]) * way
        assert abs(slope - float(terms.sum())) <= 2e-5 * float(terms.abs().sum())


def test_scan_minus_infinity_forgets():
    """exp(-inf) = 0: nothing of the earlier state remains, nor of its gradient."""
    x, g = rand(1, 200, 16, seed=1), gates(1, 200, 16, seed=2)
    g[0, [0, 63, 64, 130]] = -torch.inf
    check_scan(1, 200, 16, F32, F32, x=x, g=g)
    g[0, 70:90] = -80.0  # products that underflow
    check_scan(1, 200, 16, F32, F32, x=x, g=g)


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_scan_sequences_do_not_touch_each_other(poison):
    """NaN and infinities in one sequence, its initial state and the rows
    behind the last sequence change no bit of the others."""
    cu = [0, 30, 100, 170, 340]
    cut = torch.tensor(cu, device=dev())
    x, g, h0 = rand(1, 360, 40, seed=1), gates(1, 360, 40, seed=2), rand(4, 40, seed=3)
    do, dht = rand(1, 360, 40, seed=4), rand(4, 40, seed=5)

    def both(x, g, h0, do, dht):
        leaves = [t.detach().clone().requires_grad_() for t in (x, g, h0)]
        o, ht = cg.gated_linear_recurrence(*leaves, output_final_state=True, cu_seqlens=cut)
        return (o, ht) + torch.autograd.grad((o, ht), leaves, (do, dht))

    clean = both(x, g, h0, do, dht)
    for t in (x, g, do):
        t[0, 100:170] = poison
        t[0, 340:] = poison
    h0[2], dht[2] = poison, poison
    dirty = both(x, g, h0, do, dht)
    rows, seqs = [*range(100), *range(170, 360)], [0, 1, 3]
    for k in (0, 2, 3):
        assert torch.equal(clean[k][0, rows], dirty[k][0, rows])
        assert not dirty[k][0, 340:].any()
    for k in (1, 4):
        assert torch.equal(clean[k][seqs], dirty[k][seqs])


def test_scan_is_deterministic_and_split_calls_agree():
    x, g = rand(1, 1000, 512, seed=1, dtype=BF), gates(1, 1000, 512, seed=2)
    o, ht = cg.gated_linear_recurrence(x, g, output_final_state=True)
    for _ in range(3):
        o2, ht2 = cg.gated_linear_recurrence(x, g, output_final_state=True)
        assert torch.equal(o, o2) and torch.equal(ht, ht2)
    a, mid = cg.gated_linear_recurrence(x[:, :333], g[:, :333], output_final_state=True)
    b, end = cg.gated_linear_recurrence(x[:, 333:], g[:, 333:], mid, output_final_state=True)
    val, err = R.linear_recurrence(x, g)
    within(torch.cat([a, b], 1), val["o"], R.rounded(err["o"], val["o"], BF), "two calls")
    within(end, val["ht"], R.rounded(err["ht"], val["ht"], F32), "two calls' state")


def test_scan_empty():
    x = torch.empty(2, 0, 8, device=dev(), requires_grad=True)
    h0 = rand(2, 8, seed=1).requires_grad_()
    o, ht = cg.gated_linear_recurrence(x, x.detach(), h0, output_final_state=True)
    assert o.shape == (2, 0, 8) and torch.equal(ht, h0)
    dx, dh0 = torch.autograd.grad((o, ht), (x, h0), (torch.empty_like(o), h0.detach()))
    assert dx.shape == x.shape and torch.equal(dh0, h0)


def test_scan_graph_and_streams():
    """Forward and backward captured together and replayed on new inputs; the
    same call on another stream."""
    x, g = rand(1, 500, 256, seed=1, dtype=BF), gates(1, 500, 256, seed=2)
    do = rand(1, 500, 256, seed=3, dtype=BF)

    def both():
        leaves = [t.detach().requires_grad_() for t in (x, g)]
        o, ht = cg.gated_linear_recurrence(*leaves, output_final_state=True)
        return (o, ht) + torch.autograd.grad(o, leaves, do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ref = both()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(ref, both()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for seed in (10, 20):
        x.copy_(rand(1, 500, 256, seed=seed, dtype=BF))
        graph.replay()
        for a, b in zip(out, both()):
            assert torch.equal(a, b)


def guarded(shape, dtype, fill=7.0):
    """A tensor inside a buffer of guards, and a check that the guards stand."""
    n = 1
    for s in shape:
        n *= s
    buf = torch.full((n + 512,), fill, dtype=dtype, device=dev())

    def check():
        assert (buf[:256].float() == fill).all() and (buf[256 + n:].float() == fill).all()
    return buf[256:256 + n].view(shape), check


@pytest.mark.parametrize("D", [40, 33])
@pytest.mark.parametrize("T,cu", [(130, None), (1, None), (130, [0, 0, 65, 65, 128, 128])])
def test_scan_writes_stay_inside(T, cu, D):
    lib, N = _lib.load(), 1 if cu is None else len(cu) - 1
    x, g = rand(1, T, D, seed=1, dtype=BF), gates(1, T, D, seed=2)
    cut = None if cu is None else torch.tensor(cu, device=dev())
    outs = [guarded((1, T, D), BF), guarded((N, D), F32), guarded((1, -(-T // 128), D), F32)]
    grads = [guarded((1, T, D), BF), guarded((1, T, D), F32), guarded((N, D), F32)]
    assert lib.cgdrGatedLinearRecurrence(_view(x), _view(g), None, _view(cut), *[_view(t) for t, _ in outs], None) == 0
    assert lib.cgdrGatedLinearRecurrenceBackward(_view(x), _view(g), None, _view(cut), _view(outs[2][0]), _view(x), None,
                                                 *[_view(t) for t, _ in grads], None) == 0
    torch.cuda.synchronize()
    for _, check in outs + grads:
        check()


@pytest.mark.parametrize("cu", [[0, 500, 40], [0, -3, 20], [5, 3, 1000], [0, 2 ** 40, 7]])
def test_scan_survives_inconsistent_bounds(cu):
    """Bounds past T, negative or decreasing: no read or write outside the tensors."""
    lib, T, D = _lib.load(), 100, 36
    x, g = rand(1, T, D, seed=1, dtype=BF), gates(1, T, D, seed=2)
    cut = torch.tensor(cu, device=dev())
    outs = [guarded((1, T, D), BF), guarded((2, D), F32), guarded((1, 1, D), F32)]
    outs[2][0].zero_()
    grads = [guarded((1, T, D), BF), guarded((1, T, D), F32), guarded((2, D), F32)]
    assert lib.cgdrGatedLinearRecurrence(_view(x), _view(g), None, _view(cut), *[_view(t) for t, _ in outs], None) == 0
    assert lib.cgdrGatedLinearRecurrenceBackward(_view(x), _view(g), None, _view(cut), _view(outs[2][0]), _view(x), None,
                                                 *[_view(t) for t, _ in grads], None) == 0
    torch.cuda.synchronize()
    for _, check in outs + grads:
        check()


# ---- one token a row ------------------------------------------------------------------------

@pytest.mark.parametrize("x_type,g_type", TYPES)
@pytest.mark.parametrize("B,D", [(1, 1), (3, 128), (5, 33), (70, 1028), (300, 40)])
def test_step(B, D, x_type, g_type):
    x, g = rand(B, D, seed=1, dtype=x_type), gates(B, D, seed=2, dtype=g_type)
    state, check = guarded((B + 7, D), F32)
    state.copy_(rand(B + 7, D, seed=3))
    before = state.clone()
    for dtype in (torch.int32, torch.int64):
        state.copy_(before)
        idx = torch.randperm(B + 7, generator=torch.Generator().manual_seed(4))[:B].to(dtype).to(dev())
        idx[1::3] = -1
        o = cg.gated_linear_recurrence_step(x, g, state, state_indices=idx, check_device_status=True)
        want, ref, bound = R.d(before), torch.zeros(B, D, dtype=torch.float64), torch.zeros(B, D, dtype=torch.float64)
        pool = torch.zeros_like(want)
        for b, i in enumerate(idx.tolist()):
            if i >= 0:
                bound[b] = 8 * R.U * (R.d(g)[b].exp() * want[i].abs() + R.d(x)[b].abs())
                want[i] = ref[b] = R.d(g)[b].exp() * want[i] + R.d(x)[b]
                pool[i] = bound[b]
        within(o, ref, R.rounded(bound, ref, x_type), "o")
        within(state, want, pool, "state")
        check()
    state.copy_(before)
    o = cg.gated_linear_recurrence_step(x, g, state)
    val, err = R.linear_recurrence(x[:, None], g[:, None], before[:B])
    within(o, val["ht"], R.rounded(err["ht"], val["ht"], x_type), "without indices")
    assert torch.equal(state[B:], before[B:])


def test_step_bad_indices_are_reported():
    x, g, state = rand(5, 64, seed=1), gates(5, 64, seed=2), rand(6, 64, seed=3)
    before = state.clone()
    idx = torch.tensor([2, 6, 2, -1, 0], device=dev())
    with pytest.raises(RuntimeError, match="named twice"):
        cg.gated_linear_recurrence_step(x, g, state, state_indices=idx, check_device_status=True)
    assert torch.equal(state[[1, 3, 4, 5]], before[[1, 3, 4, 5]])
    once = before.clone()
    o = cg.gated_linear_recurrence_step(x, g, once, state_indices=torch.tensor([2, -1, -1, -1, 0], device=dev()))
    assert torch.equal(state, once) and not o[1:4].any()


# ---- the gated delta rule ---------------------------------------------------------------------

def delta_inputs(lens, Nk, Nv, Dk, Dv, x_type, s_type, slots, seed):
    T = sum(lens)
    unit = lambda t: (t.float() / t.float().norm(dim=-1, keepdim=True) * 0.99).to(x_type)  # noqa: E731
    return dict(query=unit(rand(T, Nk, Dk, seed=seed)), key=unit(rand(T, Nk, Dk, seed=seed + 1)),
                value=rand(T, Nv, Dv, seed=seed + 2, dtype=x_type),
                beta=torch.sigmoid(rand(T, Nv, seed=seed + 3)).to(x_type), g=gates(T, Nv, seed=seed + 4),
                state=rand(slots, Nv, Dv, Dk, seed=seed + 5, dtype=s_type, scale=0.1))


def check_delta(t, lens, idx, scale=None, with_g=True, with_lens=True):
    before = t["state"].clone()
    dev_lens = torch.tensor(lens, dtype=torch.int32, device=dev()) if with_lens else None
    dev_idx = None if idx is None else torch.tensor(idx, dtype=torch.int32, device=dev())
    g = t["g"] if with_g else None
    o = cg.recurrent_gated_delta_rule(t["query"], t["key"], t["value"], t["beta"], t["state"], dev_lens, scale, g,
                                      state_indices=dev_idx, check_device_status=True)
    (ref, pool), (eo, es) = R.delta_rule(t["query"], t["key"], t["value"], t["beta"], before, lens, g, idx, scale)
    within(o, ref, R.rounded(eo, ref, o.dtype), "o")
    touched = (es.flatten(1).amax(1) > 0)[:, None, None, None]
    bound = torch.where(touched, R.rounded(es, pool, t["state"].dtype), 0.0)
    within(t["state"], pool, bound, "state")
    return o


@pytest.mark.parametrize("x_type,s_type", [(BF, F32), (BF, BF), (F16, F32), (F16, BF), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("Nk,Nv,Dk,Dv", [(2, 4, 128, 128), (1, 1, 64, 32), (2, 2, 96, 80), (1, 3, 50, 33),
                                         (1, 2, 256, 256), (2, 4, 8, 8), (1, 1, 1, 1), (1, 2, 132, 70)])
def test_delta_shapes(Nk, Nv, Dk, Dv, x_type, s_type):
    lens = [1, 0, 3, 1, 6]
    t = delta_inputs(lens, Nk, Nv, Dk, Dv, x_type, s_type, 8, seed=Dk + Dv)
    check_delta(t, lens, [6, 1, 0, -1, 3])
    t = delta_inputs([1] * 5, Nk, Nv, Dk, Dv, x_type, s_type, 6, seed=Dk)
    check_delta(t, [1] * 5, None, scale=0.3, with_g=False, with_lens=False)


def test_delta_full_batches():
    """Grids that take two state rows a lane group, and many rows before the last one."""
    t = delta_inputs([1] * 90, 2, 4, 128, 128, BF, F32, 100, seed=1)
    check_delta(t, [1] * 90, [(7 * i) % 100 for i in range(90)], with_lens=False)
    lens = [(i * 5 + 2) % 4 for i in range(600)]
    t = delta_inputs(lens, 1, 1, 64, 64, BF, F32, 600, seed=2)
    check_delta(t, lens, list(range(599, -1, -1)))


def test_delta_float32_beta_and_inference_mode():
    t = delta_inputs([1] * 3, 2, 4, 64, 64, BF, F32, 5, seed=11)
    t["beta"] = torch.sigmoid(rand(3, 4, seed=12))
    with torch.inference_mode():
        check_delta(t, [1] * 3, [4, 1, 0])
        x, g, state = rand(3, 64, seed=1), gates(3, 64, seed=2), rand(5, 64, seed=3)
        assert torch.isfinite(cg.gated_linear_recurrence_step(x, g, state)).all()
        assert torch.isfinite(cg.gated_linear_recurrence(x[None], g[None])[0]).all()


def test_updates_are_seen_by_autograd():
    """A pool that a graph has saved and a step then changes is refused by the
    backward pass, as after any in-place operation."""
    state = rand(3, 64, seed=3).requires_grad_()
    pool = state * 1.0
    loss = pool.square().sum()
    with torch.no_grad():
        cg.gated_linear_recurrence_step(rand(3, 64, seed=1), gates(3, 64, seed=2), pool)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_second_derivatives_are_refused():
    x, g = rand(1, 5, 8, seed=1).requires_grad_(), gates(1, 5, 8, seed=2)
    o, _ = cg.gated_linear_recurrence(x, g)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(o.sum(), x, create_graph=True)


def test_delta_long_sequence():
    t = delta_inputs([700, 1], 1, 2, 64, 64, F32, F32, 2, seed=3)
    check_delta(t, [700, 1], [1, 0])


def test_delta_strided_views():
    t = delta_inputs([1] * 4, 2, 4, 64, 64, BF, F32, 6, seed=4)
    wide = rand(4, 3, 4, 80, seed=9, dtype=BF)
    wide[:, 0, :, :64] = t["value"]
    t["value"] = wide[:, 0, :, :64]
    t["key"] = torch.cat([t["key"], t["query"]], dim=-1)[..., :64]
    t["query"] = t["query"].transpose(0, 1).contiguous().transpose(0, 1)
    t["state"] = rand(6, 4, 3, 64, 64, seed=10, scale=0.1)[:, :, 1]
    check_delta(t, [1] * 4, [5, 4, 1, 0])
    t = delta_inputs([1] * 4, 2, 4, 64, 64, BF, F32, 6, seed=4)  # rows that are not 8-byte aligned
    t["key"] = torch.cat([t["query"][..., :1], t["key"]], dim=-1)[..., 1:]
    check_delta(t, [1] * 4, [5, 4, 1, 0])


def test_delta_behind_the_last_sequence_and_bad_rows():
    lens = [2, 1]
    t = delta_inputs([2, 1, 4], 1, 2, 64, 40, BF, F32, 3, seed=5)
    before = t["state"].clone()
    args = (t["query"], t["key"], t["value"], t["beta"], t["state"])
    n = torch.tensor(lens, dtype=torch.int32, device=dev())
    with pytest.raises(RuntimeError, match="lengths"):
        cg.recurrent_gated_delta_rule(*args, n, g=t["g"], check_device_status=True)
    o = cg.recurrent_gated_delta_rule(*args, n, g=t["g"])
    assert not o[3:].any() and o[:3].any()
    assert torch.equal(t["state"][2], before[2])
    for idx in ([0, 0], [0, 3], [0, 2 ** 30]):
        state = before.clone()
        idx = torch.tensor(idx, device=dev())
        args = (t["query"], t["key"], t["value"], t["beta"], state)
        with pytest.raises(RuntimeError, match="named twice"):
            cg.recurrent_gated_delta_rule(*args, n, g=t["g"], state_indices=idx, check_device_status=True)
        assert torch.equal(state[1:], before[1:])
        alone = before.clone()
        cg.recurrent_gated_delta_rule(*args[:4], alone, n, g=t["g"], state_indices=torch.tensor([0, -1], device=dev()))
        assert torch.equal(state, alone)
    for bad in ([-5, 1], [9, 1], [2 ** 31 - 1, 2 ** 31 - 1]):  # cut to what T holds
        with pytest.raises(RuntimeError, match="lengths"):
            cg.recurrent_gated_delta_rule(*args, torch.tensor(bad, dtype=torch.int32, device=dev()), g=t["g"],
                                          check_device_status=True)


def test_delta_empty():
    t = delta_inputs([0], 1, 2, 64, 40, BF, F32, 3, seed=5)
    before = t["state"].clone()
    o = cg.recurrent_gated_delta_rule(t["query"], t["key"], t["value"], t["beta"], t["state"], g=t["g"],
                                      check_device_status=True)
    assert o.shape == (0, 2, 40) and torch.equal(t["state"], before)


def test_delta_nan_stays_in_its_sequence():
    t = delta_inputs([1] * 4, 2, 4, 64, 64, BF, F32, 6, seed=6)
    clean = {n: v.clone() for n, v in t.items()}
    for n in ("query", "key", "value", "beta", "g"):
        t[n][2] = float("nan")
    t["state"][4] = float("nan")  # no row's state
    idx = torch.tensor([5, 0, 1, 2], device=dev())
    outs = [cg.recurrent_gated_delta_rule(s["query"], s["key"], s["value"], s["beta"], s["state"], g=s["g"],
                                          state_indices=idx) for s in (clean, t)]
    assert torch.equal(outs[0][[0, 1, 3]], outs[1][[0, 1, 3]]) and torch.isnan(outs[1][2]).all()
    assert torch.equal(clean["state"][[5, 0, 2, 3]], t["state"][[5, 0, 2, 3]])


def test_delta_large_pool_offsets():
    """State offsets past 32 bits: a pool of 2^32 and more bytes and elements."""
    per = 32 * 128 * 128
    slots = (1 << 32) // per + 40  # 2^32 elements, 8 GiB in bfloat16, and 40 states behind them
    state = torch.zeros(slots, 32, 128, 128, dtype=BF, device=dev())
    t = delta_inputs([1, 1], 16, 32, 128, 128, BF, BF, 1, seed=7)
    idx = [slots - 1, 0]
    init = rand(2, 32, 128, 128, seed=8, dtype=BF, scale=0.1)
    state[idx] = init
    o = cg.recurrent_gated_delta_rule(t["query"], t["key"], t["value"], t["beta"], state, g=t["g"],
                                      state_indices=torch.tensor(idx, device=dev()))
    small = init.clone()
    o2 = cg.recurrent_gated_delta_rule(t["query"], t["key"], t["value"], t["beta"], small, g=t["g"])
    assert torch.equal(o, o2) and torch.equal(state[idx], small)
    assert not state[1:slots - 1].any()


def test_delta_graph_replays_update_the_pool():
    t = delta_inputs([1] * 3, 2, 4, 64, 64, BF, F32, 5, seed=8)
    idx = torch.tensor([4, 0, -1], device=dev())
    eager = t["state"].clone()
    run = lambda s: cg.recurrent_gated_delta_rule(t["query"], t["key"], t["value"], t["beta"], s, g=t["g"],  # noqa: E731
                                                  state_indices=idx)
    run(eager.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = run(t["state"])
    assert torch.equal(t["state"], eager)
    for _ in range(3):
        graph.replay()
        assert torch.equal(o, run(eager)) and torch.equal(t["state"], eager)
        t["value"].mul_(0.5)
        idx.copy_(torch.tensor([1, 4, 3], device=dev()))


def test_status_pointer_through_the_c_entry():
    """The status word is set and cleared in stream order."""
    lib = _lib.load()
    x, g, state = rand(2, 16, seed=1), gates(2, 16, seed=2), rand(2, 16, seed=3)
    status = torch.full((1,), -1, dtype=torch.int32, device=dev())
    for idx, want in (([0, 0], _lib.DEVICE_BAD_STATE_INDEX), ([0, 1], 0)):
        i = torch.tensor(idx, device=dev())
        st = lib.cgdrGatedLinearRecurrenceStep(_view(x), _view(g), _view(state), _view(i), _view(torch.empty_like(x)),
                                               status.data_ptr(), ctypes.c_void_p(0))
        assert st == 0
        assert int(status.item()) == want
