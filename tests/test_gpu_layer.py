"""The operators in a run together, as a recurrent layer uses them: a prompt
through the chunked gated delta rule, its final states into the pool, decode
steps token by token, the gated norm in 8 bits behind each; and a training
step through norm, diagonal recurrence and gated norm."""

from __future__ import annotations

import pytest
import torch

from oracle import recurrent as R
from test_gpu_recurrence import BF, F32, delta_inputs, dev, gates, rand, within

pytestmark = pytest.mark.gpu

cg = pytest.importorskip("cann_operator_challenge_august_b200")


def test_prompt_then_decode():
    """Against the float64 rule over the whole sequences.  The chunked prompt
    rounds its operands to bfloat16, so its states are within 2^-6 of the
    largest state value; the steps keep that distance (the rule does not
    expand), and each output adds its own rounding."""
    lens, steps, Nk, Nv, D = [70, 130, 5], 4, 2, 4, 128
    B, T = len(lens), sum(lens)
    t = delta_inputs([n + steps for n in lens], Nk, Nv, D, D, BF, F32, 6, seed=3)
    cut = [0]
    for n in lens:
        cut.append(cut[-1] + n + steps)
    prompt = torch.cat([torch.arange(cut[b], cut[b] + lens[b]) for b in range(B)]).to(dev())
    pool = torch.full((6, Nv, D, D), float("nan"), device=dev())
    slots = torch.tensor([4, 0, 3], device=dev())
    zero = torch.zeros(B, Nv, D, D, device=dev())
    n = torch.tensor(lens, dtype=torch.int32, device=dev())
    out, final = cg.chunk_gated_delta_rule(*[t[k][prompt] for k in ("query", "key", "value", "beta")], zero, n,
                                           g=t["g"][prompt], check_device_status=True)
    assert out.shape == (T, Nv, D)
    pool[slots] = final
    (ref, states), _ = R.delta_rule(t["query"], t["key"], t["value"], t["beta"], zero, [k + steps for k in lens],
                                    t["g"], None, None)
    w = 1 + 0.1 * rand(D, seed=8)
    gate = rand(B, Nv, D, seed=9, dtype=BF)
    for j in range(steps):
        at = torch.tensor([cut[b] + lens[b] + j for b in range(B)], device=dev())
        o = cg.recurrent_gated_delta_rule(*[t[k][at] for k in ("query", "key", "value", "beta")], pool, g=t["g"][at],
                                          state_indices=slots, check_device_status=True)
        want = ref[at.cpu()]
        within(o, want, 2.0 ** -6 * float(ref.abs().max()), f"step {j}")
        q, scale = cg.rms_norm_fp8(o, w, gate=gate)      # one scale a head
        val, _ = R.rms_norm(o, w, 1e-6, None, gate)
        assert q.shape == (B, Nv, D) and scale.shape == (B, Nv, 1)
        # half a step of e4m3 at the group's largest value, and fp32's own error
        within(q.float() * scale, val["y"], (2.0 ** -4 + 1e-5) * val["y"].abs().amax(-1, keepdim=True), "8-bit output")
    within(pool[slots], states, 2.0 ** -6 * float(states.abs().max()), "states")
    assert torch.isnan(pool[[1, 2, 5]]).all()


def test_training_step():
    """norm(x + residual) -> recurrence -> gated norm, forwards and backwards in
    fp32 against float64 autograd of the definitions.  Every operator's own
    gradient is held to derived bounds elsewhere; here the chain is held to
    1e-5 of the largest gradient (three operators, each within about 1e-6)."""
    B, T, D = 2, 150, 64
    cu = [0, 100, 100, 150]
    x, res, gate, g = (rand(1, T, D, seed=k) for k in range(4))
    g = gates(1, T, D, seed=5)
    w1, w2, h0 = 1 + 0.1 * rand(D, seed=6), 1 + 0.1 * rand(D, seed=7), rand(3, D, seed=8)
    dy, dz = rand(1, T, D, seed=9), rand(1, T, D, seed=10)
    args = (x, res, gate, g, w1, w2, h0)

    def plain(x, res, gate, g, w1, w2, h0):
        z = x + res
        n = z * (z.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w1
        rows = []
        for k in range(3):
            h = h0[k]
            for t in range(cu[k], cu[k + 1]):
                h = g[0, t].exp() * h + n[0, t]
                rows.append(h)
        o = torch.stack(rows)[None]
        return o * (o.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w2 * torch.nn.functional.silu(gate), z

    wide = [R.d(t).requires_grad_() for t in args]
    want_outs = plain(*wide)
    want = torch.autograd.grad(want_outs, wide, (R.d(dy), R.d(dz)))
    leaves = [t.requires_grad_() for t in args]
    x, res, gate, g, w1, w2, h0 = leaves
    n, z = cg.rms_norm(x, w1, residual=res)
    o, _ = cg.gated_linear_recurrence(n, g, h0, cu_seqlens=torch.tensor(cu, device=dev()))
    y = cg.rms_norm(o, w2, gate=gate)
    got = torch.autograd.grad((y, z), leaves, (dy, dz))
    for a, b, what in zip((y, z) + got, want_outs + want, ("y", "z", "dx", "dres", "dgate", "dg", "dw1", "dw2", "dh0")):
        within(a, b.detach(), 1e-5 * float(b.detach().abs().max()), what)
