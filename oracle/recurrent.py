"""Float64 evaluations of the token-by-token recurrences and the norm --
TEST INFRASTRUCTURE ONLY (a measuring stick, never the product).

Each function takes torch tensors of any type, evaluates the definition in
float64 on the CPU without intermediate rounding, and returns float64
tensors together with what bounds the error of an fp32 evaluation.  ``U`` is
the unit roundoff of fp32.
"""

from __future__ import annotations

import torch

U = 2.0 ** -24
FP8_MAX = 448.0


def d(t):
    return None if t is None else t.detach().cpu().double()


def half_step(dtype) -> float:
    """Relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def least_step(dtype) -> float:
    """Half the spacing of the subnormal numbers: the absolute part of one rounding."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def rounded(bound, ref, dtype):
    """The bound of a value that is `bound` off `ref` and then rounded to `dtype`."""
    return bound + half_step(dtype) * (ref.abs() + bound) + least_step(dtype)


# ---- the diagonal recurrence ----------------------------------------------------------

def spans(B, T, cu):
    """(batch row, first, end, sequence) of every sequence"""
    if cu is None:
        return [(b, 0, T, b) for b in range(B)]
    cu = [int(c) for c in cu]
    return [(0, cu[n], cu[n + 1], n) for n in range(len(cu) - 1)]


def linear_recurrence(x, g, h0=None, cu=None, d_out=None, d_ht=None):
    """Values {o, ht[, dx, dg, dh0]} and bounds of the same names.

    Bounds.  One step h = a h + x in fp32 multiplies the state by a factor
    within 4 U of exp(g) (expf is within 2 ulp) and rounds product and sum;
    joining chunks multiplies by a product of such factors, again one rounding
    a factor.  With m the recurrence of absolute values, a step adds at most
    8 U m: e_t = a e_{t-1} + 8 U m_t.  The gradients are the same recurrence
    backwards; dg is a product of two such values and a factor."""
    x, g, h0, d_out, d_ht = d(x), d(g), d(h0), d(d_out), d(d_ht)
    a = g.exp()
    B, T, D = x.shape
    N = B if cu is None else len(cu) - 1
    init = torch.zeros(N, D, dtype=torch.float64) if h0 is None else h0
    o, eo = torch.zeros_like(x), torch.zeros_like(x)
    ht, eht = init.clone(), torch.zeros_like(init)
    val, err = {"o": o, "ht": ht}, {"o": eo, "ht": eht}
    backward = d_out is not None or d_ht is not None
    if backward:
        dx, edx, dg, edg = (torch.zeros_like(x) for _ in range(4))
        dh0, edh0 = (torch.zeros_like(init) for _ in range(2))
        val.update(dx=dx, dg=dg, dh0=dh0)
        err.update(dx=edx, dg=edg, dh0=edh0)
    for b, first, end, n in spans(B, T, cu):
        h, m, e = init[n], init[n].abs(), torch.zeros(D, dtype=torch.float64)
        prev, prev_e = [], []
        for t in range(first, end):
            prev.append(h)
            prev_e.append(e)
            h, m = a[b, t] * h + x[b, t], a[b, t] * m + x[b, t].abs()
            e = a[b, t] * e + 8 * U * m
            o[b, t], eo[b, t] = h, e
        ht[n], eht[n] = h, e
        if not backward:
            continue
        u = torch.zeros(D, dtype=torch.float64) if d_ht is None else d_ht[n]
        m, e = u.abs(), torch.zeros(D, dtype=torch.float64)
        for t in reversed(range(first, end)):
            up = 0 if d_out is None else d_out[b, t]
            dh, m = u + up, m + (0 if d_out is None else up.abs())
            e = e + 8 * U * m
            dx[b, t], edx[b, t] = dh, e
            h, eh = prev[t - first], prev_e[t - first]
            dg[b, t] = dh * a[b, t] * h
            edg[b, t] = a[b, t] * (e * h.abs() + dh.abs() * eh + e * eh) + 8 * U * dg[b, t].abs()
            u, m, e = a[b, t] * dh, a[b, t] * m, a[b, t] * e + 8 * U * a[b, t] * m
        dh0[n], edh0[n] = u, e
    return val, err


# ---- the gated delta rule --------------------------------------------------------------

def delta_rule(q, k, v, beta, state, lens, g, idx, scale):
    """Values (out, pool) and bounds of the same, for rows of a pool.

    Bounds, for |k| <= 1, 0 <= beta <= 1 and g <= 0: the update of a state row
    s (length Dk) is then no expansion, so its error grows by at most what one
    token adds.  Dot products of length Dk are within (Dk + 3) U |s| |k|;
    with the factor exp(g) (4 U) and the roundings of d and of the update, a
    token adds at most U ((Dk + 14) |s| + 6 |v|), and its output, scale (a s.q
    + d k.q), at most scale |q| (what the row had + U (2 Dk + 20) (|s| + |v|))."""
    q, k, v, beta, pool, g = d(q), d(k), d(v), d(beta), d(state), d(g)
    T, Nv, Dv = v.shape
    Dk, rep = q.shape[2], Nv // q.shape[1]
    scale = Dk ** -0.5 if scale is None else scale
    out, eout, epool = torch.zeros_like(v), torch.zeros_like(v), torch.zeros_like(pool)
    t, taken = 0, set()
    for b, n in enumerate(lens):
        slot = b if idx is None else int(idx[b])
        bad = slot < 0 or slot >= pool.shape[0] or slot in taken
        taken.add(slot)
        if bad:
            t += n
            continue
        s = pool[slot]
        e = torch.zeros(Nv, Dv, dtype=torch.float64)
        for _ in range(n):
            kt, qt = k[t].repeat_interleave(rep, 0), q[t].repeat_interleave(rep, 0)
            norm = s.norm(dim=-1)
            s = s * (torch.ones(Nv, dtype=torch.float64) if g is None else g[t].exp())[:, None, None]
            diff = beta[t][:, None] * (v[t] - (s * kt[:, None]).sum(-1))
            s = s + diff[..., None] * kt[:, None]
            out[t] = scale * (s * qt[:, None]).sum(-1)
            norm = torch.maximum(norm, s.norm(dim=-1))
            e = e + U * ((Dk + 14) * norm + 6 * v[t].abs())
            eout[t] = scale * qt.norm(dim=-1)[:, None] * (e + U * (2 * Dk + 20) * (norm + v[t].abs()))
            t += 1
        pool[slot], epool[slot] = s, e[..., None].expand_as(s)
    return (out, pool), (eout, epool)


# ---- the norm --------------------------------------------------------------------------

def rms_norm(x, w, eps, residual=None, gate=None, dy=None, dz=None):
    """Values {y, z[, dx, dw, dgate]} and bounds of the same names.

    Bounds.  A row's sum of squares is taken in at most 32 terms a lane and
    ten joins, all positive, so it is within 64 U; with the division, the sum
    with eps and rsqrt (2 ulp) r is within 40 U.  silu(gate) through the
    hardware's exponential and reciprocal is within (16 + 4 |gate|) U, and a
    sigmoid below 2^-126 (gate below -87.3), whose denominator 1 + e^-gate is
    past 2^126, comes out as 0 (the documented result of __fdividef there): an
    absolute error of at most 2^-126 |gate| in silu.  z is
    rounded to its type, which is part of the definition: in float64 it is
    rounded from the exact sum, and the fp32 sum of two values of at most 24
    bits rounds to the same one or, at a tie of fp32, to its neighbour."""
    shape, kind = x.shape, x.dtype
    x, w, residual, gate, dy, dz = (None if t is None else d(t) for t in (x, w, residual, gate, dy, dz))
    z = x if residual is None else (x + residual).to(kind).double()
    D = shape[-1]
    r = (z.square().mean(-1, keepdim=True) + eps).rsqrt()
    one = torch.ones_like(z)
    sig = one if gate is None else torch.sigmoid(gate)
    act = one if gate is None else gate * sig
    ea = 0 * one if gate is None else (16 + 4 * gate.abs()) * U
    lost = 0 * one if gate is None else gate.abs() * 2.0 ** -126
    n = z * r
    y = n * w * act
    val, err = {"y": y, "z": z}, {"y": y.abs() * (48 * U + ea) + (n * w).abs() * lost, "z": 0 * z}
    if dy is not None:
        flat = lambda t: t.reshape(-1, D)  # noqa: E731
        u = dy * w * act
        eu = u.abs() * (4 * U + ea) + (dy * w).abs() * lost
        mean, emean = (u * n).mean(-1, keepdim=True), (u * n).abs().mean(-1, keepdim=True)
        core = u - n * mean
        val["dx"] = r * core + (0 if dz is None else dz)
        # both sums are within 80 U of their absolute values' sums, r within 40 U
        err["dx"] = r * (eu + (eu * n.abs()).mean(-1, keepdim=True) * n.abs()
                         + 170 * U * n.abs() * emean + 44 * U * u.abs()) + 4 * U * val["dx"].abs()
        terms = flat(dy * act * n)
        rows = terms.shape[0]
        val["dw"] = terms.sum(0)
        err["dw"] = ((rows + 100) * U + flat(ea + 48 * U).amax(0)) * terms.abs().sum(0) + flat(
            (dy * n).abs() * lost).sum(0)
        if gate is not None:
            slope = sig + act * (1 - sig)
            val["dgate"] = dy * n * w * slope
            # 1 - sig is off by ea, absolutely; so is the slope's other term
            err["dgate"] = (dy * n * w).abs() * ((48 * U) * (sig + act.abs()) + 3 * ea * (1 + gate.abs()) + 2.0 ** -126
                                                 + lost)
    return val, err
