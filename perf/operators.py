"""The operators around the chunked gated delta rule, as they are measured.

* ``recurrence``: the diagonal gated recurrence h_t = exp(g_t) h_{t-1} + x_t over
  whole sequences, forward, or forward and backward.
* ``recurrence_step``: the same for one token a row, on a pool of states.
* ``delta_step``: the gated delta rule token by token, on a pool of states.
* ``norm``: root-mean-square norm, with the residual's addition or a silu gate,
  forward, or forward and backward.
* ``norm_fp8``: the same forward with an e4m3 output and fp32 scales.

``run`` computes the plain form in float32 unless ``own`` is true; then it
calls this package.  ``exact`` evaluates the definitions in float64.
"""

from __future__ import annotations

import math

import torch

own = False

BF, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
TYPES = {"bf16": BF, "fp16": F16, "fp32": F32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
FP8_MAX = 448.0


# ---- cases ------------------------------------------------------------------------

def listed():
    return [
        # training step of a layer of 32 heads x 128 channels on 4 x 8192 tokens
        {"name": "recurrence_train_4x8192", "op": "recurrence", "B": 4, "T": 8192, "D": 4096, "N": 0, "tail": 0,
         "x": "bf16", "g": "bf16", "state": True, "backward": True},
        # training on 16 packed ragged sequences, gates kept in float32, some padding behind the last one
        {"name": "recurrence_train_packed", "op": "recurrence", "B": 1, "T": 32768, "D": 2048, "N": 16, "tail": 37,
         "x": "bf16", "g": "fp32", "state": True, "backward": True},
        # long-context evaluation: one sequence of 65536 tokens, forward only
        {"name": "recurrence_long_65536", "op": "recurrence", "B": 1, "T": 65536, "D": 4096, "N": 0, "tail": 0,
         "x": "bf16", "g": "bf16", "state": False, "backward": False},
        # one decode step of a batch of 64 rows (two of them padding) on a pool of 96 states
        {"name": "recurrence_step_64", "op": "recurrence_step", "B": 64, "pad": 2, "slots": 96, "D": 4096, "x": "bf16",
         "g": "bf16"},
        # one decode step of a full server, float32 gates, rows that are no multiple of 16 bytes
        {"name": "recurrence_step_1000", "op": "recurrence_step", "B": 1000, "pad": 100, "slots": 1024, "D": 4100,
         "x": "bf16", "g": "fp32"},
        # one decode step of a single user: 32 heads of 128 x 128
        {"name": "delta_step_1", "op": "delta_step", "B": 1, "pad": 0, "slots": 4, "Nk": 16, "Nv": 32, "Dk": 128,
         "Dv": 128, "most": 1, "x": "bf16", "state": "fp32"},
        # one decode step of a full serving batch
        {"name": "delta_step_256", "op": "delta_step", "B": 256, "pad": 3, "slots": 260, "Nk": 16, "Nv": 32, "Dk": 128,
         "Dv": 128, "most": 1, "x": "bf16", "state": "fp32"},
        # drafted tokens taken in at once: 0 to 8 a sequence, bfloat16 states, odd head widths
        {"name": "delta_step_drafts", "op": "delta_step", "B": 48, "pad": 1, "slots": 64, "Nk": 4, "Nv": 8, "Dk": 96,
         "Dv": 80, "most": 8, "x": "bf16", "state": "bf16"},
        # a training step's residual norm on 4 x 8192 tokens
        {"name": "norm_residual_train", "op": "norm", "rows": 32768, "D": 4096, "form": "residual", "x": "bf16",
         "w": "fp32", "backward": True},
        # a training step's gated norm of every head of 8192 tokens
        {"name": "norm_gated_train", "op": "norm", "rows": 262144, "D": 128, "form": "gated", "x": "bf16", "w": "bf16",
         "backward": True},
        # a layer's output for an 8-bit projection: every head of 4 x 8192 tokens, one scale a head
        {"name": "norm_fp8_gated", "op": "norm_fp8", "rows": 1048576, "D": 128, "group": 128, "form": "gated",
         "x": "bf16", "w": "bf16"},
        # a decode step's residual norm for an 8-bit projection, one scale a token
        {"name": "norm_fp8_residual", "op": "norm_fp8", "rows": 65, "D": 2000, "group": 2000, "form": "residual",
         "x": "bf16", "w": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence_step", "delta_step", "norm", "norm_fp8"])
    x = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "recurrence":
        D = _log(rng, 64, 512) * 8 if rng.random() < 0.75 else _log(rng, 33, 4000)
        N = rng.choice([0, 0, _log(rng, 1, 64)])
        B = 1 if N else _log(rng, 1, 8)
        T = _log(rng, 1, min(65536, 50_000_000 // (D * B)))
        return {"op": op, "B": B, "T": max(T, N), "D": D, "N": N, "tail": rng.randrange(min(T, 40)) if N else 0,
                "x": x, "g": rng.choice([x, "fp32"]), "state": rng.random() < 0.5, "backward": rng.random() < 0.6}
    if op == "recurrence_step":
        B = _log(rng, 1, 1024)
        return {"op": op, "B": B, "pad": rng.randrange(B) if rng.random() < 0.3 else 0, "slots": B + _log(rng, 1, 64),
                "D": _log(rng, 16, 1024) * 8 if rng.random() < 0.75 else _log(rng, 33, 8000), "x": x,
                "g": rng.choice([x, "fp32"])}
    if op == "delta_step":
        wide = [64, 96, 128, 128, 256, 72, 50]
        Nk, Dk, Dv = rng.choice([1, 2, 4, 8, 16]), rng.choice(wide), rng.choice(wide)
        Nv = Nk * rng.choice([1, 2, 4])
        B = _log(rng, 1, min(256, 200_000_000 // (Nv * Dk * Dv)))
        return {"op": op, "B": B, "pad": rng.randrange(min(B, 4)), "slots": B + _log(rng, 1, 16), "Nk": Nk,
                "Nv": Nv, "Dk": Dk, "Dv": Dv, "most": rng.choice([1, 1, 1, 4, 9]), "x": x, "state": rng.choice(["fp32", "fp32", "bf16"])}
    D = rng.choice([64, 128, 128, 256, _log(rng, 256, 8192), 8 * _log(rng, 64, 1024)])
    rows = _log(rng, 1, 60_000_000 // D)
    form = rng.choice(["residual", "gated", "plain"])
    if op == "norm":
        return {"op": op, "rows": rows, "D": D, "form": form, "x": x, "w": rng.choice([x, "fp32"]),
                "backward": rng.random() < 0.6}
    return {"op": op, "rows": rows, "D": D, "group": 128 if D % 128 == 0 and rng.random() < 0.5 else D, "form": form,
            "x": x, "w": rng.choice([x, "fp32"])}


def work(c):
    if c["op"] == "recurrence":
        n, e, ge = c["B"] * c["T"] * c["D"], BYTES[c["x"]], BYTES[c["g"]]
        states = 4 * (c["N"] or c["B"]) * c["D"]
        nbytes = n * (2 * e + ge) + states * (1 + c["state"])
        if c["backward"]:  # x, g and the output's gradient in, two gradients out
            nbytes += n * (3 * e + 2 * ge) + states * (1 + 2 * c["state"])
        return {"bytes": nbytes, "flops": n * (3 + 8 * c["backward"])}
    if c["op"] == "recurrence_step":
        live = c["B"] - c["pad"]
        return {"bytes": live * c["D"] * (2 * BYTES[c["x"]] + BYTES[c["g"]] + 8), "flops": 3 * live * c["D"]}
    if c["op"] == "delta_step":
        lens = _lengths(c)
        tokens = sum(lens)
        live = sum(1 for n in lens[: c["B"] - c["pad"]] if n)
        e = BYTES[c["x"]]
        row = 2 * c["Nk"] * c["Dk"] * e + c["Nv"] * (2 * c["Dv"] * e + e + 4)
        head = c["Nv"] * c["Dk"] * c["Dv"]
        return {"bytes": tokens * row + 2 * live * head * BYTES[c["state"]], "flops": 8 * tokens * head}
    n, e = c["rows"] * c["D"], BYTES[c["x"]]
    extra = {"residual": 2 * e, "gated": e, "plain": 0}[c["form"]]
    if c["op"] == "norm_fp8":
        return {"bytes": n * (e + extra + 1) + 4 * n // c["group"], "flops": 8 * n}
    nbytes = n * (2 * e + extra) + c["D"] * BYTES[c["w"]]
    if c["backward"]:
        nbytes += n * (3 * e + {"residual": e, "gated": 2 * e, "plain": 0}[c["form"]]) + 2 * c["D"] * BYTES[c["w"]]
    return {"bytes": nbytes, "flops": n * (6 + 14 * c["backward"])}


# ---- inputs -----------------------------------------------------------------------

def _lengths(c):
    """Tokens of each row of a delta_step: 1, or 0 to `most` in a fixed pattern."""
    if c["most"] == 1:
        return [1] * c["B"]
    return [(5 * i + 3) % (c["most"] + 1) for i in range(c["B"])]


def _bounds(c, gen):
    """cu_seqlens of `N` packed sequences in T - tail tokens, at random places."""
    cuts = torch.randint(0, c["T"] - c["tail"] + 1, (c["N"] - 1,), generator=gen).sort().values
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([c["T"] - c["tail"]])])


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=F32):
        # in pieces, so that the float32 values of a large input need little room
        out = torch.empty(*shape, dtype=dtype, device=dev)
        for piece in out.view(-1).split(1 << 26):
            piece.copy_(torch.randn(piece.numel(), generator=gen, device=dev).mul_(scale))
        return out

    def gates(*shape, dtype=F32):
        out = torch.empty(*shape, dtype=dtype, device=dev)
        for piece in out.view(-1).split(1 << 26):
            piece.copy_(torch.nn.functional.logsigmoid(torch.randn(piece.numel(), generator=gen, device=dev) + 2))
        return out

    def slots(rows, pad, pool):
        idx = torch.randperm(pool, generator=host)[:rows].to(torch.int32)
        if pad:
            idx[rows - pad:] = -1
        return idx.to(dev)

    s = {"case": c}
    if c["op"] == "recurrence":
        B, T, D, X, G = c["B"], c["T"], c["D"], TYPES[c["x"]], TYPES[c["g"]]
        rows = c["N"] or B
        s["x"], s["g"] = randn(B, T, D, scale=0.5, dtype=X), gates(B, T, D, dtype=G)
        s["h0"] = randn(rows, D, scale=0.5) if c["state"] else None
        s["cu"] = _bounds(c, host).to(dev) if c["N"] else None
        if c["backward"]:
            s["do"], s["dht"] = randn(B, T, D, dtype=X), randn(rows, D)
            for name in ("x", "g", "h0"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif c["op"] == "recurrence_step":
        s["x"] = randn(c["B"], c["D"], scale=0.5, dtype=TYPES[c["x"]])
        s["g"] = gates(c["B"], c["D"], dtype=TYPES[c["g"]])
        s["state"] = randn(c["slots"], c["D"])
        s["idx"] = slots(c["B"], c["pad"], c["slots"])
    elif c["op"] == "delta_step":
        X, lens = TYPES[c["x"]], _lengths(c)
        T = sum(lens)
        unit = lambda t: (t / t.norm(dim=-1, keepdim=True)).to(X)  # noqa: E731
        s["q"], s["k"] = unit(randn(T, c["Nk"], c["Dk"])), unit(randn(T, c["Nk"], c["Dk"]))
        s["v"] = randn(T, c["Nv"], c["Dv"], dtype=X)
        s["beta"] = torch.sigmoid(randn(T, c["Nv"])).to(X)
        s["g"] = gates(T, c["Nv"])
        s["state"] = randn(c["slots"], c["Nv"], c["Dv"], c["Dk"], scale=0.1, dtype=TYPES[c["state"]])
        s["idx"] = slots(c["B"], c["pad"], c["slots"])
        s["lens"] = None if c["most"] == 1 else torch.tensor(lens, dtype=torch.int32, device=dev)
    else:
        X, W = TYPES[c["x"]], TYPES[c["w"]]
        n, D = c["rows"], c["D"]
        s["x"] = randn(n, D, dtype=X)
        s["w"] = (1 + 0.1 * randn(D)).to(W)
        s["residual"] = randn(n, D, scale=2.0, dtype=X) if c["form"] == "residual" else None
        s["gate"] = randn(n, D, dtype=X) if c["form"] == "gated" else None
        if c.get("backward"):
            s["dy"] = randn(n, D, dtype=X)
            s["dz"] = randn(n, D, dtype=X) if c["form"] == "residual" else None
            for name in ("x", "w", "residual", "gate"):
                if s[name] is not None:
                    s[name].requires_grad_()
    return s


# ---- one pass ---------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    with torch.no_grad():
        return {"recurrence": _recurrence, "recurrence_step": _recurrence_step, "delta_step": _delta_step,
                "norm": _norm, "norm_fp8": _norm_fp8}[op](s)


def _own(s, op):
    import cann_operator_challenge_august_b200 as cg

    if op == "recurrence":
        o, ht = cg.gated_linear_recurrence(s["x"], s["g"], s["h0"], output_final_state=True, cu_seqlens=s["cu"])
        out = {"o": o, "ht": ht}
        if s["case"]["backward"]:
            leaves = [n for n in ("x", "g", "h0") if s[n] is not None]
            grads = torch.autograd.grad((o, ht), [s[n] for n in leaves], (s["do"], s["dht"]))
            out.update(("d" + n, t) for n, t in zip(leaves, grads))
        return out
    if op == "recurrence_step":
        return {"o": cg.gated_linear_recurrence_step(s["x"], s["g"], s["state"], state_indices=s["idx"]),
                "state": s["state"]}
    if op == "delta_step":
        o = cg.recurrent_gated_delta_rule(s["q"], s["k"], s["v"], s["beta"], s["state"], s["lens"], g=s["g"],
                                          state_indices=s["idx"])
        return {"o": o, "state": s["state"]}
    if op == "norm_fp8":
        got = cg.rms_norm_fp8(s["x"], s["w"], EPS, residual=s["residual"], gate=s["gate"],
                              group_size=s["case"]["group"])
        return dict(zip(("q", "scale", "z"), got))
    y = cg.rms_norm(s["x"], s["w"], EPS, residual=s["residual"], gate=s["gate"])
    y, z = y if s["residual"] is not None else (y, None)
    out = {"y": y} if z is None else {"y": y, "z": z}
    if s["case"]["backward"]:
        leaves = [n for n in ("x", "w", "residual", "gate") if s[n] is not None]
        outs, grads = ((y,), (s["dy"],)) if z is None else ((y, z), (s["dy"], s["dz"]))
        got = torch.autograd.grad(outs, [s[n] for n in leaves], grads)
        out.update(("d" + n, t) for n, t in zip(leaves, got))
    return out


# ---- the plain forms: float32, rounded once at the end ------------------------------

def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t along dim 1, by doubling (a and x are overwritten)."""
    d = 1
    while d < x.shape[1]:
        x[:, d:] += a[:, d:] * x[:, :-d]
        a[:, d:] *= a[:, :-d].clone()
        d *= 2
    return x


def _ends(s):
    """(batch row, first token, last token, sequence) of the sequences that have tokens, on the device."""
    x, cu = s["x"], s["cu"]
    if cu is None:
        b = torch.arange(x.shape[0], device=x.device)
        return b, torch.zeros_like(b), torch.full_like(b, x.shape[1] - 1), b
    n = torch.nonzero(cu[1:] > cu[:-1])[:, 0]
    return torch.zeros_like(n), cu[n], cu[n + 1] - 1, n


def _recurrence(s):
    c, x, a = s["case"], s["x"].float(), s["g"].float().exp()
    B, T, D = x.shape
    row, first, last, seq = _ends(s)
    h0 = s["h0"]
    start = x.new_zeros(c["N"] or B, D) if h0 is None else h0.detach()
    # a sequence's first token has nothing before it but the initial state
    cut, h = a.clone(), x if s["x"].dtype != F32 else x.clone()
    h[row, first] += a[row, first] * start[seq]
    cut[row, first] = 0
    if c["N"]:  # rows behind the last sequence belong to none
        h[:, T - c["tail"]:] = 0
        cut[:, T - c["tail"]:] = 0
    h = _scan(cut, h)
    ht = start.clone()
    ht[seq] = h[row, last]
    out = {"o": h.to(s["x"].dtype), "ht": ht}
    if not c["backward"]:
        return out
    # the gradient of h_t: what comes from o_t, from the final state, and from h_{t+1}
    dh = s["do"].float().clone()
    dh[row, last] += s["dht"][seq]
    back = a.clone()
    back[row, first] = 0
    if c["N"]:
        dh[:, T - c["tail"]:] = 0
    back = torch.cat([back[:, 1:], back.new_zeros(B, 1, D)], dim=1).flip(1)
    dh = _scan(back, dh.flip(1)).flip(1)
    del back
    before = torch.cat([h.new_zeros(B, 1, D), h[:, :-1]], dim=1)
    before[row, first] = start[seq]
    out["dx"] = dh.to(s["x"].dtype)
    out["dg"] = (dh * a * before).to(s["g"].dtype)
    if h0 is not None:
        dh0 = s["dht"].clone()
        dh0[seq] = (dh * a)[row, first]
        out["dh0"] = dh0
    return out


def _recurrence_step(s):
    live = s["idx"] >= 0
    at = s["idx"].clamp(min=0).long()
    h = s["g"].float().exp() * s["state"][at] + s["x"].float()
    o = (h * live[:, None]).to(s["x"].dtype)
    # a padded row has no state: it writes what a live row's slot holds
    pad = torch.where(live, at, at[0])
    s["state"][pad] = torch.where(live[:, None], h, h[0])
    return {"o": o, "state": s["state"]}


def _delta_step(s):
    c, state = s["case"], s["state"]
    B, Nv, rep = c["B"], c["Nv"], c["Nv"] // c["Nk"]
    q, k = (s[n].float().repeat_interleave(rep, dim=1) for n in ("q", "k"))
    v, beta, a = s["v"].float(), s["beta"].float(), s["g"].float().exp()
    lens = torch.ones(B, dtype=torch.int64, device=q.device) if s["lens"] is None else s["lens"].long()
    begin = lens.cumsum(0) - lens
    live = s["idx"] >= 0
    at = torch.where(live, s["idx"], s["idx"][0]).long()
    S = state[at].float()
    o = torch.zeros_like(v)
    for j in range(c["most"]):
        go = (lens > j) & live
        t = torch.where(go, begin + j, 0)
        new = S * a[t][:, :, None, None]
        delta = beta[t][..., None] * (v[t] - (new * k[t][:, :, None, :]).sum(-1))
        new = new + delta[..., None] * k[t][:, :, None, :]
        out = (new * q[t][:, :, None, :]).sum(-1) * c["Dk"] ** -0.5
        o.index_add_(0, t, out * go[:, None, None])
        S = torch.where(go[:, None, None, None], new, S)
    # a padded row has no state: it writes what the first row's slot holds
    state[at] = torch.where(live[:, None, None, None], S, S[0]).to(state.dtype)
    return {"o": o.to(s["v"].dtype), "state": state}


def _normed(s):
    """(stored residual stream, its float32 values, 1 / rms, silu(gate) or 1)"""
    z = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    f = z.float()
    r = (f.square().mean(-1, keepdim=True) + EPS).rsqrt()
    act = 1.0 if s["gate"] is None else s["gate"].float() * torch.sigmoid(s["gate"].float())
    return z, f, r, act


def _norm(s):
    z, f, r, act = _normed(s)
    n, w = f * r, s["w"].float()
    out = {"y": (n * w * act).to(s["x"].dtype)}
    if s["residual"] is not None:
        out["z"] = z
    if s["case"]["backward"]:
        dy = s["dy"].float()
        dn = dy * w * act
        dz = r * (dn - n * (dn * n).mean(-1, keepdim=True))
        if s["residual"] is not None:
            dz = dz + s["dz"].float()
            out["dresidual"] = dz.to(s["x"].dtype)
        out["dx"] = dz.to(s["x"].dtype)
        out["dw"] = (dy * act * n).sum(0).to(s["w"].dtype)
        if s["gate"] is not None:
            sig = torch.sigmoid(s["gate"].float())
            out["dgate"] = (dy * n * w * (sig + act * (1 - sig))).to(s["x"].dtype)
    return out


def _norm_fp8(s):
    z, f, r, act = _normed(s)
    y = (f * r * s["w"].float() * act).view(f.shape[0], -1, s["case"]["group"])
    scale = y.abs().amax(-1).clamp(min=1e-12) / FP8_MAX
    q = (y / scale[..., None]).clamp(-FP8_MAX, FP8_MAX).view(f.shape).to(torch.float8_e4m3fn)
    return {"q": q, "scale": scale} if s["residual"] is None else {"q": q, "scale": scale, "z": z}


# ---- the definitions in float64 -----------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        return {"recurrence": _exact_recurrence, "recurrence_step": _exact_recurrence_step,
                "delta_step": _exact_delta_step, "norm": _exact_norm, "norm_fp8": _exact_norm}[c["op"]](s)


def _exact_recurrence(s):
    """Token by token, forwards and then backwards; a sequence's state is put in place before its first token."""
    c, x = s["case"], s["x"].detach().double()
    a = s["g"].detach().double().exp_()
    B, T, D = x.shape
    init = x.new_zeros(c["N"] or B, D) if s["h0"] is None else s["h0"].detach().double()
    cu = None if s["cu"] is None else s["cu"].tolist()
    final, o = init.clone(), torch.zeros_like(x)
    spans = [(slice(0, B), 0, T, slice(0, B))] if cu is None else [
        (slice(0, 1), cu[n], cu[n + 1], slice(n, n + 1)) for n in range(c["N"]) if cu[n + 1] > cu[n]]
    for b, first, end, n in spans:
        h = init[n]
        for t in range(first, end):
            h = torch.addcmul(x[b, t], a[b, t], h, out=o[b, t])
        final[n] = h
    out = {"o": o, "ht": final}
    if c["backward"]:
        dx, dg, dh0 = torch.zeros_like(x), torch.zeros_like(x), s["dht"].double().clone()
        do = s["do"].double()
        for b, first, end, n in spans:
            dh = dh0[n].clone()
            for t in reversed(range(first, end)):
                dh = torch.add(dh, do[b, t], out=dx[b, t]).clone()
                dh.mul_(a[b, t])
                torch.mul(dh, o[b, t - 1] if t > first else init[n], out=dg[b, t])
            dh0[n] = dh
        out.update({"dx": dx, "dg": dg})
        if s["h0"] is not None:
            out["dh0"] = dh0
    return out


def _exact_recurrence_step(s):
    state, o = s["state"].double(), torch.zeros_like(s["x"], dtype=F64)
    for b, slot in enumerate(s["idx"].tolist()):
        if slot >= 0:
            state[slot] = torch.exp(s["g"][b].double()) * state[slot] + s["x"][b].double()
            o[b] = state[slot]
    return {"o": o, "state": state}


def _exact_delta_step(s):
    c, state = s["case"], s["state"].double()
    o = torch.zeros_like(s["v"], dtype=F64)
    t, heads = 0, [j // (c["Nv"] // c["Nk"]) for j in range(c["Nv"])]
    for slot, n in zip(s["idx"].tolist(), _lengths(c)):
        for _ in range(n):
            if slot >= 0:
                k, q = s["k"][t, heads].double(), s["q"][t, heads].double()
                S = state[slot] * torch.exp(s["g"][t].double())[:, None, None]
                err = s["v"][t].double() - torch.einsum("hvk,hk->hv", S, k)
                S = S + torch.einsum("hv,hk->hvk", s["beta"][t].double()[:, None] * err, k)
                state[slot] = S
                o[t] = torch.einsum("hvk,hk->hv", S, q) / math.sqrt(c["Dk"])
            t += 1
    return {"o": o, "state": state}


def _exact_norm(s):
    c, x, w = s["case"], s["x"].detach().double(), s["w"].detach().double()
    z = x if s["residual"] is None else (x + s["residual"].detach().double()).to(s["x"].dtype).double()
    inv = 1 / torch.sqrt((z * z).sum(-1, keepdim=True) / c["D"] + EPS)
    g = None if s["gate"] is None else s["gate"].detach().double()
    silu = 1 if g is None else g / (1 + torch.exp(-g))
    y = z * inv * w * silu
    if c["op"] == "norm_fp8":
        per = y.reshape(c["rows"], c["D"] // c["group"], c["group"])
        scale = per.abs().amax(2).clamp(min=1e-12) / FP8_MAX
        out = {"q": (per / scale.unsqueeze(2)).reshape(y.shape), "scale": scale}
    else:
        out = {"y": y}
    if s["residual"] is not None:
        out["z"] = z
    if c.get("backward"):
        dy = s["dy"].double()
        up = dy * w * silu
        dz = inv * up - z * inv ** 3 * (up * z).sum(-1, keepdim=True) / c["D"]
        if s["residual"] is not None:
            dz = dz + s["dz"].double()
            out["dresidual"] = dz
        out["dx"], out["dw"] = dz, (dy * silu * z * inv).sum(0)
        if g is not None:
            sg = 1 / (1 + torch.exp(-g))
            out["dgate"] = dy * z * inv * w * sg * (1 + g * (1 - sg))
    return out
