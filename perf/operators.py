"""The recurrent block's operators as a user calls them: cases, inputs, plain forms and exact values.

Six entry points of ``theorem_b200.ops``, all channel-last:

* ``gated_scan``            h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t,
                            a_t = exp(-decay sigmoid(r_t)), per channel
* ``gated_scan_bwd``        its gradients
* ``group_norm``            per-token norm of groups of channels, with SiLU or a SiLU gate
* ``group_norm_bwd``        its gradients
* ``causal_conv1d_step``    the depthwise causal conv continued from a carried state
* ``causal_conv1d_bwd``     its gradients

``run`` takes the plain forms (elementary torch operations in 32 bits, sums over all tokens in 64)
unless ``own`` is true; ``exact`` evaluates the definitions in 64 bits, token by token.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One decoded token for 64 sequences: the state moves on by a step; latency counts.
        dict(name="scan_token", op="scan", B=64, T=1, D=2048, dtype="bf16", packed=0, states=False, sliced=True),
        # The forward pass of a training batch, its chunk states kept for the backward pass.
        dict(name="scan_train", op="scan", B=16, T=8192, D=2048, dtype="bf16", packed=0, states=True, sliced=True),
        # Prefill of one long sequence: few channels, so the work has to be split along time.
        dict(name="scan_long", op="scan", B=1, T=131072, D=2048, dtype="bf16", packed=0, states=False, sliced=False),
        # Prompts of many lengths packed into one row range, fp32, a width that is no power of two.
        dict(name="scan_packed", op="scan", B=1, T=20011, D=1000, dtype="f32", packed=37, states=False, sliced=False),
        # The backward pass of a training batch.
        dict(name="scan_bwd_train", op="scan_bwd", B=8, T=4096, D=2048, dtype="bf16", packed=0, sliced=True),
        # The backward pass over long documents packed into one row range.
        dict(name="scan_bwd_packed", op="scan_bwd", B=1, T=65537, D=2048, dtype="bf16", packed=5, sliced=False),
        # Per-head RMS norm with a SiLU gate on one decoded token of 64 sequences.
        dict(name="norm_token", op="norm", R=64, C=2048, G=128, dtype="bf16", center=False, gate=True, act=True),
        # The same on a layer's whole output.
        dict(name="norm_heads", op="norm", R=131072, C=2048, G=128, dtype="bf16", center=False, gate=True, act=True),
        # Its backward pass in training.
        dict(name="norm_bwd_heads", op="norm_bwd", R=32768, C=2048, G=128, dtype="bf16", center=False, gate=True,
             act=True),
        # Mean and variance over odd groups, SiLU after it, fp32: no power of two anywhere.
        dict(name="norm_bwd_odd", op="norm_bwd", R=7777, C=1960, G=49, dtype="f32", center=True, gate=False, act=True),
        # The conv's one decoded token for 64 sequences.
        dict(name="conv_token", op="conv_step", B=64, S=1, D=2048, W=4, dtype="bf16", act=True),
        # The conv's backward pass in training.
        dict(name="conv_bwd_train", op="conv_bwd", B=8, S=8192, D=2048, W=4, dtype="bf16", act=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Channels: mostly whole vectors, sometimes odd."""
    d = _log(rng, lo, hi)
    return d if rng.random() < 0.25 else max(8, d // 8 * 8)


def draw(rng):
    op = rng.choice(["scan", "scan", "scan_bwd", "scan_bwd", "norm", "norm_bwd", "conv_step", "conv_bwd"])
    dt = rng.choice(["bf16", "bf16", "f32"])
    half = 2 if dt == "f32" else 1
    if op in ("scan", "scan_bwd"):
        D = _width(rng, 24, 4096)
        most = (1 << 27 if op == "scan" else 1 << 26) // half // D
        packed = rng.choice([0, 0, _log(rng, 1, 100)])
        rows = _log(rng, 1, min(most, 131072))
        if packed:
            c = dict(op=op, B=1, T=rows, D=D, dtype=dt, packed=packed)
        else:
            B = _log(rng, 1, min(64, rows))
            c = dict(op=op, B=B, T=max(1, rows // B), D=D, dtype=dt, packed=0)
        c["sliced"] = rng.random() < 0.5
        if op == "scan":
            c["states"] = rng.random() < 0.5
        return c
    if op in ("norm", "norm_bwd"):
        G = rng.choice([16, 32, 64, 128, 256, _log(rng, 8, 4096)])
        groups = _log(rng, 1, max(1, 4096 // G))
        R = _log(rng, 1, min(131072, (1 << 27 if op == "norm" else 1 << 26) // half // (G * groups)))
        return dict(op=op, R=R, C=G * groups, G=G, dtype=dt, center=rng.random() < 0.5, gate=rng.random() < 0.5,
                    act=rng.random() < 0.7)
    D = _width(rng, 24, 4096)
    W = rng.choice([2, 3, 4, 4, 4])
    if op == "conv_step":
        return dict(op=op, B=_log(rng, 1, 512), S=_log(rng, 1, 32), D=D, W=W, dtype=dt, act=rng.random() < 0.5)
    rows = _log(rng, 1, min(131072, (1 << 27) // half // D))
    B = _log(rng, 1, min(64, rows))
    return dict(op=op, B=B, S=max(1, rows // B), D=D, W=W, dtype=dt, act=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    t = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    return t.mul_(scale) if scale != 1.0 else t


def _offsets(case, seed):
    """Row offsets of the packed sequences: ragged lengths, some empty, and a few rows behind the last."""
    n, total = case["packed"], case["T"]
    c = torch.Generator().manual_seed(int(seed) * 7919 + 17)
    cuts = torch.randint(0, total + 1, (n,), generator=c).tolist()
    cuts[-1] = total - min(total // 50, 100)
    return [0] + sorted(min(v, cuts[-1]) for v in cuts)


def prepare(case, seed):
    g = _gen(seed)
    dt = _DT[case["dtype"]]
    s = dict(case)
    if case["op"] in ("scan", "scan_bwd"):
        B, T, D = case["B"], case["T"], case["D"]
        s["x"] = _randn(g, B, T, D, dtype=dt)
        if case["sliced"]:  # both gates out of one projection
            both = _randn(g, B, T, 2 * D, dtype=dt)
            s["r"], s["i"] = both[..., :D], both[..., D:]
        else:
            s["r"], s["i"] = _randn(g, B, T, D, dtype=dt), _randn(g, B, T, D, dtype=dt)
        # Memory of about 2 to 250 tokens at an open half of the gate.
        s["decay"] = torch.exp(torch.rand(D, generator=g, device="cuda") * 4.6 - 4.8)
        n = case["packed"] or B
        s["h0"] = _randn(g, n, D)
        off = _offsets(case, seed) if case["packed"] else None
        s["off"] = off
        s["cu"] = torch.tensor(off, dtype=torch.int32, device="cuda") if off else None
        if case["op"] == "scan_bwd":
            s["dy"] = _randn(g, B, T, D, dtype=dt)
            s["dfinal"] = _randn(g, n, D)
            if own:  # the states that the forward pass kept
                from theorem_b200 import ops
                s["states"] = ops.gated_scan(s["x"], s["r"], s["i"], s["decay"], h0=s["h0"], cu_seqlens=s["cu"],
                                             want_states=True)[2]
    elif case["op"] in ("norm", "norm_bwd"):
        R, C = case["R"], case["C"]
        s["x"] = _randn(g, R, C, dtype=dt)
        s["z"] = _randn(g, R, C, dtype=dt) if case["gate"] else None
        s["w"] = 1.0 + _randn(g, C, scale=0.1)
        s["b"] = _randn(g, C, scale=0.1) if case["center"] else None
        if case["op"] == "norm_bwd":
            s["dy"] = _randn(g, R, C, dtype=dt)
    else:
        B, S, D, W = case["B"], case["S"], case["D"], case["W"]
        s["x"] = _randn(g, B, S, D, dtype=dt)
        s["w"] = _randn(g, D, W, scale=0.5)
        s["b"] = _randn(g, D, scale=0.3)
        if case["op"] == "conv_step":
            s["state"] = _randn(g, B, W - 1, D, dtype=dt)
        else:
            s["dy"] = _randn(g, B, S, D, dtype=dt)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"scan": _scan, "scan_bwd": _scan_bwd, "norm": _norm, "norm_bwd": _norm_bwd, "conv_step": _conv_step,
            "conv_bwd": _conv_bwd}[s["op"]](s)


def _run_own(s):
    from theorem_b200 import ops
    op = s["op"]
    act = "silu" if s.get("act") else None
    if op == "scan":
        y, final, states = ops.gated_scan(s["x"], s["r"], s["i"], s["decay"], h0=s["h0"], cu_seqlens=s["cu"],
                                          want_states=s["states"])
        if not s["states"]:
            return y, final
        return y, final, states
    if op == "scan_bwd":
        return ops.gated_scan_bwd(s["x"], s["r"], s["i"], s["decay"], s["states"], s["dy"], dfinal=s["dfinal"],
                                  cu_seqlens=s["cu"])
    if op == "norm":
        return ops.group_norm(s["x"], s["G"], s["w"], s["b"], gate=s["z"], activation=act, center=s["center"], eps=EPS)
    if op == "norm_bwd":
        out = ops.group_norm_bwd(s["x"], s["dy"], s["G"], s["w"], s["b"], gate=s["z"], activation=act,
                                 center=s["center"], eps=EPS)
        return tuple(t for t in out if t is not None)
    if op == "conv_step":
        return ops.causal_conv1d_step(s["x"], s["state"], s["w"], s["b"], activation=act)
    return ops.causal_conv1d_bwd(s["x"], s["w"], s["b"], s["dy"], activation=act)


def _sequences(s):
    """(batch entries, their rows of h0, first row, length): a dense batch's sequences at once, packed ones singly."""
    if s["off"] is None:
        return [(slice(0, s["B"]), slice(0, s["B"]), 0, s["T"])]
    return [(slice(0, 1), slice(n, n + 1), a, e - a) for n, (a, e) in enumerate(zip(s["off"], s["off"][1:]))]


def _doubling(a, b):
    """All h_t = a_t h_{t-1} + b_t along axis 1, by doubling the span that each row has summed up; a, b are used up."""
    T, k = a.shape[1], 1
    while k < T:
        b[:, k:] = a[:, k:] * b[:, :-k] + b[:, k:]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return b


def _gates(s):
    sr = torch.sigmoid(s["r"].float())
    L = sr * s["decay"]
    a = torch.exp(-L)
    p = torch.sigmoid(s["i"].float())
    m = torch.sqrt(-torch.expm1(-2.0 * L))
    return sr, L, a, p, m


def _states_of(s):
    """a_t, h_t of every row; rows that no sequence holds have h = 0."""
    _, _, a, p, m = _gates(s)
    b = m * p * s["x"].float()
    del p, m
    aa = a.clone()
    for e, n, lo, ln in _sequences(s):
        if ln:
            b[e, lo] = aa[e, lo] * s["h0"][n] + b[e, lo]
            aa[e, lo] = 0.0
    if s["off"] is not None:
        b[:, s["off"][-1]:] = 0.0
        aa[:, s["off"][-1]:] = 0.0
    return a, _doubling(aa, b)


def _finals(s, h):
    return torch.cat([(h[e, lo + ln - 1] if ln else s["h0"][n].to(h.dtype)) for e, n, lo, ln in _sequences(s)])


def _chunk_states(s, h):
    """The state that enters each 64-row chunk of each sequence, [B, ceil(T/64), D]."""
    first = torch.cat([s["h0"].to(h.dtype)[:, None], h[:, 63:-1:64]], 1) if s["T"] > 64 else s["h0"].to(h.dtype)[:, None]
    return first[:, :(s["T"] + 63) // 64].contiguous()


def _scan(s):
    _, h = _states_of(s)
    final = _finals(s, h)
    y = h.to(s["x"].dtype)
    if not s["states"]:
        return y, final
    if s["packed"]:
        return y, final, _packed_states(s, h)
    return y, final, _chunk_states(s, h)


def _packed_states(s, h):
    """Packed: sequence n's chunks stand from slot offset[n] // 64 + n on; the other slots are 0."""
    st = torch.zeros(1, s["T"] // 64 + s["packed"], s["D"], device=h.device, dtype=h.dtype)
    for k, (e, n, lo, ln) in enumerate(_sequences(s)):
        if ln:
            at = lo // 64 + k
            st[:, at] = s["h0"][n]
            st[:, at + 1:at + (ln + 63) // 64] = h[:, lo + 63:lo + ln - 1:64]
    return st


def _before(s, h):
    """h_{t-1} of every row."""
    prev = torch.empty_like(h)
    prev[:, 1:] = h[:, :-1]
    prev[:, 0] = 0.0
    for e, n, lo, ln in _sequences(s):
        if ln:
            prev[e, lo] = s["h0"][n]
    return prev


def _scan_bwd(s):
    a, h = _states_of(s)
    prev = _before(s, h)
    del h
    # dh_t = dy_t + a_{t+1} dh_{t+1}, from the back.
    d = s["dy"].float()
    nxt = torch.zeros_like(a)
    nxt[:, :-1] = a[:, 1:]
    dh0 = torch.empty_like(s["h0"])
    for e, n, lo, ln in _sequences(s):
        if ln:
            d[e, lo + ln - 1] += s["dfinal"][n]
            nxt[e, lo + ln - 1] = 0.0
    if s["off"] is not None:
        d[:, s["off"][-1]:] = 0.0
        nxt[:, s["off"][-1]:] = 0.0
    dh = _doubling(nxt.flip(1), d.flip(1)).flip(1)
    del nxt, d
    for e, n, lo, ln in _sequences(s):
        dh0[n] = a[e, lo] * dh[e, lo] if ln else s["dfinal"][n]
    sr, L, a, p, m = _gates(s)
    x = s["x"].float()
    dx = dh * m * p
    di = dh * m * x * p * (1.0 - p)
    dL = dh * (a * a / m * p * x - a * prev)
    dr = dL * L * (1.0 - sr)
    ddecay = (dL * sr).sum((0, 1), dtype=torch.float64).float()
    dt = s["x"].dtype
    return dx.to(dt), dr.to(dt), di.to(dt), ddecay, dh0


def _norm_parts(s):
    R, C, G = s["R"], s["C"], s["G"]
    xg = s["x"].float().reshape(R, C // G, G)
    if s["center"]:
        xg = xg - xg.mean(-1, keepdim=True)
    rs = torch.rsqrt((xg * xg).mean(-1, keepdim=True) + EPS)
    return xg * rs, rs


def _norm(s):
    xh, _ = _norm_parts(s)
    u = xh.reshape(s["R"], s["C"]) * s["w"]
    if s["b"] is not None:
        u = u + s["b"]
    if s["z"] is not None:
        z = s["z"].float()
        u = u * (z * torch.sigmoid(z) if s["act"] else z)
    elif s["act"]:
        u = u * torch.sigmoid(u)
    return u.to(s["x"].dtype)


def _norm_bwd(s):
    R, C, G = s["R"], s["C"], s["G"]
    xh3, rs = _norm_parts(s)
    xh = xh3.reshape(R, C)
    u = xh * s["w"]
    if s["b"] is not None:
        u = u + s["b"]
    dy = s["dy"].float()
    out = []
    if s["z"] is not None:
        z = s["z"].float()
        sg = torch.sigmoid(z)
        du = dy * (z * sg if s["act"] else z)
        dz = dy * u * (sg * (1.0 + z * (1.0 - sg)) if s["act"] else 1.0)
        out.append(dz.to(s["x"].dtype))
    elif s["act"]:
        sg = torch.sigmoid(u)
        du = dy * sg * (1.0 + u * (1.0 - sg))
    else:
        du = dy
    dw = (du * xh).sum(0, dtype=torch.float64).float()
    dxh = (du * s["w"]).reshape(R, C // G, G)
    dx = dxh - xh3 * (dxh * xh3).mean(-1, keepdim=True)
    if s["center"]:
        dx = dx - dxh.mean(-1, keepdim=True)
    out.insert(0, (dx * rs).reshape(R, C).to(s["x"].dtype))
    out.append(dw)
    if s["b"] is not None:
        out.append(du.sum(0, dtype=torch.float64).float())
    return tuple(out)


def _taps(xp, w, b, S):
    """bias + sum_k w[:, k] xp[:, t + k], xp with its W - 1 rows before the first token."""
    u = b.expand(xp.shape[0], S, -1).clone()
    for k in range(w.shape[1]):
        u += w[:, k] * xp[:, k:k + S]
    return u


def _conv_step(s):
    xp = torch.cat([s["state"], s["x"]], 1)
    u = _taps(xp.float(), s["w"], s["b"], s["S"])
    if s["act"]:
        u = u * torch.sigmoid(u)
    return u.to(s["x"].dtype), xp[:, s["S"]:].contiguous()


def _conv_bwd(s):
    S, W = s["S"], s["W"]
    x = s["x"].float()
    xp = torch.cat([x.new_zeros(x.shape[0], W - 1, x.shape[2]), x], 1)
    du = s["dy"].float()
    if s["act"]:
        u = _taps(xp, s["w"], s["b"], S)
        sg = torch.sigmoid(u)
        du = du * sg * (1.0 + u * (1.0 - sg))
        del u, sg
    dx = torch.zeros_like(x)
    dw = []
    for k in range(W):
        lag = W - 1 - k
        if lag < S:
            dx[:, :S - lag] += s["w"][:, k] * du[:, lag:]
        dw.append((du * xp[:, k:k + S]).sum((0, 1), dtype=torch.float64).float())
    return dx.to(s["x"].dtype), torch.stack(dw, 1), du.sum((0, 1), dtype=torch.float64).float()


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op in ("scan", "scan_bwd"):
        n = case["B"] * case["T"] * case["D"]
        seqs = case["packed"] or case["B"]
        st = 4 * case["D"] * (case["T"] // 64 + seqs if case["packed"] else seqs * ((case["T"] + 63) // 64))
        ends = 8 * seqs * case["D"] + 4 * case["D"]
        if op == "scan":  # x, r, i in, y out; h0 in, final out
            return {"bytes": 4 * e * n + ends + (st if case["states"] else 0), "flops": 20 * n}
        # x, r, i, dy in, dx, dr, di out; states, dfinal in, dh0 and ddecay out
        return {"bytes": 7 * e * n + ends + st + 4 * case["D"], "flops": 50 * n}
    if op in ("norm", "norm_bwd"):
        n = case["R"] * case["C"]
        par = 4 * case["C"] * (2 if case["center"] else 1)
        if op == "norm":
            return {"bytes": (3 if case["gate"] else 2) * e * n + par, "flops": 12 * n}
        return {"bytes": (5 if case["gate"] else 3) * e * n + 2 * par, "flops": 25 * n}
    n = case["B"] * case["S"] * case["D"]
    par = 4 * case["D"] * (case["W"] + 1)
    if op == "conv_step":
        return {"bytes": 2 * e * n + 2 * e * case["B"] * (case["W"] - 1) * case["D"] + par,
                "flops": (2 * case["W"] + 6) * n}
    return {"bytes": 3 * e * n + 2 * par, "flops": (6 * case["W"] + 10) * n}


# ---------------------------------------------------------------------------
# exact values: the definitions in 64 bits, token by token
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "scan_bwd": _exact_scan_bwd, "norm": _exact_norm, "norm_bwd": _exact_norm_bwd,
            "conv_step": _exact_conv_step, "conv_bwd": _exact_conv_bwd}[case["op"]](s)


def _exact_gates(s):
    f = torch.float64
    sr = 1.0 / (1.0 + torch.exp(-s["r"].to(f)))
    loga = -(s["decay"].to(f) * sr)
    inject = torch.sqrt(-torch.expm1(loga + loga)) / (1.0 + torch.exp(-s["i"].to(f)))
    return sr, loga, inject


def _exact_walk(s):
    """h_t of every row (0 where no sequence is), walked forward one token at a time."""
    _, loga, inject = _exact_gates(s)
    a = loga.exp_()
    h = inject.mul_(s["x"].to(torch.float64))
    if s["off"] is not None:
        h[:, s["off"][-1]:] = 0.0
    for eb, en, lo, ln in _sequences(s):
        prev = s["h0"][en].to(torch.float64)
        rows_h, rows_a = h[eb].unbind(1), a[eb].unbind(1)
        for t in range(lo, lo + ln):
            rows_h[t].addcmul_(rows_a[t], prev)
            prev = rows_h[t]
    return a, h


def _exact_scan(s):
    _, h = _exact_walk(s)
    out = (h, _finals(s, h))
    if s["states"]:
        out += ((_packed_states(s, h) if s["packed"] else _chunk_states(s, h)),)
    return out


def _exact_scan_bwd(s):
    f = torch.float64
    a, h = _exact_walk(s)
    dh = s["dy"].to(f)
    if s["off"] is not None:
        dh[:, s["off"][-1]:] = 0.0
    dh0 = s["dfinal"].to(f).clone()
    for eb, en, lo, ln in _sequences(s):
        carry = dh0[en]
        rows_d, rows_a = dh[eb].unbind(1), a[eb].unbind(1)
        for t in range(lo + ln - 1, lo - 1, -1):
            rows_d[t].add_(carry)
            carry = rows_a[t] * rows_d[t]
        dh0[en] = carry
    prev = _before(dict(s, h0=s["h0"].to(f)), h)
    del h
    da = dh * prev
    del prev
    sr, loga, inject = _exact_gates(s)
    x, p = s["x"].to(f), 1.0 / (1.0 + torch.exp(-s["i"].to(f)))
    dx = dh * inject
    di = dx * x * (1.0 - p)
    # inject = p sqrt(1 - a^2): d inject / d a = -a p / sqrt(1 - a^2) = -a p^2 / inject.
    da -= dh * x * a * p * p / inject
    dloga = da * a
    ddecay = -(dloga * sr).sum((0, 1))
    dr = dloga * loga * (1.0 - sr)
    return dx, dr, di, ddecay, dh0


def _exact_norm_of(s, x, w, b, z):
    g = x.unflatten(-1, (s["C"] // s["G"], s["G"]))
    if s["center"]:
        v, mu = torch.var_mean(g, -1, correction=0, keepdim=True)
        g = (g - mu) / torch.sqrt(v + EPS)
    else:
        g = g / torch.sqrt(g.square().mean(-1, keepdim=True) + EPS)
    u = g.flatten(-2) * w
    if b is not None:
        u = u + b
    if z is not None:
        return u * (z / (1.0 + torch.exp(-z)) if s["act"] else z)
    return u / (1.0 + torch.exp(-u)) if s["act"] else u


def _exact_norm(s):
    f = torch.float64
    return _exact_norm_of(s, s["x"].to(f), s["w"].to(f), None if s["b"] is None else s["b"].to(f),
                          None if s["z"] is None else s["z"].to(f))


def _exact_norm_bwd(s):
    f = torch.float64
    x, z, w, b = [None if s[k] is None else s[k].to(f).requires_grad_() for k in ("x", "z", "w", "b")]
    y = _exact_norm_of(s, x, w, b, z)
    return torch.autograd.grad(y, [t for t in (x, z, w, b) if t is not None], s["dy"].to(f))


def _exact_conv_of(x, before, w, b, act):
    xp = torch.cat([before, x], 1)
    S = x.shape[1]
    u = b + sum(xp[:, k:k + S] * w[:, k] for k in range(w.shape[1]))
    return u / (1.0 + torch.exp(-u)) if act else u


def _exact_conv_step(s):
    f = torch.float64
    y = _exact_conv_of(s["x"].to(f), s["state"].to(f), s["w"].to(f), s["b"].to(f), s["act"])
    return y, torch.cat([s["state"], s["x"]], 1)[:, s["S"]:].to(f)


def _exact_conv_bwd(s):
    f = torch.float64
    x, w, b = (s[k].to(f).requires_grad_() for k in ("x", "w", "b"))
    before = torch.zeros(s["B"], s["W"] - 1, s["D"], dtype=f, device=x.device)
    return torch.autograd.grad(_exact_conv_of(x, before, w, b, s["act"]), [x, w, b], s["dy"].to(f))
