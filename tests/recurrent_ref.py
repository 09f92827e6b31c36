"""Error bounds of the recurrent block's kernels against the float64 oracle.

u = 2^-24 is half an fp32 step, so one rounded operation is off by at most u of its result.
Every bound below adds up, per output, what each rounded operation contributes, with the
magnitudes that the float64 oracle gives; an output in bf16 adds half a bf16 step of its value.

Elementary functions, as CUDA documents them: expf 1 ulp, fp32 divide and square root
correctly rounded, rsqrtf 2 ulp; __expf(x) 2 + 1.173 |x| ulp, __fdividef 2 ulp. An ulp is up
to 2 u of the value.
"""
import numpy as np
import torch

from oracle import ops as orc

U = 2.0 ** -24


def rounded(err, ref, dtype):
    """The bound of a value off by err before it is rounded to the output type: half a step of
    that value, which is |ref| + err at most."""
    return err + (np.abs(ref) + err) * (torch.finfo(dtype).eps / 2)


def assert_within(got, ref, bound, what):
    got = got.detach().double().cpu().numpy()
    assert got.shape == ref.shape, f"{what}: shape {got.shape} != {ref.shape}"
    assert np.isfinite(got).all() or not np.isfinite(ref).all(), f"{what}: not finite"
    err = np.abs(got - ref)
    bad = err > bound + 1e-30
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} outside the bound, worst error "
                           f"{err[bad].max():.3e} at bound {np.broadcast_to(bound, err.shape)[bad][err[bad].argmax()]:.3e}")


def sigmoid_rel(x, dtype):
    """Relative error of sigmoid(x) = 1 / (1 + e^-x): the exponential's, times 1 - s <= 1 of
    it that reaches the sum, the sum's and the reciprocal's (rcp.approx: 1 ulp)."""
    x = np.abs(orc._f64(x))
    x = np.where(np.isfinite(x), x, 0.0)  # sigmoid(+-inf) is exact; NaN stands only where it is not used
    if dtype == torch.bfloat16:
        return (2 * (2 + 1.173 * x) + 1 + 4) * U
    return np.full(x.shape, 2 + 1 + 2) * U


def p_floor(dtype):
    """The bf16 kernels' sigmoid(i) does not fall below 2^-62."""
    return 2.0 ** -62 if dtype == torch.bfloat16 else 0.0


def scan_errors(x, r, i, decay, h0, dtype, bwd=False):
    """Relative errors of a_t and of the injected term, and the bound E_t on |h_t's error|.

    L = decay s carries s's error and a rounding; a = e^-L turns L's relative error into L
    times as much and adds the exponential's (its reduction k ln 2 + f rounds at L u, its
    polynomial and sum at 2 u; 2 (2 + 1.173 L) u covers both). The products of a over a run of
    tokens that the scan forms instead of single steps round once a token: u.
    m^2 = -t (2 + t), t = a - 1 to a relative (1.3e-8 = 0.3 u) + 4 u: 10 u; m has half of that,
    half of L's error times L a^2 / m^2 <= 1/2, and the root's 4 u (as m^2 rsqrt(m^2): 4 + 1 u).
    Then the products with p and x: 2 u, and p's own error.
    E_t = a_t E_{t-1} + da a_t |h|_{t-1} + db |b_t| + 2 u (...), |h| the recurrence of the
    magnitudes; twice that covers the products of errors. The bf16 kernels keep e^-i under 2^62, so
    p is off by an absolute 2^-62 below that (1e-12 of a rounding step of a state of size x).
    The backward kernels keep t and take a as 1 + t, which adds an absolute u to a.
    """
    s, L, a, p, m, xv = orc.scan_gates(x, r, i, decay)
    dL = sigmoid_rel(r, dtype) + U
    da = dL * L + 2 * (2 + 1.173 * L) * U + U
    if bwd:
        da = da + U / np.maximum(a, 1e-37)
    db = (12 + 5 + 2) * U + dL + sigmoid_rel(i, dtype)
    b = np.abs(m * p * xv)
    flush = p_floor(dtype) * np.abs(m * xv)
    B, T, D = b.shape
    H = np.zeros((B, D)) if h0 is None else np.abs(orc._f64(h0))
    E = np.zeros((B, D))
    Es, Hs = np.zeros((B, T, D)), np.zeros((B, T, D))
    for t in range(T):
        E = a[:, t] * E + da[:, t] * a[:, t] * H + db[:, t] * b[:, t] + flush[:, t]
        H = a[:, t] * H + b[:, t]
        E = E + 2 * U * H
        Es[:, t], Hs[:, t] = 2 * E, H
    return dict(s=s, L=L, a=a, p=p, m=m, x=xv, da=da, db=db, dL=dL, E=Es, H=Hs)


def scan_bwd_bounds(x, r, i, decay, h0, dy, dfinal, dtype):
    """The oracle's gradients and their bounds. dh has the recurrence of magnitudes of h with dy in
    place of b; the rest is the product rule over the factors of each gradient, 1 - s and 1 - p
    being off by an absolute 8 u at most."""
    e = scan_errors(x, r, i, decay, h0, dtype, bwd=True)
    s, L, a, p, m, xv = (e[k] for k in ("s", "L", "a", "p", "m", "x"))
    ref = orc.gated_scan_bwd(x, r, i, decay, h0, dy, dfinal)
    B, T, D = s.shape
    dyv = np.abs(orc._f64(dy))
    G = np.zeros((B, D)) if dfinal is None else np.abs(orc._f64(dfinal))  # magnitude of a dh from behind
    Eg = np.zeros((B, D))
    dh, Edh = np.zeros((B, T, D)), np.zeros((B, T, D))
    for t in range(T - 1, -1, -1):
        dh[:, t] = dyv[:, t] + G
        Edh[:, t] = Eg + 2 * U * dh[:, t]
        G = a[:, t] * dh[:, t]
        Eg = a[:, t] * Edh[:, t] + (e["da"][:, t] + 2 * U) * G
    Edh = 2 * Edh
    first = np.zeros((B, 1, D)) if h0 is None else orc._f64(h0)[:, None]
    H = np.concatenate([np.abs(first), e["H"][:, :-1]], 1)
    EH = np.concatenate([np.zeros((B, 1, D)), e["E"][:, :-1]], 1)
    im = np.where(L == 0, 0.0, 1.0 / np.where(L == 0, 1.0, m))
    q = a * a * im * p * np.abs(xv)
    Eq = q * (2 * e["da"] + e["db"] + 8 * U)
    EaH = a * EH + a * H * (e["da"] + 2 * U)
    dL = dh * (q + a * H)
    EdL = Edh * (q + a * H) + dh * (Eq + EaH) + 4 * U * dL
    f = np.abs(m * p)
    b_dx = Edh * f + dh * f * (e["db"] + 4 * U)
    b_di = (Edh * f + dh * f * (e["db"] + 4 * U)) * np.abs(xv) * (1 - p) + 8 * U * dh * f * np.abs(xv)
    b_dr = EdL * L * (1 - s) + dL * L * ((1 - s) * (e["dL"] + 4 * U) + 8 * U)
    n = B * T
    pf = p_floor(dtype) * dh
    b_dx, b_di, b_dr = b_dx + pf * m, b_di + pf * m * np.abs(xv), b_dr + pf * a * a * im * np.abs(xv) * L
    flushed = (pf * a * a * im * np.abs(xv) * s).sum((0, 1))
    b_dd = flushed + (EdL * s + dL * s * (e["dL"] + 4 * U)).sum((0, 1)) + min(n, 4096) * U * (dL * s).sum((0, 1))
    bounds = [rounded(b_dx, ref[0], dtype), rounded(b_dr, ref[1], dtype), rounded(b_di, ref[2], dtype), b_dd,
              2 * Eg + 2 * U * G]
    return ref, bounds
