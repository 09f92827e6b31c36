"""numpy (float64) restatement of the reference's hot-path ops -- TEST INFRASTRUCTURE.

Every function cites the reference file:line it restates (paths are relative
to the yhinai/Theorem checkout). Inputs may be numpy arrays or torch CPU
tensors of any float dtype; everything is computed in float64 and returned as
float64 numpy arrays. Callers that compare against bf16 kernels pass the
bf16-rounded inputs, so the oracle sees exactly what the kernel saw.

Layouts follow the reference:
    conv   x [B, D, S] (``layout="bds"``) or channel-last x [B, S, D] (``"bsd"``)
    q,k    [B, T, H, K];  v, u, w-like [B, T, H, V|K];  beta, g [B, T, H]
    A      [B, T, H, BT]  (row t of the chunk's 64x64 matrix at position t)
    h      [B, NT, H, K, V]
"""
from __future__ import annotations

import numpy as np

BT = 64  # chunk length (kernels/recompute_w_u/reference.py:31, chunk_fwd_h/reference.py:13)


def _f64(x):
    if x is None:
        return None
    if hasattr(x, "detach"):  # torch tensor
        x = x.detach().to("cpu").float().numpy()
    return np.asarray(x, dtype=np.float64)


# --------------------------------------------------------------------------
# causal_conv1d
# --------------------------------------------------------------------------
def silu(x):
    x = _f64(x)
    return x / (1.0 + np.exp(-x))


def causal_conv1d(x, weight, bias, activation: str | None = None, layout: str = "bds"):
    """Depthwise causal conv, zero left-pad of W-1.

    out[b,d,t] = bias[d] + sum_k weight[d,k] * x[b,d,t-W+1+k]
    Restates kernels/causal_conv1d/reference.py:55-81 (F.pad + grouped
    F.conv1d) in the per-tap form of scripts/cpu_reference.py:40-63.
    ``activation="silu"`` applies SiLU to the output (
    the reference has no activation). ``layout="bsd"`` takes/returns the
    channel-last [B, S, D] tensor of the gated-DeltaNet chain.
    """
    x, w, b = _f64(x), _f64(weight), _f64(bias)
    if layout == "bsd":
        x = x.transpose(0, 2, 1)
    B, D, S = x.shape
    Dw, W = w.shape
    assert D == Dw and b.shape == (D,)
    xp = np.pad(x, ((0, 0), (0, 0), (W - 1, 0)))
    out = np.broadcast_to(b[None, :, None], (B, D, S)).copy()
    for k in range(W):
        out += w[None, :, k, None] * xp[:, :, k:k + S]
    if activation == "silu":
        out = silu(out)
    elif activation not in (None, "none"):
        raise ValueError(f"unknown activation {activation!r}")
    if layout == "bsd":
        out = out.transpose(0, 2, 1)
    return np.ascontiguousarray(out)


def l2norm(x, eps: float = 1e-6):
    """x / sqrt(sum(x^2) + eps) over the last axis (the chain's q/k norm)."""
    x = _f64(x)
    return x / np.sqrt((x * x).sum(-1, keepdims=True) + eps)


# --------------------------------------------------------------------------
# helpers: [B, T, H, X] <-> per-chunk [B, NT, H, BT, X]
# --------------------------------------------------------------------------
def _to_chunks(x):
    B, T, H = x.shape[:3]
    rest = x.shape[3:]
    NT = T // BT
    y = x.reshape((B, NT, BT, H) + rest)
    if rest:
        return np.ascontiguousarray(y.transpose(0, 1, 3, 2, 4))
    return np.ascontiguousarray(y.transpose(0, 1, 3, 2))


def _from_chunks(y):
    B, NT, H, bt, X = y.shape
    return np.ascontiguousarray(y.transpose(0, 1, 3, 2, 4).reshape(B, NT * bt, H, X))


def _decay(gc):
    """exp(g_i - g_j) for j <= i, 0 above the diagonal; gc [..., BT]."""
    d = gc[..., :, None] - gc[..., None, :]
    mask = np.tril(np.ones((gc.shape[-1],) * 2, dtype=bool))
    return np.where(mask, np.exp(np.where(mask, d, 0.0)), 0.0)


# --------------------------------------------------------------------------
# WY matrix and recompute_w_u
# --------------------------------------------------------------------------
def build_A(k, beta, g, sign: int = -1):
    """Per-chunk WY matrix, returned in the reference's [B, T, H, BT] storage.

    M = strict_tril(beta_i * (k_i . k_j) * exp(g_i - g_j))
    sign=-1: A = (I - M)^-1  -- kernels/recompute_w_u/reference.py:48-91
             (the reference's upstream producer ``_build_A``);
    sign=+1: A = (I + M)^-1  -- the gated-DeltaNet (FLA) convention written
             in BASELINE.json config 2.
    """
    assert sign in (-1, 1)
    k, beta, g = _f64(k), _f64(beta), _f64(g)
    B, T, H, K = k.shape
    assert T % BT == 0
    kc, bc, gc = _to_chunks(k), _to_chunks(beta), _to_chunks(g)
    kkt = kc @ kc.swapaxes(-1, -2)
    M = np.tril(kkt * bc[..., :, None] * _decay(gc), -1)
    eye = np.eye(BT)
    L = eye + sign * M
    Ainv = np.linalg.solve(L, np.broadcast_to(eye, L.shape))
    Ainv = np.tril(Ainv)  # exact zeros above the diagonal
    return _from_chunks(Ainv)


def recompute_w_u(k, v, beta, A, g):
    """w = A @ (k * beta * exp(g)), u = A @ (v * beta), per 64-chunk.

    Restates kernels/recompute_w_u/reference.py:118-149 (ref_kernel).
    Returns (w [B,T,H,K], u [B,T,H,V]).
    """
    k, v, beta, A, g = map(_f64, (k, v, beta, A, g))
    kc, vc, bc, gc, Ac = map(_to_chunks, (k, v, beta, g, A))
    ks = kc * (bc * np.exp(gc))[..., None]
    vs = vc * bc[..., None]
    return _from_chunks(Ac @ ks), _from_chunks(Ac @ vs)


# --------------------------------------------------------------------------
# chunk_fwd_h
# --------------------------------------------------------------------------
def chunk_fwd_h(k, v, g):
    """Reference inter-chunk recurrence; h[b,c,h] is the POST-update state.

    state = state * exp(g_end) + k_c^T @ (v_c * exp(g_end - g_c))
    Restates kernels/chunk_fwd_h/reference.py:50-97 (vectorised over b, h).
    Returns h [B, NT, H, K, V].
    """
    k, v, g = map(_f64, (k, v, g))
    B, T, H, K = k.shape
    V = v.shape[-1]
    NT = T // BT
    kc, vc, gc = _to_chunks(k), _to_chunks(v), _to_chunks(g)
    h = np.zeros((B, NT, H, K, V))
    state = np.zeros((B, H, K, V))
    for c in range(NT):
        gend = gc[:, c, :, -1]                                   # [B,H]
        vg = vc[:, c] * np.exp(gend[..., None] - gc[:, c])[..., None]
        state = state * np.exp(gend)[..., None, None] + kc[:, c].swapaxes(-1, -2) @ vg
        h[:, c] = state
    return h


def chunk_fwd_h_delta(k, w, u, g, h0=None):
    """Gated delta-rule recurrence (extension, no reference).

    For each chunk c (h_c = state entering the chunk, h_0 = h0):
        v_new_c = u_c - w_c @ h_c
        h_{c+1} = exp(g_last) h_c + (k_c * exp(g_last - g_c))^T @ v_new_c
    Extends the loop of kernels/chunk_fwd_h/reference.py:75-95: with w = 0,
    u = v, h0 = 0 it reduces to it (h_{c+1} here == h[c] there).
    Returns (h_pre [B,NT,H,K,V] with h_pre[:,c] = h_c, v_new [B,T,H,V],
    final [B,H,K,V] = h_NT).
    """
    k, w, u, g = map(_f64, (k, w, u, g))
    B, T, H, K = k.shape
    V = u.shape[-1]
    NT = T // BT
    kc, wc, uc, gc = map(_to_chunks, (k, w, u, g))
    h = np.zeros((B, NT, H, K, V))
    vnew = np.zeros((B, NT, H, BT, V))
    state = np.zeros((B, H, K, V)) if h0 is None else _f64(h0).copy()
    for c in range(NT):
        h[:, c] = state
        vn = uc[:, c] - wc[:, c] @ state
        vnew[:, c] = vn
        gl = gc[:, c, :, -1]
        vs = vn * np.exp(gl[..., None] - gc[:, c])[..., None]
        state = state * np.exp(gl)[..., None, None] + kc[:, c].swapaxes(-1, -2) @ vs
    return h, _from_chunks(vnew), state


# --------------------------------------------------------------------------
# chunk_fwd_o
# --------------------------------------------------------------------------
def chunk_fwd_o(q, k, v, g, h, scale):
    """o = scale * (tril((q k^T) * exp(g_t - g_s)) v + (q * exp(g)) h[c]).

    Restates kernels/chunk_fwd_o/reference.py:80-142: the reference forms
    q*exp(g) and v*exp(-g) and a causal (s <= t) mask; the decay is applied
    here as exp(g_t - g_s) on the masked tile, which is the same quantity.
    h[:, c] is used for chunk c exactly as given (reference.py:113).
    Returns o [B, T, H, V].
    """
    q, k, v, g, h = map(_f64, (q, k, v, g, h))
    qc, kc, vc, gc = map(_to_chunks, (q, k, v, g))
    P = (qc @ kc.swapaxes(-1, -2)) * _decay(gc)
    local = P @ vc
    glob = (qc * np.exp(gc)[..., None]) @ h                 # h [B,NT,H,K,V]
    return _from_chunks(scale * (local + glob))


# --------------------------------------------------------------------------
# chained gated-DeltaNet layer forward (extension)
# --------------------------------------------------------------------------
def gated_delta_chain(xq, xk, xv, wq, bq, wk, bk, wv, bv, beta, g, H, K, V,
                      h0=None, scale=None, sign: int = 1, act: str = "silu",
                      round_bf16=None):
    """causal_conv1d(+SiLU) on q/k/v projections [B,T,D] -> l2norm(q,k) ->
    WY (A, w, u) -> delta-rule h (h0) -> chunk_fwd_o with v_new and h entering
    each chunk. ``round_bf16`` (callable or None) is applied to every
    intermediate the CUDA chain stores in bf16 (conv outputs, w, u, v_new), so
    the oracle sees the same rounded operands. Returns (o [B,T,H,V], final).
    """
    rnd = round_bf16 if round_bf16 is not None else (lambda a: a)
    B, T, D = _f64(xq).shape
    q = causal_conv1d(xq, wq, bq, act, "bsd").reshape(B, T, H, K)
    k = causal_conv1d(xk, wk, bk, act, "bsd").reshape(B, T, H, K)
    v = rnd(causal_conv1d(xv, wv, bv, act, "bsd").reshape(B, T, H, V))
    q = rnd(l2norm(q))
    k = rnd(l2norm(k))
    A = build_A(k, beta, g, sign)
    w, u = recompute_w_u(k, v, beta, A, g)
    w, u = rnd(w), rnd(u)
    h, vnew, final = chunk_fwd_h_delta(k, w, u, g, h0)
    vnew = rnd(vnew)
    if scale is None:
        scale = K ** -0.5
    o = chunk_fwd_o(q, k, vnew, g, h, scale)
    return o, final


# --------------------------------------------------------------------------
# recurrent block: gated scan, group norm, conv step and gradients (extensions, no reference)
# --------------------------------------------------------------------------
def _sigmoid(x):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-x))


def scan_gates(x, r, i, decay):
    """(s, L, a, p, m, x) of every token; a token with r < -43 or L = 0 holds the state (L = p = x = 0)."""
    x, r, i, decay = map(_f64, (x, r, i, decay))
    with np.errstate(invalid="ignore"):
        s = _sigmoid(r)
        L = np.where(r < -43.0, 0.0, decay * s)
        held = L == 0.0
        a = np.exp(-L)
        p = np.where(held, 0.0, _sigmoid(i))
        m = np.sqrt(-np.expm1(-2.0 * L))
        return s, L, a, p, m, np.where(held, 0.0, x)


def gated_scan(x, r, i, decay, h0=None):
    """h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t, a_t = exp(-decay sigmoid(r_t)).

    x, r, i [B, T, D], decay [D], h0 [B, D]. Returns (y [B, T, D], final [B, D],
    states [B, ceil(T / 64), D]: the state entering each 64-token chunk)."""
    _, _, a, p, m, x = scan_gates(x, r, i, decay)
    B, T, D = x.shape
    h = np.zeros((B, D)) if h0 is None else _f64(h0).copy()
    y = np.zeros((B, T, D))
    states = np.zeros((B, (T + BT - 1) // BT, D))
    for t in range(T):
        if t % BT == 0:
            states[:, t // BT] = h
        h = a[:, t] * h + m[:, t] * p[:, t] * x[:, t]
        y[:, t] = h
    return y, h, states


def gated_scan_bwd(x, r, i, decay, h0, dy, dfinal=None):
    """Gradients of gated_scan: (dx, dr, di, ddecay, dh0). A held token's are zero."""
    s, L, a, p, m, xv = scan_gates(x, r, i, decay)
    B, T, D = xv.shape
    y, _, _ = gated_scan(x, r, i, decay, h0)
    first = np.zeros((B, 1, D)) if h0 is None else _f64(h0)[:, None]
    prev = np.concatenate([first, y[:, :-1]], 1) if T else y
    dy = _f64(dy)
    carry = np.zeros((B, D)) if dfinal is None else _f64(dfinal).copy()
    dh = np.zeros((B, T, D))
    for t in range(T - 1, -1, -1):
        dh[:, t] = dy[:, t] + carry
        carry = a[:, t] * dh[:, t]
    inv_m = np.where(L == 0.0, 0.0, 1.0 / np.where(L == 0.0, 1.0, m))
    dL = dh * (a * a * inv_m * p * xv - a * prev)
    dx = dh * m * p
    di = dh * m * xv * p * (1.0 - p)
    return dx, dL * L * (1.0 - s), di, (dL * s).sum((0, 1)), carry


def group_norm(x, group, weight=None, bias=None, gate=None, activation=None, center=True, eps=1e-5):
    """u = xh weight + bias over runs of ``group`` channels; act(u), or u act(gate)."""
    x = _f64(x)
    C = x.shape[-1]
    g = x.reshape(x.shape[:-1] + (C // group, group))
    if center:
        g = g - g.mean(-1, keepdims=True)
    u = (g / np.sqrt((g * g).mean(-1, keepdims=True) + eps)).reshape(x.shape)
    if weight is not None:
        u = u * _f64(weight)
    if bias is not None:
        u = u + _f64(bias)
    if gate is not None:
        z = _f64(gate)
        return u * (silu(z) if activation == "silu" else z)
    return silu(u) if activation == "silu" else u


def silu_grad(x):
    s = _sigmoid(x)
    return s * (1.0 + x * (1.0 - s))


def group_norm_bwd(x, dy, group, weight=None, bias=None, gate=None, activation=None, center=True, eps=1e-5):
    """Gradients of group_norm: (dx, dgate or None, dweight or None, dbias or None)."""
    x, dy = _f64(x), _f64(dy)
    C = x.shape[-1]
    shape3 = x.shape[:-1] + (C // group, group)
    g = x.reshape(shape3)
    if center:
        g = g - g.mean(-1, keepdims=True)
    rs = 1.0 / np.sqrt((g * g).mean(-1, keepdims=True) + eps)
    xh3 = g * rs
    xh = xh3.reshape(x.shape)
    w = np.ones(C) if weight is None else _f64(weight)
    u = xh * w + (0.0 if bias is None else _f64(bias))
    silu_on = activation == "silu"
    dgate = None
    if gate is not None:
        z = _f64(gate)
        dgate = dy * u * (silu_grad(z) if silu_on else 1.0)
        du = dy * (silu(z) if silu_on else z)
    else:
        du = dy * (silu_grad(u) if silu_on else 1.0)
    axes = tuple(range(x.ndim - 1))
    dxh = (du * w).reshape(shape3)
    dx = dxh - xh3 * (dxh * xh3).mean(-1, keepdims=True)
    if center:
        dx = dx - dxh.mean(-1, keepdims=True)
    return ((dx * rs).reshape(x.shape), dgate, None if weight is None else (du * xh).sum(axes),
            None if bias is None else du.sum(axes))


def causal_conv1d_step(x, state, weight, bias, activation=None):
    """causal_conv1d ("bsd") continued from the W - 1 inputs before x: (out, new state)."""
    z = np.concatenate([_f64(state), _f64(x)], 1)
    W = _f64(weight).shape[1]
    out = causal_conv1d(z, weight, bias, activation, "bsd")[:, W - 1:]
    return out, z[:, z.shape[1] - (W - 1):]


def causal_conv1d_bwd(x, weight, bias, dy, activation=None):
    """Gradients of causal_conv1d ("bsd"): (dx, dweight [D, W], dbias [D])."""
    x, w, dy = _f64(x), _f64(weight), _f64(dy)
    B, S, D = x.shape
    W = w.shape[1]
    du = dy
    if activation == "silu":
        du = dy * silu_grad(causal_conv1d(x, w, bias, None, "bsd"))
    xp = np.concatenate([np.zeros((B, W - 1, D)), x], 1)
    dup = np.concatenate([du, np.zeros((B, W - 1, D))], 1)
    dx = sum(w[:, k] * dup[:, W - 1 - k:W - 1 - k + S] for k in range(W))
    dw = np.stack([(du * xp[:, k:k + S]).sum((0, 1)) for k in range(W)], 1)
    return dx, dw, du.sum((0, 1))
