"""GPU parity of group_norm and group_norm_bwd against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import ops as orc
from tests import recurrent_ref as rr

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U = rr.U


def _inputs(R, C, dtype, seed, gate, affine, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, C, generator=g) + offset).to(dtype)
    dy = torch.randn(R, C, generator=g).to(dtype)
    z = (2 * torch.randn(R, C, generator=g)).to(dtype) if gate else None
    w = 1 + 0.3 * torch.randn(C, generator=g) if affine else None
    b = 0.3 * torch.randn(C, generator=g) if affine else None
    return x, dy, z, w, b


def _parts(x, G, center, eps):
    """|xh|'s stand-in for error bounds and its error. The mean is a sum of G terms in at most
    32 steps per thread and 10 + 32 across threads: 74 u of mean|x|; so x - mu is off by
    e = u |x| + 76 u mean|x|. rs: the squares' mean 77 u and twice e against the deviation's root
    mean square, half of it, and rsqrt's 4 u."""
    x = orc._f64(x)
    g = x.reshape(x.shape[0], -1, G)
    ax = np.abs(g).mean(-1, keepdims=True)
    d = g - g.mean(-1, keepdims=True) if center else g
    rs = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    e = (2 * np.abs(g) + 76 * ax) * U if center else 0 * np.abs(g)
    rel = 45 * U + (e * np.abs(d)).mean(-1, keepdims=True) * rs * rs
    xh = d * rs
    exh = rs * e + np.abs(xh) * (rel + U)
    return xh, exh, rs, rel


def _flat(a, like):
    return np.broadcast_to(a, a.shape).reshape(like)


def _check(x, dy, z, w, b, G, act, center, eps, y, grads, dtype):
    shape = tuple(x.shape)
    xh3, exh3, rs, rel = _parts(x, G, center, eps)
    xh, exh = xh3.reshape(shape), exh3.reshape(shape)
    W = np.ones(shape[1]) if w is None else orc._f64(w)
    Bb = np.zeros(shape[1]) if b is None else orc._f64(b)
    u = xh * W + Bb
    eu = np.abs(W) * exh + 2 * U * (np.abs(xh * W) + np.abs(u))
    # silu is 1.1-Lipschitz, silu' 0.5-Lipschitz; a sigmoid is off by an absolute 8 u at most
    # (its relative error times s (1 - s), which |x| of the exponential's error stays under).
    if z is not None:
        zz = orc._f64(z)
        f, df = (orc.silu(zz), orc.silu_grad(zz)) if act else (zz, np.ones_like(zz))
        ef, edf = (12 * U * np.abs(zz), 12 * U * (1 + np.abs(zz))) if act else (0.0, 0.0)
        ref = u * f
        ey = eu * np.abs(f) + np.abs(u) * ef + 2 * U * np.abs(ref)
    else:
        ref = orc.silu(u) if act else u
        ey = 1.1 * eu + 12 * U * np.abs(u) if act else eu
    assert np.allclose(ref, orc.group_norm(x, G, w, b, z, activation=act, center=center, eps=eps), rtol=1e-12, atol=1e-12)
    rr.assert_within(y, ref, rr.rounded(ey, ref, dtype), "y")
    if grads is None:
        return
    rdx, rdz, rdw, rdb = orc.group_norm_bwd(x, dy, G, w, b, z, activation=act, center=center, eps=eps)
    g = orc._f64(dy)
    if z is not None:
        du, edu = g * f, np.abs(g) * (ef + 2 * U * np.abs(f))
        ez = np.abs(g) * (eu * np.abs(df) + np.abs(u) * (edf + 4 * U * np.abs(df)))
        rr.assert_within(grads[1], rdz, rr.rounded(ez, rdz, dtype), "dgate")
    else:
        assert grads[1] is None
        d1 = orc.silu_grad(u) if act else np.ones_like(u)
        du = g * d1
        edu = np.abs(g) * ((0.5 * eu + 12 * U * (1 + np.abs(u))) if act else 0.0) + 2 * U * np.abs(du)
    # dx = rs (dxh - mean(dxh) - xh mean(dxh xh)): each mean's own error, 76 u of its magnitudes.
    dxh, edxh = du * W, edu * np.abs(W) + U * np.abs(du * W)
    d3, e3 = dxh.reshape(xh3.shape), edxh.reshape(xh3.shape)
    mean = lambda a: a.mean(-1, keepdims=True)  # noqa: E731
    m1, em1 = (mean(np.abs(d3)), mean(e3) + 76 * U * mean(np.abs(d3))) if center else (0.0, 0.0)
    m2 = mean(np.abs(d3 * xh3))
    em2 = mean(e3 * np.abs(xh3) + np.abs(d3) * exh3) + 78 * U * m2
    mag = np.abs(d3) + m1 + np.abs(xh3) * m2
    edx = rs * (e3 + em1 + exh3 * m2 + np.abs(xh3) * em2 + (4 * U + rel) * mag)
    rr.assert_within(grads[0], rdx, rr.rounded(edx.reshape(shape), rdx, dtype), "dx")
    R = shape[0]
    if w is not None:
        bound = (edu * np.abs(xh) + np.abs(du) * exh).sum(0) + (R + 2) * U * np.abs(du * xh).sum(0)
        rr.assert_within(grads[2], rdw, bound, "dweight")
    if b is not None:
        rr.assert_within(grads[3], rdb, edu.sum(0) + (R + 2) * U * np.abs(du).sum(0), "dbias")


SHAPES = [  # rows, channels, group
    (1, 1, 1), (1, 128, 128), (64, 2048, 128), (5, 48, 16), (3, 40, 8), (7, 6, 2), (300, 64, 64), (9, 196, 49),
    (33, 96, 3), (4, 1024, 1024), (3, 1032, 1032), (2, 4096, 4096), (5, 4095, 4095), (3, 2050, 1025), (11, 129, 129),
    (6, 260, 130), (2, 8192, 256), (40, 392, 49), (21, 808, 101), (3, 5416, 677),
    (5, 2600, 650), (2, 8184, 4092), (9, 264, 33), (4, 1960, 490), (1500, 24, 12), (2, 3000, 1500), (257, 520, 260),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("gate,act", [(False, None), (False, "silu"), (True, None), (True, "silu")])
@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("R,C,G", SHAPES)
def test_matches_oracle(R, C, G, center, gate, act, dtype):
    from theorem_b200 import ops
    affine = (R + G) % 3 != 0
    x, dy, z, w, b = _inputs(R, C, dtype, R + C + G, gate, affine)
    dx, ddy, dz, dw, db = [None if t is None else t.to(DEV) for t in (x, dy, z, w, b)]
    kw = dict(gate=dz, activation=act, center=center, eps=1e-5)
    y = ops.group_norm(dx, G, dw, db, **kw)
    grads = ops.group_norm_bwd(dx, ddy, G, dw, db, **kw)
    if G == 1:
        # A one-channel group: centred, xh = 0; not centred, dx is all cancellation.
        grads_ref = orc.group_norm_bwd(x, dy, G, w, b, z, activation=act, center=center, eps=1e-5)
        assert np.isfinite(grads[0].float().cpu().numpy()).all() and np.isfinite(grads_ref[0]).all()
    _check(x, dy, z, w, b, G, act, center, 1e-5, y, grads, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_row_strides_and_unaligned_addresses(shift, dtype):
    """x, gate and dy as slices of wider projections, [B, T, C] with a common row stride."""
    from theorem_b200 import ops
    B, T, C, G = 2, 19, 128, 32
    x, dy, z, w, b = _inputs(B * T, C, dtype, shift, True, True)
    wide = torch.zeros(B, T, 3 * C + 8, device=DEV, dtype=dtype)
    views = []
    for k, t in enumerate((x, dy, z)):
        v = wide[..., shift + k * C: shift + (k + 1) * C]
        v.copy_(t.view(B, T, C).to(DEV))
        views.append(v)
    kw = dict(gate=views[2], activation="silu", center=False, eps=1e-5)
    y = ops.group_norm(views[0], G, w.to(DEV), b.to(DEV), **kw)
    grads = ops.group_norm_bwd(views[0], views[1], G, w.to(DEV), b.to(DEV), **kw)
    assert y.shape == (B, T, C) and y.is_contiguous()
    _check(x, dy, z, w, b, G, "silu", False, 1e-5, y.view(-1, C), [g.view(-1, C) if g.dim() == 3 else g for g in grads],
           dtype)


def test_in_place():
    from theorem_b200 import ops
    x, _, z, w, b = [t.to(DEV) for t in _inputs(500, 384, BF, 6, True, True)]
    kw = dict(activation="silu", center=False)
    want = ops.group_norm(x, 128, w, b, gate=z, **kw)
    for k in range(2):
        xs, zs = x.clone(), z.clone()
        out = (xs, zs)[k]
        assert ops.group_norm(xs, 128, w, b, gate=zs, out=out, **kw) is out and torch.equal(out, want)


def test_offsets_past_32_bits():
    from theorem_b200 import ops
    C, tail = 4096, 300
    R = (1 << 19) + tail
    x = torch.randn(R, C, device=DEV, dtype=BF, generator=torch.Generator(DEV).manual_seed(0))
    w = torch.ones(C, device=DEV)
    kw = dict(activation="silu", center=False)
    xt = x[-tail:].clone()
    assert torch.equal(ops.group_norm(x, 128, w, gate=x, **kw)[-tail:], ops.group_norm(xt, 128, w, gate=xt, **kw))
    a = ops.group_norm_bwd(x, x, 128, w, gate=x, **kw)
    b = ops.group_norm_bwd(xt, xt, 128, w, gate=xt, **kw)
    assert torch.equal(a[0][-tail:], b[0]) and torch.equal(a[1][-tail:], b[1])


def test_large_mean_keeps_the_variance():
    """A mean 1000 times the deviation: the centred sum keeps what a difference of sums loses."""
    from theorem_b200 import ops
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 256, generator=g) + 1000.0
    y = ops.group_norm(x.to(DEV), 128)
    _check(x, x, None, None, None, 128, None, True, 1e-5, y, None, F32)


def test_constant_rows_and_zero_rows():
    """No deviation: xh is 0 centred; zeros stay zeros and gradients stay finite."""
    from theorem_b200 import ops
    x = torch.full((4, 64), 3.0, device=DEV)
    x[2:] = 0
    y = ops.group_norm(x, 32)
    assert (y == 0).all()
    for center in (True, False):
        g = ops.group_norm_bwd(x, torch.ones_like(x), 32, center=center)[0]
        assert torch.isfinite(g).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_groups_that_cut_vectors_keep_to_themselves(dtype):
    """NaN in a neighbouring group that shares a 16-byte vector reaches neither sums nor gradients, in
    place as well."""
    from theorem_b200 import ops
    R, C, G = 70, 392, 49
    x, dy, z, w, b = [t.to(DEV) for t in _inputs(R, C, dtype, 3, True, True)]
    kw = dict(activation="silu", center=True)
    y, g = ops.group_norm(x, G, w, b, gate=z, **kw), ops.group_norm_bwd(x, dy, G, w, b, gate=z, **kw)
    own = slice(49, 98)
    bad = [t.clone() for t in (x, dy, z)]
    for t in bad:
        t[:, 98:] = float("nan")
        t[:, :49] = float("inf")
    y2, g2 = ops.group_norm(bad[0], G, w, b, gate=bad[2], **kw), ops.group_norm_bwd(bad[0], bad[1], G, w, b, gate=bad[2], **kw)
    assert torch.equal(y2[:, own], y[:, own])
    assert all(torch.equal(p[..., own], q[..., own]) for p, q in zip(g2, g))
    assert torch.equal(ops.group_norm(x, G, w, b, gate=z, out=x, **kw), y)


def test_non_finite_values_stay_in_their_group():
    from theorem_b200 import ops
    x = torch.randn(6, 96, device=DEV)
    clean = ops.group_norm(x, 32)
    x[2, 40] = float("nan")
    x[4, 5] = float("inf")
    y = ops.group_norm(x, 32)
    touched = torch.zeros(6, 96, dtype=torch.bool, device=DEV)
    touched[2, 32:64] = True
    touched[4, :32] = True
    assert torch.isnan(y[2, 32:64]).all() and torch.equal(y[~touched], clean[~touched])


def test_empty_and_repeated_and_captured():
    from theorem_b200 import ops
    w = torch.ones(64, device=DEV)
    e = torch.empty(0, 64, device=DEV)
    assert ops.group_norm(e, 16, w, w).shape == (0, 64)
    dx, dz, dw, db = ops.group_norm_bwd(e, e, 16, w, w)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    x, dy, z, w, b = [t.to(DEV) for t in _inputs(3000, 512, BF, 4, True, True)]
    step = lambda: (ops.group_norm(x, 128, w, b, gate=z, activation="silu"),  # noqa: E731
                    *ops.group_norm_bwd(x, dy, 128, w, b, gate=z, activation="silu"))
    a = step()
    assert all(torch.equal(p, q) for p, q in zip(a, step()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            o = step()
        g.replay()
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, o))


def test_refusals():
    from theorem_b200 import ops
    x = torch.zeros(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    bad = [
        lambda: ops.group_norm(x, 48),
        lambda: ops.group_norm(x, 0),
        lambda: ops.group_norm(x.half(), 16),
        lambda: ops.group_norm(x, 16, w.bfloat16()),
        lambda: ops.group_norm(x, 16, w[:32]),
        lambda: ops.group_norm(x, 16, gate=x.bfloat16()),
        lambda: ops.group_norm(x, 16, activation="relu"),
        lambda: ops.group_norm(x.t(), 4),
        lambda: ops.group_norm(torch.zeros(4, 6, 64, device=DEV).transpose(0, 1), 16),
        lambda: ops.group_norm(torch.zeros(1, 8192, device=DEV), 8192),
        lambda: ops.group_norm(x, 16, out=torch.zeros(4, 128, device=DEV)[:, :64]),
        lambda: ops.group_norm_bwd(x, x[:2], 16),
        lambda: ops.group_norm_bwd(x, x.bfloat16(), 16),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"refusal {k} did not raise")
