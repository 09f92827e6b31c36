"""The recurrent block's oracle on the CPU: its gradients against central differences in
float64, and the identities that tie its forms together."""
import numpy as np
import pytest

from oracle import ops as orc


def _diff(f, arr, cot, eps=1e-6, n=12, seed=0):
    """Directional derivatives of sum(cot * f) along unit vectors of arr, by central differences."""
    rng = np.random.default_rng(seed)
    flat = arr.reshape(-1)
    for k in rng.choice(flat.size, size=min(n, flat.size), replace=False):
        old = flat[k]
        flat[k] = old + eps
        up = sum((c * o).sum() for c, o in zip(cot, f()))
        flat[k] = old - eps
        dn = sum((c * o).sum() for c, o in zip(cot, f()))
        flat[k] = old
        yield k, (up - dn) / (2 * eps)


# Central differences of f at step 1e-6: the third derivative's share is of the order 1e-12 f''',
# the rounding of the sums 1e-16 |sum| / 1e-6; both stay under 1e-6 for values of order 1 to 100.
TOL = 1e-6


def _check(grad, f, arr, cot):
    for k, d in _diff(f, arr, cot):
        assert abs(grad.reshape(-1)[k] - d) <= TOL * max(1.0, abs(d)) * 10, (k, grad.reshape(-1)[k], d)


@pytest.mark.parametrize("T", [1, 3, 65])
def test_gated_scan_gradients_match_differences(T):
    rng = np.random.default_rng(T)
    B, D = 2, 3
    x, r, i, dy = (rng.standard_normal((B, T, D)) for _ in range(4))
    decay = np.exp(rng.uniform(-3, 0, D))
    h0, df = rng.standard_normal((2, B, D))
    f = lambda: orc.gated_scan(x, r, i, decay, h0)[:2]  # noqa: E731
    dx, dr, di, dd, dh0 = orc.gated_scan_bwd(x, r, i, decay, h0, dy, df)
    for g, arr in ((dx, x), (dr, r), (di, i), (dd, decay), (dh0, h0)):
        _check(g, f, arr, (dy, df))


def test_gated_scan_continues_and_holds():
    rng = np.random.default_rng(7)
    x, r, i = rng.standard_normal((3, 1, 130, 4))
    decay = np.full(4, 0.3)
    y, fin, st = orc.gated_scan(x, r, i, decay)
    y1, f1, _ = orc.gated_scan(x[:, :64], r[:, :64], i[:, :64], decay)
    y2, f2, _ = orc.gated_scan(x[:, 64:], r[:, 64:], i[:, 64:], decay, f1)
    assert np.allclose(np.concatenate([y1, y2], 1), y, rtol=0, atol=1e-14) and np.allclose(f2, fin, rtol=0, atol=1e-14)
    assert np.array_equal(st[:, 1], f1)
    r[:, 100:] = -np.inf
    x[:, 100:] = np.nan
    i[:, 100:] = np.nan
    yh, fh, _ = orc.gated_scan(x, r, i, decay)
    assert np.array_equal(fh, y[:, 99]) and np.array_equal(yh[:, :100], y[:, :100])
    g = orc.gated_scan_bwd(x, r, i, decay, None, np.ones_like(x))
    assert all(np.isfinite(a).all() for a in g) and not g[0][:, 100:].any() and not g[1][:, 100:].any()


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("center", [False, True])
def test_group_norm_gradients_match_differences(center, act, gate):
    rng = np.random.default_rng(3)
    x, dy, z = rng.standard_normal((3, 4, 12))
    z = z if gate else None
    w, b = rng.standard_normal((2, 12))
    kw = dict(activation=act, center=center, eps=1e-3)
    f = lambda: (orc.group_norm(x, 6, w, b, z, **kw),)  # noqa: E731
    g = orc.group_norm_bwd(x, dy, 6, w, b, z, **kw)
    for grad, arr in zip(g, (x, z, w, b)):
        if arr is not None:
            _check(grad, f, arr, (dy,))


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("S,W", [(1, 4), (2, 4), (9, 3), (5, 1)])
def test_conv_gradients_match_differences(S, W, act):
    rng = np.random.default_rng(S * 10 + W)
    x, dy = rng.standard_normal((2, 2, S, 3))
    w, b = rng.standard_normal((3, W)), rng.standard_normal(3)
    f = lambda: (orc.causal_conv1d(x, w, b, act, "bsd"),)  # noqa: E731
    for grad, arr in zip(orc.causal_conv1d_bwd(x, w, b, dy, act), (x, w, b)):
        _check(grad, f, arr, (dy,))


@pytest.mark.parametrize("W", [1, 2, 4])
def test_conv_step_continues_the_conv(W):
    rng = np.random.default_rng(W)
    x = rng.standard_normal((2, 11, 3))
    w, b = rng.standard_normal((3, W)), rng.standard_normal(3)
    whole = orc.causal_conv1d(x, w, b, "silu", "bsd")
    st = np.zeros((2, W - 1, 3))
    outs = []
    for lo, hi in ((0, 1), (1, 4), (4, 11)):
        o, st = orc.causal_conv1d_step(x[:, lo:hi], st, w, b, "silu")
        outs.append(o)
    assert np.allclose(np.concatenate(outs, 1), whole, rtol=0, atol=1e-15)
    assert np.array_equal(st, x[:, 11 - (W - 1):])
