"""GPU parity of causal_conv1d_step and causal_conv1d_bwd against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import ops as orc
from tests import recurrent_ref as rr

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U = rr.U


def _inputs(B, S, D, W, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x, dy = (torch.randn(B, S, D, generator=g).to(dtype) for _ in range(2))
    w = 0.5 * torch.randn(D, W, generator=g)
    b = 0.3 * torch.randn(D, generator=g)
    st = torch.randn(B, W - 1, D, generator=g).to(dtype)
    return x, dy, w, b, st


def _u_error(z, w, b):
    """W fused steps from the bias: each rounds the running sum, at most the sum of magnitudes."""
    mag = orc.causal_conv1d(np.abs(orc._f64(z)), np.abs(orc._f64(w)), np.abs(orc._f64(b)), None, "bsd")
    return (orc._f64(w).shape[1] + 1) * U * mag


def _check_step(x, w, b, st, act, out, st2, dtype):
    ref, rst = orc.causal_conv1d_step(x, st, w, b, act)
    W = w.shape[1]
    z = np.concatenate([orc._f64(st), orc._f64(x)], 1)
    u = orc.causal_conv1d(z, w, b, None, "bsd")[:, W - 1:]
    e = _u_error(z, w, b)[:, W - 1:]
    if act:  # silu is 1.1-Lipschitz; the sigmoid is off by an absolute 8 u at most
        e = 1.1 * e + 12 * U * np.abs(u)
    rr.assert_within(out, ref, rr.rounded(e, ref, dtype), "out")
    assert np.array_equal(st2.double().cpu().numpy(), rst), "state"


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("B,S,D,W", [(1, 1, 1, 4), (64, 1, 2048, 4), (3, 2, 66, 4), (2, 5, 128, 3), (5, 64, 40, 2),
                                     (2, 3, 36, 1), (3, 4, 33, 8), (2, 2, 64, 7), (2, 0, 64, 4), (2, 6, 20, 5)])
def test_step_matches_oracle(B, S, D, W, act, dtype):
    from theorem_b200 import ops
    x, _, w, b, st = _inputs(B, S, D, W, dtype, seed=B + S + D + W)
    dx, dw, db, dst = (t.to(DEV) for t in (x, w, b, st))
    out, st2 = ops.causal_conv1d_step(dx, dst, dw, db, activation=act)
    _check_step(x, w, b, st, act, out, st2, dtype)
    assert torch.equal(dst.cpu(), st), "the given state changed"
    out3, st3 = ops.causal_conv1d_step(dx, dst, dw, db, activation=act, state_out=dst)
    assert st3.data_ptr() == dst.data_ptr() and torch.equal(st3, st2) and torch.equal(out3, out)


@pytest.mark.parametrize("act", [None, "silu"])
def test_steps_continue_the_whole_conv(act):
    """Prefill through causal_conv1d, then token by token from the last W - 1 inputs, within two
    roundings of the whole conv's outputs (each path rounds its own sum once; their SiLUs differ
    by the tanh form's relative 2^-11 that the whole conv uses for bf16)."""
    from theorem_b200 import ops
    B, S, D, W, n = 3, 40, 128, 4, 30
    x, _, w, b, _ = (t.to(DEV) for t in _inputs(B, S, D, W, BF, seed=2))
    whole = ops.causal_conv1d(x, w, b, act, "bsd").double()
    st = x[:, n - (W - 1):n].contiguous()
    for t in range(n, S):
        out, _ = ops.causal_conv1d_step(x[:, t:t + 1], st, w, b, activation=act, state_out=st)
        d = (out[:, 0].double() - whole[:, t]).abs()
        u = orc.causal_conv1d(x.float().cpu(), w.cpu(), b.cpu(), None, "bsd")[:, t]
        lim = 2 * (torch.finfo(BF).eps / 2) * whole[:, t].abs() + torch.from_numpy(np.abs(u)).to(DEV) * 2 ** -10
        assert (d <= lim).all()


BWD = [(1, 1, 1, 4), (2, 1, 64, 4), (1, 2, 8, 4), (2, 3, 130, 4), (3, 15, 40, 3), (2, 16, 256, 4), (2, 17, 129, 4),
       (1, 64, 36, 2), (2, 127, 64, 1), (2, 129, 132, 4), (1, 1023, 24, 4), (2, 1024, 68, 4), (1, 1500, 33, 3),
       (2, 700, 64, 8), (1, 5000, 20, 5), (9, 40, 512, 6), (1, 300, 31, 7)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("B,S,D,W", BWD)
def test_bwd_matches_oracle(B, S, D, W, act, dtype):
    from theorem_b200 import ops
    x, dy, w, b, _ = _inputs(B, S, D, W, dtype, seed=B + S + D + W)
    _check_bwd(x, dy, w, b, act, ops.causal_conv1d_bwd(*(t.to(DEV) for t in (x, w, b, dy)), activation=act), dtype)


def _check_bwd(x, dy, w, b, act, got, dtype):
    B, S, D = x.shape
    W = w.shape[1]
    g = np.abs(orc._f64(dy))
    ref = orc.causal_conv1d_bwd(x, w, b, dy, act)
    if act:
        u = orc.causal_conv1d(x, w, b, None, "bsd")
        du = g * np.abs(orc.silu_grad(u))
        edu = g * (0.5 * _u_error(x, w, b) + 12 * U * (1 + np.abs(u))) + 2 * U * du  # silu' is 0.5-Lipschitz
    else:
        du, edu = g, 0 * g
    z = np.zeros((D, 1))
    flip = lambda a: orc.causal_conv1d(a[:, ::-1], np.abs(orc._f64(w)), z[:, 0], None, "bsd")[:, ::-1]  # noqa: E731
    edx = flip(edu) + (W + 1) * U * flip(du)
    rr.assert_within(got[0], ref[0], rr.rounded(edx, ref[0], dtype), "dx")
    xp = np.abs(np.concatenate([np.zeros((B, W - 1, D)), orc._f64(x)], 1))
    n = B * S
    for k in range(W):
        xs = xp[:, k:k + S]
        bound = (edu * xs).sum((0, 1)) + (n + 1) * U * (du * xs).sum((0, 1))
        rr.assert_within(got[1][:, k], ref[1][:, k], bound, f"dweight[{k}]")
    rr.assert_within(got[2], ref[2], edu.sum((0, 1)) + (n + 1) * U * du.sum((0, 1)), "dbias")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_strided_and_unaligned_inputs(shift, dtype):
    from theorem_b200 import ops
    B, S, D, W = 2, 37, 72, 4
    x, dy, w, b, st = _inputs(B, S, D, W, dtype, seed=shift)
    wide = torch.zeros(B, S, 2 * D + 8, device=DEV, dtype=dtype)
    xv, gv = wide[..., shift:shift + D], wide[..., shift + D:shift + 2 * D]
    xv.copy_(x.to(DEV))
    gv.copy_(dy.to(DEV))
    _check_bwd(x, dy, w, b, "silu", ops.causal_conv1d_bwd(xv, w.to(DEV), b.to(DEV), gv, activation="silu"), dtype)
    xt = x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    out, st2 = ops.causal_conv1d_step(xt, st.to(DEV), w.to(DEV), b.to(DEV), activation="silu")
    _check_step(x, w, b, st, "silu", out, st2, dtype)
    out, st2 = ops.causal_conv1d_step(xv, st.to(DEV), w.to(DEV), b.to(DEV))
    _check_step(x, w, b, st, None, out, st2, dtype)


def test_time_major_inputs():
    from theorem_b200 import ops
    x, dy, w, b, _ = _inputs(3, 200, 64, 4, BF, seed=3)
    tm = [t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1) for t in (x, dy)]
    _check_bwd(x, dy, w, b, "silu", ops.causal_conv1d_bwd(tm[0], w.to(DEV), b.to(DEV), tm[1], activation="silu"), BF)


def test_offsets_past_32_bits():
    from theorem_b200 import ops
    D, tail = 2048, 500
    S = (1 << 20) + tail
    x = torch.randn(1, S, D, device=DEV, dtype=BF, generator=torch.Generator(DEV).manual_seed(0))
    w, b = torch.full((D, 4), 0.25, device=DEV), torch.zeros(D, device=DEV)
    xt = x[:, -tail:].contiguous()
    a = ops.causal_conv1d_bwd(x, w, b, x, activation="silu")[0][:, -tail + 3:]  # 3 rows see what came before
    c = ops.causal_conv1d_bwd(xt, w, b, xt, activation="silu")[0][:, 3:]
    assert torch.equal(a, c)


def test_empty_repeat_and_capture():
    from theorem_b200 import ops
    e = torch.empty(0, 5, 64, device=DEV)
    w, b = torch.ones(64, 4, device=DEV), torch.ones(64, device=DEV)
    dx, dw, db = ops.causal_conv1d_bwd(e, w, b, e)
    assert dx.shape == e.shape and (dw == 0).all() and (db == 0).all()
    assert ops.causal_conv1d_step(e, torch.empty(0, 3, 64, device=DEV), w, b)[0].shape == e.shape
    x, dy, w, b, _ = (t.to(DEV) for t in _inputs(3, 1500, 256, 4, BF, seed=1))
    step = lambda: ops.causal_conv1d_bwd(x, w, b, dy, activation="silu")  # noqa: E731
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
    x = torch.zeros(2, 4, 16, device=DEV)
    w, b = torch.zeros(16, 4, device=DEV), torch.zeros(16, device=DEV)
    st = torch.zeros(2, 3, 16, device=DEV)
    bad = [
        lambda: ops.causal_conv1d_step(x, st[:, :2], w, b),
        lambda: ops.causal_conv1d_step(x, st.bfloat16(), w, b),
        lambda: ops.causal_conv1d_step(torch.zeros(2, 65, 16, device=DEV), st, w, b),
        lambda: ops.causal_conv1d_step(x, torch.zeros(2, 8, 16, device=DEV), torch.zeros(16, 9, device=DEV), b),
        lambda: ops.causal_conv1d_step(x, st, w.bfloat16(), b),
        lambda: ops.causal_conv1d_step(x, st, w, b, activation="relu"),
        lambda: ops.causal_conv1d_step(x.transpose(1, 2), st, w[:4], b[:4]),
        lambda: ops.causal_conv1d_bwd(x, w, b, x[:1]),
        lambda: ops.causal_conv1d_bwd(x, w, b, x.bfloat16()),
        lambda: ops.causal_conv1d_bwd(x, torch.zeros(16, 9, device=DEV), b, x),
        lambda: ops.causal_conv1d_bwd(x, w, b[:8], x),
        lambda: ops.causal_conv1d_bwd(x.half(), w, b, x.half()),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"refusal {k} did not raise")
