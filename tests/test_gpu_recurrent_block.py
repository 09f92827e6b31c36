"""The recurrent block's operators together, as they are used: forward, backward, prefill then single
tokens, against the float64 oracle; and the DeltaNet layer with its output norm."""
import numpy as np
import pytest
import torch

from oracle import ops as orc
from tests.harness import assert_close
from tests.synth import deltanet_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
# The framework's tolerances: 1e-4 for fp32, 1e-2 for bf16 (rtol = atol). The oracle rounds what the
# block stores in bf16 (u, h, and the gradients dh, du between the operators).
TOL = {F32: 1e-4, BF: 1e-2}


def _rnd(dtype):
    if dtype == F32:
        return lambda a: a
    return lambda a: torch.from_numpy(np.asarray(a)).to(BF).double().numpy()


def _params(D, W, seed, bias):
    g = torch.Generator().manual_seed(seed)
    return dict(conv_weight=torch.randn(D, W, generator=g) * 0.5, conv_bias=torch.randn(D, generator=g) * 0.3,
                decay=torch.exp(torch.rand(D, generator=g) * 3 - 4), norm_weight=1 + 0.1 * torch.randn(D, generator=g),
                norm_bias=0.1 * torch.randn(D, generator=g) if bias else None)


def _inputs(B, T, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, T, D, generator=g).to(dtype) for _ in range(5)]  # x, r, i, z, dy


def _oracle(p, group, center, x, r, i, z, rnd, state=None):
    u = orc.causal_conv1d(x, p["conv_weight"], p["conv_bias"], "silu", "bsd")
    u = rnd(u)
    h, fin, _ = orc.gated_scan(u, r, i, p["decay"], state)
    h = rnd(h)
    y = orc.group_norm(h, group, p["norm_weight"], p["norm_bias"], z, activation="silu", center=center)
    return u, h, fin, y


def _block(p, group, center):
    from theorem_b200.recurrent import GatedRecurrentBlock
    q = {k: None if v is None else v.to(DEV) for k, v in p.items()}
    return GatedRecurrentBlock(**q, norm_group=group, center=center)


def _np(t):
    return torch.from_numpy(np.ascontiguousarray(t))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,D,W,group,center", [(2, 1, 64, 4, 64, False), (3, 130, 192, 4, 64, False),
                                                  (1, 517, 128, 3, 128, True), (2, 64, 100, 2, 20, True)])
def test_forward_and_backward_match_oracle(B, T, D, W, group, center, dtype):
    p = _params(D, W, seed=T + D, bias=center)
    x, r, i, z, dy = _inputs(B, T, D, dtype, seed=T)
    blk = _block(p, group, center)
    dev = [t.to(DEV) for t in (x, r, i, z, dy)]
    y, st, saved = blk(*dev[:4], want_grad=True)
    rnd, tol = _rnd(dtype), TOL[dtype]
    u, h, fin, ry = _oracle(p, group, center, x, r, i, z, rnd)
    assert_close(y.double().cpu(), _np(ry), tol, tol, "y")
    assert_close(st.h.double().cpu(), _np(fin), tol, tol, "final state")
    y2, st2 = blk(*dev[:4])
    assert torch.equal(y2, y) and torch.equal(st2.h, st.h) and torch.equal(st2.conv, st.conv)
    df = torch.randn(B, D, generator=torch.Generator().manual_seed(1))
    got = blk.backward(saved, dev[4], dfinal=df.to(DEV))
    dh, dz, dnw, dnb = orc.group_norm_bwd(h, dy, group, p["norm_weight"], p["norm_bias"], z, activation="silu",
                                          center=center)
    du, dr, di, dd, _ = orc.gated_scan_bwd(u, r, i, p["decay"], None, rnd(dh), df)
    dx, dcw, dcb = orc.causal_conv1d_bwd(x, p["conv_weight"], p["conv_bias"], rnd(du), "silu")
    want = dict(x=dx, r=dr, i=di, z=dz, conv_weight=dcw, conv_bias=dcb, decay=dd, norm_weight=dnw)
    if center:
        want["norm_bias"] = dnb
    assert set(got) == set(want)
    # Sums over tokens: their absolute tolerance is that of a term, times the root of the number of
    # terms (the terms' roundings are independent).
    for k, w in want.items():
        atol = tol * (max(1.0, (B * T) ** 0.5) if w.ndim < 3 else max(1.0, float(np.abs(w).max()) / 4))
        assert_close(got[k].double().cpu(), _np(w), tol, atol, k)


def test_gradients_match_differences_of_the_composed_oracle():
    """fp32 gradients against central differences of the whole block in float64."""
    B, T, D, W, group = 2, 70, 32, 4, 16
    p = _params(D, W, seed=3, bias=False)
    x, r, i, z, dy = _inputs(B, T, D, F32, seed=4)
    blk = _block(p, group, False)
    _, _, saved = blk(*(t.to(DEV) for t in (x, r, i, z)), want_grad=True)
    got = blk.backward(saved, dy.to(DEV))
    vals = {"x": x, "r": r, "i": i, "z": z, **{k: v for k, v in p.items() if v is not None}}
    vals = {k: v.double().numpy().copy() for k, v in vals.items()}
    cot = dy.double().numpy()

    def loss():
        q = {k: vals.get(k) for k in ("conv_weight", "conv_bias", "decay", "norm_weight", "norm_bias")}
        return float((cot * _oracle(q, group, False, vals["x"], vals["r"], vals["i"], vals["z"], lambda a: a)[3]).sum())

    rng = np.random.default_rng(0)
    for k, v in vals.items():
        d = rng.standard_normal(v.shape)
        d /= np.sqrt((d * d).sum())
        base = v.copy()
        eps = 1e-5
        v[...] = base + eps * d
        up = loss()
        v[...] = base - eps * d
        dn = loss()
        v[...] = base
        want = (up - dn) / (2 * eps)
        have = float((got[k].double().cpu().numpy() * d).sum())
        assert abs(have - want) <= 1e-4 * max(1.0, abs(want)), (k, have, want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prefill_then_tokens_match_the_whole_sequence(dtype):
    B, T, D, W = 3, 150, 128, 4
    p = _params(D, W, seed=9, bias=False)
    x, r, i, z, _ = (t.to(DEV) for t in _inputs(B, T, D, dtype, seed=5))
    blk = _block(p, 64, False)
    whole, end = blk(x, r, i, z)
    cut = lambda a, b: [t[:, a:b].contiguous() for t in (x, r, i, z)]  # noqa: E731
    y, st = blk(*cut(0, 40))
    parts = [y]
    y, st = blk(*cut(40, 140), state=st)          # a long continuation
    parts.append(y)
    y, st = blk(*cut(140, 144), state=st)         # a short one
    parts.append(y)
    for t in range(144, T):                       # tokens, in place
        parts.append(blk.step(*cut(t, t + 1), st))
    # The short forms round the conv's SiLU once from another (more exact) form of it: u may differ by a
    # bf16 step, which the tolerance of the block covers.
    tol = TOL[dtype]
    assert_close(torch.cat(parts, 1), whole, tol, tol, "y")
    assert_close(st.h, end.h, tol, tol, "state")
    assert torch.equal(st.conv, end.conv)


def test_short_sequences_and_new_state():
    D, W = 64, 4
    p = _params(D, W, seed=2, bias=False)
    blk = _block(p, 64, False)
    x, r, i, z, _ = (t.to(DEV) for t in _inputs(2, 2, D, BF, seed=1))
    _, st = blk(x, r, i, z)
    assert st.conv.shape == (2, 3, D) and (st.conv[:, 0] == 0).all() and torch.equal(st.conv[:, 1:], x)
    st0 = blk.new_state(2)
    ys = [blk.step(*(t[:, k:k + 1].contiguous() for t in (x, r, i, z)), st0) for k in range(2)]
    assert torch.equal(st0.conv, st.conv)
    assert_close(torch.cat(ys, 1), blk(x, r, i, z)[0], 1e-2, 1e-2, "y")


def test_training_step_and_decode_step_replay_in_graphs():
    B, T, D = 2, 200, 128
    p = _params(D, 4, seed=1, bias=False)
    blk = _block(p, 64, False)
    x, r, i, z, dy = (t.to(DEV) for t in _inputs(B, T, D, BF, seed=2))

    def train():
        y, st, saved = blk(x, r, i, z, want_grad=True)
        return [y, st.h, *blk.backward(saved, dy).values()]

    eager = train()
    tok = [t[:, :1].contiguous() for t in (x, r, i, z)]
    st_eager = blk.new_state(B)
    toks_eager = [blk.step(*tok, st_eager).clone() for _ in range(5)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1, stream=side):
            out = train()
        st = blk.new_state(B)
        with torch.cuda.graph(g2, stream=side):
            ytok = blk.step(*tok, st)
        got = []
        for k in range(5):
            g2.replay()
            got.append(ytok.clone())
            g1.replay()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, out))
    assert all(torch.equal(a, b) for a, b in zip(toks_eager, got)) and torch.equal(st.h, st_eager.h)


def test_two_streams_at_once():
    """Training steps of two blocks interleaved on two streams give what each gives alone."""
    blocks, ins, alone = [], [], []
    for k, (B, T, D) in enumerate(((1, 3000, 256), (6, 400, 512))):
        blocks.append(_block(_params(D, 4, seed=k, bias=False), 64, False))
        ins.append([t.to(DEV) for t in _inputs(B, T, D, BF, seed=k)])

    def step(k):
        x, r, i, z, dy = ins[k]
        y, st, saved = blocks[k](x, r, i, z, want_grad=True)
        return [y, st.h, *blocks[k].backward(saved, dy).values()]

    for k in range(2):
        alone.append(step(k))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(step(k))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(alone[k], g))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_inputs_are_left_as_they_are(dtype):
    """No call writes into what it is given, and passes on one state repeat with others in between."""
    from theorem_b200 import ops
    B, T, D = 2, 200, 72
    g = torch.Generator(DEV).manual_seed(0)
    rn = lambda *s, dt=dtype: torch.randn(*s, generator=g, device=DEV, dtype=dt)  # noqa: E731

    def make():
        f = torch.float32
        return dict(x=rn(B, T, D), r=rn(B, T, D), i=rn(B, T, D), dy=rn(B, T, D), h0=rn(B, D, dt=f), df=rn(B, D, dt=f),
                    decay=rn(D, dt=f).abs(), w=rn(D, dt=f), b=rn(D, dt=f), cw=rn(D, 4, dt=f), st=rn(B, 3, D))

    def run(s):
        y, fin, states = ops.gated_scan(s["x"], s["r"], s["i"], s["decay"], h0=s["h0"], want_states=True)
        kw = dict(gate=s["r"], activation="silu")
        return [y, fin, states,
                *ops.gated_scan_bwd(s["x"], s["r"], s["i"], s["decay"], states, s["dy"], dfinal=s["df"]),
                ops.group_norm(s["x"], 24, s["w"], s["b"], **kw),
                *ops.group_norm_bwd(s["x"], s["dy"], 24, s["w"], s["b"], **kw),
                *ops.causal_conv1d_step(s["x"][:, :8], s["st"], s["cw"], s["b"], activation="silu"),
                *ops.causal_conv1d_bwd(s["x"], s["cw"], s["b"], s["dy"], activation="silu")]

    one, two = make(), make()
    before = {k: v.clone() for k, v in one.items()}
    first = run(one)
    run(two)
    again = run(one)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert all(torch.equal(one[k], v) for k, v in before.items())


def test_arguments_by_name():
    from theorem_b200 import ops
    x = torch.randn(2, 40, 64, device=DEV)
    dec = torch.full((64,), 0.1, device=DEV)
    a = ops.gated_scan(x, x, x, dec)[0]
    assert torch.equal(a, ops.gated_scan(x=x, r=x, i=x, decay=dec)[0])
    assert torch.equal(ops.group_norm(x, 16), ops.group_norm(x=x, group=16))


@pytest.mark.parametrize("K", [128, 64])
@pytest.mark.parametrize("gated", [True, False])
def test_deltanet_layer_with_output_norm(K, gated):
    """chain.GatedDeltaNetForward with norm_weight: its own output, normed by the oracle."""
    from theorem_b200.chain import GatedDeltaNetForward
    B, T, H = 2, 128, 2
    d = deltanet_inputs(B, T, H, K, K, seed=K)
    D = H * K
    g = torch.Generator().manual_seed(K)
    xs = [torch.randn(B, T, D, generator=g).to(BF).to(DEV) for _ in range(3)]
    cw = [(torch.randn(D, 4, generator=g) * 0.5).to(DEV) for _ in range(3)]
    cb = [(torch.randn(D, generator=g) * 0.3).to(DEV) for _ in range(3)]
    beta, gg = d["beta"].to(DEV), d["g"].to(DEV)
    z = torch.randn(B, T, D, generator=g).to(BF) if gated else None
    w = 1 + 0.1 * torch.randn(K, generator=g)
    plain = GatedDeltaNetForward(H, K, K, cw, cb)
    normed = GatedDeltaNetForward(H, K, K, cw, cb, norm_weight=w.to(DEV))
    o, fin = plain(*xs, beta, gg)
    on, finn = normed(*xs, beta, gg, gate=None if z is None else z.to(DEV))
    assert torch.equal(fin, finn) and on.shape == o.shape
    ref = orc.group_norm(o.float().cpu().reshape(B, T, D), K, w.repeat(H), None, z, activation="silu" if gated else None,
                         center=False)
    assert_close(on.reshape(B, T, D).double().cpu(), _np(ref), 1e-2, 1e-2, "normed output")
    with pytest.raises(AssertionError):
        plain(*xs, beta, gg, gate=xs[0])


def test_refusals():
    from theorem_b200.recurrent import GatedRecurrentBlock
    p = {k: None if v is None else v.to(DEV) for k, v in _params(64, 4, 0, False).items()}
    with pytest.raises(AssertionError):
        GatedRecurrentBlock(**{**p, "conv_weight": torch.zeros(64, 9, device=DEV)})
    with pytest.raises(AssertionError):
        GatedRecurrentBlock(**{**p, "conv_weight": torch.zeros(66, 4, device=DEV)})
    blk = GatedRecurrentBlock(**p, norm_group=64)
    x = torch.zeros(1, 8, 64, device=DEV, dtype=BF)
    with pytest.raises(AssertionError):
        blk(x, x, x, x, state=blk.new_state(1), want_grad=True)
    with pytest.raises(AssertionError):
        blk(x[..., :32], x, x, x)
