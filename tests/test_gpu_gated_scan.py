"""GPU parity of gated_scan and gated_scan_bwd against the float64 oracle, within the bounds of
tests/recurrent_ref.py."""
import numpy as np
import pytest
import torch

from oracle import ops as orc
from tests import recurrent_ref as rr

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _inputs(B, T, D, dtype, seed, n=None, spread=4.6):
    g = torch.Generator().manual_seed(seed)
    x, r, i, dy = (torch.randn(B, T, D, generator=g).to(dtype) for _ in range(4))
    decay = torch.exp(torch.rand(D, generator=g) * spread - 4.8)
    h0, df = (torch.randn(n or B, D, generator=g) for _ in range(2))
    return x, r, i, decay, h0, dy, df


def _d(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _check_fwd(x, r, i, decay, h0, out, dtype, what=""):
    y, fin, st = out
    ry, rf, rs = orc.gated_scan(x, r, i, decay, h0)
    e = rr.scan_errors(x, r, i, decay, h0, dtype)
    B, T, D = ry.shape
    rr.assert_within(y, ry, rr.rounded(e["E"], ry, dtype), what + "y")
    ef = e["E"][:, -1] if T else np.zeros((B, D))
    rr.assert_within(fin, rf, ef, what + "final")
    if st is not None:
        es = np.concatenate([np.zeros((B, 1, D)), e["E"][:, 63:T - 1:64]], 1) if T else np.zeros((B, 0, D))
        rr.assert_within(st, rs, es, what + "states")


def _check_bwd(x, r, i, decay, h0, dy, df, out, dtype, what=""):
    ref, bounds = rr.scan_bwd_bounds(x, r, i, decay, h0, dy, df, dtype)
    for name, o, rf, bd in zip(("dx", "dr", "di", "ddecay", "dh0"), out, ref, bounds):
        rr.assert_within(o, rf, bd, what + name)


SHAPES = [
    (1, 1, 1), (2, 1, 64), (64, 1, 200), (3, 2, 66), (1, 7, 63), (2, 33, 65), (2, 63, 128), (2, 64, 128), (1, 65, 130),
    (3, 127, 72), (2, 200, 321), (1, 513, 64), (1, 1030, 96), (2, 2047, 40), (1, 4097, 2), (70, 130, 64), (1, 700, 2050),
    (70000, 1, 8), (16, 321, 2048), (300, 47, 130), (300, 49, 130), (2, 4, 70), (2, 14, 70), (2, 15, 70), (1, 4200, 64), (2, 2500, 72),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_matches_oracle(B, T, D, dtype):
    from theorem_b200 import ops
    x, r, i, decay, h0, dy, df = _inputs(B, T, D, dtype, seed=B * 1000 + T + D)
    dx, dr_, di, dd, dh0, ddy, ddf = _d(x, r, i, decay, h0, dy, df)
    out = ops.gated_scan(dx, dr_, di, dd, h0=dh0, want_states=True)
    _check_fwd(x, r, i, decay, h0, out, dtype)
    grads = ops.gated_scan_bwd(dx, dr_, di, dd, out[2], ddy, dfinal=ddf)
    _check_bwd(x, r, i, decay, h0, dy, df, grads, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [3, 300])
def test_decays_past_the_plain_range(T, dtype):
    """Decays over 1 and under 1e-6, in some warps' channels only and in all of one's."""
    from theorem_b200 import ops
    B, D = 2, 200
    x, r, i, decay, h0, dy, df = _inputs(B, T, D, dtype, seed=T)
    decay[:64] *= 20.0
    decay[70] = 3.0
    decay[130] = 1e-7
    args = _d(x, r, i, decay)
    out = ops.gated_scan(*args, h0=h0.to(DEV), want_states=True)
    _check_fwd(x, r, i, decay, h0, out, dtype)
    grads = ops.gated_scan_bwd(*args, out[2], dy.to(DEV), dfinal=df.to(DEV))
    _check_bwd(x, r, i, decay, h0, dy, df, grads, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [5, 200])
def test_large_decay_behind_a_closed_gate(T, dtype):
    """A decay of hundreds with a nearly closed gate is an ordinary memory: decay sigmoid(r) counts,
    not decay."""
    from theorem_b200 import ops
    B, D = 2, 64
    x, r, i, decay, h0, dy, df = _inputs(B, T, D, dtype, seed=T)
    decay = 100.0 + 40.0 * torch.arange(D).float()
    r = (r - 8.0).to(dtype)
    args = _d(x, r, i, decay)
    out = ops.gated_scan(*args, h0=h0.to(DEV), want_states=True)
    _check_fwd(x, r, i, decay, h0, out, dtype)
    grads = ops.gated_scan_bwd(*args, out[2], dy.to(DEV), dfinal=df.to(DEV))
    _check_bwd(x, r, i, decay, h0, dy, df, grads, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 100])
def test_defaults_without_h0_and_dfinal(T, dtype):
    from theorem_b200 import ops
    x, r, i, decay, _, dy, _ = _inputs(2, T, 96, dtype, seed=T)
    dx, dr_, di, dd, ddy = _d(x, r, i, decay, dy)
    y, fin, none = ops.gated_scan(dx, dr_, di, dd)
    assert none is None
    _check_fwd(x, r, i, decay, None, (y, fin, None), dtype)
    st = ops.gated_scan(dx, dr_, di, dd, want_states=True)[2]
    _check_bwd(x, r, i, decay, None, dy, None, ops.gated_scan_bwd(dx, dr_, di, dd, st, ddy), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 5, 300])
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_strided_and_unaligned_inputs(T, shift, dtype):
    """Slices of a wider projection, a transposed batch, an address off any vector."""
    from theorem_b200 import ops
    B, D = 3, 70
    x, r, i, decay, h0, dy, df = _inputs(B, T, D, dtype, seed=T * 10 + shift)
    wide = torch.zeros(B, T, 3 * D + 5, dtype=dtype, device=DEV)
    views = []
    for k, t in enumerate((x, r, i)):
        v = wide[..., shift + k * D: shift + (k + 1) * D]
        v.copy_(t.to(DEV))
        views.append(v)
    gy = dy.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)  # [T, B, D] storage
    assert gy.stride(1) == B * D or T == 1
    out = ops.gated_scan(*views, decay.to(DEV), h0=h0.to(DEV), want_states=True)
    _check_fwd(x, r, i, decay, h0, out, dtype)
    grads = ops.gated_scan_bwd(*views, decay.to(DEV), out[2], gy, dfinal=df.to(DEV))
    _check_bwd(x, r, i, decay, h0, dy, df, grads, dtype)


@pytest.mark.parametrize("T", [65, 1100])
def test_time_major_and_expanded_inputs(T):
    """A [T, B, D] tensor seen as [B, T, D], and a gate that all sequences share (stride 0)."""
    from theorem_b200 import ops
    B, D = 3, 64
    x, r, i, decay, h0, dy, df = _inputs(B, T, D, BF, seed=T)
    i = i[:1].expand(B, T, D)
    tm = [t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1) for t in (x, r, dy)]
    ie = i[:1].to(DEV).expand(B, T, D)
    out = ops.gated_scan(tm[0], tm[1], ie, decay.to(DEV), h0=h0.to(DEV), want_states=True)
    assert out[0].is_contiguous()
    _check_fwd(x, r, i, decay, h0, out, BF)
    grads = ops.gated_scan_bwd(tm[0], tm[1], ie, decay.to(DEV), out[2], tm[2], dfinal=df.to(DEV))
    _check_bwd(x, r, i, decay, h0, dy, df, grads, BF)


@pytest.mark.parametrize("T", [1, 40, 3000])
def test_final_in_place_of_h0(T):
    """Short runs, single blocks and chains of blocks: the state moves on in its own buffer."""
    from theorem_b200 import ops
    x, r, i, decay, h0, _, _ = _inputs(1, T, 128, BF, seed=T)
    args = _d(x, r, i, decay)
    y, fin, _ = ops.gated_scan(*args, h0=h0.to(DEV))
    st = h0.to(DEV)
    y2, fin2, _ = ops.gated_scan(*args, h0=st, final=st)
    assert fin2 is st and torch.equal(st, fin) and torch.equal(y, y2)


def test_offsets_past_32_bits():
    """More than 2^31 elements a tensor: the last rows equal the same rows run on their own from the
    chunk state that entered them, and so do their gradients."""
    from theorem_b200 import ops
    D, tail = 2048, 640
    T = (1 << 20) + 64 * 17
    assert T * D > 1 << 31
    x = torch.randn(1, T, D, device=DEV, dtype=BF, generator=torch.Generator(DEV).manual_seed(0))
    dec = torch.full((D,), 0.2, device=DEV)
    y, fin, st = ops.gated_scan(x, x, x, dec, want_states=True)
    xt = x[:, -tail:]
    y2, fin2, st2 = ops.gated_scan(xt, xt, xt, dec, h0=st[:, -tail // 64].contiguous(), want_states=True)
    e = 1e-5  # two orders of the same fp32 sums; y also by one bf16 step of its value
    assert (fin - fin2).abs().max() <= e and (st[:, -tail // 64:] - st2).abs().max() <= e
    assert ((y[:, -tail:].float() - y2.float()).abs() <= e + 2 ** -7 * y2.float().abs()).all()
    del y, y2
    df = torch.ones(1, D, device=DEV)
    a = ops.gated_scan_bwd(x, x, x, dec, st, x, dfinal=df)
    b = ops.gated_scan_bwd(xt, xt, xt, dec, st2, xt, dfinal=df)
    for p, q in zip(a[:3], b[:3]):
        assert ((p[:, -tail:].float() - q.float()).abs() <= e + 2 ** -7 * q.float().abs()).all()


PACKS = [  # row offsets, rows
    ([0, 1, 2, 3], 3), ([0, 0, 0], 5), ([0, 64, 64, 191, 200], 200), ([3, 10, 10, 75, 331], 400),
    ([0, 129, 130, 700, 701], 777), ([0, 1500], 1500),
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("off,T", PACKS)
@pytest.mark.parametrize("given", [False, True])
def test_packed_sequences(off, T, dtype, given):
    from theorem_b200 import ops
    D, n = 72, len(off) - 1
    x, r, i, decay, h0, dy, df = _inputs(1, T, D, dtype, seed=T + n, n=n)
    cu = torch.tensor(off, dtype=torch.int32, device=DEV)
    mark = -7.0
    full = lambda: torch.full((1, T, D), mark, dtype=dtype, device=DEV)  # noqa: E731
    args = _d(x, r, i, decay)
    y, fin, st = ops.gated_scan(*args, h0=h0.to(DEV), cu_seqlens=cu, want_states=True, y=full() if given else None)
    outs = [full() for _ in range(3)] if given else [None] * 3
    grads = ops.gated_scan_bwd(*args, st, dy.to(DEV), dfinal=df.to(DEV), cu_seqlens=cu, dx=outs[0], dr=outs[1],
                               di=outs[2])
    assert st.shape == (1, T // 64 + n, D)
    rest = torch.ones(T, dtype=torch.bool)
    used = torch.zeros(st.shape[1], dtype=torch.bool)
    dd, dd_bound = 0.0, 0.0
    for k, (a, b) in enumerate(zip(off, off[1:])):
        rest[a:b] = False
        sl = slice(a, b)
        nc = (b - a + 63) // 64
        slot = slice(a // 64 + k, a // 64 + k + nc)
        used[slot] = True
        one = (x[:, sl], r[:, sl], i[:, sl], decay, h0[k:k + 1])
        _check_fwd(*one, (y[:, sl], fin[k:k + 1], st[:, slot]), dtype, f"sequence {k} ")
        ref, bd = rr.scan_bwd_bounds(*one, dy[:, sl], df[k:k + 1], dtype)
        for name, o, rf, bb in zip(("dx", "dr", "di"), grads[:3], ref, bd):
            rr.assert_within(o[:, sl], rf, bb, f"sequence {k} {name}")
        rr.assert_within(grads[4][k:k + 1], ref[4], bd[4], f"sequence {k} dh0")
        dd, dd_bound = dd + ref[3], dd_bound + bd[3] + n * rr.U * np.abs(ref[3])
    rr.assert_within(grads[3], dd + np.zeros(D), dd_bound + np.zeros(D), "ddecay")
    for t in (y, *grads[:3]):
        assert (t[:, rest.to(DEV)] == (mark if given else 0.0)).all(), "rows of no sequence"
    assert (st[:, ~used.to(DEV)] == 0).all()


def test_out_of_range_offsets_are_clamped():
    """Offsets past the rows, or descending, touch nothing outside the tensors: the rows that
    they do name give the clamped sequences' results."""
    from theorem_b200 import ops
    T, D = 100, 64
    x, r, i, decay, h0, _, _ = _inputs(1, T, D, F32, seed=5, n=2)
    cu = torch.tensor([-4, 70, 5000], dtype=torch.int32, device=DEV)
    y, fin, _ = ops.gated_scan(*_d(x, r, i, decay), h0=h0.to(DEV), cu_seqlens=cu)
    good = torch.tensor([0, 70, 100], dtype=torch.int32, device=DEV)
    y2, fin2, _ = ops.gated_scan(*_d(x, r, i, decay), h0=h0.to(DEV), cu_seqlens=good)
    assert torch.equal(y, y2) and torch.equal(fin, fin2)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [4, 150])
def test_held_tokens_ignore_what_they_hold(T, dtype):
    """r = -inf holds the state: padding may hold NaN and infinities, and its gradients are 0."""
    from theorem_b200 import ops
    B, D = 3, 66
    x, r, i, decay, h0, dy, df = _inputs(B, T, D, dtype, seed=T)
    lens = [T, T // 2, 0]
    for b, ln in enumerate(lens):
        r[b, ln:] = -float("inf")
        x[b, ln:] = float("nan")
        x[b, ln:, ::2] = float("inf")
        i[b, ln:] = float("nan")
    args = _d(x, r, i, decay)
    out = ops.gated_scan(*args, h0=h0.to(DEV), want_states=True)
    _check_fwd(x, r, i, decay, h0, out, dtype)
    assert torch.equal(out[1][2].cpu(), h0[2])
    grads = ops.gated_scan_bwd(*args, out[2], dy.to(DEV), dfinal=df.to(DEV))
    _check_bwd(x, r, i, decay, h0, dy, df, grads, dtype)
    for b, ln in enumerate(lens):
        for g in grads[:3]:
            assert (g[b, ln:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_extreme_gates(dtype):
    """Gates at the ends of their range: saturated logits, long and no memory, tiny decay, 0."""
    from theorem_b200 import ops
    B, T, D = 2, 140, 64
    x, r, i, decay, h0, dy, df = _inputs(B, T, D, dtype, seed=9)
    r[:, ::7] = 30.0
    r[:, 1::7] = -30.0
    r[:, 2::11] = -100.0
    r[:, 3::11] = float("inf")
    i[:, ::5] = -40.0
    i[:, 1::5] = 60.0
    i[:, 2::13] = -float("inf")
    decay[:8] = 50.0
    decay[8:16] = 1e-4
    decay[16:24] = 1e-6
    decay[24:32] = 0.0
    args = _d(x, r, i, decay)
    out = ops.gated_scan(*args, h0=h0.to(DEV), want_states=True)
    _check_fwd(x, r, i, decay, h0, out, dtype)
    grads = ops.gated_scan_bwd(*args, out[2], dy.to(DEV), dfinal=df.to(DEV))
    assert all(torch.isfinite(g).all() for g in grads)
    _check_bwd(x, r, i, decay, h0, dy, df, grads, dtype)


def test_nan_spreads_only_along_its_own_channel():
    from theorem_b200 import ops
    x, r, i, decay, h0, _, _ = _inputs(2, 200, 64, BF, seed=1)
    clean = ops.gated_scan(*_d(x, r, i, decay), h0=h0.to(DEV))[0]
    x[1, 100, 5] = float("nan")
    y = ops.gated_scan(*_d(x, r, i, decay), h0=h0.to(DEV))[0]
    nan = torch.isnan(y)
    want = torch.zeros_like(nan)
    want[1, 100:, 5] = True
    assert torch.equal(nan, want) and torch.equal(y[~want], clean[~want])


def test_token_by_token_in_place_continues_the_long_pass():
    from theorem_b200 import ops
    B, T, D = 4, 130, 130
    x, r, i, decay, h0, _, _ = _inputs(B, T, D, BF, seed=3)
    args = _d(x, r, i)
    dec, state = decay.to(DEV), h0.to(DEV)
    y, fin, _ = ops.gated_scan(*(t[:, :100] for t in args), dec, h0=state, final=state)
    assert fin.data_ptr() == state.data_ptr()
    parts = [y]
    for t in range(100, T):
        y1, _, _ = ops.gated_scan(*(a[:, t:t + 1] for a in args), dec, h0=state, final=state)
        parts.append(y1)
    _check_fwd(x, r, i, decay, h0, (torch.cat(parts, 1), state, None), BF)


def test_zero_tokens():
    from theorem_b200 import ops
    e = torch.empty(3, 0, 40, device=DEV, dtype=BF)
    h0 = torch.randn(3, 40, device=DEV)
    dec = torch.ones(40, device=DEV)
    y, fin, st = ops.gated_scan(e, e, e, dec, h0=h0, want_states=True)
    assert y.shape == e.shape and torch.equal(fin, h0) and st.shape == (3, 0, 40)
    assert (ops.gated_scan(e, e, e, dec)[1] == 0).all()
    df = torch.randn(3, 40, device=DEV)
    dx, dr, di, dd, dh0 = ops.gated_scan_bwd(e, e, e, dec, st, e, dfinal=df)
    assert dx.shape == e.shape and (dd == 0).all() and torch.equal(dh0, df)
    e = torch.empty(0, 8, 40, device=DEV, dtype=BF)
    y, fin, st = ops.gated_scan(e, e, e, dec, want_states=True)
    assert y.shape == e.shape and fin.shape == (0, 40)
    assert (ops.gated_scan_bwd(e, e, e, dec, st, e)[3] == 0).all()


def test_repeats_bit_for_bit_and_replays_in_a_graph():
    from theorem_b200 import ops
    x, r, i, decay, h0, dy, df = _d(*_inputs(2, 700, 320, BF, seed=8))

    def step():
        y, fin, st = ops.gated_scan(x, r, i, decay, h0=h0, want_states=True)
        return (y, fin, st, *ops.gated_scan_bwd(x, r, i, decay, st, dy, dfinal=df))

    a, b = step(), step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step())
            graphs.append(g)
        for g in graphs:
            g.replay()
        for _ in range(3):
            graphs[1].replay()
            graphs[0].replay()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(a, o))


def test_refusals():
    from theorem_b200 import ops
    x = torch.zeros(2, 8, 16, device=DEV)
    dec = torch.ones(16, device=DEV)
    cu = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    st = torch.zeros(2, 1, 16, device=DEV)
    bad = [
        lambda: ops.gated_scan(x.half(), x.half(), x.half(), dec),
        lambda: ops.gated_scan(x, x.bfloat16(), x, dec),
        lambda: ops.gated_scan(x, x[:, :4], x, dec),
        lambda: ops.gated_scan(x[0], x[0], x[0], dec),
        lambda: ops.gated_scan(x, x, x, dec.double()),
        lambda: ops.gated_scan(x, x, x, dec[:8]),
        lambda: ops.gated_scan(x, x, x, dec, h0=torch.zeros(3, 16, device=DEV)),
        lambda: ops.gated_scan(x, x, x, dec, h0=torch.zeros(2, 16, device=DEV, dtype=torch.bfloat16)),
        lambda: ops.gated_scan(x.transpose(1, 2), x.transpose(1, 2), x.transpose(1, 2), torch.ones(8, device=DEV)),
        lambda: ops.gated_scan(x, x, x, dec, cu_seqlens=cu),              # two batch entries
        lambda: ops.gated_scan(x[:1], x[:1], x[:1], dec, cu_seqlens=cu.long()),
        lambda: ops.gated_scan(x[:1], x[:1], x[:1], dec, cu_seqlens=cu[:1]),
        lambda: ops.gated_scan(x[:1], x[:1], x[:1], dec, cu_seqlens=cu.cpu()),
        lambda: ops.gated_scan(x, x, x, dec, y=torch.zeros(2, 8, 32, device=DEV)[..., :16]),
        lambda: ops.gated_scan(x, x, x, dec, final=torch.zeros(2, 16, device=DEV, dtype=torch.float64)),
        lambda: ops.gated_scan_bwd(x, x, x, dec, st[:1], x),
        lambda: ops.gated_scan_bwd(x, x, x, dec, st, x.bfloat16()),
        lambda: ops.gated_scan_bwd(x, x, x, dec, st, x, dx=torch.zeros_like(x)),
        lambda: ops.gated_scan_bwd(x, x, x, dec, st, x, dfinal=torch.zeros(2, 8, device=DEV)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"refusal {k} did not raise")
