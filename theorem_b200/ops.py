"""Functional host API over the C ABI (torch tensors in, torch tensors out).

Each function validates like the reference launcher it replaces (asserts on
device, dtype, contiguity and shape), allocates its outputs with
``torch.empty`` on the input's device, and launches on torch's current CUDA
stream. Nothing here computes on the CPU.
"""
from __future__ import annotations

import functools

import torch

from . import _lib as L

BT = 64
_ACT = {None: L.THM_ACT_NONE, "none": L.THM_ACT_NONE, "silu": L.THM_ACT_SILU}


def _on_input_device(fn):
    """Run the op with its first tensor argument's device current, so the
    launch (which goes to the current device) and the pointers agree even when
    the caller's current device is another GPU."""
    @functools.wraps(fn)
    def wrapped(*args, **kw):
        t = args[0] if args else None
        if not isinstance(t, torch.Tensor):
            t = next((a for a in (*args, *kw.values()) if torch.is_tensor(a)), None)
        if t is not None and t.is_cuda and t.get_device() != torch.cuda.current_device():
            with torch.cuda.device(t.device):
                return fn(*args, **kw)
        return fn(*args, **kw)
    return wrapped


def _on_gpu(x):
    """x is a CUDA tensor (the others are checked against its device)."""
    assert x.is_cuda, "theorem_b200 ops need CUDA tensors (there is no CPU fallback)"


def _cuda(*ts):
    for t in ts:
        if t is not None:
            assert t.is_cuda, "theorem_b200 ops need CUDA tensors (there is no CPU fallback)"


def _contig(*ts):
    for t in ts:
        if t is not None:
            assert t.is_contiguous(), "inputs must be contiguous"


@_on_input_device
def causal_conv1d(x, weight, bias, activation=None, layout: str = "bds", l2norm_group: int = 0,
                  out=None):
    """Depthwise causal conv (kernels/causal_conv1d/kernel.py:170-230 contract).

    layout "bds": x [B, D, S] fp32 (reference). layout "bsd": x [B, S, D] fp32 or
    bf16 (channel-last chain). weight [D, W], bias [D] fp32. Optional SiLU and
    per-``l2norm_group`` L2 norm (bsd only).
    """
    _cuda(x, weight, bias)
    _contig(x, weight, bias)
    assert weight.dtype == torch.float32 and bias.dtype == torch.float32, "weight/bias must be float32"
    assert x.dim() == 3, "x must be rank 3"
    if layout == "bds":
        B, D, S = x.shape
        lay = L.THM_LAYOUT_BDS
    elif layout == "bsd":
        B, S, D = x.shape
        lay = L.THM_LAYOUT_BSD
    else:
        raise AssertionError(f"unknown layout {layout!r}")
    Dw, W = weight.shape
    assert D == Dw, f"channel mismatch: x has D={D}, weight has D={Dw}"
    assert bias.shape == (D,), f"bias shape {tuple(bias.shape)} != ({D},)"
    if out is None:
        out = torch.empty_like(x)
    st = L.stream_of(x)
    L.check(L.load().thm_causal_conv1d_fwd(L.ptr(x), L.ptr(weight), L.ptr(bias), L.ptr(out), B, D, S, W,
                                           lay, L.dtype_code(x), _ACT[activation], int(l2norm_group), st),
            "thm_causal_conv1d_fwd")
    return out


@_on_input_device
def causal_conv1d_pair(x0, weight0, bias0, x1, weight1, bias1, activation=None, l2norm_group: int = 0,
                       out0=None, out1=None):
    """Two channel-last convs of the same shape in one launch (the layer's q and k
    projections): equal bit for bit to ``causal_conv1d(x0, weight0, bias0, activation,
    "bsd", l2norm_group)`` and the same for x1. x0, x1 [B, S, D] fp32 or bf16 of one
    dtype; weights [D, W] and biases [D] fp32. Returns (out0, out1)."""
    _cuda(x0, weight0, bias0, x1, weight1, bias1, out0, out1)
    _contig(x0, weight0, bias0, x1, weight1, bias1)
    for t in (weight0, bias0, weight1, bias1):
        assert t.dtype == torch.float32, "weight/bias must be float32"
    assert x0.dim() == 3 and x1.shape == x0.shape, "x0, x1 must be [B, S, D] of one shape"
    assert x1.dtype == x0.dtype and x1.device == x0.device, "x0, x1 must share dtype and device"
    B, S, D = x0.shape
    W = weight0.shape[1]
    for wt, bt in ((weight0, bias0), (weight1, bias1)):
        assert wt.shape == (D, W), f"weight shape {tuple(wt.shape)} != ({D}, {W})"
        assert bt.shape == (D,), f"bias shape {tuple(bt.shape)} != ({D},)"
    outs = []
    for o in (out0, out1):
        if o is None:
            o = torch.empty_like(x0)
        assert o.shape == x0.shape and o.dtype == x0.dtype and o.is_contiguous() and o.device == x0.device, \
            "out must match x in shape, dtype and device and be contiguous"
        outs.append(o)
    st = L.stream_of(x0)
    L.check(L.load().thm_causal_conv1d_pair_fwd(L.ptr(x0), L.ptr(weight0), L.ptr(bias0), L.ptr(outs[0]),
                                                L.ptr(x1), L.ptr(weight1), L.ptr(bias1), L.ptr(outs[1]),
                                                B, D, S, W, L.dtype_code(x0), _ACT[activation], int(l2norm_group), st),
            "thm_causal_conv1d_pair_fwd")
    return outs[0], outs[1]


@_on_input_device
def recompute_w_u(k, v, beta, A, g, a_mode: int = 0, w=None, u=None, A_out=None):
    """w = A (k beta e^g), u = A (v beta) per 64-chunk (kernels/recompute_w_u/kernel.py:192-248).

    a_mode 0 reads ``A`` [B,T,H,64] fp32; a_mode -1 / +1 computes
    A = (I -/+ M)^-1 in-kernel (``A`` may be None; ``A_out`` receives it).
    """
    _cuda(k, v, beta, A, g)
    _contig(k, v, beta, A, g)
    B, T, H, K = k.shape
    V = v.shape[-1]
    assert v.shape == (B, T, H, V) and v.dtype == k.dtype
    assert beta.shape == (B, T, H) and g.shape == (B, T, H)
    assert beta.dtype == torch.float32 and g.dtype == torch.float32, "beta / g must be float32"
    assert T % BT == 0, "T must be a multiple of BT (=64)"
    if a_mode == 0:
        assert A is not None and A.shape == (B, T, H, BT) and A.dtype == torch.float32
    w = torch.empty_like(k) if w is None else w
    u = torch.empty_like(v) if u is None else u
    st = L.stream_of(k)
    L.check(L.load().thm_recompute_w_u_fwd(L.ptr(k), L.ptr(v), L.ptr(beta), L.ptr(A) if a_mode == 0 else None,
                                           L.ptr(g), L.ptr(w), L.ptr(u), L.ptr(A_out), B, T, H, K, V,
                                           L.dtype_code(k), int(a_mode), st),
            "thm_recompute_w_u_fwd")
    return w, u


@_on_input_device
def recompute_w_u_conv(k, xv, conv_weight, conv_bias, beta, g, activation=None, a_mode: int = 1, w=None, u=None,
                       A_out=None):
    """recompute_w_u with v = act(causal_conv1d(xv)) formed in the same kernel.

    The layer's v projection ``xv`` [B,T,H*V] bf16 goes through the depthwise causal
    conv (``conv_weight`` [H*V, 4], ``conv_bias`` [H*V] fp32, optional SiLU) and straight
    into u = A (v beta): the chain kernels/causal_conv1d -> kernels/recompute_w_u
    (kernel.py:192-248) without v in HBM. a_mode +1 / -1 computes A in-kernel.
    """
    _cuda(k, xv, conv_weight, conv_bias, beta, g)
    _contig(k, xv, conv_weight, conv_bias, beta, g)
    B, T, H, K = k.shape
    assert k.dtype == torch.bfloat16 and xv.dtype == torch.bfloat16, "bf16 only"
    assert xv.dim() == 3 and xv.shape[:2] == (B, T) and xv.shape[2] % H == 0
    V = xv.shape[2] // H
    Dw, W = conv_weight.shape
    assert Dw == H * V and conv_bias.shape == (H * V,)
    assert conv_weight.dtype == torch.float32 and conv_bias.dtype == torch.float32, "conv weight/bias must be float32"
    assert beta.shape == (B, T, H) and g.shape == (B, T, H)
    assert beta.dtype == torch.float32 and g.dtype == torch.float32, "beta / g must be float32"
    assert T % BT == 0, "T must be a multiple of BT (=64)"
    assert a_mode in (1, -1), "the conv-fused path computes A in-kernel"
    w = torch.empty_like(k) if w is None else w
    u = torch.empty(B, T, H, V, device=k.device, dtype=k.dtype) if u is None else u
    for name, t, shape, dt in (("w", w, (B, T, H, K), k.dtype), ("u", u, (B, T, H, V), k.dtype),
                               ("A_out", A_out, (B, T, H, BT), torch.float32)):
        if t is not None:
            assert t.shape == shape and t.dtype == dt, f"{name} must be {tuple(shape)} {dt}"
            assert t.is_contiguous() and t.device == k.device, f"{name} must be contiguous on {k.device}"
    st = L.stream_of(k)
    L.check(L.load().thm_recompute_w_u_conv_fwd(L.ptr(k), L.ptr(xv), L.ptr(conv_weight), L.ptr(conv_bias),
                                                L.ptr(beta), L.ptr(g), L.ptr(w), L.ptr(u), L.ptr(A_out), B, T, H,
                                                K, V, W, _ACT[activation], int(a_mode), st),
            "thm_recompute_w_u_conv_fwd")
    return w, u


@_on_input_device
def chunk_fwd_h(k, v, g, w=None, h0=None, mode: int = 0, want_v_new: bool = False,
                want_final: bool = False, h=None, v_new=None, h_dtype=torch.float32, want_h: bool = True):
    """Inter-chunk state recurrence (kernels/chunk_fwd_h/kernel.py:141-191).

    mode 0: reference recurrence, returns h [B,NT,H,K,V] of post-update states.
    mode 1: gated delta rule (``v`` is u, ``w`` required), returns
    (h of states entering each chunk, v_new or None, final or None).
    h is stored in ``h_dtype`` (float32, or bfloat16 for the chain); the state
    itself is carried in fp32. ``want_h=False`` (mode 1) writes no per-chunk
    states and returns None for h.
    """
    _cuda(k, v, g, w, h0)
    _contig(k, v, g, w, h0)
    B, T, H, K = k.shape
    V = v.shape[-1]
    assert T % BT == 0, f"T={T} must be divisible by {BT}"
    assert v.shape == (B, T, H, V) and v.dtype == k.dtype and g.shape == (B, T, H)
    assert g.dtype == torch.float32
    NT = T // BT
    assert want_h or mode == 1, "the reference recurrence (mode 0) always returns h"
    if h is None and want_h:
        h = torch.empty(B, NT, H, K, V, device=k.device, dtype=h_dtype)
    if h is not None:
        assert h.shape == (B, NT, H, K, V) and h.dtype in (torch.float32, torch.bfloat16) and h.is_contiguous()
    final = None
    if mode == 1:
        assert w is not None and w.shape == k.shape and w.dtype == k.dtype
        if h0 is not None:
            assert h0.shape == (B, H, K, V) and h0.dtype == torch.float32
        if v_new is not None:
            assert v_new.shape == v.shape and v_new.dtype == v.dtype and v_new.is_contiguous()
        elif want_v_new:
            v_new = torch.empty_like(v)
        if want_final:
            final = torch.empty(B, H, K, V, device=k.device, dtype=torch.float32)
    else:
        assert w is None and h0 is None and v_new is None
    st = L.stream_of(k)
    L.check(L.load().thm_chunk_fwd_h_fwd(L.ptr(k), L.ptr(w), L.ptr(v), L.ptr(g), L.ptr(h0), L.ptr(h),
                                         L.ptr(v_new), L.ptr(final), B, T, H, K, V, L.dtype_code(k),
                                         L.dtype_code(h) if h is not None else L.dtype_code(k), int(mode), st),
            "thm_chunk_fwd_h_fwd")
    if mode == 1:
        return h, v_new, final
    return h


@_on_input_device
def chunk_fwd_o(q, k, v, g, h, scale: float, o=None):
    """Chunkwise output (kernels/chunk_fwd_o/kernel.py:146-212)."""
    _cuda(q, k, v, g, h)
    _contig(q, k, v, g, h)
    B, T, H, K = q.shape
    V = v.shape[-1]
    assert k.shape == q.shape and k.dtype == q.dtype and v.dtype == q.dtype
    assert v.shape == (B, T, H, V) and g.shape == (B, T, H) and g.dtype == torch.float32
    assert T % BT == 0, f"T={T} must be divisible by BT={BT}"
    NT = T // BT
    assert h.shape == (B, NT, H, K, V) and h.dtype in (torch.float32, torch.bfloat16), \
        "h must be [B,NT,H,K,V] float32 (or bfloat16 with bfloat16 q/k/v)"
    if o is None:
        o = torch.empty(B, T, H, V, dtype=q.dtype, device=q.device)
    st = L.stream_of(q)
    L.check(L.load().thm_chunk_fwd_o_fwd(L.ptr(q), L.ptr(k), L.ptr(v), L.ptr(g), L.ptr(h), L.ptr(o),
                                         float(scale), B, T, H, K, V, L.dtype_code(q), L.dtype_code(h), st),
            "thm_chunk_fwd_o_fwd")
    return o


@_on_input_device
def gated_delta_fwd_ho(q, k, w, u, g, scale: float, h0=None, want_final: bool = False, o=None):
    """chunk_fwd_h (delta rule) and chunk_fwd_o fused in one kernel: returns
    (o, final state or None). Same result as
    ``chunk_fwd_h(k, u, g, w=w, h0=h0, mode=1, want_v_new=True, h_dtype=bf16)``
    followed by ``chunk_fwd_o(q, k, v_new, g, h, scale)``, without writing h or
    v_new (kernels/chunk_fwd_h/kernel.py:141-191 + kernels/chunk_fwd_o/kernel.py:146-212).
    Built for bf16, K = V = 128."""
    _cuda(q, k, w, u, g, h0)
    _contig(q, k, w, u, g, h0)
    B, T, H, K = q.shape
    V = u.shape[-1]
    assert k.shape == q.shape and w.shape == q.shape and u.shape == (B, T, H, V)
    assert k.dtype == q.dtype and w.dtype == q.dtype and u.dtype == q.dtype
    assert g.shape == (B, T, H) and g.dtype == torch.float32
    assert T % BT == 0, f"T={T} must be divisible by BT={BT}"
    if h0 is not None:
        assert h0.shape == (B, H, K, V) and h0.dtype == torch.float32
    if o is None:
        o = torch.empty(B, T, H, V, dtype=q.dtype, device=q.device)
    assert o.shape == (B, T, H, V) and o.dtype == q.dtype and o.is_contiguous()
    final = torch.empty(B, H, K, V, device=q.device, dtype=torch.float32) if want_final else None
    st = L.stream_of(q)
    L.check(L.load().thm_gated_delta_fwd_ho(L.ptr(q), L.ptr(k), L.ptr(w), L.ptr(u), L.ptr(g), L.ptr(h0), L.ptr(o),
                                            L.ptr(final), float(scale), B, T, H, K, V, L.dtype_code(q), st),
            "thm_gated_delta_fwd_ho")
    return o, final


@_on_input_device
def sp_prefix_fold(Ms, Ss, x0=None, nout: int | None = None, out=None):
    """States entering consecutive segments: out[0] = x0 (or 0), out[r+1] =
    Ms[r] out[r] + Ss[r]. Ms [R, BH, K, K], Ss [R, BH, K, V], x0 [BH, K, V] fp32;
    returns out [nout, BH, K, V] (nout <= R + 1, default R + 1). One launch; the
    state of each (bh, 32-column tile) stays in shared memory across the steps."""
    _cuda(Ms, Ss, x0)
    _contig(Ms, Ss, x0)
    R, BH, K, V = Ss.shape
    assert Ms.shape == (R, BH, K, K), f"Ms shape {tuple(Ms.shape)} != {(R, BH, K, K)}"
    assert Ms.dtype == torch.float32 and Ss.dtype == torch.float32, "segment maps must be float32"
    if x0 is not None:
        assert x0.shape == (BH, K, V) and x0.dtype == torch.float32
    nout = R + 1 if nout is None else int(nout)
    assert 1 <= nout <= R + 1
    if out is None:
        out = torch.empty(nout, BH, K, V, device=Ss.device, dtype=torch.float32)
    assert out.shape == (nout, BH, K, V) and out.dtype == torch.float32 and out.is_contiguous()
    st = L.stream_of(Ss)
    L.check(L.load().thm_sp_prefix_fold(L.ptr(Ms), L.ptr(Ss), L.ptr(x0), L.ptr(out), nout, BH, K, V, st),
            "thm_sp_prefix_fold")
    return out


@_on_input_device
def build_A(k, beta, g, sign: int = -1, out=None):
    """Per-chunk WY matrix A = (I + sign*M)^-1, M = strict_tril(beta_i k_i.k_j e^{g_i-g_j})
    (kernels/recompute_w_u/reference.py:48-91 ``_build_A`` is sign = -1). Returns
    A [B,T,H,64] fp32 -- the ``A`` input of ``recompute_w_u`` with a_mode 0."""
    _cuda(k, beta, g)
    _contig(k, beta, g)
    B, T, H, K = k.shape
    assert T % BT == 0, f"T={T} must be divisible by BT={BT}"
    assert beta.shape == (B, T, H) and g.shape == (B, T, H)
    assert beta.dtype == torch.float32 and g.dtype == torch.float32
    assert sign in (-1, 1)
    if out is None:
        out = torch.empty(B, T, H, BT, device=k.device, dtype=torch.float32)
    assert out.shape == (B, T, H, BT) and out.dtype == torch.float32 and out.is_contiguous()
    st = L.stream_of(k)
    L.check(L.load().thm_build_A_fwd(L.ptr(k), L.ptr(beta), L.ptr(g), L.ptr(out), B, T, H, K, L.dtype_code(k),
                                     int(sign), st), "thm_build_A_fwd")
    return out


@_on_input_device
def chunk_local_cumsum(g_inc, scale: float = 1.0, out=None):
    """g[b, c*64+i, h] = scale * sum_{j<=i} g_inc[b, c*64+j, h] per 64-token chunk: the
    chunk-local cumulative gate the reference's generators build
    (kernels/chunk_fwd_h/reference.py:41-45). ``out`` may be ``g_inc`` (in place)."""
    _cuda(g_inc)
    _contig(g_inc)
    assert g_inc.dtype == torch.float32 and g_inc.dim() == 3, "g_inc must be [B,T,H] float32"
    B, T, H = g_inc.shape
    assert T % BT == 0, f"T={T} must be divisible by BT={BT}"
    if out is None:
        out = torch.empty_like(g_inc)
    assert out.shape == g_inc.shape and out.dtype == torch.float32 and out.is_contiguous()
    st = L.stream_of(g_inc)
    L.check(L.load().thm_chunk_local_cumsum_fwd(L.ptr(g_inc), L.ptr(out), B, T, H, float(scale), st),
            "thm_chunk_local_cumsum_fwd")
    return out


# ---------------------------------------------------------------------------
# Recurrent block: gated scan, group norm, the conv's carried-state form and gradients
# ---------------------------------------------------------------------------
# These calls serve single tokens too, where the launch takes 2 to 3 us on the GPU and the host
# sets the pace: the checks are plain comparisons, and messages are only formed on failure.
def _like(name, t, ref):
    """t's strides; t has ref's shape, dtype and device, and unit stride over channels."""
    assert t.shape == ref.shape and t.dtype is ref.dtype and t.get_device() == ref.get_device(), \
        f"{name} must be {tuple(ref.shape)} {ref.dtype} on {ref.device}"
    st = t.stride()
    assert st[-1] == 1 or t.shape[-1] <= 1, f"{name} must have unit stride over channels"
    return st


def _dense(name, t, ref, shape, dtype):
    """t is a contiguous ``shape`` of ``dtype`` on ref's device."""
    assert t.shape == shape and t.dtype is dtype and t.get_device() == ref.get_device() and t.is_contiguous(), \
        f"{name} must be a contiguous {tuple(shape)} {dtype} on {ref.device}"


def _empty(ref, shape, dtype):
    """An uninitialised contiguous tensor on ref's device (empty_like is the cheaper call)."""
    if ref.shape == shape and ref.dtype == dtype and ref.is_contiguous():
        return torch.empty_like(ref)
    return torch.empty(shape, dtype=dtype, device=ref.device)


def _channel_last(x):
    """x's strides; x is fp32 or bf16 with unit stride over channels."""
    assert x.dtype is torch.bfloat16 or x.dtype is torch.float32, f"unsupported dtype {x.dtype} (float32 or bfloat16)"
    st = x.stride()
    assert st[-1] == 1 or x.shape[-1] <= 1, "x must have unit stride over channels"
    return st


def _scan_args(x, r, i, decay, cu_seqlens):
    """(B, T, D, sequences, shape of the chunk states, batch and time strides of x, r, i)."""
    _on_gpu(x)
    shape = x.shape
    assert len(shape) == 3, "x must be [B, T, D]"
    strides = _channel_last(x)[:2] + _like("r", r, x)[:2] + _like("i", i, x)[:2]
    B, T, D = shape
    _dense("decay", decay, x, (D,), torch.float32)
    if cu_seqlens is None:
        return B, T, D, B, (B, (T + BT - 1) // BT, D), strides
    assert B == 1, "packed sequences share one batch entry: x must be [1, T, D]"
    assert cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 2, "cu_seqlens must hold N + 1 >= 2 row offsets"
    n = cu_seqlens.numel() - 1
    _dense("cu_seqlens", cu_seqlens, x, (n + 1,), torch.int32)
    return B, T, D, n, (B, T // BT + n, D), strides


@_on_input_device
def gated_scan(x, r, i, decay, h0=None, cu_seqlens=None, want_states: bool = False, y=None, final=None):
    """Per-channel gated linear recurrence over time (no reference counterpart: the
    per-channel sibling of ``chunk_fwd_h``), channel-last:

        a_t = exp(-decay sigmoid(r_t)),  h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t

    x, r, i [B, T, D] fp32 or bf16 of one dtype, unit stride over D, any strides over B and
    T; decay [D] fp32, finite and >= 0; h0 [N, D] fp32 (zeros if None). Any T: T = 1 with ``final=h0`` is
    the in-place single-token step. A token with r < -43 (sigmoid(r) < 2^-62, -inf) holds the
    state, whatever x and i hold there (pad a batch with it and ``final`` is each sequence's own).

    ``cu_seqlens`` [N + 1] int32: N packed sequences, rows cu[n] .. cu[n+1] of a batch of one,
    each from its h0; cu[0] may be > 0 and sequences may be empty (final = h0). Rows before the
    first sequence and behind the last are 0 in a fresh y and left as they are in a given one.

    Returns (y [B, T, D] in x's dtype, final [N, D] fp32, states). The state is carried in fp32; a
    given y must not overlap the inputs.
    ``want_states`` keeps the state entering each 64-token chunk for ``gated_scan_bwd``:
    [B, ceil(T / 64), D] fp32; packed, sequence n's start at slot cu[n] // 64 + n of
    [1, T // 64 + N, D] and unused slots are 0.
    """
    B, T, D, n, sshape, strides = _scan_args(x, r, i, decay, cu_seqlens)
    if h0 is not None:
        _dense("h0", h0, x, (n, D), torch.float32)
    fresh = y is None
    if fresh:
        y = _empty(x, x.shape, x.dtype)
    else:
        _dense("y", y, x, x.shape, x.dtype)
    if final is not None:
        _dense("final", final, x, (n, D), torch.float32)
    elif h0 is not None:
        final = torch.empty_like(h0)
    else:
        final = torch.empty(n, D, device=x.device, dtype=torch.float32)
    states = None
    if want_states:
        make = torch.zeros if cu_seqlens is not None else torch.empty
        states = make(sshape, device=x.device, dtype=torch.float32)
    ptr = L.ptr
    L.check(L.load().thm_gated_scan_fwd(x.data_ptr(), r.data_ptr(), i.data_ptr(), decay.data_ptr(), ptr(h0),
                                        ptr(cu_seqlens), y.data_ptr(), final.data_ptr(), ptr(states), *strides, B, T, D,
                                        n, int(fresh), L.dtype_code(x), L.stream_of(x)), "thm_gated_scan_fwd")
    return y, final, states


@_on_input_device
def gated_scan_bwd(x, r, i, decay, states, dy, dfinal=None, cu_seqlens=None, dx=None, dr=None, di=None):
    """Gradients of ``gated_scan``: (dx, dr, di [B, T, D] in x's dtype, ddecay [D], dh0 [N, D] fp32).

    ``states`` is what the forward pass returned for the same inputs with want_states; dy like
    y (any strides over B and T), dfinal [N, D] fp32 the gradient of ``final`` (None: zeros).
    Tokens that held the state (r < -43) get zero gradients. Rows that no sequence holds are
    treated as in ``gated_scan``. Sums over tokens are in fp32 in a fixed order, so results
    repeat bit for bit.
    """
    B, T, D, n, sshape, strides = _scan_args(x, r, i, decay, cu_seqlens)
    strides += _like("dy", dy, x)[:2]
    _dense("states", states, x, sshape, torch.float32)
    if dfinal is not None:
        _dense("dfinal", dfinal, x, (n, D), torch.float32)
    outs = (dx, dr, di)
    fresh = all(t is None for t in outs)
    assert fresh or all(t is not None for t in outs), "dx, dr, di are given together or not at all"
    if fresh:
        dx, dr, di = (_empty(x, x.shape, x.dtype) for _ in range(3))
    else:
        for name, t in zip(("dx", "dr", "di"), outs):
            _dense(name, t, x, x.shape, x.dtype)
    ddecay = torch.empty_like(decay)
    dh0 = torch.empty(n, D, device=x.device, dtype=torch.float32) if dfinal is None else torch.empty_like(dfinal)
    parts = L.load().thm_gated_scan_bwd_parts(T, D, n, int(cu_seqlens is not None), L.dtype_code(x))
    work = torch.empty(parts, D, device=x.device, dtype=torch.float32)
    L.check(L.load().thm_gated_scan_bwd(L.ptr(x), L.ptr(r), L.ptr(i), L.ptr(decay), L.ptr(states), L.ptr(dy),
                                        L.ptr(dfinal), L.ptr(cu_seqlens), L.ptr(dx), L.ptr(dr), L.ptr(di),
                                        L.ptr(ddecay), L.ptr(dh0), L.ptr(work), *strides, B, T, D, n, int(fresh),
                                        L.dtype_code(x), L.stream_of(x)), "thm_gated_scan_bwd")
    return dx, dr, di, ddecay, dh0


def _rows(name, t):
    """(rows, row stride) of a [..., C] tensor whose leading dimensions collapse to one."""
    C = t.shape[-1]
    if t.is_contiguous():
        return (t.numel() // C if C else 0), C
    rows, stride = 1, None
    for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size != 1:
            assert stride is None or rows == 0 or st == stride * rows, \
                f"{name}'s leading dimensions must collapse to rows"
            stride = st if stride is None else stride
        rows *= size
    return rows, (C if stride is None else stride)


def _norm_args(x, group, weight, bias, gate, activation):
    _on_gpu(x)
    assert x.dim() >= 1, "x must be [..., C]"
    _channel_last(x)
    C = x.shape[-1]
    assert group >= 1 and C % group == 0, f"C={C} is not a multiple of the group size {group}"
    if gate is not None:
        _like("gate", gate, x)
    if weight is not None:
        _dense("weight", weight, x, (C,), torch.float32)
    if bias is not None:
        _dense("bias", bias, x, (C,), torch.float32)
    assert activation in _ACT, f"unknown activation {activation!r}"
    return C


@_on_input_device
def group_norm(x, group: int, weight=None, bias=None, gate=None, activation=None, center: bool = True,
               eps: float = 1e-5, out=None):
    """Norm over runs of ``group`` consecutive channels of each token, channel-last (no
    reference counterpart; torch's group_norm on [tokens, C] with C / group groups):

        u = xh weight + bias,  y = act(u),  or y = u act(gate) with a gate

    xh = (x - mean) / sqrt(var + eps), or x / sqrt(mean(x^2) + eps) with ``center=False``
    (RMS norm per head). x, gate [..., C] fp32 or bf16 of one dtype, unit stride over C, the
    leading dimensions collapsible to rows (any row stride); weight, bias [C] fp32 or None;
    activation None or "silu"; group <= 4096. Statistics in fp32, variance from centred
    values. Returns y, contiguous, like x; ``out`` may be x or gate (in place).
    """
    C = _norm_args(x, group, weight, bias, gate, activation)
    R, xs = _rows("x", x)
    zs = _rows("gate", gate)[1] if gate is not None else 0
    if out is None:
        out = _empty(x, x.shape, x.dtype)
    else:
        _dense("out", out, x, x.shape, x.dtype)
    L.check(L.load().thm_group_norm_fwd(L.ptr(x), L.ptr(gate), L.ptr(weight), L.ptr(bias), L.ptr(out), xs, zs, R, C,
                                        int(group), int(bool(center)), _ACT[activation], float(eps), L.dtype_code(x),
                                        L.stream_of(x)), "thm_group_norm_fwd")
    return out


@_on_input_device
def group_norm_bwd(x, dy, group: int, weight=None, bias=None, gate=None, activation=None, center: bool = True,
                   eps: float = 1e-5):
    """Gradients of ``group_norm``: (dx, dgate, dweight, dbias), None for what was None.

    Statistics are recomputed from x; dweight and dbias are fp32 sums over all tokens in a
    fixed order, so results repeat bit for bit.
    """
    C = _norm_args(x, group, weight, bias, gate, activation)
    _like("dy", dy, x)
    R, xs = _rows("x", x)
    gs = _rows("dy", dy)[1]
    zs = _rows("gate", gate)[1] if gate is not None else 0
    dev = x.device
    dx = _empty(x, x.shape, x.dtype)
    dgate = _empty(x, x.shape, x.dtype) if gate is not None else None
    dweight = torch.empty_like(weight) if weight is not None else None
    dbias = torch.empty_like(bias) if bias is not None else None
    work = None
    if weight is not None or bias is not None:
        work = torch.empty(L.load().thm_group_norm_bwd_parts(R, C, int(group)), 2, C, device=dev, dtype=torch.float32)
    L.check(L.load().thm_group_norm_bwd(L.ptr(x), L.ptr(gate), L.ptr(weight), L.ptr(bias), L.ptr(dy), L.ptr(dx),
                                        L.ptr(dgate), L.ptr(dweight), L.ptr(dbias), L.ptr(work), xs, zs, gs, R, C,
                                        int(group), int(bool(center)), _ACT[activation], float(eps), L.dtype_code(x),
                                        L.stream_of(x)), "thm_group_norm_bwd")
    return dx, dgate, dweight, dbias


def _conv_args(x, weight, bias, activation):
    _on_gpu(x)
    assert x.dim() == 3, "x must be [B, S, D]"
    strides = _channel_last(x)[:2]
    B, S, D = x.shape
    assert weight.dim() == 2 and weight.shape[1] >= 1, "weight must be [D, W]"
    W = weight.shape[1]
    _dense("weight", weight, x, (D, W), torch.float32)
    _dense("bias", bias, x, (D,), torch.float32)
    assert activation in _ACT, f"unknown activation {activation!r}"
    return B, S, D, W, strides


@_on_input_device
def causal_conv1d_step(x, state, weight, bias, activation=None, out=None, state_out=None):
    """``causal_conv1d(..., "bsd")`` continued from the inputs before x, for decoding:
    x [B, S, D] (S <= 64: one token, a few drafted ones), state [B, W - 1, D] in x's dtype.

    Returns (out [B, S, D], the state after x: the last W - 1 rows of [state; x]).
    ``state_out`` may be ``state`` (in place). A zero state is a sequence's start; after a
    prefill it is the last W - 1 rows of its input. x has unit stride over D, any strides over
    B and S; W <= 8; weight, bias fp32 (kernels/causal_conv1d/kernel.py:170-230 from zeros).
    """
    B, S, D, W, strides = _conv_args(x, weight, bias, activation)
    assert S <= 64, f"S={S}: the carried-state form takes at most 64 tokens (causal_conv1d takes long runs)"
    _dense("state", state, x, (B, W - 1, D), x.dtype)
    if out is None:
        out = _empty(x, x.shape, x.dtype)
    else:
        _dense("out", out, x, x.shape, x.dtype)
    if state_out is None:
        state_out = torch.empty_like(state)
    else:
        _dense("state_out", state_out, x, (B, W - 1, D), x.dtype)
    L.check(L.load().thm_causal_conv1d_step(L.ptr(x), L.ptr(state), L.ptr(weight), L.ptr(bias), L.ptr(out),
                                            L.ptr(state_out), *strides, B, S, D, W, L.dtype_code(x),
                                            _ACT[activation], L.stream_of(x)), "thm_causal_conv1d_step")
    return out, state_out


@_on_input_device
def causal_conv1d_bwd(x, weight, bias, dy, activation=None):
    """Gradients of ``causal_conv1d(x, weight, bias, activation, "bsd")`` without the L2
    norm: (dx [B, S, D] in x's dtype, dweight [D, W], dbias [D] fp32).

    x, dy [B, S, D] fp32 or bf16 of one dtype, unit stride over D, any strides over B and S;
    W <= 8. Sums over tokens are in fp32 in a fixed order, so results repeat bit for bit.
    """
    B, S, D, W, strides = _conv_args(x, weight, bias, activation)
    strides += _like("dy", dy, x)[:2]
    dx = _empty(x, x.shape, x.dtype)
    dweight, dbias = torch.empty_like(weight), torch.empty_like(bias)
    parts = L.load().thm_causal_conv1d_bwd_parts(B, S, D)
    work = torch.empty(max(parts, 0), W + 1, D, device=x.device, dtype=torch.float32)
    L.check(L.load().thm_causal_conv1d_bwd(L.ptr(x), L.ptr(weight), L.ptr(bias), L.ptr(dy), L.ptr(dx), L.ptr(dweight),
                                           L.ptr(dbias), L.ptr(work), *strides, B, S, D, W, L.dtype_code(x), _ACT[activation],
                                           L.stream_of(x)), "thm_causal_conv1d_bwd")
    return dx, dweight, dbias
