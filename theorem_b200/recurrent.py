"""The gated recurrent block: causal conv -> gated scan -> gated group norm, for training and serving.

The per-channel sibling of ``chain.GatedDeltaNetForward`` (no reference counterpart; the reference's
conv is kernels/causal_conv1d, forward only):

    u = act(conv(x))                      depthwise causal conv, width W
    a = exp(-decay sigmoid(r))            per channel and token
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) u_t
    y = norm_group(h) w (+ b) * silu(z)

x, r, i, z are channel-last projections [B, T, D] of one dtype (fp32 or bf16), which the caller's
linear layers make; r, i and z may be slices of a wider projection. Every call is a few launches on
torch's current stream, captures into CUDA graphs, and keeps nothing between calls but what it
returns. There is no autograd through these ops: ``backward`` returns the gradients.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops


@dataclass
class RecurrentState:
    """What a sequence carries on: the last W - 1 conv inputs [B, W - 1, D] in x's dtype and the
    scan's state [B, D] fp32."""
    conv: torch.Tensor
    h: torch.Tensor


class GatedRecurrentBlock:
    """Holds the parameters: conv_weight [D, W], conv_bias [D], decay [D] >= 0, norm_weight [D],
    norm_bias [D] or None, all fp32; ``norm_group`` channels share a norm (RMS unless ``center``)."""

    def __init__(self, conv_weight, conv_bias, decay, norm_weight, norm_bias=None, norm_group: int = 128,
                 activation: str | None = "silu", center: bool = False, eps: float = 1e-5):
        D, self.W = conv_weight.shape
        assert 2 <= self.W <= 8, f"conv width {self.W}: 2 to 8 have a carried state and gradients"
        assert D % 4 == 0, f"D={D} must be a multiple of 4 (causal_conv1d, channel-last)"
        self.D = D
        self.conv_weight, self.conv_bias = conv_weight.float().contiguous(), conv_bias.float().contiguous()
        self.decay = decay.float().contiguous()
        self.norm_weight = norm_weight.float().contiguous()
        self.norm_bias = None if norm_bias is None else norm_bias.float().contiguous()
        self.group, self.activation, self.center, self.eps = int(norm_group), activation, bool(center), float(eps)

    def new_state(self, B: int, dtype=torch.bfloat16) -> RecurrentState:
        """The state at a sequence's start."""
        dev = self.conv_weight.device
        return RecurrentState(torch.zeros(B, self.W - 1, self.D, device=dev, dtype=dtype),
                              torch.zeros(B, self.D, device=dev, dtype=torch.float32))

    def _norm(self, h, z, out=None):
        return ops.group_norm(h, self.group, self.norm_weight, self.norm_bias, gate=z, activation="silu",
                              center=self.center, eps=self.eps, out=out)

    def __call__(self, x, r, i, z, state: RecurrentState | None = None, want_grad: bool = False):
        """A whole sequence, or the next part of one after ``state``: (y [B, T, D], state after it),
        and with ``want_grad`` what ``backward`` needs (training starts at the sequence's start).
        The given state is left as it is."""
        B, T, D = x.shape
        assert D == self.D, f"x has {D} channels, the block {self.D}"
        assert not (want_grad and state is not None), "gradients are for whole sequences: no state is given"
        tail = self.W - 1
        if state is None:
            u = ops.causal_conv1d(x, self.conv_weight, self.conv_bias, self.activation, "bsd")
            conv = torch.cat([x.new_zeros(B, max(tail - T, 0), D), x[:, max(T - tail, 0):]], 1)
        elif T <= 64:
            u, conv = ops.causal_conv1d_step(x, state.conv, self.conv_weight, self.conv_bias,
                                             activation=self.activation)
        else:
            xs = torch.cat([state.conv, x], 1)
            u = ops.causal_conv1d(xs, self.conv_weight, self.conv_bias, self.activation, "bsd")[:, tail:]
            conv = xs[:, T:].contiguous()
        h, final, states = ops.gated_scan(u, r, i, self.decay, h0=None if state is None else state.h,
                                          want_states=want_grad)
        y = self._norm(h, z, out=None if want_grad else h)
        after = RecurrentState(conv, final)
        return (y, after, (x, r, i, z, u, h, states)) if want_grad else (y, after)

    def step(self, x, r, i, z, state: RecurrentState):
        """The next token of every sequence: x, r, i, z [B, 1, D] (or a few, [B, S <= 64, D]); ``state``
        moves on in place. Returns y like x."""
        u, _ = ops.causal_conv1d_step(x, state.conv, self.conv_weight, self.conv_bias, activation=self.activation,
                                      state_out=state.conv)
        h, _, _ = ops.gated_scan(u, r, i, self.decay, h0=state.h, final=state.h)
        return self._norm(h, z, out=h)

    def backward(self, saved, dy, dfinal=None) -> dict:
        """Gradients for dy [B, T, D] (and dfinal [B, D] fp32 of the final scan state): x, r, i, z in
        their dtype, the parameters in fp32 (``norm_bias`` only if there is one)."""
        x, r, i, z, u, h, states = saved
        dh, dz, dnw, dnb = ops.group_norm_bwd(h, dy, self.group, self.norm_weight, self.norm_bias, gate=z,
                                              activation="silu", center=self.center, eps=self.eps)
        du, dr, di, ddecay, _ = ops.gated_scan_bwd(u, r, i, self.decay, states, dh, dfinal=dfinal)
        dx, dcw, dcb = ops.causal_conv1d_bwd(x, self.conv_weight, self.conv_bias, du, activation=self.activation)
        grads = dict(x=dx, r=dr, i=di, z=dz, conv_weight=dcw, conv_bias=dcb, decay=ddecay, norm_weight=dnw)
        if dnb is not None:
            grads["norm_bias"] = dnb
        return grads
