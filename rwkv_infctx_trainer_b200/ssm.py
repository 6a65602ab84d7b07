"""Selective state space scan and the short causal convolution in front of it: a second recurrence with a carried
state, with the contract of the WKV ops (state in, state out, the gradient of both, segments chained).

``causal_conv(x, weight, bias=None, state=None, silu=True) -> (y, state)``
    one filter of W = 2, 3 or 4 taps per channel over time: ``s_t = bias + sum_j weight[:, j] x_{t-W+1+j}``,
    ``y = silu(s)`` or ``s``.  x [B,T,D]; weight [D,W] (or [D,1,W]); bias [D]; state [B,W-1,D]: the inputs before the
    first token (None: zeros), returned: the last W-1 inputs, in x's type.

``selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True, state=None) -> (y, state)``
    ``dt = softplus(delta + delta_bias)``, ``h_t = exp(dt A) h_{t-1} + dt u_t B_t``, ``y_t = (C_t . h_t + D u_t) silu(z_t)``
    per channel and state.  u, delta, z [B,T,D]; B, C [B,T,N] or [B,T,G,N] (channel d uses group d // (D / G));
    A [D,N], 1 <= N <= 64; D, delta_bias [D]; state fp32 [B,D,N] (None: zeros).  Without z there is no gate.  An A of -inf forgets
    the state at any step above 1e-36; a step of zero keeps it.

Both are differentiable w.r.t. every tensor, the state included (once, and not in forward mode: anything else is refused).  Any T >= 0
up to 2^31 - 273.

``causal_conv_step(x, state, weight, bias=None, silu=True) -> y``
``selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, delta_softplus=True) -> y``
    one token (x, u, delta, z [B,D]; B, C [B,N] or [B,G,N]) with the state updated in place; no gradient.  (A state made in
    ``torch.inference_mode()`` is updated there only.)

Activations in bf16, fp16 or fp32 (of one type within a call); parameters in any float type; the scan's state in fp32.
A view of a wider tensor along the channels (the halves of a projection) is read where it lies.
"""
from __future__ import annotations

from . import _lib as L


def causal_conv(x, weight, bias=None, state=None, silu=True):
    return L.native().causal_conv(x, weight, bias, state, silu)


def causal_conv_step(x, state, weight, bias=None, silu=True):
    return L.native().causal_conv_step(x, state, weight, bias, silu)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=True, state=None):
    return L.native().selective_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, state)


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, delta_softplus=True):
    return L.native().selective_scan_step(u, delta, A, B, C, state, D, z, delta_bias, delta_softplus)
