"""Matrix products with what stands behind them, in one kernel: the projections around a recurrence and the feed-forward
block's first half.

``linear_act(x, weight, bias=None, activation="none", mul=None, residual=None) -> y``
    ``y = act(x weight^T + bias) * mul + residual``.  x [..., K]; weight [N,K]; bias [N] in any float type; mul, residual [..., N].
    A channel mix of the WKV models is ``k = linear_act(xk, w_key, activation="relu2")``, ``kv = linear_act(k, w_value)``,
    ``linear_act(xr, w_receptance, activation="sigmoid", mul=kv)``.

``gated_linear(x, w_gate, w_up, activation="silu") -> y``
    ``y = act(x w_gate^T) * (x w_up^T)``, both products in one kernel.  w_gate, w_up [N,K].

activation: ``"none"``, ``"silu"`` (z sigmoid(z)), ``"gelu"`` (z Phi(z), with the error function), ``"relu2"`` (max(z, 0)^2) or
``"sigmoid"``.  Differentiable w.r.t. every tensor (once, and not in forward mode: anything else is refused).

x, the matrices, mul, residual and y in bf16 or fp16 (of one type within a call; fp32 is refused: the tensor cores would take it
at 10 bits).  Sums, bias, activation, product and residual are in fp32 and rounded once.  For the backward pass the
pre-activations are kept in fp32 (where an activation or ``mul`` needs them); their gradient is rounded to x's type once, as an operand of the
products (the bias' gradient is summed before that; in fp16 what is above 65504 there is an infinity).  Kept is what the wanted
gradients need: x for those of the matrices, the matrices for that of x, ``mul`` and the pre-activations for any but the residual's.  Any size and
alignment is taken; rows whose length or stride is no multiple of 8 elements are copied first, except in calls of few rows
(up to 16, or 32 of a small matrix).
"""
from __future__ import annotations

from . import _lib as L


def linear_act(x, weight, bias=None, activation="none", mul=None, residual=None):
    return L.native().linear_act(x, weight, bias, activation, mul, residual)


def gated_linear(x, w_gate, w_up, activation="silu"):
    return L.native().gated_linear(x, w_gate, w_up, activation)
