"""Gated linear recurrence: one state per channel whose decay and input stand behind gates, with the contract of the other
recurrences (state in, state out, the gradient of both, segments chained).

``gated_recurrence(x, input_gate, decay_gate, decay, z=None, state=None, c=8.0) -> (y, state)``
    ``a_t = exp(-c softplus(decay) sigmoid(decay_gate_t))``,
    ``h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(input_gate_t) x_t``, ``y_t = h_t silu(z_t)``, without z ``y_t = h_t``.
    x, input_gate, decay_gate, z [B,T,D]; decay [D]; state fp32 [B,D] (None: zeros); 0 < c <= 1e6.  Differentiable w.r.t. every
    tensor, the state included (once, and not in forward mode: anything else is refused).  Any T >= 0 up to 2^31 - 4097.  A decay
    gate of minus infinity keeps the state and takes nothing in: what padding is masked with (an x of any finite value).

``gated_recurrence_step(x, input_gate, decay_gate, decay, state, z=None, c=8.0) -> y``
    one token (x, input_gate, decay_gate, z [B,D]) with the state updated in place; no gradient.  (A state made in
    ``torch.inference_mode()`` is updated there only.)

Activations in bf16, fp16 or fp32 (of one type within a call); decay in any float type; the state in fp32.  A view of a wider
tensor along the channels (the two gates of one projection) is read where it lies.  The gradient of the gates is exact where a
decay is 1, too: the slope of the square root, which has no bound there, only enters as a product that goes to zero.
"""
from __future__ import annotations

from . import _lib as L


def gated_recurrence(x, input_gate, decay_gate, decay, z=None, state=None, c=8.0):
    return L.native().gated_recurrence(x, input_gate, decay_gate, decay, z, state, float(c))


def gated_recurrence_step(x, input_gate, decay_gate, decay, state, z=None, c=8.0):
    return L.native().gated_recurrence_step(x, input_gate, decay_gate, decay, state, z, float(c))
