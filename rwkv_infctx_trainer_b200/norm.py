"""Root-mean-square norm with the residual's addition, in one CUDA pass.

``rms_norm(x, weight, residual=None, eps=1e-6)``
    ``y = weight * h / sqrt(mean(h^2) + eps)`` over the last dimension, ``h = x + residual``.  Returns ``y``, and with
    a residual ``(y, h)``: ``h`` is the new residual stream.  Differentiable w.r.t. x, weight and residual, with a
    gradient on both outputs.

``rms_norm_q8(x, weight, residual=None, eps=1e-6, group=None)``
    the same with ``y`` in 8 bits: ``(q, scale)`` or ``(q, scale, h)``; ``q`` is float8_e4m3fn of x's shape and stands
    for ``q * scale``, ``scale`` is float32 ``[..., 1]``, or with ``group`` (32, 64, 128 or 256 channels) ``[..., C / group]``
    rounded up.  ``scale = max|y| / 448``, 1 where the maximum is below 2^-100.  No gradient.

x [..., C] in bf16, fp16 or fp32, 1 <= C <= 16384; the residual (and ``h``) in x's type or in fp32, ``y`` in x's type;
weight [C] in any float type.  Sums are fp32; ``y`` and the gradients are formed from ``h`` before it is rounded to the
residual's type.  There are no second derivatives and no forward-mode derivatives: both are refused.
"""
from __future__ import annotations

from . import _lib as L


def rms_norm(x, weight, residual=None, eps=1e-6):
    out = L.native().rms_norm(x, weight, residual, float(eps))
    return tuple(out) if residual is not None else out[0]


def rms_norm_q8(x, weight, residual=None, eps=1e-6, group=None):
    return tuple(L.native().rms_norm_q8(x, weight, residual, float(eps), group))
