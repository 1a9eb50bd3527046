"""The residual step between two blocks of a transformer with norms on both sides of a block (csrc/rnorm.hip): the
norm after the finished block, its gate and residual scale, the residual sum and the norm before the next block in one
pass, with all gradients. The text encoder's own residual steps are ``LayerNorm(x + y)`` (``text_encoder.Encoder``); its bucket form
(``text_encoder.BucketEncoder``) takes this one.
"""
from __future__ import annotations

from ._lib import ops


def residual_norm(x, y, post_weight, pre_weight, post_bias=None, pre_bias=None, gate=None, scale=1.0, eps=1e-5,
                  kind="layer", lengths=None):
    """``out = x + scale * gate * N1(y)``, ``h = N2(out)``; returns ``(out, h)``.

    x (residual stream) and y (block output) ``[B, T, C]``, float32, bfloat16 or float16, B <= 65535, C <= 8192. N is a layer norm
    (``kind="layer"``) or root-mean-square norm (``"rms"``) over the channels with float32 weights ``[C]`` and optional
    biases ``[C]``; gate: float32 ``[C]``, or ``[B, C]`` for one of each batch entry, or None (1). All of them are
    differentiable (once: second derivatives raise). lengths: integers ``[B]``; rows ``t >= lengths[b]`` are not read,
    their outputs and gradients are zero. Statistics and parameter gradients are float32 sums in a fixed order. Works on the current stream; may be
    captured into a graph (with gradients only once no eager autograd graph of the same parameters is alive: refused
    otherwise). Needs a HIP device."""
    if not x.is_cuda and x.device.type != "meta":
        raise RuntimeError("residual_norm needs a HIP (MI355X) device; there is no CPU path")
    if kind not in ("layer", "rms"):
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    return ops().residual_norm(x, y, gate, post_weight, post_bias, pre_weight, pre_bias, lengths, scale, eps,
                               kind == "rms")[:2]


__all__ = ["residual_norm"]
