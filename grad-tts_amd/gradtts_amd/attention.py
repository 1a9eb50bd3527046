"""Attention with a learned relative position bias by buckets (csrc/battn_fwd.hip, csrc/battn_bwd.hip), with all
gradients.

The text encoder's own attention (``text_encoder.MultiHeadAttention``) learns an embedding for each offset within a
window of a few tokens and treats everything beyond alike; here every offset has a learned bias for each head, one for
each small distance and one for each of some logarithmically wider ranges up to ``max_distance``, the last for all
beyond. ``text_encoder.TextEncoder(n_buckets=...)`` is built on it.
"""
from __future__ import annotations

import torch

from ._lib import lib, ops


def bucket_attention(q, k, v, table, lengths=None, q_lengths=None, q_start=None, causal=False, max_distance=128,
                     scale=None):
    """``softmax(q k^T scale + table[bucket(j - pos_i)]) v`` for every head; returns ``[B, Tq, Hq, D]`` of q's type.

    q ``[B, Tq, Hq, D]``, k and v ``[B, Tk, Hkv, D]`` (Hq a multiple of Hkv, D <= 128; any strides, best with contiguous
    channels and rows on 16 bytes), table ``[n_buckets, Hq]``; all float32, bfloat16 or float16 and differentiable (once:
    second derivatives raise). lengths, q_lengths, q_start: integers ``[B]``. Keys ``j >= lengths[b]`` are neither seen
    nor read; rows ``i >= q_lengths[b]`` give zeros and pass no gradient, as do rows that see no key. Query i stands at
    ``pos_i = q_start[b] + i`` (q_start 0 if None): a decoding step over a cache passes ``q_start = lengths - Tq``.
    causal: keys ``j > pos_i`` are not seen (nor, past the last query, read) and the buckets cover distances
    ``pos_i - j``; otherwise each direction has half of them (n_buckets even). scale: 1 / sqrt(D) if None, else in
    [2^-20, 2^20]. Table entries below -2^17 (or -inf) shut their bucket off.

    Products take q's type: the probabilities and score gradients that enter them are rounded to it; sums and statistics
    are float32. An infinity or NaN in v may also reach rows of its head and batch entry that see other keys only (zero
    times infinity). Calls of equal shapes repeat bit for bit; an entry's last digits may depend on the batch around it,
    whose size chooses the kernel. Scores that rise by some 69 and more past those of a row's first keys make the forward
    take about twice as long (float16: never). Works on the current stream; may be captured into a graph (with gradients
    only once no eager autograd graph of the same parameters is alive: refused otherwise). Needs a HIP device."""
    if not q.is_cuda and q.device.type != "meta":
        raise RuntimeError("bucket_attention needs a HIP (MI355X) device; there is no CPU path")
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return ops().bucket_attention(q, k, v, table, lengths, q_lengths, q_start, causal, max_distance, scale)[0]


def relative_bucket(offset, n_buckets, causal=False, max_distance=128):
    """Bucket of one offset (key position - query position), as ``bucket_attention`` uses them (host integers)."""
    b = lib().gt_relative_bucket(int(causal), n_buckets, max_distance, offset)
    if b < 0:
        raise ValueError(f"no buckets for n_buckets {n_buckets}, max_distance {max_distance}, causal {causal}")
    return b


__all__ = ["bucket_attention", "relative_bucket"]
