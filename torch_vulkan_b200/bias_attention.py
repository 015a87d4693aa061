"""Attention with a learned relative position bias by buckets (text encoders whose positions enter as one scalar per
head and bucket of distances), forward and backward, with padding and causal masks and a form for few query rows
against a long cache. CUDA tensors only."""

from __future__ import annotations

import math

import torch


def relative_position_bucket(rel: int, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True) -> int:
    """Bucket of a relative position (key position - query position). The first half of a direction's buckets hold one
    distance each, the others are spaced by the logarithm of the distance up to max_distance (computed exactly);
    bidirectional: the upper half of the buckets is for keys after the query, else those share bucket 0."""
    return int(torch.ops.b2.bias_bucket(int(rel), int(num_buckets), int(max_distance), bool(bidirectional)))


def bucket_bias_attention(q, k, v, table, key_mask=None, max_distance=128, bidirectional=True, causal=False, scale=None,
                          q_offset=0):
    """softmax(scale * q k^T + table[bucket(j - i - q_offset)]) v.

    q [B, H, Sq, D], k and v [B, Hk, Sk, D] with H a multiple of Hk (query head h reads key/value head h // (H // Hk)),
    D at most 128, bf16, f16 or fp32, any strides; table [num_buckets, H], float, where an entry of -inf (or below -2.3e38)
    hides its bucket. The 16-bit backward is many times slower where max_distance is above 591 (D up to 64) or 471 and the
    table wants its gradient. key_mask bool [B, Sk], true where a
    key may be attended to; causal hides keys after the query's position i + q_offset (a decoder's new token against a
    cache of Sk keys has q_offset = Sk - Sq). scale defaults to 1 / sqrt(D). A query whose keys are all masked gets
    zeros and zero gradients; what k and v hold at masked positions, or (causal) past the last query's, is never used.
    Differentiable (once) in q, k, v and table; every sum has a fixed order, so results are the same bits on every call."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return torch.ops.b2.bucket_bias_attention(q, k, v, table, key_mask, max_distance, bidirectional, causal, scale, q_offset)
