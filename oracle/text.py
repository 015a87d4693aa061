"""Float64 restatements of the 4-bit (MXFP4) quantisation and of the relative-position-bias attention with its
gradients, from their formulas."""

from __future__ import annotations

import math

import numpy as np
import torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mx4_quantize(x: torch.Tensor):
    """(codes [rows, cols] 0..15, scale codes [rows, ceil(cols/32)] 0..255) of a matrix."""
    a = x.detach().cpu().double().numpy()
    rows, cols = a.shape
    nb = (cols + 31) // 32
    pad = np.zeros((rows, nb * 32))
    pad[:, :cols] = a
    blk = pad.reshape(rows, nb, 32)
    bad = ~np.isfinite(blk).all(-1)
    mag = np.where(np.isfinite(blk), np.abs(blk), 0.0)
    _, e = np.frexp(mag.max(-1))  # mantissa in [0.5, 1): floor(log2) = e - 1
    scale = np.where(mag.max(-1) > 0, np.clip(e - 1 - 2 + 127, 0, 254), 0)
    unit = np.ldexp(1.0, scale - 127)[..., None]
    v = np.minimum(mag / unit, 6.0)
    dist = np.abs(v[..., None] - E2M1)
    dist[..., 1::2] += 1e-12  # a tie goes to the even code
    code = dist.argmin(-1)
    code = np.where(bad[..., None], 0, code | (np.signbit(blk) * 8))
    scale = np.where(bad, 255, scale)
    return torch.from_numpy(code.reshape(rows, -1)[:, :cols].copy()), torch.from_numpy(scale.copy())


def mx4_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    grid = torch.from_numpy(np.concatenate([E2M1, -E2M1]))
    s = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales - 127)
    s[scales == 255] = math.nan
    return grid[codes] * s.repeat_interleave(32, 1)[:, :codes.shape[1]]


def mx4_round(x: torch.Tensor) -> torch.Tensor:
    """The values the quantised matrix stands for."""
    return mx4_values(*mx4_quantize(x))


def bucket(rel: int, num_buckets: int, max_distance: int, bidirectional: bool) -> int:
    """Relative position bucket, whole-number arithmetic throughout."""
    nb = num_buckets // 2 if bidirectional else num_buckets
    n = abs(rel) if bidirectional else max(-rel, 0)
    side = nb if bidirectional and rel > 0 else 0
    first = nb // 2
    if n < first:
        return n + side
    span, t = nb - first, 0
    # the largest t < span with (n / first)^span >= (max_distance / first)^t
    while t + 1 < span and n ** span * first ** (t + 1) >= max_distance ** (t + 1) * first ** span:
        t += 1
    return first + t + side


def bias_attention(q, k, v, table, key_mask=None, max_distance=128, bidirectional=True, causal=False, scale=None,
                   q_offset=0, go=None):
    """o, and with go a dict of o, dq, dk, dv, dtable; dtable_abs: what the rounding of o to a relative precision eps
    can move dtable by, over eps; ds_abs: the sum of |dS| by bucket; dq_abs, dk_abs: the gradients' sums with every
    term of dP - delta taken by its magnitude."""
    q, k, v, table = (t.detach().cpu().double() for t in (q, k, v, table))
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    rel = torch.arange(Sk)[None, :] - torch.arange(Sq)[:, None] - q_offset
    lo, hi = int(rel.min()), int(rel.max())
    lut = torch.tensor([bucket(r, table.shape[0], max_distance, bidirectional) for r in range(lo, hi + 1)])
    bk = lut[rel - lo]
    keep = torch.ones(B, 1, Sq, Sk, dtype=torch.bool)
    if causal:
        keep = keep & (rel <= 0)
    if key_mask is not None:
        m = key_mask.cpu()
        keep = keep & m[:, None, None, :]
        k, v = (torch.where(m[:, None, :, None], t, 0.0) for t in (k, v))
    x = scale * (q @ k.transpose(-1, -2)) + table[bk].permute(2, 0, 1)
    x = torch.where(keep, x, -math.inf)
    some = keep.any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, x, 0.0), -1), 0.0)
    o = p @ v
    if go is None:
        return o
    go = go.detach().cpu().double()
    delta = (go * o).sum(-1, keepdim=True)
    ds = p * (go @ v.transpose(-1, -2) - delta)
    mag = p * (go.abs() @ v.abs().transpose(-1, -2) + (go * o).abs().sum(-1, keepdim=True))
    grp = lambda t: t.view(B, Hk, H // Hk, Sk, D).sum(2)  # noqa: E731
    by_bucket = lambda t: torch.zeros_like(table).index_add_(0, bk.flatten(), t.sum(0).flatten(1).t())  # noqa: E731
    return {"o": o, "dq": scale * (ds @ k), "dk": scale * grp(ds.transpose(-1, -2) @ q), "dv": grp(p.transpose(-1, -2) @ go),
            "dtable": by_bucket(ds), "dtable_abs": by_bucket(p * (go.abs() * o.abs()).sum(-1, keepdim=True)),
            "ds_abs": by_bucket(ds.abs()), "dq_abs": scale * (mag @ k.abs()),
            "dk_abs": scale * grp(mag.transpose(-1, -2) @ q.abs())}
