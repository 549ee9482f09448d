"""Streaming operators restated in float64 (torch): rotary positions over several axes, the
append to a paged cache, and attention under the causal / block / window / sinks rule. Test
infrastructure only; written from the definitions, a row or a head at a time."""
from __future__ import annotations

import math

import torch


def turn(x, positions, sections, theta, paired=True, shared=False, inverse=False):
    """x [..., N, 128], positions [N, axes] (or broadcastable [..., N, axes]) -> float64."""
    x = x.double()
    angles = []
    for axis, dims in enumerate(sections):
        done = sum(sections[:axis]) // 2
        for i in range(dims // 2):
            power = 2.0 * (done + i) / 128 if shared else 2.0 * i / dims
            angles.append(positions[..., axis].double() * math.pow(theta, -power))
    angle = torch.stack(angles, -1)
    c, s = angle.cos(), angle.sin() * (-1 if inverse else 1)
    out = torch.empty_like(x)
    first, second = (slice(0, 128, 2), slice(1, 128, 2)) if paired else (slice(0, 64), slice(64, 128))
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., first] * s + x[..., second] * c
    return out


def sees(first, tokens, keys, window, sinks, block, device=None):
    """bool [tokens, keys] for queries at positions first, first + 1, ..."""
    p = first + torch.arange(tokens, device=device)[:, None]
    j = torch.arange(keys, device=device)[None]
    e = torch.where(p < 0, 0, (p // block + 1) * block)
    seen = j < e
    if window is not None:
        seen &= (j >= e - window) | (j < sinks)
    return seen


def attend(q, k, v, *, window=None, sinks=0, block=1, first=None):
    """q [N, H, 128] over k, v [K, Hk, 128], the queries the last N of the K positions ->
    float64 (o [N, H, 128], base-2 lse [N, H], a [N, H, 128] = the same weights over |v|)."""
    n, heads, _ = q.shape
    keys, kv = k.shape[0], k.shape[1]
    first = keys - n if first is None else first
    seen = sees(first, n, keys, window, sinks, block, q.device)
    o = torch.zeros(n, heads, 128, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
    if n == 0 or keys == 0:
        return o, lse, a
    for h in range(heads):
        kh, vh = k[:, h * kv // heads].double(), v[:, h * kv // heads].double()
        s = (q[:, h].double() @ kh.T * 128 ** -0.5).masked_fill(~seen, -math.inf)
        l = torch.logsumexp(s, -1, keepdim=True)
        w = torch.where(seen, torch.exp(s - torch.where(l == -math.inf, 0.0, l)), 0.0)
        o[:, h], a[:, h] = w @ vh, w @ vh.abs()
        lse[:, h] = l[:, 0] / math.log(2.0)
    return o, lse, a


def rows_of(cache, page_table, length):
    """[length, kv_heads, 128] of one sequence's pages [pages, kv_heads, page_size, 128]."""
    size = cache.shape[2]
    used = page_table[: -(-length // size)].long()
    return cache[used].transpose(1, 2).flatten(0, 1)[:length]
