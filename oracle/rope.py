"""64-bit ground truth of the operators around the attention that have no counterpart among the
reference's samples: query / key norm with rotation by position, its gradient, the append to a
paged cache and the attention over it.  Plain formulas, one row, pair or sequence at a time where
that is the definition; every function takes tensors of any type and returns float64."""
from __future__ import annotations

import math

import torch

__all__ = ["qk_rope_ref", "qk_rope_grad_ref", "paged_append_ref", "paged_attention_ref"]


def _pairs(rotary: int, interleaved: bool):
    i = torch.arange(rotary // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def _angles(cos, sin, positions):
    """(B, T) positions -> (B, 1, T, R / 2) cos, sin; NaN where the table has no such row."""
    pos = positions.long()
    bad = (pos < 0) | (pos >= cos.shape[0])
    at = pos.clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[at], sin.double()[at]
    c[bad], s[bad] = math.nan, math.nan
    return c[:, None], s[:, None]


def _unit(x, eps):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def _rotate(n, c, s, interleaved):
    first, second = (i.to(n.device) for i in _pairs(2 * c.shape[-1], interleaved))
    y = n.clone()
    y[..., first] = n[..., first] * c - n[..., second] * s
    y[..., second] = n[..., second] * c + n[..., first] * s
    return y


def qk_rope_ref(x, weight, cos, sin, positions, eps=1e-6, interleaved=False):
    """(y, scale): rows (B, H, T, D) normed and rotated, and for every element the sum of the
    magnitudes that its rotation adds up (what fp32 rounding errors are relative to)."""
    x = x.double()
    n = x if weight is None else _unit(x, eps) * weight.double()
    if cos is None:
        return n, n.abs()
    c, s = _angles(cos, sin, positions)
    first, second = (i.to(n.device) for i in _pairs(2 * c.shape[-1], interleaved))
    scale = n.abs()
    both = scale[..., first] + scale[..., second]
    scale[..., first], scale[..., second] = both, both.clone()
    return _rotate(n, c, s, interleaved), scale


def qk_rope_grad_ref(dy, x, weight, cos, sin, positions, eps=1e-6, interleaved=False):
    """(dx, dw, scale of dx, scale of dw)"""
    x, dy = x.double(), dy.double()
    c, s = _angles(cos, sin, positions)
    g = _rotate(dy, c, -s, interleaved)
    first, second = (i.to(g.device) for i in _pairs(2 * c.shape[-1], interleaved))
    mag = dy.abs()
    both = mag[..., first] + mag[..., second]
    mag[..., first], mag[..., second] = both, both.clone()
    if weight is None:
        return g, None, mag, None
    w = weight.double()
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    u = x * r
    h = g * w
    dx = r * (h - u * (h * u).mean(-1, keepdim=True))
    hm = mag * w.abs()
    return (dx, (g * u).sum((0, 1, 2)), r * (hm + u.abs() * (hm * u.abs()).mean(-1, keepdim=True)),
            (mag * u.abs()).sum((0, 1, 2)))


def paged_append_ref(new, cache, page_table, cache_lens, new_lens=None):
    """cache (pages, H, slots, D) after the rows (B, H, T, D) were stored; tokens without a page
    are left out.  Returns the cache in the rows' type."""
    cache = cache.clone().to(new.dtype)
    size = cache.shape[2]
    for b in range(new.shape[0]):
        count = new.shape[2] if new_lens is None else max(0, min(int(new_lens[b]), new.shape[2]))
        for t in range(count):
            at = int(cache_lens[b]) + t
            if at < 0 or at // size >= page_table.shape[1]:
                continue
            page = int(page_table[b, at // size])
            if 0 <= page < cache.shape[0]:
                cache[page, :, at % size] = new[b, :, t]
    return cache


def paged_attention_ref(q, k_cache, v_cache, page_table, cache_lens, new_lens=None, tree_mask=None, qk_scale=None):
    """(out, weight): float64 attention of (B, Hq, T, D) queries, and sum_p softmax_p |v_p|, the
    magnitude that rounding errors of the weights are relative to.  Padding rows are zero."""
    b_, hq, t_, d = q.shape
    hkv, size = k_cache.shape[1], k_cache.shape[2]
    scale = 1.0 / math.sqrt(d) if qk_scale is None else qk_scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for b in range(b_):
        have = int(cache_lens[b])
        n = t_ if new_lens is None else max(0, min(int(new_lens[b]), t_))
        if n == 0:
            continue
        at = torch.arange(have + n, device=q.device)
        pages = page_table[b].long()[at // size]
        sees = torch.ones(n, have + n, dtype=torch.bool, device=q.device)
        if tree_mask is None:
            sees[:, have:] = torch.ones(n, n, device=q.device).tril().bool()
        else:
            sees[:, have:] = (tree_mask if tree_mask.dim() == 2 else tree_mask[b])[:n, :n]
        for h in range(hq):
            hk = h // (hq // hkv)
            keys, values = (c[pages, hk, at % size].double() for c in (k_cache, v_cache))
            if bool(torch.isfinite(keys).all() and torch.isfinite(values).all()):
                score = q[b, h, :n].double() @ keys.T * scale
                p = torch.softmax(score.masked_fill(~sees, -math.inf), dim=1)
                p[~sees.any(1)] = 0.0
                out[b, h, :n], mag[b, h, :n] = p @ values, p @ values.abs()
                continue
            for t in range(n):               # only what the query sees takes part, row by row
                who = sees[t]
                if bool(who.any()):
                    p = torch.softmax(keys[who] @ q[b, h, t].double() * scale, dim=0)
                    out[b, h, t], mag[b, h, t] = p @ values[who], p @ values[who].abs()
    return out, mag
