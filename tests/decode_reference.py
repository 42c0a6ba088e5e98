"""Plain 64-bit forms of the operators around the MoE layer, for the tests."""
from __future__ import annotations

import numpy as np
import torch


def rotate(x, positions, inv_freq, interleaved):
    """x [T, heads, dim] -> float64, the first 2 * len(inv_freq) columns turned."""
    x = x.double().clone()
    a = positions.double()[:, None] * inv_freq.double()
    cos, sin = a.cos()[:, None], a.sin()[:, None]
    n = inv_freq.numel()
    first = torch.arange(n, device=x.device) * 2 if interleaved else torch.arange(n, device=x.device)
    second = first + (1 if interleaved else n)
    p, r = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = p * cos - r * sin, r * cos + p * sin
    return x


def keys_of(cache, pages, n):
    """The first n rows of a list of pages: [heads, n, dim] float64; a page
    outside the cache gives None rows (second result: visible)."""
    ps = cache.shape[2]
    rows = torch.zeros(cache.shape[1], n, cache.shape[3], dtype=torch.float64, device=cache.device)
    seen = torch.zeros(n, dtype=torch.bool, device=cache.device)
    for i, p in enumerate(pages[:-(-n // ps)]):
        lo, hi = i * ps, min(n, (i + 1) * ps)
        if 0 <= p < cache.shape[0]:
            rows[:, lo:hi] = cache[p, :, :hi - lo].double()
            seen[lo:hi] = True
    return rows, seen


def attention(q, k_cache, v_cache, tables, lens, prefix_pages, prefix_len, q_start, scale):
    """(out, lse, sum of p |v|, largest sum of |q k| scale a row) in float64."""
    T, hq, d = q.shape
    hk = k_cache.shape[1]
    g = hq // hk
    dev = q.device
    out = torch.zeros(T, hq, d, dtype=torch.float64, device=dev)
    lse = torch.full((T, hq), float("-inf"), dtype=torch.float64, device=dev)
    mass, size = torch.zeros_like(out), torch.zeros_like(lse)
    tables, lens = tables.tolist(), lens.tolist()
    starts = list(range(len(lens) + 1)) if q_start is None else q_start.tolist()
    pp = [] if prefix_pages is None else prefix_pages.tolist()
    kp, sp = keys_of(k_cache, pp, prefix_len)
    vp, _ = keys_of(v_cache, pp, prefix_len)
    for b, c in enumerate(lens):
        lo, hi = starts[b], min(starts[b + 1], T)
        n = hi - lo
        if n <= 0:
            continue
        ko, so = keys_of(k_cache, tables[b], c)
        vo, _ = keys_of(v_cache, tables[b], c)
        k, v = torch.cat([kp, ko], 1), torch.cat([vp, vo], 1)
        see = torch.cat([sp, so])
        if k.shape[1] == 0:
            continue
        qq = q[lo:hi].double().view(n, hk, g, d)
        s = torch.einsum("nhgd,hkd->nhgk", qq, k) * scale
        a = torch.einsum("nhgd,hkd->nhgk", qq.abs(), k.abs()) * abs(scale)
        pos = torch.arange(k.shape[1], device=dev)
        last = prefix_len + c - n + torch.arange(n, device=dev)
        ok = see[None] & ((pos[None] < prefix_len) | (pos[None] <= last[:, None]))
        s = s.masked_fill(~ok[:, None, None], float("-inf"))
        some = ok.any(1)
        p = torch.where(some[:, None, None, None], torch.softmax(s, -1), 0.0)
        out[lo:hi] = torch.einsum("nhgk,hkd->nhgd", p, v).reshape(n, hq, d)
        mass[lo:hi] = torch.einsum("nhgk,hkd->nhgd", p, v.abs()).reshape(n, hq, d)
        lse[lo:hi] = torch.logsumexp(s, -1).reshape(n, hq)
        size[lo:hi] = torch.where(ok[:, None, None], a, 0.0).amax(-1).reshape(n, hq)
    return out, lse, mass, size


def sample(x, u, temperature, top_k, top_p, min_p):
    """One row (numpy float64), settings float32 numbers."""
    x = np.where(np.isnan(x), -np.inf, x)
    if not (x > -np.inf).any():
        return -1
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0])
    order = order[x[order] > -np.inf]
    if top_k >= 1:
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(temperature)))
    keep = w >= np.float64(min_p)
    if top_p < 1:
        keep &= np.concatenate([[0.0], np.cumsum(w)[:-1]]) < np.float64(top_p) * w.sum()
    keep[0] = True
    chosen = order[keep]
    by = np.argsort(chosen)
    c = np.cumsum(w[keep][by])
    return int(chosen[by][min(np.searchsorted(c, np.float64(u) * c[-1], side="right"), len(by) - 1)])
