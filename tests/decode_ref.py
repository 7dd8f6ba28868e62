"""The operators between a layer's projections from their definitions in 64 bits, on the CPU (imported by tests only)."""
import numpy as np
import torch


def norm_rope(x, weight, eps, positions, inv_freq, interleaved, unit=False):
    """x [T, H, D] -> float64 results and, for error bounds, the sum of the absolute terms of every element"""
    y = x.detach().cpu().double()
    if weight is not None:
        w = weight.detach().cpu().double() + (1.0 if unit else 0.0)
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
    out, size = y.clone(), y.abs()
    if inv_freq is not None and inv_freq.numel():
        half = inv_freq.numel()
        angle = (positions.cpu().double()[:, None] * inv_freq.cpu().double())[:, None]
        a_at = torch.arange(0, 2 * half, 2) if interleaved else torch.arange(half)
        b_at = a_at + (1 if interleaved else half)
        a, b = y[..., a_at], y[..., b_at]
        out[..., a_at] = a * angle.cos() - b * angle.sin()
        out[..., b_at] = b * angle.cos() + a * angle.sin()
        size[..., a_at] = a.abs() + b.abs()
        size[..., b_at] = a.abs() + b.abs()
    return out, size


def attention(q, k_cache, v_cache, table, cu, prefix, seen, scale):
    """q [T, Hq, D]; seen: one [n, n] truth array per sequence (which new tokens a new token sees).  Positions of pages outside the cache count
    as zeros, positions behind the block table do not exist.  Returns float64 [T, Hq, D] (rows in no sequence NaN) and, for error bounds, the same
    with |v| for v and the largest sum of a score's absolute terms [T, Hq, 1]."""
    q = q.detach().cpu().double()
    pages, page, kv, D = k_cache.shape
    group = q.shape[1] // kv
    out, size, terms = torch.full(q.shape, float("nan"), dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2] + (1,), dtype=torch.float64)
    for b in range(len(cu) - 1):
        lo, n = int(cu[b]), int(cu[b + 1] - cu[b])
        length = min(int(prefix[b]) + n, table.shape[1] * page)
        at = torch.arange(length)
        ids = table[b].cpu().long()[at // page] if length else at
        good = (ids >= 0) & (ids < pages)
        ids = torch.where(good, ids, 0)
        see = torch.ones((n, int(prefix[b]) + n), dtype=torch.bool)
        see[:, int(prefix[b]):] = torch.as_tensor(seen[b])
        see = see[:, :length]
        for h in range(q.shape[1]):
            if h % group == 0:
                k, v = [c[ids.to(c.device), (at % page).to(c.device), h // group].cpu().double() for c in (k_cache, v_cache)]
                k, v = [torch.where(good[:, None], c, 0.0) for c in (k, v)]
            for t in range(n):
                m = see[t]
                if not m.any():
                    out[lo + t, h] = 0
                    continue
                s = (k[m] @ q[lo + t, h]) * scale
                p = (s - s.max()).exp()
                p = p / p.sum()
                out[lo + t, h] = p @ v[m]
                size[lo + t, h] = p @ v[m].abs()
                terms[lo + t, h] = (k[m].abs() @ q[lo + t, h].abs()).max() * scale
    return out, size, terms


def ancestors(parents):
    """truth values [n, n]: token j is token i or one of its ancestors (parents[i] < i; below 0: a root)"""
    n = len(parents)
    seen = np.eye(n, dtype=bool)
    for i in range(n):
        if parents[i] >= 0:
            seen[i] |= seen[parents[i]]
    return seen


def sample(logits, u, temperature, top_k, top_p, min_p):
    """one row, in float64 (the definition in the header)"""
    x = np.asarray(logits, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    if len(x) == 0 or x.max() == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.argmax(x))
    top = x.max()
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / np.float64(np.float32(temperature))) if np.isfinite(top) else 0.0)
    w[w < 2.0 ** -52] = 0
    order = np.lexsort((np.arange(len(x)), -x))
    if 0 < top_k < len(x):
        w[order[top_k:]] = 0
    p = float(np.float32(top_p))
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])])
        w[order[max(1, int(np.searchsorted(before, p * before[-1], "left"))):]] = 0
    w[w < min(float(np.float32(min_p)), 1.0)] = 0
    up_to = np.cumsum(w)
    i = int(np.searchsorted(up_to, float(np.float32(u)) * up_to[-1], "right"))
    return min(i, int(np.nonzero(w)[0][-1]))
