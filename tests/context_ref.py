"""The operators over images and long contexts from their definitions in 64 bits, on the CPU (imported by tests only)."""
import numpy as np
import torch


def norm_rope_axes(x, weight, eps, positions, axes, inv_freq, interleaved, unit=False):
    """x [T, H, D], positions [A, T], axes [rot / 2] -> float64 results and, for error bounds, the sum of the absolute terms of every element.  A pair
    whose axis is not there stays."""
    y = x.detach().cpu().double()
    if weight is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (weight.detach().cpu().double() + (1.0 if unit else 0.0))
    out, size = y.clone(), y.abs()
    half = len(inv_freq)
    for j, (axis, f) in enumerate(zip(axes.tolist(), inv_freq.tolist())):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        if not 0 <= axis < positions.shape[0]:
            continue
        angle = (positions[axis].cpu().double() * f)[:, None]
        out[..., a] = y[..., a] * angle.cos() - y[..., b] * angle.sin()
        out[..., b] = y[..., b] * angle.cos() + y[..., a] * angle.sin()
        size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, size


def adjust(x, said=(), prompt=0, repetition=1.0, presence=0.0, frequency=0.0, bias=(), allowed=None):
    """one row of logits in float64: `said` the tokens in front (the first `prompt` of them given, the others chosen), bias (token, value) pairs of which a token's last
    one counts, allowed: truth values.  Returns the results and, for error bounds, the sum of each one's absolute terms."""
    x = np.asarray(x, np.float64).copy()
    size = np.abs(x)
    said = [int(t) for t in said]
    inside = [t for t in said if 0 <= t < len(x)]
    with np.errstate(all="ignore"):
        for t in set(inside):
            x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
            size[t] = abs(x[t])
        chosen = [t for t in said[max(0, int(prompt)):] if 0 <= t < len(x)]
        for t, n in zip(*np.unique(chosen, return_counts=True)):
            x[int(t)] -= frequency * n + presence
            size[int(t)] += abs(frequency) * n + abs(presence)
        for t, v in {int(t): float(v) for t, v in bias}.items():
            if 0 <= t < len(x):
                x[t] += v
                size[t] += abs(v)
    if allowed is not None:
        x[~np.asarray(allowed, bool)] = -np.inf
    return x, size


def finite(x):
    """sizes of terms that are rounded: a score with an infinite one is infinite or no number, exactly"""
    return torch.where(torch.isfinite(x), x.abs(), 0.0)


def cross(q, k, v, cu, first, count, scale):
    """q [T, Hq, D]; k, v [S, Hkv, D] -> float64 [T, Hq, D] (rows in no sequence NaN) and, for error bounds, the same with |v| for v and the largest sum of a
    score's absolute terms [T, Hq, 1]"""
    q, k, v = [x.detach().cpu().double() for x in (q, k, v)]
    group = q.shape[1] // k.shape[1]
    out, size, terms = torch.full(q.shape, float("nan"), dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2] + (1,), dtype=torch.float64)
    for b in range(len(first)):
        rows = slice(int(cu[b]), int(cu[b + 1]))
        lo = min(max(int(first[b]), 0), k.shape[0])
        n = min(max(int(count[b]), 0), k.shape[0] - lo)
        for h in range(q.shape[1]):
            kh, vh, qh = k[lo:lo + n, h // group], v[lo:lo + n, h // group], q[rows, h]
            if n == 0:
                out[rows, h] = 0
                continue
            p = torch.softmax(qh @ kh.t() * scale, -1)
            out[rows, h], size[rows, h] = p @ vh, p @ vh.abs()
            if len(qh):
                terms[rows, h] = (finite(qh) @ finite(kh).t()).amax(-1, keepdim=True) * scale
    return out, size, terms


def weights(q, k_cache, table, cu, prefix, scale, max_tokens=None, max_keys=None):
    """per sequence: what its positions get, float64 [Hkv, positions], and, for error bounds, the largest sum of a score's absolute terms.  Positions of pages outside the cache count as zeros."""
    q = q.detach().cpu().double()
    pages, page, kv, D = k_cache.shape
    group, out = q.shape[1] // kv, []
    for b in range(len(cu) - 1):
        lo, n = int(cu[b]), int(cu[b + 1] - cu[b])
        length = min(int(prefix[b]) + n, table.shape[1] * page, max_keys if max_keys is not None else 1 << 62)
        at = torch.arange(length)
        ids = table[b].cpu().long()[at // page] if length else at
        good = (ids >= 0) & (ids < pages)
        k = k_cache.detach()[torch.where(good, ids, 0).to(k_cache.device), (at % page).to(k_cache.device)].cpu().double()
        k = torch.where(good[:, None, None], k, 0.0)
        got, most = torch.zeros((kv, length), dtype=torch.float64), 0.0
        for t in range(min(n, max_tokens if max_tokens is not None else n)):
            m = min(int(prefix[b]) + t + 1, length)
            for h in range(q.shape[1]):
                s = k[:m, h // group] @ q[lo + t, h] * scale
                if m == 0 or (s == -np.inf).all():
                    continue
                got[h // group, :m] += torch.softmax(s, 0)
                most = max(most, float((finite(k[:m, h // group]) @ finite(q[lo + t, h])).max() * scale))
        out.append((got, most))
    return out


def evict(mass, length, keep, first, recent):
    """one head's masses (numpy fp32): the positions that stay, in order"""
    n = len(mass[:max(0, length)])
    if n <= keep:
        return np.arange(n)
    order = sorted(range(first, n - recent), key=lambda i: (0 if np.isnan(mass[i]) else -1, 0.0 if np.isnan(mass[i]) else -float(mass[i]), i))
    return np.array(sorted(list(range(first)) + list(range(n - recent, n)) + order[:keep - first - recent]), dtype=np.int64)
