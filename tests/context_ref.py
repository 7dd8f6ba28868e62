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
                terms[rows, h] = (qh.abs() @ kh.abs().t()).amax(-1, keepdim=True) * scale
    return out, size, terms
