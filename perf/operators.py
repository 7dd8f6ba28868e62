"""The operators between the Linears of a decode step, as measurable cases: `run` computes them in plain torch operations, or
(`own`) makes the calls of mllm_amd.qlinear that a program makes.

  rope       RMSNorm of every query and key head and their rotation (a prompt's or a step's q and k, views of one projection's rows)
  append     the same on the way into a paged cache: keys normed, rotated and stored, values stored, queries handed back
  attention  softmax(scale * q K^T) V over the pages of a cache, for one token a sequence, a tree of drafted tokens, or a chunk of a prompt
  sample     a token from logits by temperature, top-k, top-p, min-p and a given uniform number

Head counts and widths are those of the Qwen3 shaped layers that the benchmark and the tests use (32 query heads, 8 of keys, 128
wide), or generic.
"""
import math
import types

import numpy as np
import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
LARGEST_BYTES = 32 * 8192 * 8 * 128 * 4  # keys and values of the largest attention case
LARGEST_PAIRS = 32 * 8192 * 64 * 32      # (sequence, key, token, query head) of it
LARGEST_LOGITS = 128 * 151936


def listed():
    return [
        # one sequence's decode token: q and k as a Q4_0 projection leaves them
        {"name": "rope_f32_1", "kind": "rope", "x": "f32", "tokens": 1, "heads": 32, "kv": 8, "d": 128, "rot": 128, "pairs": "half", "norm": True, "far": 40000},
        # a prompt of an odd length through a model with an int8 or 4-bit checkpoint
        {"name": "rope_bf16_8191", "kind": "rope", "x": "bf16", "tokens": 8191, "heads": 32, "kv": 8, "d": 128, "rot": 128, "pairs": "half", "norm": True, "far": 131072},
        # a verification step of five drafted tokens for eight sequences
        {"name": "append_f32_40", "kind": "append", "x": "f32", "tokens": 40, "heads": 32, "kv": 8, "d": 128, "rot": 128, "pairs": "half", "norm": True, "far": 8192, "page": 16, "pages": 2048},
        # a long prompt into the cache, without norms, rotated by neighbouring pairs over half of a head
        {"name": "append_bf16_6007", "kind": "append", "x": "bf16", "tokens": 6007, "heads": 16, "kv": 4, "d": 128, "rot": 64, "pairs": "next", "norm": False, "far": 8192, "page": 64, "pages": 512},
        # a decode token of one sequence
        {"name": "attention_bf16_1x1x4097", "kind": "attention", "x": "bf16", "seqs": 1, "tokens": 1, "keys": 4097, "heads": 32, "kv": 8, "d": 128, "page": 16, "tree": False},
        # a decode token of sixteen sequences of ragged lengths, fp32 queries of a Q4_0 model
        {"name": "attention_f32_16x1x8000", "kind": "attention", "x": "f32", "seqs": 16, "tokens": 1, "keys": 8000, "heads": 32, "kv": 8, "d": 128, "page": 16, "tree": False},
        # a tree of drafted tokens for eight sequences
        {"name": "attention_bf16_8x29x5000", "kind": "attention", "x": "bf16", "seqs": 8, "tokens": 29, "keys": 5000, "heads": 32, "kv": 8, "d": 128, "page": 32, "tree": True},
        # large trees for many sequences of long contexts
        {"name": "attention_bf16_32x64x8192", "kind": "attention", "x": "bf16", "seqs": 32, "tokens": 64, "keys": 8192, "heads": 32, "kv": 8, "d": 128, "page": 64, "tree": True},
        # the next token of one sequence with the usual settings
        {"name": "sample_f32_1x151936", "kind": "sample", "x": "f32", "rows": 1, "vocab": 151936, "k": 20, "p": 0.95, "min_p": 0.0, "t": 0.6},
        # eight sequences that cut by mass alone
        {"name": "sample_f32_8x151936", "kind": "sample", "x": "f32", "rows": 8, "vocab": 151936, "k": 0, "p": 0.9, "min_p": 0.0, "t": 1.0},
        # many sequences, each with settings of its own, 16-bit logits
        {"name": "sample_bf16_128x151936", "kind": "sample", "x": "bf16", "rows": 128, "vocab": 151936, "k": -1, "p": -1.0, "min_p": -1.0, "t": -1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attention", "attention", "attention", "sample", "sample"])
    x = rng.choice(["f32", "bf16"])
    if kind in ("rope", "append"):
        d = rng.choice([64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        c = {"kind": kind, "x": x, "tokens": _log(rng, 1, 4096), "heads": kv * rng.choice([1, 2, 4, 5, 7]), "kv": kv, "d": d,
             "rot": rng.choice([d, d, d // 2 // 16 * 16]), "pairs": rng.choice(["half", "half", "next"]), "norm": rng.random() < 0.7, "far": _log(rng, 64, 1 << 20)}
        if kind == "append":
            c["page"] = rng.choice([1, 8, 16, 24, 64, 256])
            c["pages"] = -(-c["tokens"] * rng.randint(2, 4) // c["page"])
        return c
    if kind == "attention":
        kv = rng.choice([1, 2, 4, 8, 8])
        heads = kv * rng.choice([1, 2, 4, 4, 5, 8])
        d = rng.choice([64, 128, 128, 128, 256])
        tokens = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 512)])
        seqs = _log(rng, 1, 48)
        keys = tokens + _log(rng, 16, 65536)
        keys = max(tokens, min(keys, LARGEST_BYTES // (seqs * kv * d * 4), LARGEST_PAIRS * 128 // (seqs * tokens * heads * d)))
        return {"kind": kind, "x": x, "seqs": seqs, "tokens": tokens, "keys": keys, "heads": heads, "kv": kv, "d": d,
                "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 256]), "tree": tokens <= 256 and rng.random() < 0.6}
    vocab = _log(rng, 1000, 260000)
    return {"kind": kind, "x": x, "rows": max(1, min(_log(rng, 1, 512), LARGEST_LOGITS // vocab)), "vocab": vocab, "k": rng.choice([-1, 0, 1, 20, 50, 400, 5000]),
            "p": rng.choice([-1.0, 1.0, 0.5, 0.9, 0.99]), "min_p": rng.choice([-1.0, 0.0, 0.0, 0.05]), "t": rng.choice([-1.0, 0.6, 1.0, 1.5])}


# --------------------------------------------------------------------------------------------------------------------- inputs
def _randn(shape, g, x):
    return torch.randn(shape, device="cuda", generator=g).to(BF16 if x == "bf16" else F32)


def _projections(s, c, g):
    """q, k and v as views of one projection's rows, weights of the norms, positions and the rotation's frequencies"""
    t, h, kv, d = c["tokens"], c["heads"], c["kv"], c["d"]
    rows = _randn((t, (h + 2 * kv) * d), g, c["x"]).view(t, h + 2 * kv, d)
    s.q, s.k, s.v = rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
    s.wq, s.wk = [1 + 0.2 * torch.randn(d, device="cuda", generator=g) if c["norm"] else None for _ in range(2)]
    first = torch.randint(0, max(1, c["far"] - t), (1,), device="cuda", generator=g)
    s.positions = (first + torch.arange(t, device="cuda")).int()
    s.inv_freq = 1e6 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])


def _ancestors(seqs, tokens, g):
    """[seqs, tokens, tokens]: whether token j is on the way from the root to token i (itself among them); a token's parent comes before it"""
    parent = (torch.rand((seqs, tokens), device="cuda", generator=g) * torch.arange(tokens, device="cuda")).long()
    near = torch.zeros((seqs, tokens, tokens), device="cuda")
    near.scatter_(2, parent[..., None], 1.0)
    near = ((near + torch.eye(tokens, device="cuda")) > 0).float()
    for _ in range(max(1, tokens - 1).bit_length()):
        near = (torch.bmm(near, near) > 0).float()
    return near > 0


def _words(seen):
    """truth values [rows, n] as int64 words of 64 bits each [rows, ceil(n / 64)], bit j % 64 of word j // 64"""
    rows, n = seen.shape
    bits = torch.zeros((rows, -(-n // 64) * 64), dtype=torch.int64, device=seen.device)
    bits[:, :n] = seen
    return (bits.view(rows, -1, 64) << torch.arange(64, device=seen.device)).sum(-1)


def _counts(seqs, tokens):
    """ragged numbers of tokens, the first sequence's the largest"""
    return np.concatenate([[tokens], np.random.RandomState(tokens).randint(max(1, tokens // 2), tokens + 1, seqs - 1)])


def prepare(case, seed):
    c, s = case, types.SimpleNamespace(case=case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 32))
    if c["kind"] in ("rope", "append"):
        _projections(s, c, g)
    if c["kind"] == "append":
        shape = (c["pages"], c["page"], c["kv"], c["d"])
        s.k_cache, s.v_cache = _randn(shape, g, "bf16"), _randn(shape, g, "bf16")
        # whole pages in the order the allocator gives them out, the last token a padded one
        pages = torch.from_numpy(r.permutation(c["pages"])).cuda()
        t = torch.arange(c["tokens"], device="cuda")
        s.slots = pages[t // c["page"]] * c["page"] + t % c["page"]
        if c["tokens"] > 1:
            s.slots[-1] = -1
    elif c["kind"] == "attention":
        b, n, keys, page = c["seqs"], c["tokens"], c["keys"], c["page"]
        # the first sequence is as long as the case says, the others from a quarter of it on
        prefix = np.concatenate([[keys - n], r.randint((keys - n) // 4, keys - n + 1, b - 1)])
        count = _counts(b, n)
        per = -(-keys // page)
        table = r.permutation(b * per).reshape(b, per)
        s.block_table = torch.from_numpy(table.astype(np.int32)).cuda()
        s.cu = torch.from_numpy(np.concatenate([[0], np.cumsum(count)]).astype(np.int32)).cuda()
        s.prefix = torch.from_numpy(prefix.astype(np.int32)).cuda()
        s.k_cache, s.v_cache = [_randn((b * per, page, c["kv"], c["d"]), g, "bf16") for _ in range(2)]
        s.q = _randn((int(count.sum()), c["heads"], c["d"]), g, c["x"]) * 1.5
        s.tree = None
        if c["tree"]:
            own_row = torch.from_numpy(np.repeat(np.arange(b), count)).cuda()
            own_token = torch.from_numpy(np.concatenate([np.arange(m) for m in count])).cuda()
            s.tree = _words(_ancestors(b, n, g)[own_row, own_token])
    elif c["kind"] == "sample":
        rows, v = c["rows"], c["vocab"]
        spread = torch.rand((rows, 1), device="cuda", generator=g) * 2 + 1.5
        s.logits = (torch.randn((rows, v), device="cuda", generator=g) * spread).to(BF16 if c["x"] == "bf16" else F32)
        s.u = torch.rand(rows, device="cuda", generator=g)
        pick = lambda value, choices: torch.tensor([value] * rows if value != -1 else r.choice(choices, rows), device="cuda")  # noqa: E731
        s.t = pick(c["t"], [0.0, 0.3, 0.7, 1.0, 1.3]).float()
        s.k = pick(c["k"], [0, 1, 20, 64, 1000]).int()
        s.p = pick(c["p"], [0.3, 0.8, 0.95, 1.0]).float()
        s.min_p = pick(c["min_p"], [0.0, 0.02, 0.1]).float()
    return s


# ----------------------------------------------------------------------------------------------------------------- plain forms
def _norm_rope(x, w, s, c):
    y = x.float()
    if w is not None:
        y = y * (w * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6))
    angle = s.positions.double()[:, None] * s.inv_freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half, rot = c["rot"] // 2, c["rot"]
    if c["pairs"] == "half":
        a, b = y[..., :half], y[..., half:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1)


def _append(s, c):
    page, kept = c["page"], (s.slots >= 0).nonzero()[:, 0]
    at = s.slots[kept]
    s.k_cache[at // page, at % page] = _norm_rope(s.k, s.wk, s, c)[kept].to(BF16)
    s.v_cache[at // page, at % page] = s.v[kept].to(BF16)
    return {"q": _norm_rope(s.q, s.wq, s, c).to(s.q.dtype), "k_cache": s.k_cache, "v_cache": s.v_cache}


def _attention(s, c):
    b, n, kv, d, page = c["seqs"], c["tokens"], c["kv"], c["d"], c["page"]
    per = s.block_table.shape[1]
    # every sequence padded to the longest: queries [b, kv, group * n, d], keys and values [b, kv, keys, d]
    k, v = [x[s.block_table.long()].view(b, per * page, kv, d).transpose(1, 2).float() for x in (s.k_cache, s.v_cache)]
    count, at = (s.cu[1:] - s.cu[:-1]).long(), s.cu[:-1].long()
    token = torch.arange(n, device="cuda")
    row = (at[:, None] + token).clamp(max=s.q.shape[0] - 1)
    q = s.q[row].float().view(b, n, kv, -1, d).permute(0, 2, 3, 1, 4)
    group = q.shape[2]
    scores = torch.matmul(q.reshape(b, kv, group * n, d), k.transpose(2, 3)).view(b, kv, group, n, -1) * d ** -0.5
    j = torch.arange(per * page, device="cuda") - s.prefix.long()[:, None]
    j = j[:, None].expand(b, n, per * page)
    if s.tree is None:
        seen = j <= token[:, None]
    else:
        word = s.tree[row].gather(2, (j.clamp(0, s.tree.shape[1] * 64 - 1) // 64))
        seen = (j < 0) | ((word >> (j.clamp(min=0) % 64)) & 1).bool()
    seen = seen & (j < count[:, None, None])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    o = torch.matmul(scores.view(b, kv, group * n, -1), v).view(b, kv, group, n, d) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, kv * group, d).to(s.q.dtype)
    return o[token < count[:, None]]


def _sample(s, c):
    x = s.logits.double()
    rows, v = x.shape
    ordered, index = torch.sort(x, dim=-1, descending=True, stable=True)
    t = s.t.double()[:, None]
    w = ((ordered - ordered[:, :1]) / torch.where(t > 0, t, torch.ones_like(t))).exp()
    w = torch.where(w < 2.0 ** -52, torch.zeros_like(w), w)
    rank = torch.arange(v, device="cuda")
    k = torch.where((s.k <= 0) | (t[:, 0] <= 0), v, s.k.long())
    k = torch.where(t[:, 0] > 0, k, torch.ones_like(k))[:, None]
    w = torch.where(rank < k, w, torch.zeros_like(w))
    mass = w.cumsum(-1)
    p = s.p.double()[:, None]
    keep = (mass - w < p * mass[:, -1:]) | (p >= 1) | (rank == 0)
    w = torch.where(keep & (w >= s.min_p.double()[:, None]), w, torch.zeros_like(w))
    by_index = torch.zeros_like(w).scatter_(1, index, w).cumsum(-1)
    target = s.u.double()[:, None] * by_index[:, -1:]
    return (by_index <= target).sum(-1).int()


def run(state):
    s, c = state, state.case
    kind = c["kind"]
    if own:
        from mllm_amd import qlinear as ql
        if kind == "rope":
            return ql.qk_norm_rope(s.q, s.k, s.positions, s.inv_freq, q_weight=s.wq, k_weight=s.wk, eps=1e-6, interleaved=c["pairs"] == "next")
        if kind == "append":
            q = ql.kv_append(s.k, s.v, s.k_cache, s.v_cache, s.slots, positions=s.positions, inv_freq=s.inv_freq, k_weight=s.wk, q=s.q, q_weight=s.wq,
                             eps=1e-6, interleaved=c["pairs"] == "next")
            return {"q": q, "k_cache": s.k_cache, "v_cache": s.v_cache}
        if kind == "attention":
            return ql.attention_paged(s.q, s.k_cache, s.v_cache, s.block_table, s.cu, s.prefix, c["tokens"], c["keys"], tree=s.tree)
        return ql.sample(s.logits, s.u, temperature=s.t, top_k=s.k, top_p=s.p, min_p=s.min_p)
    if kind == "rope":
        return tuple(_norm_rope(x, w, s, c).to(x.dtype) for x, w in ((s.q, s.wq), (s.k, s.wk)))
    return _append(s, c) if kind == "append" else _attention(s, c) if kind == "attention" else _sample(s, c)


# ------------------------------------------------------------------------------------------------------- from the definitions
def _exact_rope(x, w, s, c):
    y = x.double().cpu()
    if w is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double().cpu()
    turn = torch.outer(s.positions.cpu().double(), s.inv_freq.cpu())
    pair = torch.polar(torch.ones_like(turn), turn)[:, None]
    rot, half = c["rot"], c["rot"] // 2
    at = (range(half), range(half, rot)) if c["pairs"] == "half" else (range(0, rot, 2), range(1, rot, 2))
    z = torch.complex(y[..., list(at[0])], y[..., list(at[1])]) * pair
    out = y.clone()
    out[..., list(at[0])], out[..., list(at[1])] = z.real, z.imag
    return out


def _exact_attention(s, c):
    group, page, d = c["heads"] // c["kv"], c["page"], c["d"]
    cu, prefix, out = s.cu.tolist(), s.prefix.tolist(), torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for b in range(c["seqs"]):
        n, length = cu[b + 1] - cu[b], prefix[b] + cu[b + 1] - cu[b]
        at = torch.arange(length, device="cuda")
        pages = s.block_table[b].long()[at // page]
        seen = torch.ones((n, length), dtype=torch.bool, device="cuda")
        bits = torch.ones((n, n), device="cuda").tril().bool()
        if s.tree is not None:
            words = s.tree[cu[b]:cu[b + 1]]
            bits = torch.stack([(words[:, i // 64] >> (i % 64)) % 2 != 0 for i in range(n)], 1)
        seen[:, prefix[b]:] = bits
        for h in range(c["kv"]):
            k, v = s.k_cache[pages, at % page, h].double(), s.v_cache[pages, at % page, h].double()
            for i in range(group):
                z = s.q[cu[b]:cu[b + 1], h * group + i].double() @ k.t() / math.sqrt(d)
                z = torch.where(seen, z, torch.full_like(z, -math.inf))
                out[cu[b]:cu[b + 1], h * group + i] = torch.softmax(z, -1).nan_to_num(0.0) @ v
    return out


def _exact_sample(s):
    tokens = []
    for x, u, t, k, p, min_p in zip(s.logits.double().cpu().numpy(), s.u.tolist(), s.t.tolist(), s.k.tolist(), s.p.tolist(), s.min_p.tolist()):
        if t <= 0:
            tokens.append(int(np.argmax(x)))
            continue
        w = np.exp((x - x.max()) / t)
        w[w < 2.0 ** -52] = 0
        order = np.lexsort((np.arange(len(x)), -x))
        if 0 < k < len(x):
            w[order[k:]] = 0
        if p < 1:
            before = np.concatenate([[0.0], np.cumsum(w[order])])
            cut = max(1, int(np.searchsorted(before, p * before[-1], "left")))
            w[order[cut:]] = 0
        w[w < min_p] = 0
        up_to = np.cumsum(w)
        tokens.append(int(np.searchsorted(up_to, u * up_to[-1], "right")))
    return torch.tensor(tokens, dtype=torch.int32)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "rope":
        return _exact_rope(s.q, s.wq, s, c), _exact_rope(s.k, s.wk, s, c)
    if c["kind"] == "append":
        kc, vc = s.k_cache.double().cpu(), s.v_cache.double().cpu()
        k = _exact_rope(s.k, s.wk, s, c)
        slots, v = s.slots.cpu(), s.v.double().cpu()
        kept = slots >= 0
        kc.view(-1, c["kv"], c["d"])[slots[kept]] = k[kept]
        vc.view(-1, c["kv"], c["d"])[slots[kept]] = v[kept]
        return {"q": _exact_rope(s.q, s.wq, s, c), "k_cache": kc, "v_cache": vc}
    if c["kind"] == "attention":
        return _exact_attention(s, c)
    return _exact_sample(s) if c["rows"] * c["vocab"] <= LARGEST_LOGITS else None


def work(case):
    c = case
    wide = 4 if c["x"] == "f32" else 2
    if c["kind"] in ("rope", "append"):
        t, h, kv, d = c["tokens"], c["heads"], c["kv"], c["d"]
        moved = t * (h + kv) * d * 2 * wide if c["kind"] == "rope" else t * d * (2 * h * wide + 2 * kv * (wide + 2))
        return {"bytes": moved + t * 4, "flops": 8.0 * t * (h + kv) * d}
    if c["kind"] == "attention":
        # the other sequences' prefixes are five eighths of the longest in the mean
        count = _counts(c["seqs"], c["tokens"]).astype(float)
        held = count + (c["keys"] - c["tokens"]) * np.where(np.arange(c["seqs"]) > 0, 0.625, 1.0)
        return {"bytes": float(held.sum()) * c["kv"] * c["d"] * 4 + float(count.sum()) * c["heads"] * c["d"] * 2 * wide,
                "flops": 4.0 * float((held * count).sum()) * c["heads"] * c["d"]}
    return {"bytes": c["rows"] * (c["vocab"] * wide + 24), "flops": 4.0 * c["rows"] * c["vocab"]}
