"""Operators of a decode step over images and long contexts, as measurable cases: `run` computes them in plain torch operations, or (`own`) makes
the calls of mllm_amd.qlinear that a program makes.

  rope     RMSNorm of every query and key head and their rotation by positions of several axes (time, height, width)
  append   the same on the way into a paged cache
  cross    softmax(scale * q K^T) V over an encoder's states (no token comes before another): a decoder's tokens over them, or the encoder's own, whole or in windows
  weights  what every cached key gets of the new tokens' attention, added to what it got before
  evict    the keys with the largest such weights, the first and the latest ones among them, into the pages of another table
  adjust   penalties of tokens that a row has seen, biases, and masks of the tokens that a grammar allows, on logits

Head counts and widths are those of the Qwen3 shaped layers that the benchmark and the tests use (32 query heads, 8 of keys, 128 wide), or generic.
"""
import math
import types

import numpy as np
import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
LARGEST_PAIRS = 4900 * 4900 * 16 * 80  # (row, key, query head, element) of the largest attention case
LARGEST_ROWS = 24 * 6000 * 8 * 128     # keys' elements of the largest eviction
LARGEST_LOGITS = 96 * 151936


def listed():
    return [
        # the next token of four sequences behind images, queries and keys as a Q4_0 projection leaves them, keys and values on their way into the cache
        {"name": "append_axes_f32_4", "kind": "append", "x": "f32", "tokens": 4, "heads": 32, "kv": 8, "d": 128, "rot": 128, "axes": 3, "order": "blocks", "pairs": "half", "norm": True, "far": 9000, "page": 16, "pages": 512},
        # a prompt with images through a model with an int8 or 4-bit checkpoint
        {"name": "rope_axes_bf16_5185", "kind": "rope", "x": "bf16", "tokens": 5185, "heads": 32, "kv": 8, "d": 128, "rot": 128, "axes": 3, "order": "turns", "pairs": "half", "norm": True, "far": 40000},
        # a decode token of four sequences over one picture's states each
        {"name": "cross_f32_4x1x1601", "kind": "cross", "x": "f32", "seqs": 4, "tokens": 1, "keys": 1601, "heads": 32, "kv": 8, "d": 128},
        # prompts of three sequences over the states of several pictures
        {"name": "cross_bf16_3x700x6404", "kind": "cross", "x": "bf16", "seqs": 3, "tokens": 700, "keys": 6404, "heads": 32, "kv": 8, "d": 128},
        # an encoder's own attention in windows of 64 patches
        {"name": "cross_bf16_160x64x64", "kind": "cross", "x": "bf16", "seqs": 160, "tokens": 64, "keys": 64, "heads": 16, "kv": 16, "d": 80},
        # an encoder's own attention over all patches of a large picture
        {"name": "cross_bf16_1x4900x4900", "kind": "cross", "x": "bf16", "seqs": 1, "tokens": 4900, "keys": 4900, "heads": 16, "kv": 16, "d": 80},
        # a decode token of sixteen sequences of ragged lengths
        {"name": "weights_bf16_16x1x8000", "kind": "weights", "x": "bf16", "seqs": 16, "tokens": 1, "keys": 8000, "heads": 32, "kv": 8, "d": 128, "page": 16, "decay": 1.0},
        # the last tokens of prompts, by which their keys are judged, fp32 queries of a Q4_0 model
        {"name": "weights_f32_6x32x7000", "kind": "weights", "x": "f32", "seqs": 6, "tokens": 32, "keys": 7000, "heads": 32, "kv": 8, "d": 128, "page": 16, "decay": 0.0},
        # one long prompt cut down to a quarter
        {"name": "evict_1x16384x4096", "kind": "evict", "seqs": 1, "keys": 16384, "keep": 4096, "first": 4, "recent": 64, "kv": 8, "d": 128, "page": 16},
        # many sequences that have outgrown their share of the cache
        {"name": "evict_24x6000x2048", "kind": "evict", "seqs": 24, "keys": 6000, "keep": 2048, "first": 4, "recent": 256, "kv": 8, "d": 128, "page": 64},
        # the next token of one sequence that a grammar binds
        {"name": "adjust_f32_1x151936", "kind": "adjust", "x": "f32", "rows": 1, "vocab": 151936, "history": 900, "penalties": True, "bias": 20, "masks": 1},
        # many sequences, 16-bit logits, some of them bound by grammars
        {"name": "adjust_bf16_96x151936", "kind": "adjust", "x": "bf16", "rows": 96, "vocab": 151936, "history": 6000, "penalties": True, "bias": 64, "masks": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "cross", "cross", "weights", "weights", "evict", "adjust"])
    x = rng.choice(["f32", "bf16"])
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 4, 4, 5, 7])
    if kind in ("rope", "append"):
        d = rng.choice([64, 80, 96, 128, 128, 256])
        c = {"kind": kind, "x": x, "tokens": _log(rng, 1, 4096), "heads": heads, "kv": kv, "d": d, "rot": rng.choice([d, d, d // 2 // 16 * 16]), "axes": rng.choice([1, 2, 3, 3, 4]),
             "order": rng.choice(["blocks", "turns"]), "pairs": rng.choice(["half", "half", "next"]), "norm": rng.random() < 0.7, "far": _log(rng, 64, 1 << 20)}
        if kind == "append":
            c["page"] = rng.choice([1, 8, 16, 24, 64, 256])
            c["pages"] = -(-c["tokens"] * rng.randint(2, 4) // c["page"])
        return c
    if kind == "cross":
        d = rng.choice([64, 72, 80, 96, 128, 128, 256])
        tokens, seqs = rng.choice([1, _log(rng, 2, 64), _log(rng, 2, 2048)]), _log(rng, 1, 64)
        keys = max(1, min(_log(rng, 1, 16384), LARGEST_PAIRS // (seqs * tokens * heads * d), (1 << 30) // (seqs * kv * d)))
        return {"kind": kind, "x": x, "seqs": seqs, "tokens": tokens, "keys": keys, "heads": heads, "kv": kv, "d": d}
    if kind == "weights":
        d = rng.choice([64, 128, 128, 128, 256])
        tokens, seqs = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 512)]), _log(rng, 1, 48)
        keys = tokens + _log(rng, 1, 32768)
        keys = max(tokens, min(keys, (1 << 29) // (seqs * kv * d), LARGEST_PAIRS // (seqs * tokens * heads * d)))
        return {"kind": kind, "x": x, "seqs": seqs, "tokens": tokens, "keys": keys, "heads": heads, "kv": kv, "d": d, "page": rng.choice([1, 8, 16, 16, 24, 64, 256]),
                "decay": rng.choice([0.0, 1.0, 1.0, 0.9])}
    if kind == "evict":
        d, seqs = rng.choice([64, 80, 128, 128, 256]), _log(rng, 1, 48)
        keys = max(8, min(_log(rng, 8, 65536), LARGEST_ROWS // (seqs * kv * d)))
        keep = max(4, int(keys * rng.uniform(0.1, 0.8)))
        return {"kind": kind, "seqs": seqs, "keys": keys, "keep": keep, "first": rng.randint(0, 4), "recent": rng.randint(0, max(0, keep // 2 - 4)), "kv": kv, "d": d,
                "page": rng.choice([1, 8, 16, 16, 24, 64, 256])}
    vocab = _log(rng, 1000, 260000)
    rows = max(1, min(_log(rng, 1, 512), LARGEST_LOGITS // vocab))
    return {"kind": kind, "x": x, "rows": rows, "vocab": vocab, "history": rng.choice([0, _log(rng, 1, 16384)]), "penalties": rng.random() < 0.8, "bias": rng.choice([0, 0, 1, 50, 300]),
            "masks": rng.choice([0, 0, 1, rows, 2 * rows])}


# --------------------------------------------------------------------------------------------------------------------- inputs
def _randn(shape, g, x):
    return torch.randn(shape, device="cuda", generator=g).to(BF16 if x == "bf16" else F32)


def _int(v):
    return torch.from_numpy(np.asarray(v, np.int32)).cuda()


def _counts(seqs, most, salt=0):
    """ragged numbers, the first sequence's the largest"""
    return np.concatenate([[most], np.random.RandomState((most * 31 + salt) % (1 << 31)).randint((most + 1) // 2, most + 1, seqs - 1)])


def _projections(s, c, g):
    """q, k and v as views of one projection's rows, weights of the norms, positions, the rotation's frequencies and the axis that each turns by"""
    t, h, kv, d, half = c["tokens"], c["heads"], c["kv"], c["d"], c["rot"] // 2
    rows = _randn((t, (h + 2 * kv) * d), g, c["x"]).view(t, h + 2 * kv, d)
    s.q, s.k, s.v = rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
    s.wq, s.wk = [1 + 0.2 * torch.randn(d, device="cuda", generator=g) if c["norm"] else None for _ in range(2)]
    # text goes up by one on every axis; a picture's rows and columns go up from where it begins
    first = torch.randint(0, max(1, c["far"] - t), (1, 1), device="cuda", generator=g)
    inside = torch.randint(0, 64, (c["axes"], t), device="cuda", generator=g)
    picture = torch.rand((1, t), device="cuda", generator=g) < 0.7
    s.positions = (first + torch.where(picture, inside, torch.arange(t, device="cuda"))).int()
    j = torch.arange(half, device="cuda")
    s.axes = (j % c["axes"] if c["order"] == "turns" else j * c["axes"] // half).int()
    s.inv_freq = 1e6 ** (-2.0 * j.double() / c["rot"])


def _queries(s, c, r, g):
    """ragged new tokens and their queries"""
    count = _counts(c["seqs"], c["tokens"])
    s.cu = _int(np.concatenate([[0], np.cumsum(count)]))
    s.q = _randn((int(count.sum()), c["heads"], c["d"]), g, c["x"]) * 1.5
    return count


def prepare(case, seed):
    c, s = case, types.SimpleNamespace(case=case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 32))
    kind = c["kind"]
    if kind in ("rope", "append"):
        _projections(s, c, g)
    if kind == "append":
        shape = (c["pages"], c["page"], c["kv"], c["d"])
        s.k_cache, s.v_cache = _randn(shape, g, "bf16"), _randn(shape, g, "bf16")
        # whole pages in the order the allocator gives them out, the last token a padded one
        pages = torch.from_numpy(r.permutation(c["pages"])).cuda()
        t = torch.arange(c["tokens"], device="cuda")
        s.slots = pages[t // c["page"]] * c["page"] + t % c["page"]
        if c["tokens"] > 1:
            s.slots[-1] = -1
    elif kind == "cross":
        _queries(s, c, r, g)
        # the states of all sequences behind one another
        held = _counts(c["seqs"], c["keys"], 1)
        s.first, s.held = _int(np.cumsum(held) - held), _int(held)
        s.k, s.v = [_randn((int(held.sum()), c["kv"], c["d"]), g, "bf16") for _ in range(2)]
    elif kind == "weights":
        b, keys, page = c["seqs"], c["keys"], c["page"]
        count = _queries(s, c, r, g)
        # the first sequence is as long as the case says, the others from a quarter of it on
        most = keys - c["tokens"]
        s.prefix = _int(np.concatenate([[most], r.randint(most // 4, most + 1, b - 1)]))
        per = -(-keys // page)
        s.block_table = _int(r.permutation(b * per).reshape(b, per))
        s.k_cache = _randn((b * per, page, c["kv"], c["d"]), g, "bf16")
        s.mass = torch.rand((b, c["kv"], keys), device="cuda", generator=g)
    elif kind == "evict":
        b, keys, page, keep = c["seqs"], c["keys"], c["page"], c["keep"]
        s.lengths = _int(np.concatenate([[keys], r.randint((keys + 1) // 2, keys + 1, b - 1)]))
        per, less = -(-keys // page), -(-keep // page)
        pages = r.permutation(b * (per + less))
        s.block_table, s.to_table = _int(pages[:b * per].reshape(b, per)), _int(pages[b * per:].reshape(b, less))
        s.k_cache, s.v_cache = [_randn((b * (per + less), page, c["kv"], c["d"]), g, "bf16") for _ in range(2)]
        # few keys have most of the attention, some have none
        mass = torch.randn((b, c["kv"], keys), device="cuda", generator=g).mul_(2).exp_()
        s.mass = mass.masked_fill_(torch.rand(mass.shape, device="cuda", generator=g) < 0.05, 0.0)
    elif kind == "adjust":
        rows, v, n = c["rows"], c["vocab"], c["history"]
        s.logits = _randn((rows, v), g, c["x"]) * 3
        s.history = s.lengths = s.prompts = s.repetition = s.presence = s.frequency = s.bias_tokens = s.bias = s.masks = s.mask_of = None
        if n:
            # a few tokens come again and again, most of them seldom
            s.history = (torch.rand((rows, n), device="cuda", generator=g).pow(3) * v).clamp(max=v - 1).int()
            s.lengths = _int(r.randint(n // 2, n + 1, rows))
            s.prompts = (s.lengths * torch.rand(rows, device="cuda", generator=g)).int()
        if c["penalties"]:
            s.repetition, s.presence, s.frequency = [_row(r, rows, lo, hi) for lo, hi in ((1.0, 1.5), (0.0, 1.0), (0.0, 0.5))]
        if c["bias"]:
            s.bias_tokens = _int(np.stack([r.permutation(min(v, 4096))[:c["bias"]] for _ in range(rows)]))
            s.bias = torch.randn((rows, s.bias_tokens.shape[1]), device="cuda", generator=g) * 5
        if c["masks"]:
            # states of grammars: some allow nearly everything, some nearly nothing
            share = torch.rand((c["masks"], 1, 1), device="cuda", generator=g)
            bits = torch.rand((c["masks"], -(-v // 32), 32), device="cuda", generator=g) < share
            s.masks = (bits.long() << torch.arange(32, device="cuda")).sum(-1).int()
            s.mask_of = _int(r.randint(-1 if rows > 1 else 0, c["masks"], rows))
    return s


def _row(r, rows, lo, hi):
    return torch.from_numpy(r.uniform(lo, hi, rows).astype(np.float32)).cuda()


# ----------------------------------------------------------------------------------------------------------------- plain forms
def _norm_rope(x, w, s, c):
    y = x.float()
    if w is not None:
        y = y * (w * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6))
    angle = s.positions.double()[s.axes.long()].t() * s.inv_freq
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


def _grouped(s, c):
    """queries of every sequence, padded to the longest: [seqs, kv, group * tokens, d]; how many each has"""
    b, n, kv, d = c["seqs"], c["tokens"], c["kv"], c["d"]
    count, at = (s.cu[1:] - s.cu[:-1]).long(), s.cu[:-1].long()
    row = (at[:, None] + torch.arange(n, device="cuda")).clamp(max=s.q.shape[0] - 1)
    return s.q[row].float().view(b, n, kv, -1, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d), count


def _softmax(scores):
    """along the last axis, in place; zeros where everything is masked"""
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(torch.where(total > 0, total, torch.ones_like(total)))


def _cross(s, c):
    b, n, kv, d, keys = c["seqs"], c["tokens"], c["kv"], c["d"], c["keys"]
    j = torch.arange(keys, device="cuda")
    row = (s.first.long()[:, None] + j).clamp(max=s.k.shape[0] - 1)
    k, v = [x[row].transpose(1, 2).float() for x in (s.k, s.v)]
    q, count = _grouped(s, c)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5)
    scores.masked_fill_(j >= s.held.long()[:, None, None, None], -math.inf)
    o = torch.matmul(_softmax(scores), v).view(b, kv, -1, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, -1, d).to(s.q.dtype)
    return o[torch.arange(n, device="cuda") < count[:, None]]


def _weights(s, c):
    b, n, kv, d, page, keys = c["seqs"], c["tokens"], c["kv"], c["d"], c["page"], c["keys"]
    k = s.k_cache[s.block_table.long()].view(b, -1, kv, d)[:, :keys].transpose(1, 2).float()
    q, count = _grouped(s, c)
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(b, kv, -1, n, keys)
    j, t, prefix = torch.arange(keys, device="cuda"), torch.arange(n, device="cuda"), s.prefix.long()
    seen = (j <= prefix[:, None, None] + t[:, None]) & (t[:, None] < count[:, None, None])
    got = _softmax(scores.masked_fill_(~seen[:, None, None], -math.inf)).sum((2, 3))
    before = torch.where(j < prefix[:, None, None], s.mass * c["decay"], torch.zeros_like(got))
    s.mass.copy_(torch.where(j < (prefix + count)[:, None, None], before + got, s.mass))
    return s.mass


def _evict(s, c):
    b, kv, keys, keep, page = c["seqs"], c["kv"], c["keys"], c["keep"], c["page"]
    j, length = torch.arange(keys, device="cuda"), s.lengths.long()[:, None, None]
    worth = torch.where((j < c["first"]) | (j >= length - c["recent"]), torch.full_like(s.mass, math.inf), s.mass)
    worth = torch.where(j < length, worth, torch.full_like(worth, -math.inf))
    index = torch.sort(worth, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    place = torch.arange(keep, device="cuda").expand(b, kv, keep)
    held = place < length
    mass = torch.where(held, s.mass.gather(2, index), torch.zeros((), device="cuda"))
    seq, head = torch.arange(b, device="cuda")[:, None, None].expand_as(place)[held], torch.arange(kv, device="cuda")[:, None].expand_as(place)[held]
    source, place = index[held], place[held]
    source_page, page_to = s.block_table[seq, source // page].long(), s.to_table[seq, place // page].long()
    s.k_cache[page_to, place % page, head] = s.k_cache[source_page, source % page, head]
    s.v_cache[page_to, place % page, head] = s.v_cache[source_page, source % page, head]
    return {"kept": torch.where(held, index, -1).int(), "mass": mass, "k_cache": s.k_cache, "v_cache": s.v_cache}


def _adjust(s, c):
    rows, v = c["rows"], c["vocab"]
    x = s.logits.float()
    if s.history is not None and s.repetition is not None:
        i = torch.arange(c["history"], device="cuda")
        zeros = torch.zeros((rows, v), device="cuda")
        seen = zeros.scatter_add(1, s.history.long(), (i < s.lengths[:, None]).float()) > 0
        count = zeros.scatter_add_(1, s.history.long(), ((i < s.lengths[:, None]) & (i >= s.prompts[:, None])).float())
        r = s.repetition[:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - (s.frequency[:, None] * count + torch.where(count > 0, s.presence[:, None], torch.zeros_like(count)))
    if s.bias is not None:
        x = x.scatter_add(1, s.bias_tokens.long(), s.bias)
    if s.masks is not None:
        bits = (s.masks[s.mask_of.long().clamp(min=0)][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        banned = (bits.view(rows, -1)[:, :v] == 0) & (s.mask_of >= 0)[:, None]
        x = x.masked_fill(banned, -math.inf)
    return x.to(s.logits.dtype)


def run(state):
    s, c = state, state.case
    kind = c["kind"]
    if own:
        from mllm_amd import qlinear as ql
        if kind == "rope":
            return ql.qk_norm_rope(s.q, s.k, s.positions, s.inv_freq, q_weight=s.wq, k_weight=s.wk, eps=1e-6, interleaved=c["pairs"] == "next", axes=s.axes)
        if kind == "append":
            q = ql.kv_append(s.k, s.v, s.k_cache, s.v_cache, s.slots, positions=s.positions, inv_freq=s.inv_freq, k_weight=s.wk, q=s.q, q_weight=s.wq,
                             eps=1e-6, interleaved=c["pairs"] == "next", axes=s.axes)
            return {"q": q, "k_cache": s.k_cache, "v_cache": s.v_cache}
        if kind == "cross":
            return ql.attention_cross(s.q, s.k, s.v, s.cu, s.first, s.held, c["tokens"], c["keys"])
        if kind == "weights":
            return ql.attention_weights(s.q, s.k_cache, s.mass, s.block_table, s.cu, s.prefix, c["tokens"], c["keys"], decay=c["decay"])
        if kind == "evict":
            kept, mass = ql.kv_evict(s.k_cache, s.v_cache, s.mass, s.block_table, s.lengths, s.to_table, c["keep"], first=c["first"], recent=c["recent"])
            return {"kept": kept, "mass": mass, "k_cache": s.k_cache, "v_cache": s.v_cache}
        return ql.adjust_logits(s.logits, s.history, s.lengths, s.prompts, s.repetition, s.presence, s.frequency, s.bias_tokens, s.bias, s.masks, s.mask_of)
    if kind == "rope":
        return tuple(_norm_rope(x, w, s, c).to(x.dtype) for x, w in ((s.q, s.wq), (s.k, s.wk)))
    return {"append": _append, "cross": _cross, "weights": _weights, "evict": _evict, "adjust": _adjust}[kind](s, c)


# ------------------------------------------------------------------------------------------------------- from the definitions
def _exact_rope(x, w, s, c):
    y = x.double().cpu()
    if w is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double().cpu()
    rot, half = c["rot"], c["rot"] // 2
    turn = torch.stack([s.positions[int(a)].cpu().double() * float(f) for a, f in zip(s.axes.tolist(), s.inv_freq.tolist())], 1)
    pair = torch.polar(torch.ones_like(turn), turn)[:, None]
    at = (range(half), range(half, rot)) if c["pairs"] == "half" else (range(0, rot, 2), range(1, rot, 2))
    z = torch.complex(y[..., list(at[0])], y[..., list(at[1])]) * pair
    out = y.clone()
    out[..., list(at[0])], out[..., list(at[1])] = z.real, z.imag
    return out


def _exact_cross(s, c):
    group, cu, out = c["heads"] // c["kv"], s.cu.tolist(), torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for b, (first, held) in enumerate(zip(s.first.tolist(), s.held.tolist())):
        for h in range(c["heads"]):
            k, v = s.k[first:first + held, h // group].double(), s.v[first:first + held, h // group].double()
            out[cu[b]:cu[b + 1], h] = torch.softmax(s.q[cu[b]:cu[b + 1], h].double() @ k.t() / math.sqrt(c["d"]), -1) @ v
    return out


def _exact_weights(s, c):
    group, page, cu, mass = c["heads"] // c["kv"], c["page"], s.cu.tolist(), s.mass.double()
    for b, prefix in enumerate(s.prefix.tolist()):
        n = cu[b + 1] - cu[b]
        at = torch.arange(prefix + n, device="cuda")
        pages = s.block_table[b].long()[at // page]
        hidden = torch.ones((n, prefix + n), dtype=torch.bool, device="cuda").triu(prefix + 1)
        mass[b, :, prefix:prefix + n] = 0
        mass[b, :, :prefix] *= c["decay"]
        for h in range(c["heads"]):
            z = s.q[cu[b]:cu[b + 1], h].double() @ s.k_cache[pages, at % page, h // group].double().t() / math.sqrt(c["d"])
            mass[b, h // group, :prefix + n] += torch.softmax(z.masked_fill(hidden, -math.inf), -1).sum(0)
    return mass


def _exact_evict(s, c):
    page, keep = c["page"], c["keep"]
    kept = np.full((c["seqs"], c["kv"], keep), -1, np.int32)
    mass, source = np.zeros(kept.shape), s.mass.cpu().numpy()
    k_cache, v_cache = s.k_cache.clone(), s.v_cache.clone()
    table, to_table = s.block_table.cpu().numpy(), s.to_table.cpu().numpy()
    for b, n in enumerate(s.lengths.tolist()):
        m = min(n, keep)
        for h in range(c["kv"]):
            value = source[b, h, :n].astype(np.float64)
            value[:c["first"]] = np.inf
            value[max(0, n - c["recent"]):] = np.inf
            index = np.sort(np.lexsort((np.arange(n), -value))[:m])
            kept[b, h, :m], mass[b, h, :m] = index, source[b, h, index]
            place = np.arange(m)
            old = [torch.from_numpy(v.astype(np.int64)).cuda() for v in (table[b, index // page], index % page)]
            new = [torch.from_numpy(v.astype(np.int64)).cuda() for v in (to_table[b, place // page], place % page)]
            k_cache[new[0], new[1], h], v_cache[new[0], new[1], h] = s.k_cache[old[0], old[1], h], s.v_cache[old[0], old[1], h]
    return {"kept": torch.from_numpy(kept), "mass": torch.from_numpy(mass), "k_cache": k_cache.double(), "v_cache": v_cache.double()}


def _exact_adjust(s, c):
    out = s.logits.double().cpu().numpy()
    host = lambda x: None if x is None else x.cpu().numpy()  # noqa: E731
    history, lengths, prompts, tokens, bias, masks, mask_of = [host(x) for x in (s.history, s.lengths, s.prompts, s.bias_tokens, s.bias, s.masks, s.mask_of)]
    penalties = [host(x) for x in (s.repetition, s.presence, s.frequency)]
    for row in range(c["rows"]):
        x = out[row]
        if history is not None and c["penalties"]:
            r, presence, frequency = [float(p[row]) for p in penalties]
            said = history[row, :lengths[row]]
            for token in np.unique(said):
                x[token] = x[token] / r if x[token] > 0 else x[token] * r
            for token, count in zip(*np.unique(said[prompts[row]:], return_counts=True)):
                x[token] -= presence + frequency * count
        if bias is not None:
            x[tokens[row]] += bias[row].astype(np.float64)
        if masks is not None and mask_of[row] >= 0:
            allowed = np.unpackbits(masks[mask_of[row]].view(np.uint8), bitorder="little")[:c["vocab"]]
            x[allowed == 0] = -np.inf
    return torch.from_numpy(out)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    if kind == "rope":
        return _exact_rope(s.q, s.wq, s, c), _exact_rope(s.k, s.wk, s, c)
    if kind == "append":
        kc, vc = s.k_cache.double().cpu(), s.v_cache.double().cpu()
        slots = s.slots.cpu()
        kept = slots >= 0
        kc.view(-1, c["kv"], c["d"])[slots[kept]] = _exact_rope(s.k, s.wk, s, c)[kept]
        vc.view(-1, c["kv"], c["d"])[slots[kept]] = s.v.double().cpu()[kept]
        return {"q": _exact_rope(s.q, s.wq, s, c), "k_cache": kc, "v_cache": vc}
    return {"cross": _exact_cross, "weights": _exact_weights, "evict": _exact_evict, "adjust": _exact_adjust}[kind](s, c)


def work(case):
    c, kind = case, case["kind"]
    wide = 4 if c.get("x") == "f32" else 2
    if kind in ("rope", "append"):
        t, h, kv, d = c["tokens"], c["heads"], c["kv"], c["d"]
        moved = t * (h + kv) * d * 2 * wide if kind == "rope" else t * d * (2 * h * wide + 2 * kv * (wide + 2))
        return {"bytes": moved + t * 4 * c["axes"], "flops": 8.0 * t * (h + kv) * d}
    if kind == "adjust":
        masks = min(c["masks"], c["rows"]) * c["vocab"] / 8
        return {"bytes": c["rows"] * (c["vocab"] * 2.0 * wide + 3 * c["history"] + 8 * c["bias"]) + masks, "flops": 4.0 * c["rows"] * c["vocab"]}
    d, kv = c["d"], c["kv"]
    if kind == "evict":
        # the other sequences have three quarters of the longest in the mean
        held = c["keys"] * (1 + 0.75 * (c["seqs"] - 1))
        return {"bytes": kv * (4.0 * held + c["seqs"] * c["keep"] * (8 * d + 8)), "flops": held * kv}
    count = _counts(c["seqs"], c["tokens"]).astype(float)
    if kind == "cross":
        held = _counts(c["seqs"], c["keys"], 1).astype(float)
        return {"bytes": float(held.sum()) * kv * d * 4 + float(count.sum()) * c["heads"] * d * 2 * wide, "flops": 4.0 * float((held * count).sum()) * c["heads"] * d}
    # the other sequences' prefixes are five eighths of the longest in the mean
    held = count + (c["keys"] - c["tokens"]) * np.where(np.arange(c["seqs"]) > 0, 0.625, 1.0)
    return {"bytes": float(held.sum()) * kv * (d * 2 + 8) + float(count.sum()) * c["heads"] * d * wide, "flops": 2.0 * float((held * count).sum()) * c["heads"] * d}
