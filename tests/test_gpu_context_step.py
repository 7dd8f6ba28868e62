"""The operators over images and long contexts together, as a program uses them: an encoder's own attention over its patches with rotation by rows and columns, a prompt with positions on
three axes into a paged cache, attention over the encoder's states, eviction by what the prompt's last tokens look at, decode steps over what is left that go on adding, and the next
token under penalties and a grammar.  Against the same in 64 bits on the CPU, with what is stored in bf16 (the cache, the states) taken from the device.

Bounds.  Attention with fp32 queries is within 2^-17 of a sum of absolute terms and its own fp32 sums (see their tests); what comes before a comparison here is one rotation (24 * 2^-24) and one
product of 64 terms in fp32: 1e-4 of the largest element is asked for, 1e-3 behind two attentions and a product in a row.  Masses are sums of weights whose scores are off by as much."""
import numpy as np
import pytest
import torch

from mllm_amd import qlinear as ql
import context_ref as ref
import decode_ref
from gpu_util import announce

pytestmark = pytest.mark.gpu
HEADS, KV, D, PAGE, VOCAB = 8, 2, 64, 16, 700


def _int(v):
    return torch.from_numpy(np.asarray(v, np.int32)).cuda()


def _near(got, want, tol):
    want = want.double().cpu()
    assert torch.isfinite(got).all()
    far = (got.cpu().double() - want).abs().max() / want.abs().max()
    assert far <= tol, far.item()


def _encoder(gen, rows, columns):
    """patches of one picture through one attention: states of KV heads for the decoder, and what they are in 64 bits"""
    n, d = rows * columns, 80
    q, k, v = [torch.randn((n, 4, d), device="cuda", generator=gen) for _ in range(3)]
    freq = 1e4 ** (-torch.arange(0, d, 4, dtype=torch.float64, device="cuda") / d)
    freq, axes = torch.cat([freq, freq]), _int([0] * (d // 4) + [1] * (d // 4))
    at = torch.arange(n, device="cuda")
    pos = torch.stack([at // columns, at % columns]).int()
    rq, rk = ql.qk_norm_rope(q, k, pos, freq, axes=axes)
    _near(rq, ref.norm_rope_axes(q, None, 0, pos, axes, freq, False)[0], 1e-5)
    kb, vb = rk.bfloat16(), v.bfloat16()
    # in windows of two rows of patches, then all
    window = 2 * columns
    first = np.arange(0, n, window)
    count = np.minimum(window, n - first)
    o = ql.attention_cross(rq, kb, vb, _int(np.append(first, n)), _int(first), _int(count), window, window)
    _near(o, ref.cross(rq, kb, vb, np.append(first, n), first, count, d ** -0.5)[0], 1e-4)
    whole = ql.attention_cross(rq, kb, vb, _int([0, n]), _int([0]), _int([n]), n, n)
    _near(whole, ref.cross(rq, kb, vb, [0, n], [0], [n], d ** -0.5)[0], 1e-4)
    return ql.matmul(whole.view(n, -1), torch.randn((4 * d, 2 * KV * D), device="cuda", generator=gen) / (4 * d) ** 0.5).view(n, 2 * KV, D).bfloat16()


class Sequences:
    """two sequences with caches of their own pages, one layer"""

    def __init__(self, gen, prompts, keep, steps):
        self.gen, self.keep, self.steps = gen, keep, steps
        per, less = -(-max(prompts) // PAGE), -(-(keep + steps) // PAGE)
        ids = np.random.default_rng(1).permutation(2 * (per + less))
        self.table, self.to = ids[:2 * per].reshape(2, per), ids[2 * per:].reshape(2, less)
        shape = (2 * (per + less), PAGE, KV, D)
        self.k, self.v = [torch.full(shape, float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        self.freq = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
        self.axes = _int(np.arange(D // 2) % 3)
        self.mass = torch.full((2, KV, max(prompts)), float("nan"), device="cuda")

    def append(self, n, table, places, pos):
        """keys and values of n tokens of both sequences at these places; their rotated queries"""
        rows = torch.randn((n, HEADS + 2 * KV, D), device="cuda", generator=self.gen)
        slots = torch.tensor([int(table[b][p // PAGE]) * PAGE + p % PAGE for b, p in places], device="cuda")
        q = ql.kv_append(rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:], self.k, self.v, slots, pos, self.freq, None, rows[:, :HEADS], None, axes=self.axes)
        _near(q, ref.norm_rope_axes(rows[:, :HEADS], None, 0, pos, self.axes, self.freq, False)[0], 1e-5)
        return q


def _positions(n, first, patches, columns):
    """text, a picture of `patches`, text: on three axes"""
    t = np.arange(n)
    inside = (t >= 5) & (t < 5 + patches)
    p = t - 5
    after = np.where(t < 5, t, 5 + patches // columns + (t - 5 - patches))
    return first + np.stack([np.where(inside, 5, after), np.where(inside, 5 + p // columns, after), np.where(inside, 5 + p % columns, after)])


def test_a_prompt_with_a_picture_eviction_and_decode_steps():
    announce("context step")
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts, keep, steps, look = [150, 90], 60, 4, 8
    states = _encoder(gen, 7, 6)
    sk, sv = states[:, :KV], states[:, KV:]
    s = Sequences(gen, prompts, keep, steps)
    n = sum(prompts)
    pos = torch.from_numpy(np.concatenate([_positions(p, 0, 42, 6) for p in prompts], 1).astype(np.int32)).cuda()
    q = s.append(n, s.table, [(b, i) for b, p in enumerate(prompts) for i in range(p)], pos)
    cu = [0, prompts[0], n]
    o = ql.attention_paged(q, s.k, s.v, _int(s.table), _int(cu), _int([0, 0]), max(prompts), max(prompts))
    want, _, _ = decode_ref.attention(q, s.k, s.v, torch.from_numpy(s.table), cu, [0, 0], [np.tril(np.ones((p, p), bool)) for p in prompts], D ** -0.5)
    _near(o, want, 1e-4)
    # over the picture's states, which both sequences share
    c = ql.attention_cross(o, sk, sv, _int(cu), _int([0, 0]), _int([42, 42]), max(prompts), 42)
    _near(c, ref.cross(o, sk, sv, cu, [0, 0], [42, 42], D ** -0.5)[0], 1e-4)
    # what the last tokens look at
    late = torch.cat([q[b - look:b] for b in cu[1:]])
    prefix = [p - look for p in prompts]
    ql.attention_weights(late, s.k, s.mass, _int(s.table), _int([0, look, 2 * look]), _int(prefix), look, max(prompts), decay=0.0)
    for b, (w, _) in enumerate(ref.weights(late, s.k, torch.from_numpy(s.table), [0, look, 2 * look], prefix, D ** -0.5)):
        _near(s.mass[b, :, :prompts[b]], w, 1e-4)
    # cut down to `keep`, on pages of their own
    kept, left = ql.kv_evict(s.k, s.v, s.mass, _int(s.table), _int(prompts), _int(s.to), keep, first=4, recent=look)
    m = s.mass.cpu().numpy()
    for b in range(2):
        for h in range(KV):
            at = ref.evict(m[b, h], prompts[b], keep, 4, look)
            assert np.array_equal(kept[b, h].cpu().numpy(), at)
            page, place = torch.from_numpy(s.table[b][at // PAGE]).cuda(), torch.from_numpy(at % PAGE).cuda()
            now, where = torch.from_numpy(s.to[b][np.arange(keep) // PAGE]).cuda(), torch.arange(keep, device="cuda") % PAGE
            assert torch.equal(s.k[now, where, h], s.k[page, place, h]) and torch.equal(s.v[now, where, h], s.v[page, place, h])
    # decode steps over what is left
    mass = torch.full((2, KV, keep + steps), float("nan"), device="cuda")
    mass[..., :keep] = left
    head = torch.randn((HEADS * D, VOCAB), device="cuda", generator=gen) / (HEADS * D) ** 0.5
    history = torch.zeros((2, steps + 3), dtype=torch.int32, device="cuda")
    history[:, :3] = _int([[5, 9, 5], [0, 1, 2]])
    allowed = np.random.default_rng(2).random((1, VOCAB)) < 0.5
    masks = torch.from_numpy(np.packbits(np.pad(allowed, ((0, 0), (0, -VOCAB % 32))), axis=1, bitorder="little").view(np.int32)).cuda()
    for i in range(steps):
        pos = torch.from_numpy(np.stack([_positions(p + i + 1, 0, 42, 6)[:, -1] for p in prompts], 1).astype(np.int32)).cuda()
        q = s.append(2, s.to, [(b, keep + i) for b in range(2)], pos)
        o = ql.attention_paged(q, s.k, s.v, _int(s.to), _int([0, 1, 2]), _int([keep + i] * 2), 1, keep + steps)
        want, _, _ = decode_ref.attention(q, s.k, s.v, torch.from_numpy(s.to), [0, 1, 2], [keep + i] * 2, [np.ones((1, 1), bool)] * 2, D ** -0.5)
        _near(o, want, 1e-4)
        before = mass.clone()
        ql.attention_weights(q, s.k, mass, _int(s.to), _int([0, 1, 2]), _int([keep + i] * 2), 1, keep + steps, decay=0.9)
        for b, (w, _) in enumerate(ref.weights(q, s.k, torch.from_numpy(s.to), [0, 1, 2], [keep + i] * 2, D ** -0.5)):
            w[:, :keep + i] += float(np.float32(0.9)) * before[b, :, :keep + i].cpu().double()
            _near(mass[b, :, :keep + i + 1], w, 1e-4)
        c = ql.attention_cross(o, sk, sv, _int([0, 1, 2]), _int([0, 0]), _int([42, 42]), 1, 42)
        logits = ql.matmul(c.view(2, HEADS * D), head)
        _near(logits, ref.cross(o, sk, sv, [0, 1, 2], [0, 0], [42, 42], D ** -0.5)[0].reshape(2, -1) @ head.cpu().double(), 1e-3)
        x = ql.adjust_logits(logits, history, _int([3 + i] * 2), _int([3, 3]), torch.full((2,), 1.25, device="cuda"), torch.full((2,), 0.5, device="cuda"), torch.full((2,), 0.25, device="cuda"),
                             masks=masks, mask_of=_int([0, -1]))
        for b in range(2):
            w, size = ref.adjust(logits[b].cpu().numpy(), history[b, :3 + i].tolist(), 3, 1.25, 0.5, 0.25, (), allowed[0] if b == 0 else None)
            got, fine = x[b].cpu().double().numpy(), np.isfinite(w)
            assert np.array_equal(np.isfinite(got), fine) and (np.abs(got[fine] - w[fine]) <= 5 * 2.0 ** -24 * size[fine] + 1e-40).all()
        token = ql.sample(x, torch.tensor([0.3, 0.8], device="cuda"), top_k=_int([20, 0]), top_p=torch.tensor([1.0, 0.9], device="cuda"))
        assert allowed[0][token[0].item()] and 0 <= token[1] < VOCAB
        history[:, 3 + i] = token


def test_eviction_that_keeps_everything_changes_no_step():
    announce("context step: nothing evicted")
    gen = torch.Generator(device="cuda").manual_seed(2)
    prompts, keep = [40, 33], 44
    s = Sequences(gen, prompts, keep, 2)
    pos = torch.from_numpy(np.concatenate([_positions(p, 0, 12, 4) for p in prompts], 1).astype(np.int32)).cuda()
    s.append(sum(prompts), s.table, [(b, i) for b, p in enumerate(prompts) for i in range(p)], pos)
    s.mass.fill_(1.0)
    kept, _ = ql.kv_evict(s.k, s.v, s.mass, _int(s.table), _int(prompts), _int(s.to), keep)
    assert (kept[0, :, 40:] == -1).all() and (kept[1, :, 33:] == -1).all()
    q = torch.randn((2, HEADS, D), device="cuda", generator=gen)
    results = []
    for table in (s.table, s.to):  # a step whose key is there already, as the last of the prompt
        results.append(ql.attention_paged(q, s.k, s.v, _int(table), _int([0, 1, 2]), _int([39, 32]), 1, 48))
    assert torch.equal(*results)


def test_captured_steps_that_share_a_workspace():
    """attention over the cache, over states and the weights in one graph, every call with the same workspace, replayed while the sequences grow"""
    announce("context step: graph")
    gen = torch.Generator(device="cuda").manual_seed(3)
    pages, n = 200, 2
    k, v = [torch.randn((pages, PAGE, KV, D), device="cuda", generator=gen).bfloat16() for _ in range(2)]
    sk, sv = [torch.randn((4000, KV, D), device="cuda", generator=gen).bfloat16() for _ in range(2)]
    table = _int(np.random.default_rng(4).permutation(pages)[:n * 90].reshape(n, 90))
    q = torch.randn((n, HEADS, D), device="cuda", generator=gen)
    prefix, cu, mass = _int([1000, 1300]), _int([0, 1, 2]), torch.zeros((n, KV, 1440), device="cuda")
    work = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")

    def step(q, mass, work):
        o = ql.attention_paged(q, k, v, table, cu, prefix, 1, 1440, workspace=work)
        ql.attention_weights(q, k, mass, table, cu, prefix, 1, 1440, workspace=work)
        return ql.attention_cross(o, sk, sv, cu, _int0, counts, 1, 2000, workspace=work)

    _int0, counts = _int([0, 2000]), _int([2000, 1500])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, mass.clone(), work)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, mass, work)
    mass.zero_()
    want_mass = mass.clone()
    for i, p in enumerate(([1000, 1300], [1001, 1301], [31, 1439], [0, 1])):
        prefix.copy_(_int(p))
        q.normal_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        want = step(q, want_mass, None)
        assert torch.equal(out, want) and torch.equal(mass, want_mass), i
