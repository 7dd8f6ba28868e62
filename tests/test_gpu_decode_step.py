"""The operators between a layer's projections together, as a program uses them: a prompt in chunks, decode steps of several sequences, the verification of
a tree of drafted tokens, and the tokens that follow, through a small two-layer model whose projections are this library's matmuls and quantized Linears.

Bound of the comparisons in fp32: what is compared differs by fp32 sums (about 2^-20 of a value after one layer) and by keys and values rounded to bf16, where an
fp32 difference can move a value by one step of 2^-8; a step of one key or value in 50 or more moves an attention output by at most 2^-8 / 50 of a value's size, 1e-4,
and the layers behind it by a few times that: 2e-3 of the largest logit is asked for."""
import numpy as np
import pytest
import torch

from mllm_amd import qlinear as ql
from gpu_util import announce

pytestmark = pytest.mark.gpu
LAYERS, HIDDEN, HEADS, KV, D, VOCAB, PAGE = 2, 256, 8, 2, 64, 1000, 16


class Model:
    def __init__(self, pages, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
        self.embed = r(VOCAB, HIDDEN)
        self.layers = [dict(norm=1 + 0.1 * r(HIDDEN), qkv=r(HIDDEN, (HEADS + 2 * KV) * D) / HIDDEN ** 0.5, o=r(HEADS * D, HIDDEN) / (HEADS * D) ** 0.5, wq=1 + 0.1 * r(D),
                            wk=1 + 0.1 * r(D)) for _ in range(LAYERS)]
        self.norm = torch.ones(HIDDEN, device="cuda")
        self.head = r(HIDDEN, VOCAB) / HIDDEN ** 0.5
        self.inv_freq = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
        self.cache = [[torch.full((pages, PAGE, KV, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(LAYERS)]

    def step(self, tokens, positions, slots, table, cu, prefix, most, keys, tree=None):
        x = self.embed[tokens]
        t = len(tokens)
        for w, (kc, vc) in zip(self.layers, self.cache):
            rows = ql.matmul(ql.rmsnorm(x, w["norm"], 1e-6), w["qkv"]).view(t, HEADS + 2 * KV, D)
            q = ql.kv_append(rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:], kc, vc, slots, positions, self.inv_freq, w["wk"], rows[:, :HEADS], w["wq"])
            a = ql.attention_paged(q, kc, vc, table, cu, prefix, most, keys, tree=tree)
            x = ql.add(x, ql.matmul(a.view(t, HEADS * D), w["o"]))
        return ql.matmul(ql.rmsnorm(x, self.norm, 1e-6), self.head)


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _slots(table, places):
    return torch.tensor([table[b][p // PAGE] * PAGE + p % PAGE for b, p in places], device="cuda")


def _close(a, b):
    assert torch.isfinite(a).all() and torch.isfinite(b).all()
    assert (a - b).abs().max() <= 2e-3 * b.abs().max(), ((a - b).abs().max() / b.abs().max()).item()


def _prompt(model, table, b, tokens, chunk):
    """a sequence's prompt in chunks; the logits of all its tokens"""
    out = []
    for at in range(0, len(tokens), chunk):
        part = tokens[at:at + chunk]
        n = len(part)
        out.append(model.step(part, (at + torch.arange(n, device="cuda")).int(), _slots(table, [(b, at + i) for i in range(n)]), _int(table[b:b + 1]), _int([0, n]), _int([at]), n, at + n))
    return torch.cat(out)


def test_a_prompt_whole_in_chunks_and_token_by_token():
    announce("decode step: prompt")
    table = [[5, 1, 7, 3, 0, 2, 6, 4]]
    tokens = torch.randint(0, VOCAB, (101,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    want = _prompt(Model(8), table, 0, tokens, 101)
    for chunk in (33, 1):
        _close(_prompt(Model(8), table, 0, tokens, chunk), want)


def test_a_batch_of_ragged_sequences_equals_each_alone():
    announce("decode step: batch")
    table = [[0, 9, 3], [4, 5, 6], [11, 2, 8], [1, 7, 10]]
    g = torch.Generator(device="cuda").manual_seed(2)
    prompts = [torch.randint(0, VOCAB, (n,), device="cuda", generator=g) for n in (17, 40, 1, 31)]
    model, alone = Model(12), Model(12)
    for b, p in enumerate(prompts):
        for m in (model, alone):
            _prompt(m, table, b, p, 64)
    nxt = torch.randint(0, VOCAB, (4,), device="cuda", generator=g)
    lens = [len(p) for p in prompts]
    # two padded tokens behind the sequences: slots outside the cache, rows that belong to none
    tokens = torch.cat([nxt, nxt[:2]])
    slots = torch.cat([_slots(table, list(enumerate(lens))), torch.tensor([-1, -1], device="cuda")])
    got = model.step(tokens, _int(lens + [0, 0]), slots, _int(table), _int([0, 1, 2, 3, 4]), _int(lens), 1, 64)[:4]
    for b, n in enumerate(lens):
        want = alone.step(nxt[b:b + 1], _int([n]), _slots(table, [(b, n)]), _int(table[b:b + 1]), _int([0, 1]), _int([n]), 1, n + 1)
        _close(got[b:b + 1], want)


def test_a_tree_of_drafted_tokens_equals_its_branches_one_by_one():
    announce("decode step: tree")
    table = [[3, 0, 6, 1, 4, 2, 5]]
    g = torch.Generator(device="cuda").manual_seed(3)
    prompt = torch.randint(0, VOCAB, (53,), device="cuda", generator=g)
    parents = [-1, 0, 0, 1, 1, 2, 3, -1, 7, 5, 8]
    drafted = torch.randint(0, VOCAB, (len(parents),), device="cuda", generator=g)
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    n, at = len(parents), len(prompt)
    model = Model(7)
    _prompt(model, table, 0, prompt, 64)
    got = model.step(drafted, _int([at + d for d in depth]), _slots(table, [(0, at + i) for i in range(n)]), _int(table), _int([0, n]), _int([at]), n, at + n, ql.tree_mask(parents).cuda())
    for leaf in range(n):
        if leaf in parents:
            continue
        path = [leaf]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        single = Model(7)
        _prompt(single, table, 0, prompt, 64)
        for i, node in enumerate(path):
            want = single.step(drafted[node:node + 1], _int([at + i]), _slots(table, [(0, at + i)]), _int(table), _int([0, 1]), _int([at + i]), 1, at + i + 1)
            _close(got[node:node + 1], want)


def test_captured_steps_generate_what_eager_ones_do():
    """a step with the sampling of its tokens in one graph, replayed while the sequences grow past a page's end"""
    announce("decode step: graph")
    table = [[0, 1, 2, 3], [7, 6, 5, 4], [8, 9, 10, 11]]
    lens = [13, 30, 1]
    head = ql.PackedQWeight.synthetic(ql.Q8_0, VOCAB, HIDDEN, torch.Generator(device="cuda").manual_seed(4))

    def start():
        model = Model(12)
        for b, n in enumerate(lens):
            _prompt(model, table, b, torch.arange(n, device="cuda") * 7 % VOCAB, 64)
        s = dict(tokens=torch.tensor([1, 2, 3], device="cuda"), positions=_int(lens), slots=_slots(table, list(enumerate(lens))), prefix=_int(lens), u=torch.zeros(3, device="cuda"))
        fixed = dict(table=_int(table), cu=_int([0, 1, 2, 3]), t=torch.tensor([0.7, 0.0, 1.3], device="cuda"), k=_int([50, 0, 0]), p=torch.tensor([0.9, 1.0, 0.8], device="cuda"))

        def step():
            logits = model.step(s["tokens"], s["positions"], s["slots"], fixed["table"], fixed["cu"], s["prefix"], 1, 64)
            quantized = ql.linear_q_gemv(head, logits[:, :HIDDEN].contiguous())
            return logits, ql.sample(logits + 0.1 * quantized, s["u"], fixed["t"], fixed["k"], fixed["p"])
        return s, step

    def feed(s, i, tokens):
        s["tokens"].copy_(tokens)
        s["positions"].copy_(_int([n + i for n in lens]))
        s["prefix"].copy_(_int([n + i for n in lens]))
        s["slots"].copy_(_slots(table, [(b, n + i) for b, n in enumerate(lens)]))
        s["u"].copy_(torch.tensor(np.random.default_rng(i).random(3), dtype=torch.float32))

    said = []
    s, step = start()
    tokens = s["tokens"].clone()
    for i in range(8):
        feed(s, i, tokens)
        logits, tokens = step()
        said.append((logits.clone(), tokens.clone()))
    s, step = start()
    feed(s, 0, s["tokens"].clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, chosen = step()
    tokens = torch.tensor([1, 2, 3], device="cuda")
    for i in range(8):
        feed(s, i, tokens)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, said[i][0]) and torch.equal(chosen, said[i][1]), i
        tokens = chosen.clone()
