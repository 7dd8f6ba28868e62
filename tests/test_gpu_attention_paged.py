"""GPU parity of the attention over a paged cache against the formula in 64 bits.

Bounds, relative to size = sum_j p_j |v_j| of an element.  Scores: products of bf16 parts are exact, their fp32 sums of 3 D (fp32 queries) or D terms wander by
8 sqrt(terms) 2^-24 of the sum of the absolute terms at most (eight deviations); an error d of the scores moves the weights by 2 d.  The
exponents' single rounding and its function: 2^-19 for arguments up to 32.  Sums over keys: 8 sqrt(keys) 2^-24.  The weights go into the product with V as three bf16
parts with fp32 queries (which add up to them; 2^-17, two parts' share, is allowed) and as one with bf16 queries (2^-8, half a step), whose results are rounded once more (2^-8)."""
import numpy as np
import pytest
import torch

from mllm_amd import _lib, qlinear as ql
import decode_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu


def _bound(want, size, terms, dtype, D, keys):
    parts = 3 if dtype == torch.float32 else 1
    d = 8 * (parts * D) ** 0.5 * 2.0 ** -24 * terms
    rel = 2 * d + 2.0 ** -19 + 8 * keys ** 0.5 * 2.0 ** -24 + (2.0 ** -17 if dtype == torch.float32 else 2.0 ** -8)
    return rel * size + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0.0) + 1e-30


def _layout(pages, page, H, D, layout):
    bf = dict(dtype=torch.bfloat16, device="cuda")
    if layout == "heads":
        return [torch.empty((pages, H, page, D), **bf).transpose(1, 2) for _ in range(2)]
    if layout == "both":
        both = torch.empty((pages, 2, page, H, D + 8), **bf)
        return [both[:, i, ..., :D] for i in range(2)]
    return [torch.empty((pages, page, H, D), **bf) for _ in range(2)]


class Case:
    """sequences of `counts` new tokens behind `prefixes`; the cache holds NaN wherever no sequence has a position"""

    def __init__(self, counts, prefixes, Hq, Hkv, D, page, dtype, parents=None, layout="slots", seed=0, spare=0, stretch=1.5):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.counts, self.prefixes, self.Hq, self.D, self.page, self.dtype = counts, prefixes, Hq, D, page, dtype
        need = [-(-(p + n) // page) for p, n in zip(prefixes, counts)]
        pages = sum(need) + 2
        self.k, self.v = _layout(pages, page, Hkv, D, layout)
        self.k.fill_(float("nan"))
        self.v.fill_(float("nan"))
        ids = rng.permutation(pages)
        self.table = np.full((len(counts), max(max(need), 1) + 1), 2 ** 31 - 1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
            pos = np.arange(prefixes[b] + counts[b])
            slot = torch.from_numpy(self.table[b, pos // page].astype(np.int64)).cuda(), torch.from_numpy(pos % page).cuda()
            for c in (self.k, self.v):
                c[slot] = torch.randn((len(pos), Hkv, D), device="cuda", generator=gen).bfloat16()
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.q = (torch.randn((int(self.cu[-1]) + spare, Hq, D + 8), device="cuda", generator=gen) * stretch).to(dtype)[..., :D]
        self.seen = [np.tril(np.ones((n, n), bool)) for n in counts]
        self.tree = None
        if parents is not None:
            words = -(-max(max(counts), 1) // 64)
            tree = torch.zeros((self.q.shape[0], words), dtype=torch.int64)
            for b, n in enumerate(counts):
                par = parents(rng, n)
                self.seen[b] = ref.ancestors(par)
                if n:
                    tree[self.cu[b]:self.cu[b + 1]] = ql.tree_mask(par, words)
            self.tree = tree.cuda()
        self.scale = D ** -0.5

    def args(self):
        dev = lambda x: torch.from_numpy(np.asarray(x, np.int32)).cuda()  # noqa: E731
        return dict(q=self.q, k_cache=self.k, v_cache=self.v, block_table=dev(self.table), cu_tokens=dev(self.cu), prefix=dev(self.prefixes),
                    max_tokens=max(self.counts), max_keys=max(p + n for p, n in zip(self.prefixes, self.counts)), tree=self.tree)

    def run(self, **changed):
        args = self.args()
        args.update(changed)
        return ql.attention_paged(**args)

    def want(self):
        return ref.attention(self.q, self.k, self.v, torch.from_numpy(self.table), self.cu, self.prefixes, self.seen, self.scale)

    def check(self, got, want=None):
        out, size, terms = want or self.want()
        n = int(self.cu[-1])
        bound = _bound(out, size, terms, self.dtype, self.D, max(p + c for p, c in zip(self.prefixes, self.counts)))
        got = got[:n].cpu().double()
        assert not torch.isnan(got).any()
        far = ((got - out[:n]).abs() / bound[:n]).max().item() if n else 0.0
        assert far <= 1.0, far


def _random_tree(rng, n):
    return [int(rng.integers(-1, i)) if i else -1 for i in range(n)]


@pytest.mark.parametrize("counts,prefixes,Hq,Hkv,D,page", [
    ([1], [0], 4, 1, 128, 16), ([1], [1], 1, 1, 64, 1), ([1, 1, 1], [0, 31, 32], 8, 2, 128, 16), ([1, 1], [127, 128], 8, 8, 64, 24), ([1], [4096], 32, 8, 128, 16),
    ([1, 1], [3000, 17], 5, 1, 128, 64), ([1, 1], [700, 1900], 7, 1, 256, 16), ([2, 1, 3], [100, 5, 1000], 16, 4, 128, 32), ([5, 0, 4], [250, 40, 0], 8, 2, 128, 8),
    ([13, 8], [129, 640], 4, 2, 64, 16), ([40], [500], 4, 1, 128, 256), ([33, 17], [60, 2000], 8, 2, 64, 16), ([70, 1], [0, 90], 6, 2, 256, 16), ([129], [13], 4, 2, 128, 16)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chain(counts, prefixes, Hq, Hkv, D, page, dtype):
    announce("attention chain", counts, prefixes, Hq, Hkv, D, page, dtype)
    c = Case(counts, prefixes, Hq, Hkv, D, page, dtype, seed=sum(counts) + sum(prefixes))
    c.check(c.run())


@pytest.mark.parametrize("counts,prefixes,Hq,Hkv,D,page,layout", [
    ([5], [77], 8, 2, 128, 16, "slots"), ([8, 3, 29], [0, 1200, 40], 4, 1, 128, 16, "heads"), ([64, 63], [130, 31], 4, 1, 64, 24, "both"), ([65, 7], [300, 2], 2, 1, 128, 1, "slots"),
    ([130], [100], 2, 2, 128, 64, "both"), ([20, 9], [900, 333], 8, 4, 256, 8, "heads")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tree(counts, prefixes, Hq, Hkv, D, page, layout, dtype):
    announce("attention tree", counts, prefixes, Hq, Hkv, D, page, layout, dtype)
    c = Case(counts, prefixes, Hq, Hkv, D, page, dtype, _random_tree, layout, seed=sum(counts))
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_that_see_nothing(dtype):
    announce("attention empty rows", dtype)
    c = Case([9, 4], [0, 50], 4, 2, 128, 16, dtype, _random_tree)
    c.tree[2] = 0  # sees not even itself, and there is no prefix
    c.tree[11] = 0
    c.seen[0][2] = False
    c.seen[1][2] = False
    got = c.run()
    assert not got[2].any()
    c.check(got)


@pytest.mark.parametrize("n,Hq,D", [(12, 4, 128), (40, 8, 128), (100, 4, 64), (33, 2, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_is_not_seen_has_no_effect(n, Hq, D, dtype):
    """NaN and infinities in keys and values of new tokens reach the tokens that see them and nothing else"""
    announce("attention unseen NaN", n, Hq, D, dtype)
    for parents in (None, _random_tree):
        c = Case([n], [45], Hq, 1, D, 16, dtype, parents, seed=n)
        clean = c.want()
        place = lambda t: (int(c.table[0, (45 + t) // 16]), (45 + t) % 16)  # noqa: E731
        bad = [n // 2, n - 1]
        c.v[place(bad[0])][:, 3] = float("nan")
        c.v[place(bad[1])][:, 5] = float("inf")
        hit = np.zeros(n, bool)
        got = c.run().cpu().double()
        for b, d in zip(bad, (3, 5)):
            rows = np.nonzero(c.seen[0][:, b])[0]
            odd = got[rows, :, d]
            assert (torch.isnan(odd) if d == 3 else torch.isinf(odd)).all()
            got[rows, :, d] = clean[0][rows, :, d]
        c.check(got, clean)
        c.k[place(bad[0])] = float("nan")
        got = c.run().cpu().double()
        hit[np.nonzero(c.seen[0][:, bad[0]])[0]] = True
        assert torch.isnan(got[hit]).all()
        got[hit] = clean[0][hit]
        got[:, :, 5] = clean[0][:, :, 5]
        c.check(got, clean)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_behind_the_last_sequence_and_strided_results(dtype):
    announce("attention rows behind", dtype)
    c = Case([3, 2], [200, 10], 8, 2, 128, 16, dtype, spare=4)
    wide = torch.full((9, 8, 256), 7.0, dtype=dtype, device="cuda")
    out = wide[..., 128:]
    got = c.run(out=out)
    assert got.data_ptr() == out.data_ptr()
    c.check(got)
    assert (wide[5:] == 7).all() and (wide[..., :128] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_outside_the_cache_and_short_tables(dtype):
    announce("attention bad pages", dtype)
    c = Case([2, 1], [3000, 40], 8, 2, 128, 16, dtype)
    c.table[0, 3] = -1
    c.table[0, 100] = c.k.shape[0]
    c.table[0, 101] = -2 ** 31
    c.table[1, 0] = 2 ** 31 - 1
    c.check(c.run())
    short = c.table[:, :50]  # positions from 800 on are not there, the new tokens of the first sequence among them
    want = ref.attention(c.q, c.k, c.v, torch.from_numpy(short), c.cu, c.prefixes, c.seen, c.scale)
    c.check(c.run(block_table=torch.from_numpy(np.ascontiguousarray(short)).cuda()), want)


def test_the_hosts_bounds_decide_only_how_keys_are_cut():
    announce("attention bounds")
    c = Case([1, 3], [2500, 999], 8, 2, 128, 16, torch.float32)
    want = c.want()
    for keys in (0, 1, 300, 2501, 2502, 100000):
        c.check(c.run(max_keys=keys), want)
    c.check(c.run(max_tokens=50), want)
    # fewer than there are: the tokens behind the bound's last tile of rows are left out, the others right
    got = c.run(max_tokens=1, out=torch.zeros_like(c.q, memory_format=torch.contiguous_format))
    for row in (0, 1):
        assert ((got[row].cpu().double() - want[0][row]).abs() <= _bound(*want, torch.float32, 128, 2503)[row]).all()


def test_a_score_beyond_the_others_and_equal_scores():
    """weights that underflow beside one that is 1; keys that are all the same"""
    announce("attention extreme scores")
    c = Case([1], [1500], 4, 1, 128, 16, torch.float32, stretch=60.0)
    c.check(c.run())
    c = Case([1], [1500], 4, 1, 128, 16, torch.bfloat16)
    first = c.k[int(c.table[0, 0]), 0].clone()
    for i in range(1501):
        c.k[int(c.table[0, i // 16]), i % 16] = first
    c.check(c.run())


def test_own_scale_and_one_token_of_each_length():
    announce("attention scale")
    c = Case([1] * 9, [0, 1, 7, 8, 15, 16, 63, 64, 130], 4, 2, 128, 8, torch.float32)
    c.scale = 0.3
    c.check(c.run(scale=0.3))


def test_far_into_a_large_cache():
    """elements behind 2^32, pages of an unusual size"""
    announce("attention large cache")
    page, H, D = 48, 4, 128
    pages = (1 << 32) // (page * H * D) + 3
    k, v = [torch.empty((pages, page, H, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    for i in table[0].tolist():
        k[i], v[i] = torch.randn((2, page, H, D), device="cuda").bfloat16()
    q = torch.randn((1, 8, D), device="cuda")
    cu, prefix = [0, 1], [130]
    got = ql.attention_paged(q, k, v, table.cuda(), torch.tensor(cu, dtype=torch.int32, device="cuda"), torch.tensor(prefix, dtype=torch.int32, device="cuda"), 1, 131)
    want = ref.attention(q, k, v, table, cu, prefix, [np.ones((1, 1), bool)], D ** -0.5)
    assert ((got.cpu().double() - want[0]).abs() <= _bound(*want, torch.float32, D, 131)).all()


def test_captured_and_replayed_while_lengths_grow():
    """a captured call reads lengths, tables and cache as they are at each replay; eager work and other calls in between"""
    announce("attention graph")
    c = Case([1, 1, 1], [1800, 900, 30], 16, 4, 128, 16, torch.bfloat16)
    args = c.args()
    out = torch.empty_like(c.q, memory_format=torch.contiguous_format)
    size = _lib.lib().mllm_hip_attention_paged_workspace_bytes(ql.BF16, 3, 3, 16, 4, 128, 1, 1801)
    assert size > 0
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ql.attention_paged(**args, out=out, workspace=work)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ql.attention_paged(**args, out=out, workspace=work)
    for step, prefixes in enumerate(([1800, 900, 30], [1500, 899, 0], [10, 20, 30], [1799, 1, 29])):
        args["prefix"].copy_(torch.tensor(prefixes, dtype=torch.int32))
        c.prefixes = prefixes
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)
        eager = c.run(prefix=args["prefix"], max_keys=args["max_keys"])
        assert torch.equal(out, eager), step


def test_two_streams_at_once():
    announce("attention two streams")
    cases = [Case([1, 2], [2000, 1000], 8, 2, 128, 16, torch.float32, seed=i) for i in range(2)]
    want = [c.want() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.run())
    torch.cuda.synchronize()
    for i, c in enumerate(cases):
        c.check(got[i][0], want[i])
        assert all(torch.equal(g, got[i][0]) for g in got[i])


def test_no_tokens():
    announce("attention no tokens")
    c = Case([1], [20], 4, 2, 128, 16, torch.float32)
    none = c.q[:0]
    got = c.run(q=none, cu_tokens=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert got.shape == (0, 4, 128)
    out = torch.full((1, 4, 128), 3.0, device="cuda")
    c.run(cu_tokens=torch.zeros(2, dtype=torch.int32, device="cuda"), out=out)
    assert (out == 3).all()


def test_refusals():
    announce("refusals of attention_paged")
    c = Case([2], [30], 4, 2, 128, 16, torch.float32, _random_tree)
    a = c.args()
    for bad in (dict(q=c.q.half()), dict(q=c.q.cpu()), dict(q=c.q[0]), dict(k_cache=c.k.float()), dict(v_cache=c.v[:1]), dict(block_table=a["block_table"].long()),
                dict(block_table=a["block_table"][0]), dict(cu_tokens=a["cu_tokens"][:1]), dict(prefix=a["prefix"].long()), dict(prefix=None), dict(tree=a["tree"][:1]),
                dict(tree=a["tree"].int()), dict(out=torch.empty((1, 4, 128), device="cuda")), dict(out=c.q), dict(k_cache=c.k.transpose(1, 2))):
        with pytest.raises((AssertionError, TypeError)):
            c.run(**bad)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(max_tokens=-1), dict(max_keys=-1), dict(q=c.q[:, :3])):
        with pytest.raises(_lib.HipQLinearError):
            c.run(**bad)
    big = Case([1], [3000], 4, 2, 128, 16, torch.float32)
    with pytest.raises(_lib.HipQLinearError):
        big.run(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    wrong = Case([1], [30], 4, 2, 96, 16, torch.float32)
    with pytest.raises(_lib.HipQLinearError):
        wrong.run()


def test_workspaces_and_results_that_cannot_be_used():
    announce("refusals of workspaces and results")
    c = Case([2], [3000], 4, 2, 128, 16, torch.float32)
    wide = torch.empty((1 << 22, 2), dtype=torch.uint8, device="cuda")
    for bad in (dict(workspace=torch.empty(1 << 22, dtype=torch.uint8)), dict(workspace=wide[:, 0]), dict(out=torch.empty((1, 4, 128), device="cuda").expand(2, 4, 128))):
        with pytest.raises(AssertionError):
            c.run(**bad)


@pytest.mark.parametrize("counts,prefixes,Hq,Hkv,D,page", [
    ([700, 1, 333], [0, 900, 129], 4, 1, 128, 16), ([1300], [70], 2, 1, 64, 24), ([513], [0], 8, 8, 128, 64), ([400, 0, 260], [5, 9, 0], 6, 2, 256, 16), ([257], [1025], 3, 1, 64, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_keys", [None, 1, 40000])
def test_long_prompts(counts, prefixes, Hq, Hkv, D, page, dtype, max_keys):
    """Tiles of tokens that see all, some or none of a range of keys; partial results in a workspace that held NaNs."""
    announce("attention long prompts", counts, prefixes, Hq, Hkv, D, page, dtype, max_keys)
    c = Case(counts, prefixes, Hq, Hkv, D, page, dtype, seed=sum(counts))
    room = torch.full((1 << 28,), 0xFF, dtype=torch.uint8, device="cuda")
    c.check(c.run(workspace=room, **({} if max_keys is None else dict(max_keys=max_keys))))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("key", [0, 63, 150, 299, 639])
def test_later_tokens_of_a_prompt_have_no_effect(dtype, key):
    announce("attention later tokens", dtype, key)
    c = Case([640], [100], 4, 1, 128, 16, dtype, seed=key)
    clean = c.want()
    at = (int(c.table[0, (100 + key) // 16]), (100 + key) % 16)
    c.k[at], c.v[at] = float("nan"), float("inf")
    for max_keys in (740, 1):
        got = c.run(max_keys=max_keys).cpu().double()
        bound = _bound(*clean, dtype, 128, 740)
        assert ((got[:key] - clean[0][:key]).abs() <= bound[:key]).all()
        assert not torch.isfinite(got[key:]).any()


@pytest.mark.parametrize("Hq,Hkv,D", [(2, 1, 64), (4, 4, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tree", [None, _random_tree])
def test_many_ragged_sequences(Hq, Hkv, D, dtype, tree):
    """More sequences than a wave has lanes, some of them empty, whose tiles are cut into ranges that begin and end anywhere."""
    announce("attention many sequences", Hq, Hkv, D, dtype, tree is not None)
    rng = np.random.default_rng(Hq)
    counts = rng.choice([0, 1, 1, 2, 5], 190).tolist()
    prefixes = rng.choice([0, 1, 63, 64, 65, 300, 700], 190).tolist()
    c = Case(counts, prefixes, Hq, Hkv, D, 16, dtype, tree, seed=D)
    want = c.want()
    c.check(c.run(), want)
    c.check(c.run(max_keys=1), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_sequences_whatever_the_bound(dtype):
    """One launch, or ranges of keys over all sequences, by the host's bound of their lengths."""
    announce("attention many sequences cut and not", dtype)
    rng = np.random.default_rng(3)
    counts = rng.choice([0, 1, 1, 1, 3], 160).tolist()
    prefixes = rng.choice([0, 5, 64, 250, 900], 160).tolist()
    c = Case(counts, prefixes, 8, 8, 64, 16, dtype, seed=4)
    want = c.want()
    for max_keys in (903, 4095, 4096, 100000):
        c.check(c.run(max_keys=max_keys), want)
