"""GPU parity of the accumulated attention weights of cached keys against the formula in 64 bits.

Bound, relative to what a key gets of a call (a sum of weights, all of one sign).  Scores: as in the attention, an error d = 8 sqrt(terms) 2^-24 of the sum of a score's absolute terms moves
the weights by 2 d (their own score's and the sum's).  Exponents: one rounding and the function, 2^-19 for arguments up to 32.  Sums over keys 8 sqrt(keys) 2^-24, over rows 8 sqrt(rows)
2^-24; the reciprocal and its product 2^-23.  Then the old mass times decay and the sum: two roundings of the result, 2^-23.  A weight below 2^-126 may be 0."""
import numpy as np
import pytest
import torch

from mllm_amd import _lib, qlinear as ql
import context_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu


def _int(v):
    return torch.from_numpy(np.asarray(v, np.int32)).cuda()


class Case:
    """sequences of counts[b] new tokens behind prefixes[b] positions; the cache holds NaN wherever no sequence has a position"""

    def __init__(self, counts, prefixes, Hq, Hkv, D, page, dtype, seed=0, spare=0, stretch=1.5):
        gen, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
        self.counts, self.prefixes, self.Hq, self.Hkv, self.D, self.dtype = counts, prefixes, Hq, Hkv, D, dtype
        need = [-(-(p + n) // page) for p, n in zip(prefixes, counts)]
        pages = sum(need) + 2
        room = torch.full((pages, page, Hkv, D + 8), float("nan"), dtype=torch.bfloat16, device="cuda")
        self.k = room[..., :D]
        ids = rng.permutation(pages)
        self.table = np.full((len(counts), max(max(need), 1) + 1), 2 ** 31 - 1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
            pos = np.arange(prefixes[b] + counts[b])
            self.k[torch.from_numpy(self.table[b, pos // page].astype(np.int64)).cuda(), torch.from_numpy(pos % page).cuda()] = torch.randn((len(pos), Hkv, D), device="cuda", generator=gen).bfloat16()
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.q = (torch.randn((int(self.cu[-1]) + spare, Hq, D + 8), device="cuda", generator=gen) * stretch).to(dtype)[..., :D]
        self.keys = max(p + n for p, n in zip(prefixes, counts))
        self.old = torch.rand((len(counts), Hkv, self.keys + 5), device="cuda", generator=gen)
        self.scale = D ** -0.5

    def args(self):
        return dict(q=self.q, k_cache=self.k, block_table=_int(self.table), cu_tokens=_int(self.cu), prefix=_int(self.prefixes), max_tokens=max(self.counts), max_keys=max(1, self.keys))

    def run(self, mass=None, **changed):
        mass = self.old.clone() if mass is None else mass
        assert ql.attention_weights(mass=mass, **dict(self.args(), **changed)) is mass
        return mass

    def check(self, mass, decay=1.0, **limits):
        got, old = mass.cpu().double(), self.old.cpu().double()
        for b, (want, most) in enumerate(ref.weights(self.q, self.k, torch.from_numpy(self.table), self.cu, self.prefixes, self.scale, **limits)):
            n, p = want.shape[1], self.prefixes[b]
            if self.counts[b] == 0:
                assert torch.equal(got[b], old[b])
                continue
            assert torch.equal(got[b, :, n:], old[b, :, n:])
            d = 8 * ((3 if self.dtype == torch.float32 else 1) * self.D) ** 0.5 * 2.0 ** -24 * most
            rows = self.counts[b] * self.Hq // self.Hkv
            rel = 2 * d + 2.0 ** -19 + 8 * (self.keys ** 0.5 + rows ** 0.5) * 2.0 ** -24 + 2.0 ** -23
            total = want + torch.where(torch.arange(n) < p, old[b, :, :n] * float(np.float32(decay)), 0.0)
            far = ((got[b, :, :n] - total).abs() / (rel * want + 2.0 ** -23 * total + rows * 2.0 ** -126)).max().item() if n else 0.0
            assert far <= 1.0, (b, far)


@pytest.mark.parametrize("counts,prefixes,Hq,Hkv,D,page", [
    ([1], [0], 4, 1, 128, 16), ([1], [1], 1, 1, 64, 1), ([1, 1, 1], [0, 15, 64], 8, 2, 128, 16), ([1], [4096], 32, 8, 128, 16), ([1, 1], [3000, 17], 5, 1, 128, 64), ([2, 0, 4], [100, 5, 900], 8, 2, 80, 24),
    ([3, 1], [255, 256], 5, 1, 256, 8), ([16], [600], 1, 1, 96, 16), ([17], [300], 1, 1, 128, 16), ([40, 3], [500, 0], 4, 1, 128, 256), ([33, 0, 17], [60, 7, 2000], 8, 2, 64, 16), ([70, 1], [0, 90], 6, 2, 256, 16),
    ([129], [13], 4, 2, 72, 16), ([300], [0], 2, 2, 128, 16), ([5], [40], 16, 2, 8, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("decay", [1.0, 0.0, 0.75])
def test_against_the_formula(counts, prefixes, Hq, Hkv, D, page, dtype, decay):
    announce("attention_weights", counts, prefixes, Hq, Hkv, D, page, dtype, decay)
    c = Case(counts, prefixes, Hq, Hkv, D, page, dtype, seed=sum(counts) + sum(prefixes))
    c.check(c.run(decay=decay), decay)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("tokens,longest,Hq", [(1, 1900, 16), (2, 959, 64), (2, 961, 64), (3, 70, 8), (20, 330, 8), (70, 45, 16)])
def test_many_sequences(tokens, longest, Hq, D, dtype):
    """as many key heads as CUs and more; among the sequences some without tokens or prefix"""
    announce("attention_weights many", tokens, longest, Hq, D, dtype)
    n = 33
    counts = [tokens if b % 5 else b % 2 for b in range(n)]
    prefixes = [longest if b == 7 else (b * 97) % (longest // 2) if b % 4 else 0 for b in range(n)]
    c = Case(counts, prefixes, Hq, 8, D, 16, dtype, seed=tokens + D)
    c.check(c.run(decay=0.75), 0.75)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts,prefixes", [([3, 2], [70, 300]), ([30, 12], [70, 300])])
def test_bounds_of_tokens_keys_and_masses(counts, prefixes, dtype):
    announce("attention_weights bounds", counts, prefixes, dtype)
    c = Case(counts, prefixes, 4, 2, 64, 16, dtype, seed=1, spare=3)
    c.check(c.run(max_tokens=2), max_tokens=2)
    c.check(c.run(max_tokens=1 << 20, max_keys=1 << 12))
    c.check(c.run(max_keys=200), max_keys=200)
    c.check(c.run(max_keys=71), max_keys=71)
    whole = c.run()
    for n in (0, 1, 40, 301):  # masses of fewer positions: the others' are stored nowhere
        room = torch.full((2, 3, 500), 9.0, device="cuda")
        room[:, :2, :n] = c.old[..., :n]
        c.run(mass=room[:, :2, :n])
        assert torch.equal(room[:, :2, :n], whole[..., :n]) and (room[:, 2] == 9).all() and (room[..., n:] == 9).all()


@pytest.mark.parametrize("counts", [[2, 2], [40, 40]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_and_nans(counts, dtype):
    """in an unseen key: nothing; in a key: weight 0 or a NaN for all that its token sees; old masses of new tokens are not looked at"""
    announce("attention_weights infinite", counts, dtype)
    inf, nan = float("inf"), float("nan")
    c = Case(counts, [50, 90], 2, 1, 64, 16, dtype, seed=2)
    n = counts[0]
    c.old[0, :, 50:50 + n] = nan
    c.old[0, :, :50] = 0
    got = c.run()
    assert torch.isfinite(got[0, :, :50 + n]).all()
    place = lambda b, j: (int(c.table[b, j // 16]), j % 16)  # noqa: E731
    # the last new token's key: only it sees it
    c.k[place(0, 50 + n - 1) + (0, 5)] = nan
    c.q[n - 1] = 1.0
    got = c.run()
    assert torch.isnan(got[0, 0, :50 + n]).all() and torch.isfinite(got[1, :, :90 + n]).all()
    clean = c.run(max_tokens=n - 1, max_keys=1000)
    assert torch.isfinite(clean[0, 0, :50 + n - 1]).all()
    # an infinite element of a key: -inf scores where the queries are positive there
    c.k[place(0, 50 + n - 1) + (0, 5)] = 0.5
    c.k[place(0, 7) + (0, 3)] = -inf
    c.q[:, :, 3] = c.q[:, :, 3].abs() + 0.5
    got = c.run()
    c.old[0, :, 50:] = torch.where(torch.isnan(c.old[0, :, 50:]), torch.zeros_like(c.old[0, :, 50:]), c.old[0, :, 50:])
    c.check(got)
    assert (got[0, 0, 7] == 0).all()
    # a row that sees -inf alone adds nothing; one that has +inf makes NaN of what it sees and of nothing else
    c = Case([n, 1], [0, 5], 2, 1, 64, 16, dtype, seed=3)
    c.k[place(0, 0) + (0, 3)] = -inf
    c.q[:, :, 3] = c.q[:, :, 3].abs() + 0.5
    c.check(c.run(decay=0.0), 0.0)
    c.q[0, 0, 3] = -1
    got = c.run(decay=0.0)
    assert torch.isnan(got[0, 0, 0]) and torch.isfinite(got[0, 0, 1:n]).all() and torch.isfinite(got[1]).all()


# (sequences, tokens of the first, heads of a group, key heads, positions before them): row numbers that are no multiple of 16, with 64 keys a workgroup or more, rows in one piece or several
@pytest.mark.parametrize("seqs,tokens,group,kv,prefix", [(1, 41, 2, 1, 300), (2, 17, 1, 2, 300), (1, 7, 5, 2, 900), (1, 131, 2, 1, 300), (40, 17, 2, 8, 300), (40, 3, 7, 8, 300)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_infinite_key_and_rows_that_fill_no_sixteen(seqs, tokens, group, kv, prefix, D, dtype):
    """a key whose scores are -inf for all that see it gets nothing, whatever is behind the last row"""
    announce("attention_weights infinite, ragged rows", seqs, tokens, group, kv, prefix, D, dtype)
    c = Case([tokens - b % 2 for b in range(seqs)], [prefix] * seqs, group * kv, kv, D, 16, dtype, seed=tokens + D)
    c.q[:, :, 3] = c.q[:, :, 3].abs() + 0.5
    c.k[(c.k == c.k).all(-1)[..., None] & (torch.arange(D, device="cuda") == 3)] = 0.5  # (places of no sequence stay NaN)
    at = [(b, j) for b in range(seqs) for j in (0, 7, 100, prefix - 1)]
    for b, j in at:
        c.k[int(c.table[b, j // 16]), j % 16, :, 3] = -float("inf")
    got = c.run(decay=0.0)
    c.check(got, 0.0)
    for b, j in at:
        assert (got[b, :, j] == 0).all(), (b, j)
    # the old masses go on as they were
    got = c.run(decay=0.75)
    for b, j in at:
        assert torch.equal(got[b, :, j], c.old[b, :, j] * 0.75), (b, j)


def test_pages_outside_the_cache_and_shared_pages():
    announce("attention_weights pages")
    for counts in ([2, 2], [30, 30]):
        c = Case(counts, [100, 100], 4, 2, 128, 16, torch.bfloat16, seed=4)
        c.table[1] = c.table[0]  # the same pages for both
        c.check(c.run())
        c.table[0, 2], c.table[0, 3] = -1, 2 ** 31 - 1
        c.check(c.run())


def test_positions_behind_the_table_and_wild_lengths():
    announce("attention_weights behind the table")
    for counts in ([2, 3], [30, 20]):
        c = Case(counts, [100, 100], 4, 2, 64, 16, torch.float32, seed=5)
        c.table = c.table[:, :5].copy()  # 80 positions
        c.check(c.run())
        c.prefixes = [2 ** 31 - 1, 100]
        whole = c.run()
        c.check(whole)
        c.prefixes = [-7, 100]
        got, c.prefixes = c.run(), [0, 100]
        assert torch.equal(got, c.run())


def test_a_captured_call_over_growing_sequences_and_the_same_bits_every_time():
    announce("attention_weights graph")
    for counts in ([1, 1], [20, 20]):
        c = Case(counts, [400, 900], 8, 2, 128, 16, torch.bfloat16, seed=6)
        a = dict(c.args(), max_keys=c.keys + 100)
        mass = c.old.clone()
        need = _lib.lib().mllm_hip_attention_weights_workspace_bytes(1, sum(counts), 2, 8, 2, 128, max(counts), c.keys + 100)
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ql.attention_weights(mass=mass.clone(), workspace=work, **a)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ql.attention_weights(mass=mass, workspace=work, **a)
        mass.copy_(c.old)
        want = c.old.clone()
        for i, prefix in enumerate(([400, 900], [3, 700], [0, 64], [400, 900])):
            a["prefix"].copy_(_int(prefix))
            work.fill_(255)
            graph.replay()
            torch.cuda.synchronize()
            ql.attention_weights(mass=want, **a)
            assert torch.equal(mass, want), i


def test_keys_far_into_a_large_cache():
    """elements behind 2^32"""
    announce("attention_weights far")
    page, kv, D = 64, 8, 128
    pages = (1 << 32) // (page * kv * D) + 3
    k = torch.zeros((pages, page, kv, D), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(7)
    k[-2:] = torch.randn((2, page, kv, D), device="cuda", generator=gen).bfloat16()
    for n in (1, 40):
        q = torch.randn((n, 16, D), device="cuda", generator=gen)
        got, want = [torch.zeros((1, kv, 128), device="cuda") for _ in range(2)]
        ql.attention_weights(q, k, got, _int([[pages - 1, pages - 2]]), _int([0, n]), _int([128 - n]), n, 128)
        ql.attention_weights(q, k[-2:].clone(), want, _int([[1, 0]]), _int([0, n]), _int([128 - n]), n, 128)
        assert torch.equal(got, want) and got.sum() > 15 * n


def test_nothing_and_refusals():
    announce("attention_weights refusals")
    c = Case([2, 3], [10, 20], 4, 2, 64, 16, torch.float32)
    a = dict(c.args(), mass=c.old.clone())
    assert torch.equal(ql.attention_weights(**dict(a, q=c.q[:0], cu_tokens=_int([0, 0, 0]))), c.old)
    assert torch.equal(ql.attention_weights(**dict(a, max_keys=0)), c.old) and torch.equal(ql.attention_weights(**dict(a, max_tokens=0)), c.old)
    for bad in (dict(q=c.q.half()), dict(q=c.q.cpu()), dict(q=c.q[0]), dict(k_cache=c.k.float()), dict(k_cache=c.k[..., :32]), dict(mass=c.old.double()), dict(mass=c.old[:1]), dict(mass=c.old[:, :1]),
                dict(mass=c.old.transpose(1, 2)), dict(mass=c.old[:, :1].expand(2, 2, -1)), dict(block_table=_int(c.table).long()), dict(block_table=_int(c.table)[:1]), dict(cu_tokens=None),
                dict(prefix=_int([1]))):
        with pytest.raises((AssertionError, TypeError)):
            ql.attention_weights(**dict(a, **bad))
    for bad in (dict(q=torch.zeros((5, 3, 64), device="cuda")), dict(scale=0.0), dict(scale=float("inf")), dict(decay=-0.5), dict(decay=float("nan")), dict(max_tokens=-1), dict(max_keys=-1),
                dict(max_keys=1 << 31), dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"), max_keys=5000), dict(block_table=_int(c.table)[:, :0])):
        with pytest.raises(_lib.HipQLinearError):
            ql.attention_weights(**dict(a, **bad))
