"""GPU parity of the eviction from a paged cache: the positions that stay, their masses and rows are exact."""
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
    def __init__(self, lengths, keep, H, D, page, layout="slots", seed=0, most=None, mass="few"):
        gen, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
        B, most = len(lengths), most or max(lengths + [1])
        per, less = -(-most // page), -(-keep // page)
        pages = B * (per + less) + 1
        if layout == "heads":
            self.k, self.v = [torch.empty((pages, H, page, D), dtype=torch.bfloat16, device="cuda").transpose(1, 2) for _ in range(2)]
        elif layout == "both":
            both = torch.empty((pages, 2, page, H, D + 8), dtype=torch.bfloat16, device="cuda")
            self.k, self.v = both[:, 0, ..., :D], both[:, 1, ..., :D]
        else:
            self.k, self.v = [torch.empty((pages, page, H, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        for x in (self.k, self.v):
            x.copy_(torch.randn((pages, page, H, D), device="cuda", generator=gen))
        ids = rng.permutation(pages)
        self.table, self.to = ids[:B * per].reshape(B, per).astype(np.int32), ids[B * per:B * (per + less)].reshape(B, less).astype(np.int32)
        m = rng.standard_normal((B, H, most)).astype(np.float32)
        if mass == "few":  # few different masses: many ties
            m = np.round(m * 2) / 2
        elif mass == "near":  # masses that differ in their last bits
            m = (1 + m * 1e-6).astype(np.float32)
        elif mass == "same":
            m = np.full_like(m, 0.25)
        elif mass == "odd":
            m[rng.random(m.shape) < 0.2] = np.nan
            m[rng.random(m.shape) < 0.1] = np.inf
            m[rng.random(m.shape) < 0.1] = -np.inf
            m[rng.random(m.shape) < 0.2] = 0.0
            m[rng.random(m.shape) < 0.2] = -0.0
            m[rng.random(m.shape) < 0.1] = 1e-42
        self.mass, self.lengths, self.keep, self.page = m, lengths, keep, page

    def run(self, first=0, recent=0, **changed):
        a = dict(k_cache=self.k, v_cache=self.v, mass=torch.from_numpy(self.mass).cuda(), block_table=_int(self.table), lengths=_int(self.lengths), to_table=_int(self.to), keep=self.keep,
                 first=first, recent=recent)
        a.update(changed)
        return ql.kv_evict(**a)

    def check(self, first=0, recent=0, most=None, **changed):
        k0, v0 = self.k.clone(), self.v.clone()
        kept, mass = self.run(first, recent, **changed)
        kept_, mass_ = kept.cpu().numpy(), mass.cpu().numpy()
        B, H, n_most = self.mass.shape
        want_k, want_v = k0.clone(), v0.clone()
        for b in range(B):
            for h in range(H):
                n = max(0, min(self.lengths[b], n_most if most is None else most))
                want = ref.evict(self.mass[b, h], n, self.keep, first, recent)
                m = len(want)
                assert np.array_equal(kept_[b, h, :m], want) and (kept_[b, h, m:] == -1).all(), (b, h)
                assert np.array_equal(mass_[b, h, :m].view(np.int32), self.mass[b, h, want].view(np.int32)) and (mass_[b, h, m:] == 0).all()
                place = np.arange(m)
                dev = lambda x: torch.from_numpy(np.asarray(x, np.int64)).cuda()  # noqa: E731
                source, to = (dev(self.table[b, want // self.page]), dev(want % self.page)), (dev(self.to[b, place // self.page]), dev(place % self.page))
                want_k[to[0], to[1], h], want_v[to[0], to[1], h] = k0[source[0], source[1], h], v0[source[0], source[1], h]
        assert torch.equal(self.k, want_k) and torch.equal(self.v, want_v)
        return kept, mass


@pytest.mark.parametrize("lengths,keep,first,recent,H,D,page,layout", [
    ([1], 1, 0, 0, 1, 8, 1, "slots"), ([2], 1, 0, 0, 2, 64, 16, "heads"), ([2], 1, 1, 0, 2, 64, 16, "slots"), ([2], 1, 0, 1, 2, 64, 16, "slots"), ([64, 65, 63], 64, 4, 8, 2, 128, 16, "both"),
    ([300, 0, 12, 77], 40, 4, 16, 3, 80, 24, "both"), ([1000, 999], 512, 0, 512, 1, 256, 8, "heads"), ([1000], 999, 500, 499, 2, 64, 64, "slots"), ([5000, 2000], 1025, 4, 100, 4, 128, 16, "slots"),
    ([1025], 1024, 0, 0, 1, 72, 3, "slots"), ([700], 128, 128, 0, 2, 512, 16, "slots"), ([17000, 16384, 16385], 3000, 10, 700, 1, 64, 16, "slots")])
@pytest.mark.parametrize("mass", ["any", "few", "same"])
def test_against_the_definition(lengths, keep, first, recent, H, D, page, layout, mass):
    announce("kv_evict", lengths, keep, first, recent, H, D, page, layout, mass)
    Case(lengths, keep, H, D, page, layout, seed=sum(lengths) + keep, mass=mass).check(first, recent)


@pytest.mark.parametrize("mass", ["odd", "near"])
@pytest.mark.parametrize("keep", [1, 30, 700, 1900])
def test_odd_and_near_masses(mass, keep):
    announce("kv_evict masses", mass, keep)
    Case([2000, 1800], keep, 2, 64, 16, seed=keep, mass=mass).check(min(keep, 3), min(20, keep - min(keep, 3)))


def test_lengths_outside_and_masses_of_fewer_positions():
    announce("kv_evict lengths")
    c = Case([-5, 2 ** 31 - 1, 90], 40, 2, 64, 16, seed=1, most=100)
    c.check(2, 5)
    short = torch.from_numpy(c.mass).cuda()[..., :70]
    c.check(2, 5, most=70, mass=short)
    c.mass = c.mass[:, :, :33]
    c.check(2, 5, mass=torch.from_numpy(c.mass).cuda())


def test_pages_outside_the_cache_and_shared_pages():
    announce("kv_evict pages")
    c = Case([100, 100], 40, 2, 64, 16, seed=2)
    c.table[1] = c.table[0]  # both read the same pages
    c.check(3, 8)
    table = c.table.copy()
    table[0, 0], table[0, 1] = -1, 2 ** 31 - 1
    to = c.to.copy()
    to[1, 0] = -7
    before = c.k.clone()
    kept, _ = c.run(3, 8, block_table=_int(table), to_table=_int(to))
    kept = kept.cpu().numpy()
    for h in range(2):
        for i, j in enumerate(kept[0, h]):
            got = c.k[int(to[0, i // 16]), i % 16, h]
            assert torch.equal(got, torch.zeros_like(got) if j < 32 else before[int(table[0, j // 16]), j % 16, h])
    assert torch.equal(c.k[int(c.to[1, 0])], before[int(c.to[1, 0])])


def test_far_into_a_large_cache():
    """elements behind 2^32"""
    announce("kv_evict far")
    page, H, D = 64, 8, 128
    pages = (1 << 32) // (page * H * D) + 4
    k, v = [torch.zeros((pages, page, H, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    gen = torch.Generator(device="cuda").manual_seed(3)
    k[-2:], v[-2:] = [torch.randn((2, page, H, D), device="cuda", generator=gen).bfloat16() for _ in range(2)]
    mass = torch.rand((1, H, 128), device="cuda", generator=gen)
    kept, _ = ql.kv_evict(k, v, mass, _int([[pages - 1, pages - 2]]), _int([128]), _int([[pages - 3]]), 50)
    for h in range(H):
        at = kept[0, h].long()
        assert torch.equal(k[pages - 3, :50, h], k[pages - 1 - at // 64, at % 64, h]) and torch.equal(v[pages - 3, :50, h], v[pages - 1 - at // 64, at % 64, h])


def test_a_captured_call():
    announce("kv_evict graph")
    c = Case([900, 700], 200, 2, 64, 16, seed=4)
    mass, lengths = torch.from_numpy(c.mass).cuda(), _int(c.lengths)
    out = (torch.empty((2, 2, 200), dtype=torch.int32, device="cuda"), torch.empty((2, 2, 200), device="cuda"))
    a = dict(k_cache=c.k, v_cache=c.v, mass=mass, lengths=lengths, block_table=_int(c.table), to_table=_int(c.to), keep=200, first=4, recent=20, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ql.kv_evict(**a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ql.kv_evict(**a)
    for i, n in enumerate(([900, 700], [150, 201], [0, 800])):
        c.mass = np.random.default_rng(i).random(c.mass.shape, np.float32)
        mass.copy_(torch.from_numpy(c.mass))
        lengths.copy_(_int(n))
        c.k[torch.from_numpy(c.to.astype(np.int64)).cuda()] = 0
        graph.replay()
        torch.cuda.synchronize()
        k, kept, m = c.k.clone(), out[0].clone(), out[1].clone()
        c.k[torch.from_numpy(c.to.astype(np.int64)).cuda()] = 0
        c.lengths = n
        kept2, m2 = c.check(4, 20)
        assert torch.equal(kept, kept2) and torch.equal(m, m2) and torch.equal(k, c.k), i


def test_nothing_and_refusals():
    announce("kv_evict refusals")
    c = Case([50, 60], 20, 2, 64, 16, seed=5)
    before = c.k.clone()
    kept, mass = c.run(keep=0)
    assert kept.shape == mass.shape == (2, 2, 0) and torch.equal(c.k, before)
    m, t = torch.from_numpy(c.mass).cuda(), _int(c.table)
    for bad in (dict(k_cache=c.k.float()), dict(v_cache=c.v[:1]), dict(mass=m.double()), dict(mass=m[:1]), dict(mass=m[:, :1]), dict(block_table=t.long()), dict(lengths=None), dict(lengths=_int([1])),
                dict(to_table=_int(c.to)[:1]), dict(keep=-1), dict(out=(torch.empty((2, 2, 20), device="cuda"),) * 2), dict(out=torch.empty(1)), dict(mass=m.cpu())):
        with pytest.raises((AssertionError, TypeError)):
            c.run(**bad)
    for bad in (dict(first=21), dict(recent=21), dict(first=15, recent=6), dict(first=-1), dict(recent=-1), dict(keep=33)):
        with pytest.raises(_lib.HipQLinearError):
            c.run(**bad)
