"""GPU parity of the attention over an encoder's states against the formula in 64 bits.

Bounds, relative to size = sum_j p_j |v_j| of an element, as over the paged cache.  Scores: products of bf16 parts are exact, their fp32 sums of 3 D (fp32 queries) or D terms wander
by 8 sqrt(terms) 2^-24 of the sum of the absolute terms at most (eight deviations); an error d of the scores moves the weights by 2 d.  The exponents' single rounding
and its function: 2^-19 for arguments up to 32.  Sums over keys: 8 sqrt(keys) 2^-24.  The weights go into the product with V as three bf16 parts with fp32 queries (which add up to
them; 2^-17, two parts' share, is allowed) and as one with bf16 queries (2^-8, half a step), whose results are rounded once more (2^-8)."""
import numpy as np
import pytest
import torch

from mllm_amd import _lib, qlinear as ql
import context_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu


def _bound(want, size, terms, dtype, D, keys):
    f32 = dtype == torch.float32
    d = 8 * ((3 if f32 else 1) * D) ** 0.5 * 2.0 ** -24 * terms
    rel = 2 * d + 2.0 ** -19 + 8 * max(keys, 1) ** 0.5 * 2.0 ** -24 + (2.0 ** -17 if f32 else 2.0 ** -8)
    return rel * size + (0.0 if f32 else 2.0 ** -8 * want.abs()) + 1e-30


def _int(v):
    return torch.from_numpy(np.asarray(v, np.int32)).cuda()


class Case:
    """sequences of counts[b] tokens and held[b] keys; states that no sequence has, between them, are NaN"""

    def __init__(self, counts, held, Hq, Hkv, D, dtype, seed=0, spare=0, layout="rows", stretch=1.5):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.held = np.asarray(held, np.int32)
        self.first = (np.cumsum(self.held + 3) - self.held).astype(np.int32)
        S = int((self.held + 3).sum()) + 5
        shape = (S, Hkv, D)
        if layout == "rows":
            self.k, self.v = [torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        elif layout == "heads":
            self.k, self.v = [torch.empty((Hkv, S, D), dtype=torch.bfloat16, device="cuda").transpose(0, 1) for _ in range(2)]
        else:  # views of one projection's rows
            both = torch.empty((S, 2 * Hkv + 1, D + 8), dtype=torch.bfloat16, device="cuda")
            self.k, self.v = both[:, :Hkv, :D], both[:, Hkv:2 * Hkv, :D]
        self.k.fill_(float("nan")), self.v.fill_(float("nan"))
        for f, n in zip(self.first, self.held):
            for x in (self.k, self.v):
                x[f:f + n] = torch.randn((n, Hkv, D), device="cuda", generator=gen).bfloat16()
        self.q = (torch.randn((int(self.cu[-1]) + spare, Hq, D + 8), device="cuda", generator=gen) * stretch).to(dtype)[..., :D]
        self.dtype, self.D = dtype, D

    def args(self):
        return dict(q=self.q, k=self.k, v=self.v, cu_tokens=_int(self.cu), key_first=_int(self.first), key_count=_int(self.held), max_tokens=int(max(np.diff(self.cu))), max_keys=int(max(self.held)))

    def run(self, **changed):
        return ql.attention_cross(**dict(self.args(), **changed))

    def want(self):
        return ref.cross(self.q, self.k, self.v, self.cu, self.first, self.held, self.D ** -0.5)

    def check(self, got, want=None):
        out, size, terms = want or self.want()
        n = int(self.cu[-1])
        bound = _bound(out, size, terms, self.dtype, self.D, int(max(self.held)))
        assert got.dtype == self.dtype and got.shape == self.q.shape
        got = got[:n].cpu().double()
        assert not torch.isnan(got).any()
        far = ((got - out[:n]).abs() / bound[:n]).max().item() if n else 0.0
        assert far <= 1.0, far


@pytest.mark.parametrize("counts,held,Hq,Hkv,D", [
    ([1], [1], 1, 1, 8), ([1], [0], 4, 2, 64), ([1, 1, 1], [63, 64, 65], 8, 2, 128), ([1, 1], [1601, 700], 32, 8, 128), ([1], [6404], 5, 1, 256), ([2, 0, 3], [100, 50, 1], 16, 4, 80),
    ([7, 5], [300, 0], 7, 1, 72), ([16], [129], 1, 1, 96), ([17, 33], [200, 1000], 2, 2, 80), ([64] * 5, [64] * 5, 4, 4, 80), ([64, 64, 13], [64, 64, 13], 3, 3, 72), ([65], [65], 2, 1, 128),
    ([130], [130], 2, 2, 64), ([300, 7], [257, 640], 4, 2, 128), ([129], [500], 2, 2, 96), ([200], [77], 2, 1, 256), ([40], [4000], 4, 1, 104), ([3], [70], 2, 2, 248), ([500], [500], 1, 1, 16),
    ([150], [4097], 2, 2, 56)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_against_the_formula(counts, held, Hq, Hkv, D, dtype):
    announce("attention_cross", counts, held, Hq, Hkv, D, dtype)
    c = Case(counts, held, Hq, Hkv, D, dtype, seed=sum(counts) + sum(held))
    c.check(c.run())


@pytest.mark.parametrize("D", [40, 64, 72, 80, 88, 96])
@pytest.mark.parametrize("tokens,group,keys", [(150, 1, 800), (256, 1, 65), (66, 3, 1100), (1300, 2, 130)])
def test_many_rows_of_many_heads(D, tokens, group, keys):
    """tiles of 256 rows: partly filled, of sequences without tokens or keys, those behind the last whole round in pieces"""
    announce("attention_cross many rows", D, tokens, group, keys)
    counts, held = [tokens, 1, 0, tokens - 2, tokens // 2, 63], [keys, keys // 2, 5, 0, keys - 1, keys // 3]
    if tokens > 1000:
        counts, held = [tokens, 100], [keys, keys - 40]
    kv = 64 // (2 if tokens > 1000 else 1)
    c = Case(counts, held, kv * group, kv, D, torch.bfloat16, seed=D + tokens)
    c.check(c.run())


@pytest.mark.parametrize("D", [64, 80])
def test_many_rows_with_a_nan_and_an_infinity(D):
    """a query's NaN stays in its row, an infinite value in its sequence, head and element"""
    announce("attention_cross many rows, nan", D)
    c = Case([200, 130], [300, 190], 192, 192, D, torch.bfloat16, seed=D)
    clean = c.run()
    c.q[17, 5, 2] = float("nan")
    c.v[int(c.first[1]) + 189, 11, D - 1] = float("inf")
    got = c.run()
    assert torch.isnan(got[17, 5]).all() and not torch.isfinite(got[200:330, 11, D - 1]).any()
    got[17, 5], got[200:330, 11, D - 1] = clean[17, 5], clean[200:330, 11, D - 1]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("layout", ["rows", "heads", "both"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts,held,D", [([5, 9], [333, 90], 80), ([1], [3000], 128), ([100], [100], 72)])
def test_layouts_and_rows_of_no_sequence(counts, held, D, layout, dtype):
    announce("attention_cross layout", counts, held, D, layout, dtype)
    c = Case(counts, held, 6, 2, D, dtype, spare=4, layout=layout, seed=D)
    want = c.want()
    room = torch.full((c.q.shape[0], 9, D + 8), 3.0, device="cuda").to(dtype)
    got = c.run(out=room[:, 1:7, :D])
    c.check(got, want)
    assert (got[int(c.cu[-1]):] == 3).all() and (room[:, 0] == 3).all() and (room[:, 7:] == 3).all() and (room[..., D:] == 3).all()
    small = int(max(counts)) - 1
    if small:  # tokens behind the bound are left as they are
        got = c.run(max_tokens=small, out=torch.full_like(c.q, 7.0))
        at = int(c.cu[int(np.argmax(counts))]) + small
        assert (got[at] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bound", [1, 100, 1 << 20])
def test_any_bound_of_keys(bound, dtype):
    announce("attention_cross bound", bound, dtype)
    c = Case([2, 1, 4], [1900, 3, 700], 8, 2, 128, dtype, seed=4)
    c.check(c.run(max_keys=bound))


@pytest.mark.parametrize("D", [64, 72, 96, 128, 256])
@pytest.mark.parametrize("counts,held,group", [([64, 64, 64, 50], [64, 64, 64, 50], 1), ([49, 0, 49], [49, 3, 0], 2), ([400, 65, 1, 33], [64, 1, 33, 0], 1), ([30, 17], [63, 64], 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_tile_of_keys(counts, held, group, D, dtype):
    """and sequences that have more than the host's bound"""
    announce("attention_cross one tile", counts, held, group, D, dtype)
    c = Case(counts, held, 2 * group, 2, D, dtype, seed=D + len(counts))
    c.check(c.run())
    c = Case(counts, [n * 3 + 1 for n in held], 2 * group, 2, D, dtype, seed=D)
    for bound in (1, 64):
        c.check(c.run(max_keys=bound))


def test_sequences_that_share_keys_and_keys_that_are_not_there():
    announce("attention_cross shared")
    for dtype in (torch.float32, torch.bfloat16):
        c = Case([3, 3, 3, 2], [500, 10, 20, 30], 4, 2, 80, dtype, seed=5)
        c.first[1], c.held[1] = c.first[0], 500
        c.first[2], c.held[2] = c.first[0] + 77, 200
        S = c.k.shape[0]
        c.k[-5:], c.v[-5:] = 0.5, 0.25
        c.first[3], c.held[3] = S - 5, 2 ** 31 - 1  # no more than there are
        want = c.want()
        c.check(c.run(), want)
        c.first[3], c.held[3] = 2 ** 31 - 1, 9  # none
        assert not c.run()[9:].any()
        c.first[3], c.held[3] = S - 5, -4
        assert not c.run()[9:].any()


@pytest.mark.parametrize("tokens,keys", [(1, 700), (40, 300), (200, 130)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_and_nans(tokens, keys, dtype):
    """among a sequence's values: that element infinite or NaN; in a key: what the formula gives; in a query: its row; in states of no sequence: nothing"""
    announce("attention_cross infinite", tokens, keys, dtype)
    inf, nan = float("inf"), float("nan")
    c = Case([tokens, tokens], [keys, keys], 2, 1, 80, dtype, seed=6)
    clean = c.want()
    at = int(c.first[1])
    c.v[at + 5, 0, 3], c.v[at + keys - 1, 0, 79] = inf, nan
    got = c.run()
    assert not torch.isfinite(got[tokens:, :, [3, 79]]).any()
    c.v[at + 5, 0, 3], c.v[at + keys - 1, 0, 79] = 0, 0
    got[..., [3, 79]] = 0
    part = [x.clone() for x in clean]
    for x in part[:2]:
        x[..., [3, 79]] = 0
    c.check(got, part)
    # a key with an infinite element: weight 0 for queries of one sign there, NaN for the other
    c.k[at + 9, 0, 7] = -inf
    c.q[:, :, 7] = c.q[:, :, 7].abs() + 0.5
    got, want = c.run(), c.want()
    c.check(got, want)
    c.q[tokens, 0, 7] *= -1
    got = c.run()
    assert torch.isnan(got[tokens, 0]).all() and torch.isfinite(got[tokens, 1]).all() and torch.isfinite(got[:tokens]).all()
    c.k[at:at + keys, 0, 7] = -inf  # every score -inf: zeros
    c.q[tokens, 0, 7] *= -1
    got = c.run()
    assert not got[tokens:].any() and torch.isfinite(got[:tokens]).all()
    c.q[0, 1, 2] = nan
    got = c.run()
    assert torch.isnan(got[0, 1]).all() and torch.isfinite(got[0, 0]).all() and torch.isfinite(got[1:]).all()


@pytest.mark.parametrize("stretch", [1e-3, 30.0, 3000.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_and_large_scores(stretch, dtype):
    announce("attention_cross scores", stretch, dtype)
    c = Case([3, 70], [500, 333], 4, 2, 64, dtype, seed=7, stretch=stretch)
    got = c.run()
    assert torch.isfinite(got).all()
    if stretch < 1000:
        c.check(got)
    else:  # one key has all the weight: its values
        out, _, _ = c.want()
        assert ((got.cpu().double() - out).abs().amax(-1) < 0.05).float().mean() > 0.95


def test_a_side_stream_a_given_workspace_and_a_captured_call():
    announce("attention_cross graph")
    c = Case([4, 4], [2000, 900], 8, 2, 128, torch.bfloat16, seed=8)
    a = c.args()
    need = _lib.lib().mllm_hip_attention_cross_workspace_bytes(1, 8, 2, 8, 2, 128, 4, 2000)
    assert need > 0
    out, work = torch.empty_like(c.q), torch.empty(need, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ql.attention_cross(**a, workspace=work)
    torch.cuda.current_stream().wait_stream(side)
    c.check(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ql.attention_cross(**a, out=out, workspace=work)
    for i, held in enumerate(([2000, 900], [1, 2000], [64, 0])):
        a["key_count"].copy_(_int(held))
        work.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        # (bits: more keys than the second sequence had reach the NaNs behind them)
        assert torch.equal(out.view(torch.int16), ql.attention_cross(**a).view(torch.int16)), i


def test_far_into_many_states():
    """elements behind 2^32"""
    announce("attention_cross far")
    S = (1 << 32) // 512 + 300
    k, v = [torch.zeros((S, 4, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    gen = torch.Generator(device="cuda").manual_seed(9)
    k[-200:], v[-200:] = [torch.randn((200, 4, 128), device="cuda", generator=gen).bfloat16() for _ in range(2)]
    q = torch.randn((3, 4, 128), device="cuda", generator=gen)
    got = ql.attention_cross(q, k, v, _int([0, 3]), _int([S - 200]), _int([200]), 3, 200)
    want = ql.attention_cross(q, k[-200:].clone(), v[-200:].clone(), _int([0, 3]), _int([0]), _int([200]), 3, 200)
    assert torch.equal(got, want)


def test_nothing_and_refusals():
    announce("attention_cross refusals")
    c = Case([2, 3], [10, 20], 4, 2, 64, torch.float32)
    a = c.args()
    assert ql.attention_cross(**dict(a, q=c.q[:0], cu_tokens=_int([0, 0, 0]))).shape == (0, 4, 64)
    none = ql.attention_cross(**dict(a, k=c.k[:0], v=c.v[:0]))  # no states at all
    assert not none.any()
    kept = ql.attention_cross(**dict(a, cu_tokens=_int([0]), key_first=_int([]), key_count=_int([])), out=torch.full_like(c.q, 2.0))
    assert (kept == 2).all()
    for bad in (dict(q=c.q.half()), dict(q=c.q.cpu()), dict(q=c.q[0]), dict(k=c.k.float()), dict(v=c.v[:-1]), dict(k=c.k.transpose(1, 2)), dict(q=c.q[..., :32]), dict(cu_tokens=_int([0, 5])),
                dict(cu_tokens=a["cu_tokens"].long()), dict(key_first=_int([0])), dict(key_count=None), dict(out=c.q), dict(out=c.q[:1]), dict(workspace=torch.empty(4))):
        if "workspace" in bad:
            bad["max_keys"] = 100000
        with pytest.raises((AssertionError, TypeError)):
            ql.attention_cross(**dict(a, **bad))
    for bad in (dict(q=torch.zeros((5, 3, 64), device="cuda")), dict(scale=0.0), dict(scale=float("nan")), dict(max_tokens=-1), dict(max_keys=-1),
                dict(q=torch.zeros((5, 4, 264), device="cuda"), k=torch.zeros((9, 2, 264), device="cuda").bfloat16(), v=torch.zeros((9, 2, 264), device="cuda").bfloat16()),
                dict(q=torch.zeros((5, 4, 60), device="cuda"), k=torch.zeros((9, 2, 60), device="cuda").bfloat16(), v=torch.zeros((9, 2, 60), device="cuda").bfloat16()),
                dict(q=torch.zeros((5, 4, 66), device="cuda")[..., 2:]), dict(workspace=torch.empty(64, dtype=torch.uint8, device="cuda"), max_keys=100000)):
        with pytest.raises(_lib.HipQLinearError):
            ql.attention_cross(**dict(a, **bad))
