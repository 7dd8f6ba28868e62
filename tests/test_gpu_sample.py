"""GPU parity of the sampling against its definition in 64 bits: tokens are equal, all of them.  A row could only differ where u falls within about 1e-15
of a border of the running sum (u has 24 bits, so a border that is no short binary fraction is further away), or top_p's mass within the units' 2^-44."""
import numpy as np
import pytest
import torch

from mllm_amd import _lib, qlinear as ql
import decode_ref as ref
from gpu_util import announce

pytestmark = pytest.mark.gpu


def _want(x, u, t, k, p, m):
    return [ref.sample(x[i], u[i], t[i], k[i], p[i], m[i]) for i in range(len(x))]


def _run(x, u, t, k, p, m, dtype=torch.float32, **more):
    dev = lambda v, d: torch.from_numpy(np.ascontiguousarray(v)).to(d).cuda()  # noqa: E731
    return ql.sample(dev(x, dtype), dev(u, torch.float32), dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(m, torch.float32), **more)


def _check(x, u, t, k, p, m, dtype=torch.float32):
    got = _run(x, u, t, k, p, m, dtype).cpu().numpy()
    seen = torch.from_numpy(np.ascontiguousarray(x)).to(dtype).float().numpy()
    want = np.array(_want(seen, u, t, k, p, m))
    assert got.dtype == np.int32
    assert np.array_equal(got, want), [(i, got[i], want[i], t[i], k[i], p[i], m[i], u[i]) for i in np.nonzero(got != want)[0][:5]]


def _settings(rng, rows):
    return (rng.random(rows).astype(np.float32), rng.choice([0.0, 0.3, 0.7, 1.0, 1.7], rows).astype(np.float32), rng.choice([0, 1, 2, 20, 64, 1000, 70000], rows).astype(np.int32),
            rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 2.0], rows).astype(np.float32), rng.choice([0.0, 0.001, 0.05, 0.5], rows).astype(np.float32))


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 3), (9, 7), (40, 63), (40, 64), (40, 65), (33, 511), (33, 1000), (64, 4097), (70, 8191), (40, 32000), (24, 50257), (16, 151936),
                                        (3, 262147), (300, 997)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [3.0, 0.2])
def test_all_settings(rows, vocab, dtype, spread):
    announce("sample", rows, vocab, dtype, spread)
    rng = np.random.default_rng(rows * 7 + vocab)
    x = (rng.standard_normal((rows, vocab)) * spread).astype(np.float32)
    _check(x, *_settings(rng, rows), dtype)


@pytest.mark.parametrize("vocab", [17, 5000, 40001])
def test_each_setting_alone_and_none(vocab):
    announce("sample single settings", vocab)
    rng = np.random.default_rng(vocab)
    rows = 30
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    one, zero, none = np.ones(rows, np.float32), np.zeros(rows, np.float32), np.zeros(rows, np.int32)
    dx, du = torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
    t, k, p, m = _settings(rng, rows)[1:]
    t = np.maximum(t, np.float32(0.3))
    dev = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    for name, want in (("", (one, none, one, zero)), ("t", (t, none, one, zero)), ("k", (one, k, one, zero)), ("p", (one, none, p, zero)), ("m", (one, none, one, m))):
        args = {"t": dict(temperature=dev(t)), "k": dict(top_k=dev(k)), "p": dict(top_p=dev(p)), "m": dict(min_p=dev(m)), "": {}}[name]
        assert ql.sample(dx, du, **args).cpu().tolist() == _want(x, u, *want), name


def test_ties_at_the_border():
    """few different values: borders within long runs of equal logits, which are taken lowest index first"""
    announce("sample ties")
    rng = np.random.default_rng(5)
    for vocab in (50, 3001, 60000):
        rows = 60
        x = np.round(rng.standard_normal((rows, vocab)) * 1.5).astype(np.float32) / 2
        x[x == 0] = -0.0  # the two zeros are equal
        x[:, ::3][x[:, ::3] == 0] = 0.0
        _check(x, *_settings(rng, rows))
    x = np.full((40, 20000), 1.25, np.float32)  # all equal
    _check(x, *_settings(rng, 40))
    x[:, 7777] = 1.5
    _check(x, *_settings(rng, 40))


def test_masked_infinite_and_missing_logits():
    announce("sample special values")
    rng = np.random.default_rng(6)
    rows, vocab = 48, 9000
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    x[0:8, ::2] = -np.inf
    x[8:16, 1::2] = np.finfo(np.float32).min
    x[16:20, 5:] = np.nan
    x[20:22] = -np.inf
    x[22] = np.nan
    x[24:28, [3, 700, 8999]] = np.inf
    x[28:32, :] = -np.inf
    x[28:32, 4321] = -5.0
    x[32:36] *= 1e30
    x[36:40] *= 1e-30
    u, t, k, p, m = _settings(rng, rows)
    got = _run(x, u, t, k, p, m).cpu().tolist()
    assert got == _want(x, u, t, k, p, m)
    assert got[20] == got[21] == got[22] == -1 and got[28:32] == [4321] * 4


def test_ends_of_u_and_odd_settings():
    announce("sample ends")
    rng = np.random.default_rng(7)
    rows, vocab = 64, 3000
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    _, t, k, p, m = _settings(rng, rows)
    for u in (np.zeros(rows, np.float32), np.full(rows, 1 - 2.0 ** -24, np.float32), np.full(rows, 2.0 ** -24, np.float32)):
        _check(x, u, t, k, p, m)
    u = rng.random(rows).astype(np.float32)
    _check(x, u, np.full(rows, -1.0, np.float32), k, p, m)
    _check(x, u, t, np.full(rows, -3, np.int32), np.full(rows, -0.5, np.float32), np.full(rows, 2.0, np.float32))
    _check(x, u, np.full(rows, 1e-3, np.float32), k, p, m)
    _check(x, u, np.full(rows, 100.0, np.float32), k, p, m)


def test_frequencies_follow_the_weights():
    announce("sample frequencies")
    x = torch.log(torch.tensor([0.5, 0.25, 0.125, 0.125], device="cuda")).repeat(20000, 1)
    u = (torch.arange(20000, device="cuda") + 0.5) / 20000
    got = torch.bincount(ql.sample(x, u).long(), minlength=4).tolist()
    assert got == [10000, 5000, 2500, 2500]


def test_strided_rows_and_given_results():
    announce("sample strided")
    rng = np.random.default_rng(8)
    wide = torch.from_numpy((rng.standard_normal((9, 5003)) * 2).astype(np.float32)).cuda()
    u = torch.rand(9, device="cuda")
    for lo, hi in ((0, 5000), (1, 4999), (3, 5003), (5, 6)):
        x = wide[:, lo:hi]
        out = torch.full((9,), -7, dtype=torch.int32, device="cuda")
        got = ql.sample(x, u, top_p=torch.full((9,), 0.8, device="cuda"), out=out)
        assert got is out
        want = _want(x.cpu().numpy(), u.cpu().numpy(), [1.0] * 9, [0] * 9, [0.8] * 9, [0.0] * 9)
        assert out.cpu().tolist() == want
        half = wide.bfloat16()[:, lo:hi]
        want = _want(half.float().cpu().numpy(), u.cpu().numpy(), [1.0] * 9, [0] * 9, [0.8] * 9, [0.0] * 9)
        assert ql.sample(half, u, top_p=torch.full((9,), 0.8, device="cuda")).cpu().tolist() == want


def test_captured_replayed_and_repeated():
    announce("sample graph")
    rng = np.random.default_rng(9)
    rows, vocab = 6, 40000
    x = torch.empty((rows, vocab), device="cuda")
    u = torch.empty(rows, device="cuda")
    t, k, p, m = [torch.from_numpy(v).cuda() for v in _settings(rng, rows)[1:]]
    out = torch.empty(rows, dtype=torch.int32, device="cuda")
    work = torch.empty(_lib.lib().mllm_hip_sample_workspace_bytes(rows, vocab), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    x.normal_(), u.uniform_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ql.sample(x, u, t, k, p, m, out, work)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ql.sample(x, u, t, k, p, m, out, work)
    for _ in range(4):
        x.normal_(std=2.5), u.uniform_()
        out.fill_(-5)
        work.random_(0, 256)  # nothing is kept in the workspace from one call for the next
        graph.replay()
        torch.cuda.synchronize()
        eager = ql.sample(x, u, t, k, p, m)
        assert torch.equal(out, eager) and torch.equal(eager, ql.sample(x, u, t, k, p, m))
        assert eager.cpu().tolist() == _want(*[v.cpu().numpy() for v in (x, u, t, k, p, m)])


def test_no_rows_and_refusals():
    announce("refusals of sample")
    x, u = torch.zeros((3, 100), device="cuda"), torch.zeros(3, device="cuda")
    assert ql.sample(x[:0], u[:0]).shape == (0,)
    for bad in (dict(logits=x.half()), dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x.t()), dict(u=None), dict(u=u[:2]), dict(u=u.double()), dict(temperature=u[:1]), dict(top_k=u),
                dict(top_p=u.double()), dict(min_p=u.bfloat16()), dict(out=u), dict(logits=x[:, :0])):
        args = dict(logits=x, u=u)
        args.update(bad)
        with pytest.raises((AssertionError, TypeError)):
            ql.sample(**args)
    with pytest.raises(_lib.HipQLinearError):
        ql.sample(x, u, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))


def test_workspaces_that_cannot_be_used():
    announce("refusals of workspaces")
    x, u = torch.zeros((3, 100), device="cuda"), torch.zeros(3, device="cuda")
    for room in (torch.empty(1 << 22, dtype=torch.uint8), torch.empty((1 << 22, 2), dtype=torch.uint8, device="cuda")[:, 0]):
        with pytest.raises(AssertionError):
            ql.sample(x, u, workspace=room)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [257, 5000])
@pytest.mark.parametrize("spread", [3.0, 0.2])
def test_many_kept_of_which_a_share(dtype, k, spread):
    """The border by mass far in front of the one by count, in its step, and behind it (more kept than there are)."""
    announce("sample many kept of which a share", dtype, k, spread)
    rng = np.random.default_rng(k)
    x = (rng.standard_normal((24, 7058)) * spread).astype(np.float32)
    p = np.tile(np.array([1e-6, 0.05, 0.3, 0.6, 0.9, 0.999, 0.999999, 1.0], np.float32), 3)
    t = np.repeat(np.array([0.5, 1.0, 1.7], np.float32), 8)
    _check(x, rng.random(24).astype(np.float32), t, np.full(24, k, np.int32), p, np.zeros(24, np.float32), dtype)


@pytest.mark.parametrize("kind", ["few values", "tiny", "denormal", "huge", "one apart", "near zero", "negative", "ramp"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_of_any_size(kind, dtype):
    """Logits whose steps have hardly a number in them or nearly all, of either sign, next to zero and next to the largest there is."""
    announce("sample logits", kind, dtype)
    rng = np.random.default_rng(len(kind))
    rows, vocab = 40, 9000
    n = rng.standard_normal((rows, vocab))
    x = {"few values": np.round(n), "tiny": n * 1e-20, "denormal": n * 1e-39, "huge": np.clip(n * 2e38, -3.3e38, 3.3e38), "one apart": 1000 + n * 1e-3, "near zero": n * 10.0 ** rng.integers(-30, 1, n.shape),
         "negative": -500 - np.abs(n) * 4, "ramp": np.linspace(-20, 5, vocab)[None] + 0 * n}[kind].astype(np.float32)
    _check(x, *_settings(rng, rows), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_few_different_logits(dtype):
    """All equal, two values in turns, long runs of equals, one step's worth of many: lists that are longer than what is kept in LDS."""
    announce("sample equal logits", dtype)
    rng = np.random.default_rng(21)
    vocab = 70001
    i = np.arange(vocab)
    kinds = [0 * i, i % 2, i // 4096 % 3, (i // 512 == 7) * 2.0, np.round(rng.standard_normal(vocab)), 1 + (i % 5) / 1024, np.where(i < 60000, 3.0, -np.inf), np.where(i % 3 == 0, np.nan, 0.5)]
    x = np.repeat(np.stack(kinds).astype(np.float32), 5, 0)
    rows = len(x)
    k = np.tile(np.array([0, 50, 255, 5000, 69000], np.int32), len(kinds))
    for p in (1.0, 0.9, 0.3):
        _check(x, rng.random(rows).astype(np.float32), rng.choice([0.5, 1.0, 3.0], rows).astype(np.float32), k, np.full(rows, p, np.float32), np.zeros(rows, np.float32), dtype)
