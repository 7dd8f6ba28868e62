"""GPU parity of the rotation by positions of several axes (time, height, width), alone and on the way into a paged cache, against the formula in 64 bits.

Bounds: as of one axis (a position is picked, nothing else is computed): 24 * 2^-24 of |a| + |b| in fp32, a bf16 result in addition half a step, 2^-8 of itself."""
import pytest
import torch

from mllm_amd import _lib, qlinear as ql
from context_ref import norm_rope_axes
from gpu_util import announce

pytestmark = pytest.mark.gpu
E32, E16 = 2.0 ** -24, 2.0 ** -8


def _freq(rot, base=1e6):
    return base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)


def _check(got, want, size, dtype):
    bound = 24 * E32 * size + (E16 * want.abs() if dtype == torch.bfloat16 else 0.0) + 1e-30
    assert got.dtype == dtype
    far = ((got.cpu().double() - want).abs() / bound).max().item() if want.numel() else 0.0
    assert far <= 1.0, far


def _axes(half, A, order):
    j = torch.arange(half)
    a = {"turns": j % A, "blocks": j * A // max(1, half), "mixed": torch.randint(0, A, (half,), generator=torch.Generator().manual_seed(half))}[order]
    return a.int().cuda()


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,A,order,interleaved", [
    (1, 32, 8, 128, 128, 3, "blocks", False), (4, 28, 4, 128, 128, 3, "turns", False), (257, 5, 1, 128, 64, 2, "mixed", True), (33, 16, 16, 80, 80, 2, "blocks", False),
    (7, 3, 3, 64, 32, 4, "mixed", False), (5, 8, 4, 256, 256, 3, "turns", True), (2, 2, 1, 512, 512, 4, "turns", False), (3, 2, 2, 72, 64, 1, "blocks", False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotation_by_several_axes(T, Hq, Hkv, D, rot, A, order, interleaved, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T * 31 + D)
    announce("qk_norm_rope axes", T, Hq, Hkv, D, rot, A, order, interleaved, dtype)
    rows = torch.randn((T, Hq + Hkv, D), device="cuda", generator=gen).to(dtype)
    q, k = rows[:, :Hq], rows[:, Hq:]
    wq = 1 + 0.3 * torch.randn(D, device="cuda", generator=gen)
    f, axes = _freq(rot), _axes(rot // 2, A, order)
    for pos in (torch.randint(-100000, 1 << 20, (A, T), device="cuda", generator=gen).int(), torch.randint(0, 90, (T, A), device="cuda", generator=gen).int().t(),
                torch.randint(0, 2 ** 31 - 1, (A, 2 * T + 3), device="cuda", generator=gen).int()[:, 3::2]):
        yq, yk = ql.qk_norm_rope(q, k, pos, f, wq, None, eps=1e-5, interleaved=interleaved, axes=axes)
        _check(yq, *norm_rope_axes(q, wq, 1e-5, pos, axes, f, interleaved), dtype)
        _check(yk, *norm_rope_axes(k, None, 1e-5, pos, axes, f, interleaved), dtype)


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,A,page", [(1, 32, 8, 128, 128, 3, 16), (37, 4, 1, 80, 32, 2, 24), (130, 10, 5, 128, 128, 3, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_by_several_axes(T, Hq, Hkv, D, rot, A, page, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T + 7 * D)
    announce("kv_append axes", T, Hq, Hkv, D, rot, A, page, dtype)
    pages = -(-T * 2 // page)
    kc, vc = [torch.full((pages, page, Hkv, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    q, k, v = [torch.randn((T, h, D), device="cuda", generator=gen).to(dtype) for h in (Hq, Hkv, Hkv)]
    w = 1 + 0.3 * torch.randn(D, device="cuda", generator=gen)
    pos, axes, f = torch.randint(0, 9000, (A, T), device="cuda", generator=gen).int(), _axes(rot // 2, A, "mixed"), _freq(rot)
    slots = torch.randperm(pages * page, device="cuda", generator=gen)[:T]
    if T > 2:
        slots[1] = -1
    kept = (slots >= 0).cpu()
    y = ql.kv_append(k, v, kc, vc, slots, pos, f, w, q, None, axes=axes)
    _check(y, *norm_rope_axes(q, None, 1e-6, pos, axes, f, False), dtype)
    at = slots[kept.cuda()]
    want, size = norm_rope_axes(k, w, 1e-6, pos, axes, f, False)
    _check(kc.view(-1, Hkv, D)[at], want[kept], size[kept], torch.bfloat16)
    assert torch.equal(vc.view(-1, Hkv, D)[at], v.to(torch.bfloat16)[kept.cuda()])
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert (kc.view(-1, Hkv, D)[rest] == 7).all() and (vc.view(-1, Hkv, D)[rest] == 7).all()


def test_one_position_on_every_axis_and_axes_that_are_not_there():
    announce("qk_norm_rope axes: the same as one axis")
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k = torch.randn((19, 6, 128), device="cuda", generator=gen), torch.randn((19, 2, 128), device="cuda", generator=gen)
    pos, f = torch.randint(0, 50000, (19,), device="cuda", generator=gen).int(), _freq(128)
    want = ql.qk_norm_rope(q, k, pos, f)
    got = ql.qk_norm_rope(q, k, pos.expand(3, 19), f, axes=_axes(64, 3, "turns"))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    axes = _axes(64, 3, "turns")
    axes[5], axes[6], axes[7] = 3, -1, 2 ** 31 - 1
    pos3 = torch.randint(1, 50000, (3, 19), device="cuda", generator=gen).int()
    yq, yk = ql.qk_norm_rope(q, k, pos3, f, axes=axes)
    _check(yq, *norm_rope_axes(q, None, 1e-6, pos3, axes, f, False), torch.float32)
    for j in (5, 6, 7, 69, 70, 71):
        assert torch.equal(yq[..., j], q[..., j]) and torch.equal(yk[..., j], k[..., j])


@pytest.mark.parametrize("D,rot,interleaved", [(64, 64, False), (80, 64, False), (128, 128, False), (128, 128, True), (128, 32, False), (256, 256, True), (512, 512, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [3, 700])
def test_pairs_on_no_axis_stay_as_they_are(T, D, rot, interleaved, dtype):
    """bit for bit, whatever the other element of the pair and its frequency are; alone and on the way into a cache"""
    announce("qk_norm_rope axes: pairs on none", T, D, rot, interleaved, dtype)
    gen = torch.Generator(device="cuda").manual_seed(T + D)
    inf, half = float("inf"), rot // 2
    x = torch.randn((T, 8, D), device="cuda", generator=gen).to(dtype)
    pos, f, axes = torch.randint(1, 50000, (3, T), device="cuda", generator=gen).int(), _freq(rot), _axes(half, 3, "turns")
    still = [1, 2, half - 1]
    axes[still] = torch.tensor([3, -1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    f[1], f[half - 1] = inf, float("nan")
    first, second = [[2 * j + i if interleaved else j + i * half for j in still] for i in range(2)]
    x[0, :, first[0]], x[1, :, second[1]], x[-1, 2, first[2]], x[1, 3, second[0]], x[2, 1, first[1]] = inf, -inf, inf, float("nan"), -0.0
    q, k = x[:, :6], x[:, 6:]
    same = lambda a, b: torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))  # noqa: E731
    kc, vc = [torch.zeros((T, 1, 2, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    yq, yk = ql.qk_norm_rope(q, k, pos, f, interleaved=interleaved, axes=axes)
    zq = ql.kv_append(k, k, kc, vc, torch.arange(T, device="cuda"), pos, f, None, q, None, interleaved=interleaved, axes=axes)
    for d in first + second:
        assert same(yq[..., d], q[..., d]) and same(yk[..., d], k[..., d]) and same(zq[..., d], q[..., d]) and torch.equal(kc[:, 0, :, d].nan_to_num(9.0), k[..., d].bfloat16().nan_to_num(9.0)), d
    rest = [d for d in range(D) if d not in first + second]
    for y, x0 in ((yq, q), (yk, k), (zq, q)):
        want, size = norm_rope_axes(x0.nan_to_num(0.0, 0.0, 0.0), None, 1e-6, pos, axes, f, interleaved)
        _check(y[..., rest], want[..., rest], size[..., rest], dtype)


def test_a_captured_call_takes_new_positions():
    announce("qk_norm_rope axes in a graph")
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k = torch.randn((5, 6, 128), device="cuda", generator=gen).bfloat16(), torch.randn((5, 2, 128), device="cuda", generator=gen).bfloat16()
    pos, f, axes = torch.zeros((3, 5), dtype=torch.int32, device="cuda"), _freq(128), _axes(64, 3, "blocks")
    out = (torch.empty_like(q), torch.empty_like(k))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ql.qk_norm_rope(q, k, pos, f, out=out, axes=axes)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ql.qk_norm_rope(q, k, pos, f, out=out, axes=axes)
    for i in range(3):
        pos.copy_(torch.randint(0, 1000, (3, 5), device="cuda", generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        want = ql.qk_norm_rope(q, k, pos, f, axes=axes)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i


def test_refusals():
    announce("refusals of several axes")
    x, f = torch.zeros((2, 4, 64), device="cuda"), _freq(64)
    pos, axes = torch.zeros((3, 2), dtype=torch.int32, device="cuda"), torch.zeros(32, dtype=torch.int32, device="cuda")
    for bad in (dict(positions=pos[0]), dict(positions=pos[:, :1]), dict(positions=pos.long()), dict(axes=axes[:31]), dict(axes=axes.long()), dict(axes=axes.cpu()),
                dict(positions=None, inv_freq=None), dict(axes=None), dict(positions=pos[:0])):
        args = dict(q=x, k=x, positions=pos, inv_freq=f, axes=axes)
        args.update(bad)
        with pytest.raises(AssertionError):
            ql.qk_norm_rope(**args)
    with pytest.raises(_lib.HipQLinearError):  # more than four axes
        ql.qk_norm_rope(x, x, torch.zeros((5, 2), dtype=torch.int32, device="cuda"), f, axes=axes)
    kc = torch.zeros((2, 8, 4, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(AssertionError):
        ql.kv_append(x, x, kc, kc.clone(), torch.zeros(2, dtype=torch.int64, device="cuda"), pos[0], f, axes=axes)
