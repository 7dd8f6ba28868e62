"""GPU parity of the heads' norm and rotation and of the appending to a paged cache, against the formulas in 64 bits.

Bounds.  An fp32 result is off by: the sum of squares (up to eight fused adds in a lane and six across lanes, 14 roundings, half of it in the
root), division, addition, root and reciprocal (4), two products of the norm (2), a sine and cosine (the fraction of a turn in fp32 is within
2^-26, 2 pi of it 1.6 * 2^-24; the function 2 * 2^-24), two products and a sum (3): under 24 * 2^-24 of |a| + |b|.  A bf16 result
in addition by half a step, 2^-8 of itself."""
import numpy as np
import pytest
import torch

from mllm_amd import _lib, qlinear as ql
from decode_ref import norm_rope
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


def _heads(T, H, D, dtype, gen, wide=0):
    """views of a wider row, as a projection of several parts leaves them"""
    rows = torch.randn((T, H + wide, D), device="cuda", generator=gen).to(dtype)
    return rows[:, wide:] if wide else rows


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,interleaved,far", [
    (1, 32, 8, 128, 128, False, 0), (1, 1, 1, 64, 64, True, 1 << 20), (3, 14, 2, 64, 32, False, 131072), (257, 5, 1, 128, 128, False, 2 ** 31 - 300),
    (40, 32, 8, 128, 64, True, 4096), (7, 3, 3, 80, 80, False, 1000), (7, 3, 3, 80, 32, True, 1000), (33, 4, 2, 96, 96, False, 100000),
    (5, 8, 4, 256, 256, False, 1 << 17), (2, 2, 1, 512, 512, False, 77), (2, 2, 1, 264, 16, True, 77), (4, 6, 2, 8, 0, False, 9), (600, 16, 8, 128, 128, False, 50)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_and_rotation(T, Hq, Hkv, D, rot, interleaved, far, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T * 31 + D)
    announce("qk_norm_rope", T, Hq, Hkv, D, rot, interleaved, dtype)
    q, k = _heads(T, Hq, D, dtype, gen, 2), _heads(T, Hkv, D, dtype, gen)
    wq, wk = [1 + 0.3 * torch.randn(D, device="cuda", generator=gen) for _ in range(2)]
    pos = (far + torch.arange(T, device="cuda")).int()
    f = _freq(rot) if rot else None
    for unit, norm in ((False, True), (True, True), (False, False)):
        yq, yk = ql.qk_norm_rope(q, k, pos if rot else None, f, wq if norm else None, wk if norm else None, eps=1e-5, add_unit_offset=unit, interleaved=interleaved)
        for y, x, w in ((yq, q, wq), (yk, k, wk)):
            want, size = norm_rope(x, w if norm else None, 1e-5, pos, f, interleaved, unit)
            _check(y, want, size, dtype)


def test_in_place_negative_positions_and_one_norm_of_two():
    gen = torch.Generator(device="cuda").manual_seed(3)
    announce("qk_norm_rope in place")
    q, k = _heads(9, 12, 128, torch.float32, gen), _heads(9, 2, 128, torch.float32, gen, 3)
    w = torch.rand(128, device="cuda", generator=gen)
    pos = torch.tensor([0, -1, -2 ** 31, 2 ** 31 - 1, 5, 5, 5, 1, 2], dtype=torch.int32, device="cuda")
    f = _freq(128)
    want = [norm_rope(q, w, 1e-6, pos, f, False), norm_rope(k, None, 1e-6, pos, f, False)]
    yq, yk = ql.qk_norm_rope(q, k, pos, f, w, None, out=(q, k))
    assert yq.data_ptr() == q.data_ptr() and yk.data_ptr() == k.data_ptr()
    _check(q, *want[0], torch.float32)
    _check(k, *want[1], torch.float32)


def test_rows_that_the_norm_cannot_scale():
    """zeros stay zeros, an infinity or a NaN stays within its head"""
    announce("qk_norm_rope special rows")
    x = torch.ones((4, 2, 64), device="cuda")
    x[0, 0] = 0
    x[1, 0, 3] = float("inf")
    x[2, 1, 5] = float("nan")
    w = torch.ones(64, device="cuda")
    pos = torch.arange(4, device="cuda").int()
    y, _ = ql.qk_norm_rope(x, x, pos, _freq(64), w, w)
    y = y.cpu()
    assert (y[0, 0] == 0).all() and torch.isnan(y[1, 0]).any() and torch.isnan(y[2, 1]).all()
    clean = torch.ones((4, 2), dtype=torch.bool)
    clean[1, 0] = clean[2, 1] = False
    assert torch.isfinite(y[clean]).all()


def test_no_tokens():
    announce("qk_norm_rope no tokens")
    x = torch.empty((0, 2, 64), device="cuda")
    yq, yk = ql.qk_norm_rope(x, x, torch.empty(0, dtype=torch.int32, device="cuda"), _freq(64))
    assert yq.shape == yk.shape == (0, 2, 64)


def _cache(pages, page, H, D, layout):
    """(k_cache, v_cache) as [pages, page, H, D] of the layout, filled with numbers that must stay where nothing is stored"""
    if layout == "slots":  # heads of a slot next to each other
        k, v = torch.empty((pages, page, H, D)), torch.empty((pages, page, H, D))
    elif layout == "heads":  # slots of a head next to each other
        k, v = torch.empty((pages, H, page, D)).transpose(1, 2), torch.empty((pages, H, page, D)).transpose(1, 2)
    else:  # keys and values of a page in one tensor, rows with room behind them
        both = torch.empty((pages, 2, page, H, D + 8))
        k, v = both[:, 0, ..., :D], both[:, 1, ..., :D]
    put = lambda t: torch.empty_strided(t.shape, t.stride(), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    if layout == "both":
        both = torch.empty((pages, 2, page, H, D + 8), dtype=torch.bfloat16, device="cuda")
        k, v = both[:, 0, ..., :D], both[:, 1, ..., :D]
    else:
        k, v = put(k), put(v)
    k.copy_(torch.arange(k.numel(), device="cuda").view(k.shape) % 97 - 48)
    v.copy_(torch.arange(v.numel(), device="cuda").view(v.shape) % 89 - 44)
    return k, v


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,page,layout", [
    (1, 32, 8, 128, 128, 16, "slots"), (5, 8, 2, 64, 64, 1, "heads"), (37, 4, 1, 80, 32, 24, "both"), (130, 10, 5, 128, 128, 16, "both"),
    (64, 2, 2, 256, 64, 256, "heads"), (1000, 16, 4, 128, 64, 64, "slots")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append(T, Hq, Hkv, D, rot, page, layout, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T + 7 * D)
    announce("kv_append", T, Hq, Hkv, D, rot, page, layout, dtype)
    pages = -(-T * 2 // page)
    kc, vc = _cache(pages, page, Hkv, D, layout)
    kc0, vc0 = kc.clone(), vc.clone()
    q, k, v = _heads(T, Hq, D, dtype, gen, 1), _heads(T, Hkv, D, dtype, gen, 2), _heads(T, Hkv, D, dtype, gen, 1)
    wq, wk = [1 + 0.3 * torch.randn(D, device="cuda", generator=gen) for _ in range(2)]
    pos = torch.randint(0, 100000, (T,), device="cuda", generator=gen).int()
    slots = torch.randperm(pages * page, device="cuda", generator=gen)[:T]
    if T > 3:  # padded tokens: any number outside the cache
        slots[1], slots[2], slots[3] = -1, pages * page, 2 ** 62
    kept = ((slots >= 0) & (slots < pages * page)).cpu()
    y = ql.kv_append(k, v, kc, vc, slots, pos, _freq(rot), wk, q, wq, eps=1e-6)
    _check(y, *norm_rope(q, wq, 1e-6, pos, _freq(rot), False), dtype)
    at = slots.cpu()[kept]
    want, size = norm_rope(k, wk, 1e-6, pos, _freq(rot), False)
    _check(kc[(at // page).cuda(), (at % page).cuda()].contiguous(), want[kept], size[kept], torch.bfloat16)
    assert torch.equal(vc[(at // page).cuda(), (at % page).cuda()], v.to(torch.bfloat16)[kept.cuda()])
    for c, c0 in ((kc, kc0), (vc, vc0)):  # nothing else changed
        c[(at // page).cuda(), (at % page).cuda()] = 0
        c0[(at // page).cuda(), (at % page).cuda()] = 0
        assert torch.equal(c, c0)


def test_append_without_rotation_norm_or_queries():
    gen = torch.Generator(device="cuda").manual_seed(1)
    announce("kv_append plain")
    kc, vc = _cache(4, 8, 2, 128, "slots")
    k, v = _heads(6, 2, 128, torch.float32, gen), _heads(6, 2, 128, torch.float32, gen)
    slots = torch.arange(9, 15, device="cuda")
    assert ql.kv_append(k, v, kc, vc, slots) is None
    assert torch.equal(kc.view(-1, 2, 128)[9:15], k.to(torch.bfloat16)) and torch.equal(vc.view(-1, 2, 128)[9:15], v.to(torch.bfloat16))


def test_append_far_into_a_large_cache():
    """elements behind 2^32"""
    announce("kv_append large cache")
    page, H, D = 64, 8, 128
    pages = (1 << 32) // (page * H * D) + 3
    kc, vc = [torch.empty((pages, page, H, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k, v = [torch.randn((2, H, D), device="cuda") for _ in range(2)]
    slots = torch.tensor([pages * page - 1, 5], device="cuda")
    kc[0].zero_(), vc[0].zero_()
    ql.kv_append(k, v, kc, vc, slots)
    assert torch.equal(kc[-1, -1], k[0].to(torch.bfloat16)) and torch.equal(vc[-1, -1], v[0].to(torch.bfloat16))
    assert torch.equal(kc[0, 5], k[1].to(torch.bfloat16)) and not kc[0, :5].any() and not kc[0, 6:].any()


def test_refusals():
    announce("refusals of qk_norm_rope and kv_append")
    x, f = torch.zeros((2, 4, 64), device="cuda"), _freq(64)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    w = torch.ones(64, device="cuda")
    kc, vc = _cache(2, 8, 4, 64, "slots")
    slots = torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in (dict(q=x.cpu()), dict(q=x.half()), dict(q=x[0]), dict(k=x.bfloat16()), dict(k=x[:1]), dict(positions=pos.long()), dict(positions=pos[:1]), dict(inv_freq=f.float()),
                dict(positions=None), dict(q_weight=w.bfloat16()), dict(k_weight=w[:32]), dict(q=x.transpose(1, 2)), dict(out=(x, x[:1]))):
        args = dict(q=x, k=x, positions=pos, inv_freq=f, q_weight=w, k_weight=w)
        args.update(bad)
        with pytest.raises((AssertionError, TypeError)):
            ql.qk_norm_rope(**args)
    with pytest.raises(_lib.HipQLinearError):  # rot_dim of no whole sixteen
        ql.qk_norm_rope(x, x, pos, _freq(40))
    with pytest.raises(_lib.HipQLinearError):  # longer than a head
        ql.qk_norm_rope(x, x, pos, _freq(80))
    with pytest.raises(_lib.HipQLinearError):  # rows that are not 16-byte aligned
        ql.qk_norm_rope(torch.zeros((2, 4, 66), device="cuda")[..., :64], x, pos, f)
    for bad in (dict(k=x[:, :2]), dict(v=x.bfloat16()), dict(k_cache=kc.float()), dict(v_cache=vc[:1]), dict(k_cache=kc.transpose(1, 2)), dict(slots=slots.int()), dict(slots=None),
                dict(slots=slots[:1]), dict(q=x[:1]), dict(k_cache=kc.cpu())):
        args = dict(k=x, v=x, k_cache=kc, v_cache=vc, slots=slots)
        args.update(bad)
        with pytest.raises((AssertionError, TypeError)):
            ql.kv_append(**args)


def test_results_without_places_of_their_own_are_refused():
    announce("refusals of results in one place")
    x, f = torch.zeros((2, 4, 64), device="cuda"), _freq(64)
    pos, slots = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    one = torch.zeros((1, 4, 64), device="cuda").expand(2, 4, 64)
    y = torch.empty_like(x)
    for out in ((one, y), (y, one), (torch.zeros((2, 1, 64), device="cuda").expand(2, 4, 64), y), (y, y)):
        with pytest.raises(AssertionError):
            ql.qk_norm_rope(x, x, pos, f, out=out)
    kc, vc = (torch.zeros((1, 8, 4, 64), dtype=torch.bfloat16, device="cuda").expand(2, 8, 4, 64) for _ in range(2))
    with pytest.raises(AssertionError):
        ql.kv_append(x, x, kc, vc, slots)
    square = torch.zeros((4, 4, 64), device="cuda")  # heads and tokens in the other order, over the input itself
    with pytest.raises(_lib.HipQLinearError):
        ql.qk_norm_rope(square, torch.zeros((4, 4, 64), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), f, out=(square.transpose(0, 1), torch.empty_like(square)))
