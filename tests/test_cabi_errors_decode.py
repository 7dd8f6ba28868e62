"""Refusals of the operators between a layer's projections at the C ABI, without a GPU: made-up addresses that a refused call never reads."""
import ctypes as C

import pytest

from mllm_amd import _lib

P = 0x7F0000100000
ODD = P + 2
BADARG, SHAPE, ALIGN = -1, -2, -3
F32, BF16 = 0, 1


def _part(**changed):
    p = dict(x=P, y=P, weight=P, x_token_stride=512, x_head_stride=128, y_token_stride=512, y_head_stride=128, heads=4)
    p.update(changed)
    return _lib.Heads(**p)


def _cache(**changed):
    c = dict(k=P, v=P, page_stride=16 * 512, slot_stride=512, head_stride=128, pages=8, page_size=16, heads=4, head_dim=128)
    c.update(changed)
    return _lib.KVCache(**c)


def _rope(part=None, nparts=1, dtype=F32, T=1, D=128, pos=P, freq=P, rot=128):
    return _lib.lib().mllm_hip_qk_norm_rope(nparts, C.byref(part if part is not None else _part()), dtype, T, D, 1e-6, 0, pos, freq, rot, 0, None)


@pytest.mark.parametrize("args,want", [
    (dict(nparts=0), BADARG), (dict(nparts=5), BADARG), (dict(dtype=2), BADARG), (dict(T=-1), BADARG), (dict(T=1 << 31), SHAPE), (dict(D=0), BADARG), (dict(D=12), SHAPE),
    (dict(D=520), SHAPE), (dict(rot=-16), BADARG), (dict(rot=8), SHAPE), (dict(rot=144), SHAPE), (dict(pos=None), BADARG), (dict(freq=None), BADARG), (dict(freq=P + 4), ALIGN),
    (dict(pos=P + 1), ALIGN), (dict(part=_part(x=None)), BADARG), (dict(part=_part(y=None)), BADARG), (dict(part=_part(heads=0)), BADARG), (dict(part=_part(heads=65537)), SHAPE),
    (dict(part=_part(x=ODD)), ALIGN), (dict(part=_part(y=ODD)), ALIGN), (dict(part=_part(weight=ODD)), ALIGN), (dict(part=_part(x_token_stride=130)), ALIGN),
    (dict(part=_part(y_head_stride=2)), ALIGN), (dict(part=_part(x_head_stride=132), dtype=BF16), ALIGN), (dict(T=0), 0), (dict(T=0, pos=None, freq=None, rot=0), 0)])
def test_qk_norm_rope(args, want):
    assert _rope(**args) == want


def _append(k=None, v=None, q=None, cache=None, slots=P, T=1, dtype=BF16, rot=128, no_cache=False):
    ref = lambda s: C.byref(s) if s is not None else None  # noqa: E731
    k = _part() if k is None else k
    v = _part() if v is None else v
    return _lib.lib().mllm_hip_kv_append(ref(q), ref(k), ref(v), dtype, T, None if no_cache else ref(cache or _cache()), slots, 1e-6, 0, P, P, rot, 0, None)


@pytest.mark.parametrize("args,want", [
    (dict(no_cache=True), BADARG), (dict(slots=None), BADARG), (dict(slots=P + 4), ALIGN), (dict(cache=_cache(k=None)), BADARG), (dict(cache=_cache(v=None)), BADARG),
    (dict(cache=_cache(k=ODD)), ALIGN), (dict(cache=_cache(page_stride=100)), ALIGN), (dict(cache=_cache(slot_stride=4)), ALIGN), (dict(cache=_cache(head_stride=132)), ALIGN),
    (dict(cache=_cache(pages=0)), BADARG), (dict(cache=_cache(page_size=0)), BADARG), (dict(cache=_cache(pages=1 << 27, page_size=16)), SHAPE), (dict(cache=_cache(heads=2)), SHAPE),
    (dict(cache=_cache(head_dim=100)), SHAPE), (dict(k=_part(heads=2)), SHAPE), (dict(v=_part(heads=5)), SHAPE), (dict(k=_part(x=None)), BADARG), (dict(v=_part(x=ODD)), ALIGN),
    (dict(q=_part(y=None)), BADARG), (dict(q=_part(y=ODD)), ALIGN), (dict(k=_part(y=None), v=_part(y=None, weight=None), T=0), 0), (dict(rot=24), SHAPE), (dict(dtype=5), BADARG)])
def test_kv_append(args, want):
    assert _append(**args) == want


def _attend(q=None, cache=None, dtype=BF16, T=2, table=P, table_len=4, cu=P, prefix=P, B=1, tokens=2, keys=40, tree=None, words=0, scale=0.1, work=P, size=1 << 30, no_q=False):
    q, cache = q if q is not None else _part(heads=8), cache if cache is not None else _cache()
    return _lib.lib().mllm_hip_attention_paged(None if no_q else C.byref(q), dtype, T, C.byref(cache), table, 4, table_len, cu, prefix, B, tokens, keys, tree, words, words, scale, work, size, None)


@pytest.mark.parametrize("args,want", [
    (dict(no_q=True), BADARG), (dict(dtype=2), BADARG), (dict(T=-1), BADARG), (dict(B=-1), BADARG), (dict(tokens=-1), BADARG), (dict(keys=-1), BADARG), (dict(table=None), BADARG),
    (dict(cu=None), BADARG), (dict(prefix=None), BADARG), (dict(table_len=0), BADARG), (dict(table_len=-1), BADARG), (dict(words=-1), BADARG), (dict(scale=0.0), BADARG),
    (dict(scale=-0.1), BADARG), (dict(scale=float("nan")), BADARG), (dict(scale=float("inf")), BADARG), (dict(q=_part(heads=8, x=None)), BADARG), (dict(q=_part(heads=8, y=None)), BADARG),
    (dict(q=_part(heads=0)), BADARG), (dict(q=_part(heads=6)), SHAPE), (dict(cache=_cache(head_dim=96)), SHAPE), (dict(cache=_cache(head_dim=32)), SHAPE),
    (dict(cache=_cache(heads=0)), BADARG), (dict(cache=_cache(pages=1 << 27)), SHAPE), (dict(table_len=1 << 27), SHAPE), (dict(T=1 << 29), SHAPE), (dict(B=1 << 29), SHAPE),
    (dict(tokens=1 << 29), SHAPE), (dict(keys=(1 << 31) - 1), SHAPE), (dict(words=1 << 26), SHAPE), (dict(q=_part(heads=8, x=ODD)), ALIGN), (dict(q=_part(heads=8, y=ODD)), ALIGN),
    (dict(q=_part(heads=8, x_token_stride=516)), ALIGN), (dict(q=_part(heads=8, y_head_stride=68)), ALIGN), (dict(cache=_cache(slot_stride=4)), ALIGN), (dict(cache=_cache(v=ODD)), ALIGN),
    (dict(table=ODD), ALIGN), (dict(cu=ODD), ALIGN), (dict(prefix=ODD), ALIGN), (dict(tree=P + 4, words=1), ALIGN), (dict(work=P + 8), ALIGN),
    (dict(keys=4000, work=None), BADARG), (dict(keys=4000, size=1000), BADARG), (dict(T=0), 0), (dict(B=0), 0), (dict(tokens=0), 0)])
def test_attention_paged(args, want):
    assert _attend(**args) == want


def test_attention_workspace():
    size = _lib.lib().mllm_hip_attention_paged_workspace_bytes
    assert size(BF16, 1, 1, 32, 8, 128, 1, 100) == 0  # one range of keys
    a, b = size(BF16, 1, 1, 32, 8, 128, 1, 5000), size(F32, 1, 1, 32, 8, 128, 1, 5000)
    assert a > 0 and a == b
    assert size(BF16, 4096, 128, 32, 8, 128, 32, 5000) == 0  # rows enough for every CU
    assert size(2, 1, 1, 32, 8, 128, 1, 5000) == 0 and size(BF16, 1, 1, 30, 8, 128, 1, 5000) == 0 and size(BF16, 0, 1, 32, 8, 128, 1, 5000) == 0


def test_tree_mask():
    from mllm_amd import qlinear as ql
    assert ql.tree_mask([-1, 0, 0, 1]).tolist() == [[1], [3], [5], [11]]
    chain = ql.tree_mask(list(range(-1, 129)))
    assert chain.shape == (130, 3) and chain[63, 0] == -1 and chain[64].tolist() == [-1, 1, 0] and chain[129].tolist() == [-1, -1, 3]
    assert ql.tree_mask([], 2).shape == (0, 2) and ql.tree_mask([-5], 2).tolist() == [[1, 0]]
    with pytest.raises(ValueError):
        ql.tree_mask([0])
    with pytest.raises(ValueError):
        ql.tree_mask(list(range(-1, 64)), 1)


def _sample(x=P, dtype=F32, stride=1000, rows=2, vocab=1000, u=P, t=None, k=None, p=None, m=None, out=P, work=P, size=1 << 30):
    return _lib.lib().mllm_hip_sample(x, dtype, stride, rows, vocab, u, t, k, p, m, out, work, size, None)


@pytest.mark.parametrize("args,want", [
    (dict(x=None), BADARG), (dict(u=None), BADARG), (dict(out=None), BADARG), (dict(work=None), BADARG), (dict(dtype=2), BADARG), (dict(rows=-1), BADARG), (dict(vocab=0), BADARG),
    (dict(stride=-1), BADARG), (dict(vocab=(1 << 24) + 1), SHAPE), (dict(rows=65536), SHAPE), (dict(x=ODD), ALIGN), (dict(x=P + 1, dtype=BF16), ALIGN), (dict(u=ODD), ALIGN),
    (dict(t=ODD), ALIGN), (dict(k=ODD), ALIGN), (dict(p=ODD), ALIGN), (dict(m=ODD), ALIGN), (dict(out=ODD), ALIGN), (dict(work=P + 8), ALIGN), (dict(size=1000), BADARG),
    (dict(rows=0, x=None, u=None, out=None, work=None), 0)])
def test_sample(args, want):
    assert _sample(**args) == want


def test_sample_workspace():
    size = _lib.lib().mllm_hip_sample_workspace_bytes
    assert size(0, 100) == 0 and size(4, 0) == 0 and size(1, 1 << 25) == 0
    assert size(8, 151936) >= 8 * 151936 * 4 and size(8, 151936) % 16 == 0


@pytest.mark.parametrize("part,T,want", [
    (dict(y_token_stride=0), 2, BADARG), (dict(y_head_stride=0), 1, BADARG), (dict(x_token_stride=1024), 2, BADARG), (dict(x_head_stride=256), 1, BADARG),
    (dict(x_token_stride=0), 2, BADARG), (dict(), 1 << 24, SHAPE)])
def test_results_without_places_of_their_own_and_very_many_tokens(part, T, want):
    """Two heads of the results in one place, a result where another head's input is, more tokens than a launch has workgroups."""
    assert _rope(part=_part(**part), T=T) == want


def test_attention_over_its_queries_and_of_very_many_tokens():
    ask = lambda T=1, B=1, tokens=1, **q: _lib.lib().mllm_hip_attention_paged(  # noqa: E731
        C.byref(_part(**dict(dict(y=P + (1 << 30)), **q))), F32, T, C.byref(_cache()), P, 8, 8, P, P, B, tokens, 0, None, 0, 0, 0.1, None, 0, None)
    assert ask(y=P) == BADARG and ask(T=2, tokens=2, y_token_stride=0) == BADARG and ask(y_head_stride=0) == BADARG
    assert ask(T=1 << 22, B=1 << 22) == SHAPE


def test_a_bound_of_more_tokens_than_there_are():
    size = _lib.lib().mllm_hip_attention_paged_workspace_bytes
    assert size(BF16, 3, 2, 32, 8, 128, 4096, 5000) == size(BF16, 3, 2, 32, 8, 128, 3, 5000) > 0
