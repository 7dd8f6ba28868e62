"""Refusals of the operators over images and long contexts at the C ABI, without a GPU: made-up addresses that a refused call never reads."""
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


def _rope(T=1, pos=P, naxes=3, axes=P, freq=P, rot=128, part=None):
    return _lib.lib().mllm_hip_qk_norm_rope_axes(1, C.byref(part or _part()), F32, T, 128, 1e-6, 0, pos, 8, 1, naxes, axes, freq, rot, 0, None)


def _append(T=1, pos=P, naxes=3, axes=P, freq=P, rot=128, cache=None):
    p = _part()
    return _lib.lib().mllm_hip_kv_append_axes(None, C.byref(p), C.byref(p), BF16, T, C.byref(cache or _cache()), P, 1e-6, 0, pos, 8, 1, naxes, axes, freq, rot, 0, None)


@pytest.mark.parametrize("call", [_rope, _append])
@pytest.mark.parametrize("args,want", [
    (dict(naxes=0), BADARG), (dict(naxes=5), SHAPE), (dict(axes=None), BADARG), (dict(axes=ODD), ALIGN), (dict(pos=None), BADARG), (dict(pos=P + 1), ALIGN), (dict(freq=None), BADARG),
    (dict(rot=24), SHAPE), (dict(T=-1), BADARG), (dict(T=1 << 24), SHAPE), (dict(T=0), 0), (dict(T=0, naxes=5), SHAPE), (dict(T=0, pos=None, axes=None, freq=None), 0)])
def test_rotation_by_several_axes(call, args, want):
    assert call(**args) == want


def _adjust(dtype=F32, rows=2, vocab=1000, **changed):
    l = dict(x=P, y=P, x_stride=1000, y_stride=1000, history=P, history_stride=8, history_len=8, lengths=P, prompts=P, repetition=P, presence=P, frequency=P, bias_tokens=P, bias=P,
             bias_tokens_stride=4, bias_stride=4, biases=4, masks=P, masks_stride=32, masks_count=2, mask_of=None)
    l.update(changed)
    return _lib.lib().mllm_hip_logits_adjust(C.byref(_lib.Logits(**l)), dtype, rows, vocab, None)


@pytest.mark.parametrize("args,want", [
    (dict(dtype=2), BADARG), (dict(rows=-1), BADARG), (dict(vocab=0), BADARG), (dict(vocab=(1 << 24) + 1), SHAPE), (dict(rows=65536), SHAPE), (dict(x=None), BADARG), (dict(y=None), BADARG),
    (dict(history=None), BADARG), (dict(history_len=-1), BADARG), (dict(history_len=1 << 31), SHAPE), (dict(biases=-1), BADARG), (dict(biases=(1 << 31) - 1), SHAPE), (dict(bias=None), BADARG),
    (dict(bias_tokens=None), BADARG), (dict(masks=None), BADARG), (dict(masks_count=1), BADARG), (dict(masks_count=-1), BADARG), (dict(y_stride=999), BADARG), (dict(y_stride=0), BADARG),
    (dict(y_stride=1001), BADARG), (dict(x_stride=0), BADARG), (dict(x=ODD), ALIGN), (dict(y=P + 1, dtype=BF16), ALIGN), (dict(rows=0, x=None), 0)] +
    [({name: ODD}, ALIGN) for name in ("history", "lengths", "prompts", "repetition", "presence", "frequency", "bias_tokens", "bias", "masks", "mask_of")])
def test_logits_adjust(args, want):
    assert _adjust(**args) == want


@pytest.mark.parametrize("args", [dict(history_len=(1 << 30) + 1), dict(history_len=(1 << 31) - 1), dict(history_len=(1 << 31) - 4096, lengths=None), dict(biases=(1 << 30) + 1), dict(biases=(1 << 31) - 2)])
def test_logits_adjust_of_more_than_the_kernel_counts_to(args):
    """places are 32-bit numbers there, which go some thousands past the last: histories and biases of up to 2^30"""
    assert _adjust(**args) == SHAPE


def test_logits_adjust_without_a_struct():
    assert _lib.lib().mllm_hip_logits_adjust(None, F32, 1, 10, None) == BADARG


def _states(**changed):
    s = dict(k=P, v=P, k_stride=512, k_head_stride=128, v_stride=512, v_head_stride=128, keys=100, heads=4, head_dim=128)
    s.update(changed)
    return _lib.States(**s)


def _cross(q=None, kv=None, dtype=BF16, T=2, cu=P, first=P, count=P, B=1, tokens=2, keys=40, scale=0.1, work=P, size=1 << 30, no_q=False, no_kv=False):
    q, kv = q if q is not None else _part(heads=8, y=P + (1 << 30)), kv if kv is not None else _states()
    return _lib.lib().mllm_hip_attention_cross(None if no_q else C.byref(q), dtype, T, None if no_kv else C.byref(kv), cu, first, count, B, tokens, keys, scale, work, size, None)


@pytest.mark.parametrize("args,want", [
    (dict(no_q=True), BADARG), (dict(no_kv=True), BADARG), (dict(dtype=2), BADARG), (dict(T=-1), BADARG), (dict(B=-1), BADARG), (dict(B=1 << 23), SHAPE), (dict(B=1 << 29), SHAPE), (dict(tokens=-1), BADARG),
    (dict(keys=-1), BADARG), (dict(keys=1 << 40, size=100), BADARG), (dict(cu=None), BADARG), (dict(first=None), BADARG), (dict(count=None), BADARG), (dict(scale=0.0), BADARG),
    (dict(scale=float("nan")), BADARG), (dict(scale=float("inf")), BADARG), (dict(scale=3e38), BADARG), (dict(T=1 << 29), SHAPE), (dict(tokens=1 << 29), SHAPE),
    (dict(kv=_states(head_dim=100)), SHAPE), (dict(kv=_states(head_dim=264)), SHAPE), (dict(kv=_states(head_dim=0)), BADARG), (dict(kv=_states(heads=3)), SHAPE), (dict(kv=_states(heads=0)), BADARG),
    (dict(kv=_states(k=None)), BADARG), (dict(kv=_states(v=None)), BADARG), (dict(kv=_states(k=ODD)), ALIGN), (dict(kv=_states(v=P + 8)), ALIGN), (dict(kv=_states(k_stride=516)), ALIGN),
    (dict(kv=_states(v_head_stride=4)), ALIGN), (dict(kv=_states(keys=-1)), BADARG), (dict(kv=_states(keys=1 << 31)), SHAPE), (dict(kv=_states(k_stride=(1 << 23) + 8)), SHAPE),
    (dict(kv=_states(v_stride=-8)), SHAPE), (dict(q=_part(heads=8, x=None)), BADARG), (dict(q=_part(heads=8)), BADARG), (dict(q=_part(heads=8, x=ODD, y=P)), ALIGN),
    (dict(q=_part(heads=8, y=P + 8)), ALIGN), (dict(q=_part(heads=8, y=P + 32, y_token_stride=0)), BADARG), (dict(cu=ODD), ALIGN), (dict(first=ODD), ALIGN), (dict(count=ODD), ALIGN),
    (dict(work=P + 8), ALIGN), (dict(keys=9000, work=None), BADARG), (dict(keys=9000, size=100), BADARG), (dict(T=0), 0), (dict(B=0), 0), (dict(tokens=0), 0)])
def test_attention_cross(args, want):
    assert _cross(**args) == want


@pytest.mark.parametrize("keys", [(1 << 30) + 1, (1 << 31) - 64, (1 << 31) - 1])
@pytest.mark.parametrize("stride", [512, 0])
def test_attention_cross_of_more_keys_than_the_kernels_count_to(keys, stride):
    """places of keys are 32-bit numbers there, which go tiles past the last: states of up to 2^30 rows"""
    assert _cross(kv=_states(keys=keys, k_stride=stride, v_stride=stride)) == SHAPE


def test_attention_cross_workspace():
    size = _lib.lib().mllm_hip_attention_cross_workspace_bytes
    assert size(BF16, 1, 1, 32, 8, 128, 1, 100) == 0 and size(BF16, 1, 1, 32, 8, 128, 1, 5000) > 0
    assert size(BF16, 3, 2, 32, 8, 128, 4096, 5000) == size(BF16, 3, 2, 32, 8, 128, 3, 5000) > 0
    assert size(2, 1, 1, 32, 8, 128, 1, 5000) == 0 and size(BF16, 1, 1, 30, 8, 128, 1, 5000) == 0 and size(BF16, 0, 1, 32, 8, 128, 1, 5000) == 0 and size(BF16, 1, 1, 32, 8, 100, 1, 5000) == 0


def _weights(q=None, cache=None, dtype=BF16, T=2, mass=P, stride=2000, head=500, n=500, table=P, table_len=4, cu=P, prefix=P, B=1, tokens=2, keys=40, decay=1.0, scale=0.1, work=P, size=1 << 30,
             no_q=False, no_cache=False):
    q, cache = q if q is not None else _part(heads=8, y=None), cache if cache is not None else _cache(v=None)
    return _lib.lib().mllm_hip_attention_weights(None if no_q else C.byref(q), dtype, T, None if no_cache else C.byref(cache), mass, stride, head, n, table, 4, table_len, cu, prefix, B, tokens, keys,
                                                 decay, scale, work, size, None)


@pytest.mark.parametrize("args,want", [
    (dict(no_q=True), BADARG), (dict(no_cache=True), BADARG), (dict(dtype=2), BADARG), (dict(T=-1), BADARG), (dict(B=-1), BADARG), (dict(tokens=-1), BADARG), (dict(keys=-1), BADARG),
    (dict(keys=(1 << 30) + 1), SHAPE), (dict(mass=None), BADARG), (dict(n=-1), BADARG), (dict(table=None), BADARG), (dict(table_len=0), BADARG), (dict(table_len=-1), BADARG),
    (dict(table_len=1 << 27), SHAPE), (dict(cu=None), BADARG), (dict(prefix=None), BADARG), (dict(scale=0.0), BADARG), (dict(scale=3e38), BADARG), (dict(decay=-1.0), BADARG),
    (dict(decay=float("inf")), BADARG), (dict(decay=float("nan")), BADARG), (dict(T=1 << 29), SHAPE), (dict(B=1 << 14), SHAPE), (dict(B=2, stride=0), BADARG), (dict(head=0), BADARG),
    (dict(q=_part(heads=6)), SHAPE), (dict(q=_part(heads=8, x=None)), BADARG), (dict(q=_part(heads=8, x=ODD)), ALIGN), (dict(q=_part(heads=8, x_token_stride=516)), ALIGN),
    (dict(cache=_cache(head_dim=100)), SHAPE), (dict(cache=_cache(head_dim=264)), SHAPE), (dict(cache=_cache(k=None)), BADARG), (dict(cache=_cache(k=ODD)), ALIGN), (dict(cache=_cache(slot_stride=4)), ALIGN),
    (dict(cache=_cache(pages=0)), BADARG), (dict(cache=_cache(pages=1 << 27)), SHAPE), (dict(mass=ODD), ALIGN), (dict(table=ODD), ALIGN), (dict(cu=ODD), ALIGN), (dict(prefix=ODD), ALIGN),
    (dict(work=P + 8), ALIGN), (dict(keys=4000, work=None), BADARG), (dict(keys=4000, size=100), BADARG), (dict(T=0), 0), (dict(B=0), 0), (dict(tokens=0), 0), (dict(keys=0), 0)])
def test_attention_weights(args, want):
    assert _weights(**args) == want


def _evict(cache=None, mass=P, stride=2000, head=500, n=500, table=P, table_len=8, lengths=P, B=1, to=P, to_len=4, keep=40, first=4, recent=8, kept=P, kept_mass=P + 4096, no_cache=False):
    cache = cache if cache is not None else _cache()
    return _lib.lib().mllm_hip_kv_evict(None if no_cache else C.byref(cache), mass, stride, head, n, table, 8, table_len, lengths, B, to, 4, to_len, keep, first, recent, kept, kept_mass, None)


@pytest.mark.parametrize("args,want", [
    (dict(no_cache=True), BADARG), (dict(cache=_cache(k=None)), BADARG), (dict(cache=_cache(v=None)), BADARG), (dict(cache=_cache(v=ODD)), ALIGN), (dict(cache=_cache(head_dim=100)), SHAPE),
    (dict(cache=_cache(head_dim=520)), SHAPE), (dict(cache=_cache(heads=0)), BADARG), (dict(cache=_cache(page_stride=100)), ALIGN), (dict(cache=_cache(pages=1 << 27)), SHAPE), (dict(mass=None), BADARG),
    (dict(mass=ODD), ALIGN), (dict(n=-1), BADARG), (dict(table=None), BADARG), (dict(table=ODD), ALIGN), (dict(table_len=-1), BADARG), (dict(lengths=None), BADARG), (dict(lengths=ODD), ALIGN),
    (dict(B=-1), BADARG), (dict(B=1 << 14), SHAPE), (dict(to=None), BADARG), (dict(to=ODD), ALIGN), (dict(to_len=-1), BADARG), (dict(to_len=2), SHAPE), (dict(table_len=1 << 27), SHAPE), (dict(to_len=1 << 27), SHAPE), (dict(keep=65), SHAPE), (dict(keep=-1), BADARG),
    (dict(keep=11), BADARG), (dict(first=-1), BADARG), (dict(first=41), BADARG), (dict(recent=-1), BADARG), (dict(recent=1 << 62), BADARG), (dict(kept=None), BADARG), (dict(kept=ODD), ALIGN),
    (dict(kept_mass=None), BADARG), (dict(kept_mass=ODD), ALIGN), (dict(kept_mass=P), BADARG), (dict(B=0), 0), (dict(keep=0, first=0, recent=0), 0)])
def test_kv_evict(args, want):
    assert _evict(**args) == want


def test_attention_weights_workspace():
    size = _lib.lib().mllm_hip_attention_weights_workspace_bytes
    assert size(BF16, 1, 1, 32, 8, 128, 1, 5000) >= 32 * 5000 * 4
    assert size(F32, 640, 20, 32, 8, 128, 32, 5000) >= 640 * 32 * 8 and size(2, 1, 1, 32, 8, 128, 1, 100) == 0 and size(BF16, 0, 1, 32, 8, 128, 1, 100) == 0 and size(BF16, 1, 1, 30, 8, 128, 1, 100) == 0
