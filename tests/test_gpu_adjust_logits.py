"""GPU parity of penalties, biases and masks on logits, against the definition in 64 bits.

Bound.  fp32: a division or product, frequency times count, plus presence, the difference and the bias: five roundings, each of at most 2^-24 of a sum of the absolute
terms: 5 * 2^-24 of it.  bf16 in addition half a step of the result, 2^-8 of itself.  What nothing applies to keeps its bits."""
import numpy as np
import pytest
import torch

from mllm_amd import _lib, qlinear as ql
from context_ref import adjust
from gpu_util import announce

pytestmark = pytest.mark.gpu
E32, E16 = 2.0 ** -24, 2.0 ** -8


def _int(v):
    return torch.from_numpy(np.asarray(v, np.int32)).cuda()


def _float(v):
    return torch.from_numpy(np.asarray(v, np.float32)).cuda()


def _words(allowed):
    m, v = allowed.shape
    bits = np.zeros((m, -(-v // 32) * 32), np.uint8)
    bits[:, :v] = allowed
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).cuda()


def _check(got, want, size, dtype):
    got, want, size = got.cpu().double().numpy(), np.stack(want), np.stack(size)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    odd = ~np.isfinite(want)
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)])
    bound = 5 * E32 * size + (E16 * np.abs(np.where(odd, 0, want)) if dtype == torch.bfloat16 else 0) + 1e-40
    with np.errstate(invalid="ignore"):
        far = (np.abs(got - want) / bound)[~odd]
    assert far.size == 0 or far.max() <= 1, far.max()


def _everything(rows, vocab, L, nb, nm, seed):
    r = np.random.RandomState(seed)
    history = (r.rand(rows, L) ** 3 * vocab).astype(np.int32)
    history[r.rand(rows, L) < 0.02] = -1
    history[r.rand(rows, L) < 0.01] = vocab + 5
    lengths = r.randint(0, L + 1, rows)
    prompts = (lengths * r.rand(rows)).astype(np.int32)
    bias_tokens = r.randint(-1, vocab + 1, (rows, nb)).astype(np.int32)
    if nb > 2:
        bias_tokens[:, -1] = bias_tokens[:, 0]  # a token twice
    s = dict(history=history, lengths=lengths, prompts=prompts, repetition=r.uniform(0.8, 1.6, rows), presence=r.uniform(-0.5, 1, rows), frequency=r.uniform(-0.2, 0.5, rows),
             bias_tokens=bias_tokens, bias=r.randn(rows, nb) * 4, allowed=r.rand(nm, vocab) < r.rand(nm, 1), mask_of=r.randint(-1, nm + 1, rows))
    for name in ("repetition", "presence", "frequency", "bias"):
        s[name] = s[name].astype(np.float32)
    return s


def _want(x, s, use):
    want, size = [], []
    for i, row in enumerate(x.float().cpu().numpy()):
        said = s["history"][i, :s["lengths"][i]] if "history" in use else ()
        bias = list(zip(s["bias_tokens"][i], s["bias"][i])) if "bias" in use else ()
        m = s["mask_of"][i]
        allowed = s["allowed"][m] if "masks" in use and 0 <= m < len(s["allowed"]) else None
        w, z = adjust(row, said, s["prompts"][i], float(s["repetition"][i]), float(s["presence"][i]), float(s["frequency"][i]), bias, allowed)
        want.append(w), size.append(z)
    return want, size


def _call(x, s, use, out=None):
    a = {}
    if "history" in use:
        a.update(history=_int(s["history"]), lengths=_int(s["lengths"]), prompts=_int(s["prompts"]), repetition=_float(s["repetition"]), presence=_float(s["presence"]), frequency=_float(s["frequency"]))
    if "bias" in use:
        a.update(bias_tokens=_int(s["bias_tokens"]), bias=_float(s["bias"]))
    if "masks" in use:
        a.update(masks=_words(s["allowed"]), mask_of=_int(s["mask_of"]))
    return ql.adjust_logits(x, out=out, **a)


@pytest.mark.parametrize("rows,vocab,L,nb,nm", [(1, 1, 1, 1, 1), (1, 31, 5, 3, 1), (3, 4096, 40, 4, 2), (2, 4097, 300, 30, 3), (5, 12301, 7000, 300, 2), (1, 151936, 900, 20, 1), (130, 1000, 64, 8, 5)])
@pytest.mark.parametrize("use", ["history", "bias", "masks", "history bias masks", ""])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_against_the_definition(rows, vocab, L, nb, nm, use, dtype):
    announce("adjust_logits", rows, vocab, L, nb, nm, use, dtype)
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (torch.randn((rows, vocab), device="cuda", generator=gen) * 4).to(dtype)
    s = _everything(rows, vocab, L, nb, nm, vocab + rows)
    want, size = _want(x, s, use)
    before = x.clone()
    y = _call(x, s, use)
    assert y.dtype == dtype and y.shape == x.shape and torch.equal(x, before)
    _check(y, want, size, dtype)
    if not use:
        assert torch.equal(y, x)
    _call(x, s, use, out=x)  # in place: the same bits
    assert torch.equal(x.view(torch.int16 if dtype == torch.bfloat16 else torch.int32), y.view(torch.int16 if dtype == torch.bfloat16 else torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at,to", [(0, 0), (1, 1), (1, 0), (3, 2), (7, 7), (0, 5)])
def test_rows_anywhere(dtype, at, to):
    """rows of odd strides that begin anywhere, results in other places; what lies around them stays"""
    announce("adjust_logits strides", dtype, at, to)
    rows, vocab = 3, 5003
    gen = torch.Generator(device="cuda").manual_seed(at * 8 + to)
    x = torch.randn((rows, vocab + 12), device="cuda", generator=gen).to(dtype)[:, at:at + vocab]
    room = torch.full((rows, vocab + 29), 5.0, device="cuda").to(dtype)
    s = _everything(rows, vocab, 50, 8, 2, 3)
    want, size = _want(x, s, "history bias masks")
    y = _call(x, s, "history bias masks", out=room[:, to:to + vocab])
    _check(y, want, size, dtype)
    assert (room[:, :to] == 5).all() and (room[:, to + vocab:] == 5).all()


def test_infinities_nans_and_masks_that_leave_nothing():
    announce("adjust_logits special values")
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[inf, -inf, nan, 0.0, -0.0, 1e38, -1e38, 3.4e38] * 5] * 3, device="cuda")
    history = _int([list(range(40))] * 3)
    allowed = np.ones((3, 40), bool)
    allowed[1] = False
    allowed[2, ::2] = False
    args = dict(history=history, repetition=_float([0.5] * 3), presence=_float([0.25] * 3), masks=_words(allowed))
    y = ql.adjust_logits(x, **args)
    want = [adjust(row, range(40), 0, 0.5, 0.25, 0.0, (), m)[0] for row, m in zip(x.cpu().numpy(), allowed)]
    want = np.stack(want)
    with np.errstate(over="ignore"):
        assert np.array_equal(y.cpu().numpy(), want.astype(np.float32), equal_nan=True)
    tokens = ql.sample(y, torch.full((3,), 0.5, device="cuda"))
    assert tokens[1] == -1 and (tokens[[0, 2]] >= 0).all()


def test_shared_rows_lengths_outside_and_masks_by_row():
    """one history, one list of biases and one mask for all rows (stride 0); lengths and prompts that are outside their bounds are held to them"""
    announce("adjust_logits shared")
    rows, vocab, L = 6, 777, 9
    gen = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn((rows, vocab), device="cuda", generator=gen)
    history = _int([[5, 6, 7, 5, 5, 700, 6, 0, 776]])
    lengths, prompts = [-3, 0, 4, 9, 10, 2 ** 31 - 1], [0, 5, -7, 2, 9, 2 ** 31 - 1]
    bias_tokens, bias = _int([[1, 2]]).expand(rows, 2), _float([[0.5, -3.0]]).expand(rows, 2)
    allowed = np.random.RandomState(1).rand(1, vocab) < 0.5
    y = ql.adjust_logits(x, history.expand(rows, L), _int(lengths), _int(prompts), _float([1.3] * rows), _float([0.1] * rows), _float([0.2] * rows), bias_tokens, bias,
                         _words(allowed).expand(rows, -1))
    f = lambda v: float(np.float32(v))  # noqa: E731
    ref = [adjust(row, history[0].tolist()[:min(max(n, 0), L)], max(p, 0), f(1.3), f(0.1), f(0.2), [(1, 0.5), (2, -3.0)], allowed[0])
           for row, n, p in zip(x.cpu().numpy(), lengths, prompts)]
    _check(y, [w for w, _ in ref], [z for _, z in ref], torch.float32)


def test_a_captured_call_takes_growing_histories():
    announce("adjust_logits in a graph")
    rows, vocab, L = 4, 20000, 64
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((rows, vocab), device="cuda", generator=gen).bfloat16()
    s = _everything(rows, vocab, L, 4, 2, 9)
    a = dict(history=_int(s["history"]), lengths=_int([0] * rows), prompts=_int([3] * rows), repetition=_float(s["repetition"]), presence=_float(s["presence"]),
             frequency=_float(s["frequency"]), masks=_words(s["allowed"]), mask_of=_int([0, 1, -1, 0]))
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ql.adjust_logits(x, out=out, **a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ql.adjust_logits(x, out=out, **a)
    for i in range(4):
        a["lengths"].copy_(_int([i * 13 + 2] * rows))
        a["mask_of"].copy_(_int([i % 3 - 1] * rows))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ql.adjust_logits(x, **a)), i


def test_no_rows_and_refusals():
    announce("adjust_logits refusals")
    assert ql.adjust_logits(torch.empty((0, 9), device="cuda")).shape == (0, 9)
    x, i, f = torch.zeros((2, 64), device="cuda"), torch.zeros((2, 3), dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
    good = dict(logits=x, history=i, lengths=i[:, 0].contiguous(), repetition=f, bias_tokens=i, bias=torch.zeros((2, 3), device="cuda"), masks=i[:, :2])
    ql.adjust_logits(**good)
    for bad in (dict(logits=x.half()), dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x.t()), dict(history=i.long()), dict(history=i[:1]), dict(history=None), dict(lengths=i[:, 0]),
                dict(lengths=f), dict(repetition=f.double()), dict(repetition=f[:1]), dict(bias=None), dict(bias_tokens=None), dict(bias=torch.zeros((2, 2), device="cuda")),
                dict(masks=i), dict(masks=i[:1, :2]), dict(masks=None, mask_of=i[:, 0].contiguous()), dict(out=x.bfloat16()), dict(out=x[:1]), dict(out=x[:1].expand(2, 64))):
        with pytest.raises((AssertionError, TypeError)):
            ql.adjust_logits(**dict(good, **bad))
    with pytest.raises(_lib.HipQLinearError):  # the results over the input, rows apart by another number
        wide = torch.zeros(400, device="cuda")
        ql.adjust_logits(wide.as_strided((2, 64), (64, 1)), out=wide.as_strided((2, 64), (100, 1)))
