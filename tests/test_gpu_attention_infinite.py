"""Infinite values whose weights are 1, like the others, or too small for fp32: infinite results of their sign, whatever the form that a weight has inside
(bf16, or fp32 in parts) and whichever tile or range a position falls into.

Finite results have the bounds of test_gpu_attention_paged.py, from the inputs without their infinities."""
import pytest
import torch

from gpu_util import announce
from test_gpu_attention_paged import Case, _bound, _random_tree

pytestmark = pytest.mark.gpu
INF = float("inf")
LONG = 1 << 20  # a bound of the keys that has them cut where there are many of them; 1: never cut


def _place(c, key, b=0):
    return int(c.table[b, key // c.page]), key % c.page


@pytest.mark.parametrize("n,prefix,keys,Hq,D,tree", [
    (1, 700, [0, 63, 64, 600, 650, 699], 4, 128, False), (1, 4110, [100, 4100], 8, 64, False), (9, 300, [10, 130, 299], 4, 128, True), (20, 100, [3, 64, 99], 2, 256, True), (130, 260, [0, 255, 259], 4, 128, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_keys", [1, LONG])
def test_values_whatever_their_weight(n, prefix, keys, Hq, D, tree, dtype, max_keys):
    """An infinite value of a key whose score is the largest, is like the others, and is 150 below them (exp: 1e-65): infinite in all three."""
    announce("attention infinite values", n, prefix, keys, Hq, D, tree, dtype, max_keys)
    c = Case([n], [prefix], Hq, 1, D, 16, dtype, _random_tree if tree else None, seed=n + prefix)
    c.q[..., 0] = 8.0
    for key in keys:
        page, slot = _place(c, key)
        kept = c.k[page, slot].clone(), c.v[page, slot].clone()
        for score in (150.0, 0.0, -150.0):
            c.k[page, slot] = 0
            c.k[page, slot, :, 0] = score * D ** 0.5 / 8
            clean = c.want()
            c.v[page, slot][:, 5], c.v[page, slot][:, 33] = INF, -INF
            got = c.run(max_keys=max_keys).cpu().double()
            assert (got[..., 5] == INF).all() and (got[..., 33] == -INF).all(), (key, score)
            far = (got - clean[0]).abs() / _bound(*clean, dtype, D, prefix + n)
            far[..., [5, 33]] = 0
            assert far.max() <= 1, (key, score, far.max())
            c.k[page, slot], c.v[page, slot] = kept


@pytest.mark.parametrize("n,prefix,keys,Hq,D,tree", [(1, 700, [5, 650, 699], 4, 128, False), (1, 40, [3], 2, 64, False), (9, 300, [10, 299], 4, 128, True), (70, 130, [0, 129], 2, 256, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_keys", [1, LONG])
def test_values_of_scores_of_minus_infinity(n, prefix, keys, Hq, D, tree, dtype, max_keys):
    """The weight is 0 and the value counts all the same; the row's other elements are as if the key were not there."""
    announce("attention infinite values of scores of -inf", n, prefix, keys, Hq, D, tree, dtype, max_keys)
    c = Case([n], [prefix], Hq, 1, D, 16, dtype, _random_tree if tree else None, seed=n + prefix)
    c.q[..., 7] = 1.0
    terms = c.want()[2]
    for key in keys:
        at = _place(c, key)
        kept = c.k[at].clone(), c.v[at].clone()
        c.k[at][:, 7] = -INF
        want, size, _ = c.want()
        c.v[at][:, 5], c.v[at][:, 33] = INF, -INF
        got = c.run(max_keys=max_keys).cpu().double()
        assert (got[..., 5] == INF).all() and (got[..., 33] == -INF).all(), key
        far = (got - want).abs() / _bound(want, size, terms, dtype, D, prefix + n)
        far[..., [5, 33]] = 0
        assert far.max() <= 1, (key, far.max())
        c.k[at], c.v[at] = kept


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 8, 128), (6, 2, 256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tree", [None, _random_tree])
@pytest.mark.parametrize("max_keys", [1, LONG])
def test_other_sequences_and_heads_keep_their_bits(Hq, Hkv, D, dtype, tree, max_keys):
    announce("attention infinite values of one sequence", Hq, Hkv, D, dtype, tree is not None, max_keys)
    c = Case([3, 1, 40, 2], [70, 900, 200, 63], Hq, Hkv, D, 16, dtype, tree, seed=D, spare=3)
    out = torch.full(c.q.shape, 7.0, dtype=dtype, device="cuda")
    clean = c.run(max_keys=max_keys, out=out.clone())
    for b, key in ((1, 900), (1, 3), (2, 199), (2, 205), (2, 100)):  # new tokens and the prefix, key head 1
        c.v[_place(c, key, b)][1, 9] = INF if key % 2 else float("nan")
    got = c.run(max_keys=max_keys, out=out.clone())
    group = Hq // Hkv
    hit = torch.zeros(c.q.shape, dtype=torch.bool, device="cuda")
    hit[int(c.cu[1]):int(c.cu[3]), group:2 * group, 9] = True
    assert not torch.isfinite(got[hit]).any()
    assert torch.equal(got[~hit], clean[~hit]) and (got[int(c.cu[-1]):] == 7).all()
