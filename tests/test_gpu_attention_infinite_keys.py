"""Infinite keys: a score of -inf weighs nothing and one of inf makes NaN of its row, in whatever form a query is held inside (bf16, or fp32 in parts).

Finite results have the bounds of test_gpu_attention_paged.py, with a score's terms from the keys without their infinities."""
import pytest
import torch

import decode_ref as ref
from gpu_util import announce
from test_gpu_attention_paged import Case, _bound, _random_tree

pytestmark = pytest.mark.gpu
INF = float("inf")
LONG = 1 << 20  # a bound of the keys that has them cut where there are many of them; 1: never cut


def _place(c, key, b=0):
    return int(c.table[b, key // c.page]), key % c.page


@pytest.mark.parametrize("n,prefix,keys,Hq,D,tree", [
    (1, 40, [0, 39], 4, 128, False), (1, 700, [5, 100, 650, 699], 8, 64, False), (1, 3000, [10, 2999], 4, 256, False), (12, 200, [5, 199], 4, 128, True), (70, 130, [0, 129], 4, 128, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_keys", [1, LONG])
def test_keys(n, prefix, keys, Hq, D, tree, dtype, max_keys):
    """A score of -inf weighs nothing, one of inf makes NaN of the token's row; the query's element has few bits (bf16 holds it), many, or is infinite."""
    announce("attention infinite keys", n, prefix, keys, Hq, D, tree, dtype, max_keys)
    c = Case([n], [prefix], Hq, 1, D, 16, dtype, _random_tree if tree else None, seed=n + prefix + 1)
    c.q[..., 4] = 1.0
    c.q[..., 9] = 0.7
    c.q[:, 0, 9] = 2.0 ** -20
    terms = c.want()[2]
    for key in keys:
        at = _place(c, key)
        kept = c.k[at].clone()
        for d in (4, 9):
            c.k[at][:, d] = -INF
            want = ref.attention(c.q, c.k, c.v, torch.from_numpy(c.table), c.cu, c.prefixes, c.seen, c.scale)
            assert torch.isfinite(want[0]).all()
            got = c.run(max_keys=max_keys).cpu().double()
            far = (got - want[0]).abs() / _bound(want[0], want[1], terms, dtype, D, prefix + n)
            assert far.max() <= 1, (key, d, far.max())
            c.k[at][:, d] = INF
            assert torch.isnan(c.run(max_keys=max_keys)).all(), (key, d)
            c.k[at] = kept
    # an infinite query: scores of one sign and the other, of which only those of -inf weigh nothing
    c.q[0, 0, 4] = -INF
    want = ref.attention(c.q, c.k, c.v, torch.from_numpy(c.table), c.cu, c.prefixes, c.seen, c.scale)
    got = c.run(max_keys=max_keys).cpu().double()
    assert torch.isnan(want[0][0, 0]).all() and torch.isnan(got[0, 0]).all()
    far = (got - want[0]).abs() / _bound(want[0], want[1], terms, dtype, D, prefix + n)
    far[0, 0] = 0
    assert far.max() <= 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_of_minus_infinity_alone(dtype, D):
    announce("attention scores of -inf alone", dtype, D)
    c = Case([1, 1], [30, 2000], 2, 1, D, 16, dtype, seed=D)
    c.q[..., 7] = 0.5
    c.q[1, :, 7] = -0.5
    c.k[int(c.table[0, 0])][:, :, 7] = -INF
    c.k[int(c.table[0, 1])][:, :, 7] = -INF
    clean = c.want()
    for max_keys in (1, LONG):
        got = c.run(max_keys=max_keys).cpu().double()
        assert not got[0].any()
        assert ((got[1] - clean[0][1]).abs() <= _bound(*clean, dtype, D, 2001)[1]).all()
