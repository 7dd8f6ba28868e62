"""What is no number or infinite in the cache reaches the tokens that see it, as the formula has it, wherever its position lies: in front of the
last tile, within the one that holds the end of the prefix, in any range that the keys are cut into.

Finite results have the bounds of test_gpu_attention_paged.py."""
import numpy as np
import pytest
import torch

from gpu_util import announce
from test_gpu_attention_paged import Case, _bound, _random_tree

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")
LONG = 1 << 20  # a bound of the keys that has them cut where there are many of them; 1: never cut


def _place(c, key, b=0):
    return int(c.table[b, key // c.page]), key % c.page


def _finite(c, got, clean, skip):
    """every element but those of `skip` is within the bounds"""
    bound = _bound(*clean, c.dtype, c.D, max(p + n for p, n in zip(c.prefixes, c.counts)))
    far = (got - clean[0]).abs() / bound
    far[..., skip] = 0
    assert far.max() <= 1, far.max()


@pytest.mark.parametrize("n,prefix,keys,Hq,D,tree", [
    (1, 40, [0, 20, 39], 4, 128, False), (1, 4110, [0, 4000, 4031, 4032, 4100, 4109], 8, 128, False), (1, 45, [44], 1, 64, False), (1, 130, [127, 128, 129], 2, 256, False),
    (12, 45, [0, 44], 4, 128, True), (40, 200, [5, 191, 192, 199], 8, 128, True), (5, 3000, [17, 2943, 2944, 2999], 4, 64, True), (33, 70, [63, 64, 69], 2, 256, True),
    (70, 130, [0, 127, 128, 129], 4, 128, False), (300, 100, [63, 64, 99], 2, 64, False), (2, 1000, [959, 960, 999], 16, 128, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_keys", [1, LONG])
def test_values_of_the_prefix(n, prefix, keys, Hq, D, tree, dtype, max_keys):
    """every token sees the prefix: NaN, an infinity of either sign, and infinities of both"""
    announce("attention values of the prefix", n, prefix, keys, Hq, D, tree, dtype, max_keys)
    c = Case([n], [prefix], Hq, 1, D, 16, dtype, _random_tree if tree else None, seed=n + prefix)
    clean = c.want()
    for key in keys:
        v = c.v[_place(c, key)]
        before = v.clone()
        other = c.v[_place(c, prefix // 2)]
        kept = other.clone()
        other[:, 60] = -INF
        v[:, 3], v[:, 37], v[:, 41], v[:, 60] = NAN, INF, -INF, NAN if key == prefix // 2 else INF
        got = c.run(max_keys=max_keys).cpu().double()
        assert torch.isnan(got[..., 3]).all() and not torch.isfinite(got[..., [37, 41, 60]]).any(), key
        if dtype == torch.bfloat16:
            assert (got[..., 37] == INF).all() and (got[..., 41] == -INF).all() and torch.isnan(got[..., 60]).all(), key
        _finite(c, got, clean, [3, 37, 41, 60])
        other.copy_(kept)
        v.copy_(before)
