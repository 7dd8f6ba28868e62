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
