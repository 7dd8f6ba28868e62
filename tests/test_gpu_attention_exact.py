"""fp32 queries: the root mean square of the error against 64 bits is that of fp32 sums, which the wide bounds of the other tests do not show.

With values that are independent of one another the error of a result, relative to the results' root mean square, is the weights' relative one (both are sums over
the same weights).  In units of 2^-24: a score of up to 6 (times the scale), summed over 3 D / 32 products of four steps each: 6 * 0.3 * sqrt(96) = 18 with D 256;
the sums over up to 4097 keys in 3 * 128 steps, whose partial sums are 0.6 of the last one: 0.3 * 0.6 * sqrt(384) = 4; exponential and argument 2.  Together, as
independent ones: 18; twice that is allowed.  Queries of two bf16 parts (16 bits, cut off) would leave 214 to 355 at these sizes, weights of two parts 99 to 139."""
import pytest
import torch

from gpu_util import announce
from test_gpu_attention_paged import Case, _random_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,prefix,Hq,Hkv,D,tree,max_keys", [
    (1, 4096, 32, 8, 128, False, 4097), (1, 4096, 32, 8, 128, False, 1), (1, 1000, 32, 8, 64, False, 1001), (1, 700, 16, 2, 256, False, 701), (29, 600, 8, 2, 128, True, 629),
    (100, 200, 4, 2, 128, False, 300), (70, 50, 4, 1, 64, True, 1), (40, 300, 2, 1, 256, False, 1)])
def test_fp32(n, prefix, Hq, Hkv, D, tree, max_keys):
    announce("attention fp32 accuracy", n, prefix, Hq, Hkv, D, tree, max_keys)
    c = Case([n], [prefix], Hq, Hkv, D, 16, torch.float32, _random_tree if tree else None, seed=D + n)
    want = c.want()[0]
    got = c.run(max_keys=max_keys).cpu().double()
    rms = ((got - want).pow(2).mean() / want.pow(2).mean()).sqrt().item()
    assert rms <= 36 * 2.0 ** -24, rms * 2 ** 24
