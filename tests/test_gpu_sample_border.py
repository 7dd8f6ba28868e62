"""Where top-p's border lies in a long run of light logits: the mass that finds it is a sum of weights that are each rounded to a unit of 2^-44 (at
151 936 logits), so that what is kept may be off by half a unit for every logit of the row, V / 2 units in the sum and as much in the target."""
import numpy as np
import pytest
import torch

from mllm_amd import qlinear as ql
from gpu_util import announce

pytestmark = pytest.mark.gpu
VOCAB, PEAK, UNIT = 151936, 70000, 2.0 ** -44


def _light(units, part):
    """an fp32 logit below a peak of 0 whose weight is about `units` units and `part` of one more"""
    x = np.float32(np.log((units + part) * UNIT))
    near = [x]
    for way in (-np.inf, np.inf):
        y = x
        for _ in range(40):
            y = np.nextafter(y, np.float32(way))
            near.append(y)
    return min(near, key=lambda v: abs(np.exp(np.float64(v)) / UNIT % 1 - part))


@pytest.mark.parametrize("part", [0.45, 0.55, 0.0])
@pytest.mark.parametrize("share", [0.1, 0.5, 0.9])
def test_light_and_equal_behind_a_peak(part, share):
    announce("sample light tails", part, share)
    light = _light(2.0 ** 14, part)
    w = float(np.exp(np.float64(light)))
    x = torch.full((1, VOCAB), float(light), device="cuda")
    x[0, PEAK] = 0.0
    rest = (VOCAB - 1) * w
    p = np.float32((1 + share * rest) / (1 + rest))
    exact = int(np.ceil((float(p) * (1 + rest) - 1) / w))  # of the light ones, lowest index first
    off = int(VOCAB * UNIT / w) + 1
    for u in (1 - 2.0 ** -24, 1 - 2.0 ** -22, 1 - 2.0 ** -20, 0.0):
        got = ql.sample(x, torch.tensor([u], dtype=torch.float32, device="cuda"), top_p=torch.tensor([float(p)], device="cuda")).item()

        def token(light_ones):
            weights = np.full(VOCAB, w)
            weights[PEAK] = 1.0
            weights[light_ones + (light_ones > PEAK - 1):] = 0
            weights[PEAK] = 1.0
            up = np.cumsum(weights)
            return int(np.searchsorted(up, u * up[-1], "right"))
        assert token(exact - off) <= got <= token(exact + off), (u, got, token(exact))
