"""The heads' norm where the mean square is below the smallest normal fp32 number: 1 / sqrt is still a number there.

Bounds of test_gpu_rope_append.py, and the squares', which are multiples of 2^-149 here: each of a head's is off by half of that, and the mean of them
and its rounding by 2^-149 together, half of which (relative to the mean) is the root's."""
import pytest
import torch

from mllm_amd import qlinear as ql
from decode_ref import norm_rope
from gpu_util import announce

pytestmark = pytest.mark.gpu


def _check(got, x, want, size):
    mean = x.cpu().double().pow(2).mean(-1, keepdim=True)
    bound = (24 * 2.0 ** -24 + 2.0 ** -150 / mean) * size + (2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else 0.0)
    assert torch.isfinite(got).all()
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("exponent", [-60, -62, -63, -64, -66, -68])
@pytest.mark.parametrize("D", [64, 80, 128, 256, 512])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_heads(exponent, D, dtype):
    announce("qk_norm_rope of small heads", exponent, D, dtype)
    gen = torch.Generator(device="cuda").manual_seed(D)
    x = (torch.randn((6, 3, D), device="cuda", generator=gen) * 2.0 ** exponent).to(dtype)
    w = 1 + 0.3 * torch.randn(D, device="cuda", generator=gen)
    pos = torch.arange(6, device="cuda").int()
    f = 1e4 ** (-torch.arange(0, 16, dtype=torch.float64, device="cuda") / 16)
    want, size = norm_rope(x, w, 0.0, pos, f, False)
    q, k = ql.qk_norm_rope(x, x[:, :1], pos, f, w, w, eps=0.0)
    _check(q, x, want, size)
    _check(k, x[:, :1], want[:, :1], size[:, :1])
    k_cache, v_cache = [torch.zeros((2, 4, 3, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ql.kv_append(x, x, k_cache, v_cache, torch.arange(6, device="cuda"), pos, f, w, eps=0.0)
    _check(k_cache.view(8, 3, D)[:6], x, want, size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zeros_with_a_subnormal_epsilon(dtype):
    announce("qk_norm_rope of zeros, epsilon 1e-40", dtype)
    x, w = torch.zeros((2, 2, 128), dtype=dtype, device="cuda"), torch.ones(128, device="cuda")
    for y in ql.qk_norm_rope(x, x, None, None, w, w, eps=1e-40):
        assert not y.any()
