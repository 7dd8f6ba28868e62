"""The scales that the attention over a paged cache refuses, without a GPU: made-up addresses that a refused call never reads."""
import ctypes as C

import pytest

from mllm_amd import _lib

P = 0x7F0000100000


@pytest.mark.parametrize("scale", [2.3e38, 3e38, 3.4e38, float("inf"), float("nan"), 0.0, -0.0, -1.0])
def test_scales(scale):
    """(times log2 e, as the kernel takes it, 2.4e38 is infinite)"""
    q = _lib.Heads(P, P + (1 << 20), None, 512, 128, 512, 128, 4)
    cache = _lib.KVCache(P, P, 16 * 512, 512, 128, 8, 16, 4, 128)
    assert _lib.lib().mllm_hip_attention_paged(C.byref(q), 0, 1, C.byref(cache), P, 4, 4, P, P, 1, 1, 1, None, 0, 0, scale, None, 0, None) == -1
