"""Rows written behind a tile whose scale is below 2^-64: such a scale counts as zero, as a new one of that size does."""
import numpy as np
import pytest
import torch

import qcom_htp_b200 as qhtp
from tests.test_kv8_gpu import F32, host, i32, random_cache, same

pytestmark = pytest.mark.gpu

MIN = 2.0 ** -64


@pytest.mark.parametrize("old", [2.0 ** -65, 2.0 ** -100, 1e-40, 0.0])
@pytest.mark.parametrize("size", [0.0, 1e-30, 126 * MIN])
def test_tiny_rows_behind_a_tiny_scale(old, size):
    """Neither reaches 2^-64: the tile's scale is 0, the new codes are 0, nothing else changes."""
    cache = random_cache(3, 2, 64, 16, 1)
    cache.k_scale[1], cache.v_scale[1] = old, old
    want = host(cache)
    x = torch.linspace(-1, 1, 5 * 2 * 64, device="cuda").reshape(5, 2, 64) * size
    for dtype in (F32, torch.bfloat16):
        qhtp.kv8_write(cache, x.to(dtype), -x.to(dtype), i32([[1]]), i32([7]), seq_start=i32([0, 5]))
        got = host(cache)
        for w in range(2):
            want.scale[w][1] = 0
            want.code[w][1, :, 7:12] = 0
            same(got.scale[w], want.scale[w])
            same(got.code[w], want.code[w])
    k, v = qhtp.kv8_read(cache, i32([[1]]), i32([0]), 12, dtype=F32)
    assert (k == 0).all() and (v == 0).all()


@pytest.mark.parametrize("old", [2.0 ** -65, 1e-40])
def test_rows_behind_a_tiny_scale(old):
    """Rows of ordinary size give the tile their scale; what it held is zero in it."""
    cache = random_cache(2, 1, 128, 32, 2)
    cache.k_scale[0], cache.v_scale[0] = old, old
    x = torch.randn((3, 1, 128), device="cuda")
    qhtp.kv8_write(cache, x, x, i32([[0]]), i32([20]), seq_start=i32([0, 3]))
    for scale, code in ((cache.k_scale, cache.k), (cache.v_scale, cache.v)):
        s = np.float32(float(x.abs().max())) / np.float32(127)
        assert float(scale[0, 0]) == s
        assert (code[0, 0, :20] == 0).all()
        inv = np.float32(1) / s
        same(code[0, 0, 20:23].cpu().numpy(), np.rint(x[:, 0].cpu().numpy() * inv).astype(np.int8))


def test_the_smallest_scale_that_counts():
    """2^-64 itself is a scale like any other: a tile that has it keeps it, and codes are those of the rule."""
    cache = random_cache(1, 1, 64, 16, 3)
    cache.k_scale[0], cache.v_scale[0] = MIN, MIN
    before = cache.k[0, 0, :4].clone()
    x = (torch.arange(64, device="cuda").float() * 2 - 63).reshape(1, 1, 64) * MIN
    qhtp.kv8_write(cache, x, x, i32([[0]]), i32([4]), seq_start=i32([0, 1]))
    assert float(cache.k_scale[0, 0]) == MIN and torch.equal(cache.k[0, 0, :4], before)
    same(cache.k[0, 0, 4].cpu().numpy(), np.arange(64) * 2 - 63)
