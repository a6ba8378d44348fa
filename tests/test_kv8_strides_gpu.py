"""One sequence, one token, one head out of a projection of an odd width: its strides matter to nothing."""
import pytest
import torch

import qcom_htp_b200 as qhtp
from tests.test_kv8_gpu import BF, F32, i32, random_cache

pytestmark = pytest.mark.gpu


def odd(*shape, dtype=BF):
    """A view [1, tokens, heads, d] into rows of an odd number of elements."""
    t, h, d = shape
    base = torch.randn((3, t * h * d + 13), device="cuda").to(dtype)
    view = base.as_strided((1, t, h, d), (t * h * d + 13, h * d if t > 1 else 7, d if h > 1 else 3, 1))
    assert base.data_ptr() % 16 == 0
    return view


@pytest.mark.parametrize("t,hq,hkv", [(1, 8, 2), (5, 8, 2), (1, 1, 1), (200, 4, 1)])
def test_a_lone_sequence(t, hq, hkv):
    n = 300
    cache, other = (random_cache(20, hkv, 64, 16, 1) for _ in range(2))
    table, past = i32([list(range(20))]), i32([n - t])
    k, v, q, out = odd(t, hkv, 64), odd(t, hkv, 64), odd(t, hq, 64), odd(t, hq, 64)
    qhtp.kv8_write(cache, k, v, table, past)
    qhtp.kv8_write(other, k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format), table, past)
    assert all(torch.equal(a, b) for a, b in zip(cache, other))
    want = qhtp.kv8_attention(q.clone(memory_format=torch.contiguous_format), cache, table, i32([n]))
    assert torch.equal(qhtp.kv8_attention(q, cache, table, i32([n]), out=out), want)
    assert torch.equal(out, want)


def test_one_packed_row_in_float32():
    cache, other = (random_cache(2, 1, 64, 16, 1) for _ in range(2))
    k = odd(1, 1, 64, dtype=F32)[0]
    args = i32([[1]]), i32([3])
    qhtp.kv8_write(cache, k, k, *args, seq_start=i32([0, 1]))
    qhtp.kv8_write(other, k.clone(memory_format=torch.contiguous_format), k.clone(memory_format=torch.contiguous_format), *args, seq_start=i32([0, 1]))
    assert all(torch.equal(a, b) for a, b in zip(cache, other))
