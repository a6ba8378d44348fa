"""torch.ops.qhtp.kv8_*: the fakes' strides are the ops' own, for q in any order of its axes."""
import pytest
import torch

import qcom_htp_b200 as qhtp
from tests.test_kv8_gpu import BF, i32, random_cache, random_table

pytestmark = pytest.mark.gpu


def queries(order, b=3, t=5, h=8, d=64):
    g = torch.Generator(device="cuda").manual_seed(4)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF)
    if order == "bhtd":
        return rand(b, h, t, d).transpose(1, 2)
    if order == "fused":
        return rand(b, t, (h + 4) * d)[..., :h * d].unflatten(-1, (h, d))
    return rand(b, t, h, d)


@pytest.mark.parametrize("order", ["bthd", "bhtd", "fused"])
def test_attention_agrees_with_its_fake(order):
    q, lengths = queries(order), [40, 5, 61]
    cache, table = random_cache(12, 2, 64, 16, 1), i32(random_table(lengths, 16, 12, 2))
    args = (q, *cache, table, i32(lengths))
    torch.library.opcheck(torch.ops.qhtp.kv8_attention.default, args, test_utils=("test_schema", "test_faketensor"))
    out, _ = torch.ops.qhtp.kv8_attention(*args)
    assert out.is_contiguous()
    assert torch.equal(out, qhtp.kv8_attention(q.contiguous(), cache, table, i32(lengths)))


def test_write_and_read_agree_with_their_fakes():
    cache, table = random_cache(12, 2, 64, 16, 1), i32(random_table([40, 5, 61], 16, 12, 2))
    k, v = queries("bhtd", h=2), queries("fused", h=2)
    utils = ("test_schema", "test_faketensor")
    torch.library.opcheck(torch.ops.qhtp.kv8_write.default, (*cache, k, v, table, i32([0, 0, 7])), test_utils=utils)
    torch.library.opcheck(torch.ops.qhtp.kv8_read.default, (*cache, table, i32([0, 0, 7]), 5), test_utils=utils)


def test_a_lone_token_whose_strides_mean_nothing():
    """Axes of extent 1 may have any stride, and q counts as contiguous with it; the output's are the usual ones all the same."""
    cache, table = random_cache(4, 2, 64, 16, 1), i32([[2, 0]])
    q = torch.randn(2048, device="cuda").to(BF).as_strided((1, 1, 8, 64), (1024, 768, 64, 1))
    assert q.is_contiguous()
    args = (q, *cache, table, i32([20]))
    torch.library.opcheck(torch.ops.qhtp.kv8_attention.default, args, test_utils=("test_schema", "test_faketensor"))
    assert torch.ops.qhtp.kv8_attention(*args)[0].stride() == (512, 512, 64, 1)
