"""torch.ops.qhtp.kv8_*: registered, with shapes and types from their fake implementations."""
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import qcom_htp_b200  # noqa: F401  (registers the ops)


def test_fake_shapes():
    with FakeTensorMode():
        i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")
        bf = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")
        code = lambda: torch.empty((9, 2, 16, 64), dtype=torch.int8, device="cuda")
        scale = lambda: torch.empty((9, 2), device="cuda")
        cache = (code(), code(), scale(), scale())
        assert torch.ops.qhtp.kv8_write(*cache, bf(3, 5, 2, 64), bf(3, 5, 2, 64), i32(3, 4), i32(3)) is None
        k, v = torch.ops.qhtp.kv8_read(*cache, i32(3, 4), i32(3), 7)
        assert k.shape == v.shape == (3, 7, 2, 64) and k.dtype == v.dtype == torch.bfloat16
        k, v = torch.ops.qhtp.kv8_read(*cache, i32(3, 4), i32(3), None, i32(4), 11, None, torch.float32)
        assert k.shape == v.shape == (11, 2, 64) and k.dtype == torch.float32
        out, lse = torch.ops.qhtp.kv8_attention(bf(3, 5, 8, 64), *cache, i32(3, 4), i32(3))
        assert out.shape == (3, 5, 8, 64) and out.dtype == torch.bfloat16
        assert lse.shape == (3, 5, 8) and lse.dtype == torch.float32
        out, lse = torch.ops.qhtp.kv8_attention(bf(6, 8, 64), *cache, i32(3, 4), i32(3), None, True, 5, i32(4), 3, 64)
        assert out.shape == (6, 8, 64) and lse.shape == (6, 8)


def test_write_names_what_it_changes():
    schema = torch.ops.qhtp.kv8_write.default._schema
    changed = [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write]
    assert changed == ["cache_k", "cache_v", "k_scale", "v_scale"]
