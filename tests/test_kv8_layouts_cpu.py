"""The fake of torch.ops.qhtp.kv8_attention gives its outputs the strides that the op gives them: contiguous, whatever
the order of q's axes in memory."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import qcom_htp_b200  # noqa: F401  (registers the ops)


@pytest.mark.parametrize("order", ["bthd", "bhtd", "fused", "ragged_hnd"])
def test_fake_outputs_are_contiguous(order):
    with FakeTensorMode():
        i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")
        bf = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")
        code, scale = torch.empty((9, 2, 16, 64), dtype=torch.int8, device="cuda"), torch.empty((9, 2), device="cuda")
        start = None
        if order == "bthd":
            q = bf(3, 5, 8, 64)
        elif order == "bhtd":
            q = bf(3, 8, 5, 64).transpose(1, 2)
        elif order == "fused":
            q = bf(3, 5, 12 * 64)[..., :8 * 64].unflatten(-1, (8, 64))
        else:
            q, start = bf(8, 15, 64).transpose(0, 1), i32(4)
        out, lse = torch.ops.qhtp.kv8_attention(q, code, code, scale, scale, i32(3, 4), i32(3), seq_start=start)
        assert out.shape == q.shape and lse.shape == q.shape[:-1]
        assert out.is_contiguous() and out.stride() == torch.empty(q.shape, device="meta").stride()
        assert lse.is_contiguous()
