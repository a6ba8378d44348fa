"""What kv8.py refuses it refuses with a ValueError that says why, without a GPU."""
import pytest
import torch

from qcom_htp_b200 import kv8
from tests.test_kv8_device_cpu import CACHE, COUNT, DEV, Rows, TABLE, library  # noqa: F401  (library is a fixture)

def test_refusals_are_value_errors(library):  # noqa: F811
    q, one = Rows(3, 1, 4, 64), Rows(3, 1, 2, 64)
    start = Rows(4, dtype=torch.int32)
    attend = lambda q=q, cache=CACHE, **kw: kv8.kv8_attention(q, cache, TABLE, COUNT, out=Rows(3, 1, 4, 64), **kw)
    attend()
    no_heads = (Rows(8, 0, 16, 64, dtype=torch.int8),) * 2 + (Rows(8, 0, dtype=torch.float32),) * 2
    no_blocks = (Rows(0, 2, 16, 64, dtype=torch.int8),) * 2 + (Rows(0, 2, dtype=torch.float32),) * 2
    for cache in (no_heads, no_blocks):
        for call in (lambda: attend(cache=cache), lambda: kv8.kv8_write(cache, one, one, TABLE, COUNT),
                     lambda: kv8.kv8_read(cache, TABLE, COUNT, 3)):
            with pytest.raises(ValueError):
                call()
    for kw in (dict(window=(1 << 30) + 1), dict(window=1 << 40), dict(window=-1)):
        with pytest.raises(ValueError):
            attend(**kw)
    for bad in (Rows(64), Rows()):
        with pytest.raises(ValueError):
            kv8.kv8_attention(bad, CACHE, TABLE, COUNT, seq_start=start)
        with pytest.raises(ValueError):
            kv8.kv8_attention(bad, CACHE, TABLE, COUNT)
        with pytest.raises(ValueError):
            kv8.kv8_write(CACHE, bad, bad, TABLE, COUNT, seq_start=start)
    with pytest.raises(ValueError):
        kv8.kv8_read(CACHE, TABLE, COUNT, -1)
    with pytest.raises(ValueError):
        kv8.kv8_read(CACHE, Rows(3, dtype=torch.int32), COUNT, 3)
    with pytest.raises(ValueError):
        kv8.kv8_read(CACHE, Rows(dtype=torch.int32), COUNT, 3)


def test_a_bound_below_zero_is_zero(library, monkeypatch):  # noqa: F811
    """max_new and max_tokens are bounds of counts; both entries take one below zero alike."""
    start = Rows(4, dtype=torch.int32)
    monkeypatch.setattr(kv8, "_empty", lambda like, shape, dtype, stream: Rows(*shape, dtype=dtype))
    monkeypatch.setattr(kv8, "_like", lambda t, stream: Rows(*t.shape, dtype=t.dtype))
    kv8.kv8_write(CACHE, Rows(9, 2, 64), Rows(9, 2, 64), TABLE, COUNT, seq_start=start, max_new=-1)
    kv8.kv8_read(CACHE, TABLE, COUNT, seq_start=start, total=9, max_tokens=-1)
    assert library.calls == [("write", DEV.index)] * 2
