"""The attention workspace of packed sequences is sized by the rows that there are, not by the most rows of a sequence times
the sequences: max_new may be left at its default, all of the rows."""
import ctypes as C

import pytest

from qcom_htp_b200 import _lib as L
from tests.test_kv8_cpu import attention, cache, rows, seqs

CASES = [  # sequences, rows in all, hq, hkv, head_dim
    (8, 1400, 32, 8, 128), (16, 2400, 8, 1, 256), (64, 8192, 4, 1, 64), (300, 3000, 12, 4, 128),
]


def call(batch, total, hq, hkv, d, most, packed=True, context=8192):
    s = seqs(batch=batch, tokens=most, max_blocks=context // 64, table_stride=context // 64, seq_start=16 if packed else 0,
             total=total if packed else 0)
    return attention(cache=cache(num_blocks=batch * context // 64, kv_heads=hkv, head_dim=d), seqs=s, q=rows(), out=rows(), q_heads=hq,
                     max_len=context)


@pytest.mark.parametrize("batch,total,hq,hkv,d", CASES)
@pytest.mark.parametrize("spread", [1, 2, 7, None])
def test_packed_rows_take_what_the_rows_need(batch, total, hq, hkv, d, spread):
    """Two chunks at most of each (row, kv head): head_dim values, a maximum and a sum in float32, in tiles of 256 rows at most
    of which every sequence may leave two in part empty."""
    most = total if spread is None else min(total, spread * -(-total // batch))
    need = L.lib.qhtp_kv8_attention_workspace_bytes(C.byref(call(batch, total, hq, hkv, d, most)))
    assert need <= 2 * (total * hq // hkv + 2 * 256 * batch) * hkv * (d + 2) * 4


def test_some_of_these_have_a_workspace():
    sizes = [L.lib.qhtp_kv8_attention_workspace_bytes(C.byref(call(*c, c[1]))) for c in CASES]
    assert sum(n > 0 for n in sizes) >= 2


@pytest.mark.parametrize("total", [1 << 31, 1 << 40, (1 << 63) - 1])
def test_a_total_that_no_start_can_reach(total):
    """Starts are 32-bit: a larger total is no reason for a larger workspace, and nothing overflows."""
    c = (8, total, 32, 8, 128, 700)
    need = L.lib.qhtp_kv8_attention_workspace_bytes(C.byref(call(*c)))
    assert need <= 8 * 8 * (700 * 4 // 256 + 1) * 2 * 256 * 130 * 4  # two chunks of every sequence's row groups


def test_the_size_looks_at_numbers_and_seq_start_only():
    """No pointer but seq_start matters to the size; seq_start does (packed rows are cut by their total), and so does whether the call
    would be refused."""
    def size(**kw):
        run = call(8, 1400, 32, 8, 128, 1400)
        for name, value in kw.items():
            *path, last = name.split("__")
            at = run
            for p in path:
                at = getattr(at, p)
            setattr(at, last, value)
        return L.lib.qhtp_kv8_attention_workspace_bytes(C.byref(run))

    full = size()
    assert full > 0
    for name in ("cache__k", "cache__v", "cache__k_scale", "cache__v_scale", "seqs__block_table", "lengths", "q__data", "out__data", "stream"):
        assert size(**{name: None}) == full
    assert size(seqs__seq_start=None) != full
    for bad in (dict(scale=0.0), dict(dtype=2), dict(q_heads=31), dict(causal=0, window=5)):
        assert size(**bad) == 0
