"""The 8-bit KV cache's host side without a GPU: the packed arguments match the C structures, and the C entry
points refuse what they cannot run before they touch a device."""
import ctypes as C

import pytest
import torch

import qcom_htp_b200 as qhtp
from qcom_htp_b200 import _lib as L
from qcom_htp_b200 import kv8
from tests.kv8_helpers import HostCache


def flat(s, prefix=""):
    for name, kind in s._fields_:
        v = getattr(s, name)
        if isinstance(v, C.Structure):
            yield from flat(v, prefix + name + ".")
        else:
            yield prefix + name, v


@pytest.mark.parametrize("pack,kind,f32", [(kv8._MOVE, L.QhtpKv8Move, None), (kv8._ATTENTION, L.QhtpKv8Attention, "scale")])
def test_packed_arguments_match_the_structures(pack, kind, f32):
    assert pack.size == C.sizeof(kind)
    names = [n for n, _ in flat(kind())]
    values = [i + 1 for i in range(len(names))]
    got = dict(flat(kind.from_buffer_copy(pack.pack(*values))))
    for n, v in zip(names, values):
        assert got[n] == v, n


def cache(**kw):
    d = dict(k=16, v=16, k_scale=16, v_scale=16, num_blocks=8, kv_heads=2, head_dim=128, block_size=64)
    d.update(kw)
    return L.QhtpKv8Cache(**d)


def seqs(**kw):
    d = dict(block_table=16, table_stride=4, max_blocks=4, batch=3, tokens=2)
    d.update(kw)
    return L.QhtpKv8Seqs(**d)


def rows(**kw):
    d = dict(data=16, batch_stride=1024, token_stride=512, head_stride=128)
    d.update(kw)
    return L.QhtpKv8Rows(**d)


def move(**kw):
    d = dict(cache=cache(), seqs=seqs(), first=16, k=rows(), v=rows(), dtype=0)
    d.update(kw)
    return L.QhtpKv8Move(**d)


def attention(**kw):
    d = dict(cache=cache(), seqs=seqs(), lengths=16, q=rows(), out=rows(), q_heads=8, causal=1, scale=0.1, max_len=256)
    d.update(kw)
    return L.QhtpKv8Attention(**d)


SHAPES = [(dict(cache=cache(num_blocks=0)), L.INVALID_ARGUMENT), (dict(cache=cache(kv_heads=0)), L.INVALID_ARGUMENT),
          (dict(cache=cache(head_dim=96)), L.UNSUPPORTED), (dict(cache=cache(block_size=48)), L.UNSUPPORTED),
          (dict(cache=cache(block_size=8)), L.UNSUPPORTED), (dict(seqs=seqs(batch=65536)), L.UNSUPPORTED),
          (dict(cache=cache(num_blocks=1 << 30)), L.UNSUPPORTED), (dict(seqs=seqs(total=-1)), L.INVALID_ARGUMENT), (dict(seqs=seqs(max_blocks=1 << 28)), L.UNSUPPORTED),
          (dict(cache=cache(k=0)), L.INVALID_ARGUMENT), (dict(cache=cache(v_scale=0)), L.INVALID_ARGUMENT),
          (dict(cache=cache(v=8)), L.INVALID_ARGUMENT), (dict(seqs=seqs(block_table=0)), L.INVALID_ARGUMENT)]


@pytest.mark.parametrize("kw,status", SHAPES + [(dict(first=0), L.INVALID_ARGUMENT), (dict(dtype=3), L.UNSUPPORTED),
                                                (dict(k=rows(data=0)), L.INVALID_ARGUMENT), (dict(v=rows(data=8)), L.INVALID_ARGUMENT),
                                                (dict(v=rows(token_stride=4)), L.INVALID_ARGUMENT),
                                                (dict(k=rows(head_stride=-4)), L.INVALID_ARGUMENT)])
def test_move_refusals(kw, status):
    for fn in (L.lib.qhtp_kv8_write, L.lib.qhtp_kv8_read):
        assert fn(C.byref(move(**kw))) == status
        assert fn(None) == L.INVALID_ARGUMENT


@pytest.mark.parametrize("kw,status", SHAPES + [(dict(lengths=0), L.INVALID_ARGUMENT), (dict(dtype=2), L.UNSUPPORTED),
                                                (dict(q_heads=0), L.INVALID_ARGUMENT), (dict(q_heads=3), L.INVALID_ARGUMENT),
                                                (dict(scale=0.0), L.INVALID_ARGUMENT), (dict(scale=float("nan")), L.INVALID_ARGUMENT),
                                                (dict(window=4, causal=0), L.UNSUPPORTED), (dict(q=rows(data=8)), L.INVALID_ARGUMENT),
                                                (dict(out=rows(head_stride=4)), L.INVALID_ARGUMENT)])
def test_attention_refusals(kw, status):
    assert L.lib.qhtp_kv8_attention(C.byref(attention(**kw))) == status
    assert L.lib.qhtp_kv8_attention(None) == L.INVALID_ARGUMENT


def test_workspace_is_required():
    long = dict(cache=cache(num_blocks=10000), seqs=seqs(max_blocks=2000, batch=1, tokens=1), max_len=128000)
    need = L.lib.qhtp_kv8_attention_workspace_bytes(C.byref(attention(**long)))
    assert need > 0
    for ws in (dict(), dict(workspace=256, workspace_bytes=need - 1), dict(workspace=272, workspace_bytes=need)):
        assert L.lib.qhtp_kv8_attention(C.byref(attention(**long, **ws))) == L.INVALID_ARGUMENT
    assert b"workspace" in L.lib.qhtp_last_error_string()


def test_nothing_to_do_needs_no_device():
    for s in (seqs(batch=0), seqs(tokens=0), seqs(seq_start=16, total=0)):
        assert L.lib.qhtp_kv8_write(C.byref(move(seqs=s))) == L.OK
        assert L.lib.qhtp_kv8_read(C.byref(move(seqs=s))) == L.OK
        assert L.lib.qhtp_kv8_attention(C.byref(attention(seqs=s))) == L.OK


def test_python_refuses_a_host_cache():
    c = qhtp.Kv8Cache.empty(2, 1, 64, 16, device="cpu")
    t = torch.zeros((1, 2), dtype=torch.int32)
    r = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        qhtp.kv8_write(c, r, r, t, t[0, :1])
    with pytest.raises(ValueError):
        qhtp.kv8_attention(r, c, t, t[0, :1])
    for kw in (dict(head_dim=96), dict(block_size=24), dict(num_blocks=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            qhtp.Kv8Cache.empty(**{**dict(num_blocks=1, kv_heads=1, head_dim=64, block_size=16, device="cpu"), **kw})


def test_the_rule_keeps_values_within_half_a_step():
    """The write rule itself: values come back within half a step of the tile's scale (one and a half after growth)."""
    import numpy as np
    rng = np.random.default_rng(0)
    z = lambda *s: np.zeros(s, np.int8)
    c = HostCache(z(2, 1, 16, 64), z(2, 1, 16, 64), np.zeros((2, 1), np.float32), np.zeros((2, 1), np.float32))
    x = rng.standard_normal((20, 1, 64)).astype(np.float32)
    c.write((x[:10], x[:10]), [[1, 0]], 0, 0)
    c.write((10 * x[10:], 10 * x[10:]), [[1, 0]], 10, 0)
    k, _ = c.rows([[1, 0]], 0, 0, 20)
    step = c.scale[0]
    assert np.abs(k[:10] - x[:10]).max() <= 1.01 * step[1, 0]
    assert np.abs(k[10:16] - 10 * x[10:16]).max() <= 0.501 * step[1, 0]
    assert np.abs(k[16:] - 10 * x[16:]).max() <= 0.501 * step[0, 0]
