"""The 8-bit KV cache as it is used: through torch.ops, in the example's serving loop, and in batches whose
lengths decide how the keys are cut."""
import importlib.util
from pathlib import Path

import pytest
import torch

import qcom_htp_b200 as qhtp
from tests.test_kv8_gpu import BF, HF, attend, i32, random_cache, random_table

pytestmark = pytest.mark.gpu


def test_ops_match_the_functions():
    g = torch.Generator(device="cuda").manual_seed(5)
    cache, other = (qhtp.Kv8Cache.empty(20, 2, 64, 16) for _ in range(2))
    table, past, lengths = i32(random_table([100, 130], 16, 20, 3)), i32([0, 0]), i32([100, 100])
    k, v = (torch.randn((2, 100, 2, 64), generator=g, device="cuda").to(BF) for _ in range(2))
    torch.ops.qhtp.kv8_write(*cache, k, v, table, past)
    qhtp.kv8_write(other, k, v, table, past)
    assert all(torch.equal(a, b) for a, b in zip(cache, other))
    for a, b in zip(torch.ops.qhtp.kv8_read(*cache, table, past, 100), qhtp.kv8_read(cache, table, past, 100)):
        assert torch.equal(a, b)
    q = torch.randn((2, 100, 4, 64), generator=g, device="cuda").to(BF)
    for a, b in zip(torch.ops.qhtp.kv8_attention(q, *cache, table, lengths), qhtp.kv8_attention(q, cache, table, lengths, return_lse=True)):
        assert torch.equal(a, b)
    with pytest.raises(ValueError):
        torch.ops.qhtp.kv8_attention(q, *cache, table, lengths, window=-1)


def test_example():
    """The relative step of a code is at most 1/127 of its tile's largest value, so rounding is off by half of that and, evenly
    spread, by 1/sqrt(3) of the half; the largest of a tile's 1024 to 8192 normal values is 3 to 5 times their root mean
    square.  A tile that goes on is rounded again each time its scale grows, a few times: 0.05 bounds it all for K, and
    for outputs that are averages of V, with scores off by as little."""
    path = Path(__file__).resolve().parents[1] / "examples" / "kv8_decode.py"
    spec = importlib.util.spec_from_file_location("kv8_decode", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    r = m.run(batch=3, hidden=512, q_heads=8, kv_heads=2, head_dim=128, prompt=200, steps=20, block_size=32)
    assert 0 < r["export_error"] < 0.05
    assert 0 < r["attention_error"] < 0.05
    assert torch.isfinite(r["out"]).all()


# Lengths cut on the device: more sequences than a warp has lanes, one long among short ones, idle ones, all alike.
CUTS = [
    [1200] * 40,
    [20000] + [1] * 45,
    [0, 900, 0, 5000, 17, 0] * 9,
    [3000, 2999, 1, 0, 4096, 130] * 5 + [9000, 8000, 7],
    [1000],
]


@pytest.mark.parametrize("lengths", CUTS, ids=lambda x: f"{len(x)}_of_{max(x)}")
@pytest.mark.parametrize("hq,hkv,d,t,dtype", [(4, 2, 64, 1, BF), (8, 1, 128, 1, HF), (8, 1, 128, 5, BF), (6, 1, 256, 2, BF)])
def test_cut_by_the_lengths(lengths, hq, hkv, d, t, dtype):
    attend(lengths, [t] * len(lengths), hq, hkv, d, 32, dtype, seed=len(lengths))


@pytest.mark.parametrize("window", [0, 1500])
def test_cut_by_the_lengths_ragged(window):
    """Sequences of unlike numbers of query rows, some of none, one of several row groups."""
    news = [5, 0, 300, 1, 17, 40, 0, 9]
    lengths = [5000, 100, 2500, 1, 6000, 3000, 0, 2000]
    attend(lengths, news, 8, 1, 128, 64, BF, window=window, ragged=True, seed=3)
    attend(lengths, news, 8, 1, 256, 64, HF, window=window, ragged=True, seed=4)
    attend(lengths, news, 16, 2, 64, 16, BF, causal=window == 0, window=0, ragged=True, seed=5)


def test_cut_in_two():
    """Between one wave of row groups and one and a half, over 4096 keys and more: two chunks of half the keys."""
    attend([5000] * 5, [256] * 5, 32, 8, 128, 64, BF, seed=1)
    attend([4500, 300, 4200], [1000, 64, 1000], 24, 8, 64, 32, HF, window=4100, ragged=True, seed=2)


def test_bad_starts_give_no_rows():
    """Row ranges outside the rows, or that run backwards, are empty, also where the keys are cut by the lengths."""
    lengths = [2000, 1500, 1800]
    cache = random_cache(100, 2, 128, 64, 1)
    table, n = i32(random_table(lengths, 64, 100, 2)), i32(lengths)
    q = torch.randn((6, 8, 128), device="cuda").to(BF)
    out = torch.full_like(q, 7.0)
    qhtp.kv8_attention(q, cache, table, n, seq_start=i32([0, 2, 99, -5]), max_new=6, out=out)
    want = qhtp.kv8_attention(q[:2], cache, table[:1], n[:1], seq_start=i32([0, 2]))
    assert (out[2:] == 7.0).all()
    # two cuts of the same keys: each within a few roundings of the other
    assert (out[:2].float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
