"""Packed sequences of unlike numbers of rows whose keys are cut in two chunks: each sequence's parts lie behind those of
the sequences before it, wherever its rows begin."""
import numpy as np
import pytest
import torch

import qcom_htp_b200 as qhtp
from tests.kv8_helpers import attention64, bounds
from tests.test_kv8_gpu import BF, host, i32, random_cache, random_table

pytestmark = pytest.mark.gpu


def check(lengths, news, hq, hkv, d, bs, max_new, window=0, seed=0):
    blocks = sum(-(-n // bs) for n in lengths)
    cache, table = random_cache(blocks, hkv, d, bs, seed + 1), random_table(lengths, bs, blocks, seed + 2)
    start = np.cumsum([0] + news)
    q = torch.randn((int(start[-1]), hq, d), device="cuda").to(BF)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out, lse = qhtp.kv8_attention(q, cache, i32(table), i32(lengths), seq_start=i32(start), max_new=max_new, window=window,
                                  return_lse=True)
    torch.cuda.synchronize()
    used = torch.cuda.max_memory_allocated() - before
    h = host(cache)
    for b, (n, t) in enumerate(zip(lengths, news)):
        if t == 0:
            continue
        k, v = (torch.from_numpy(x).cuda().double() for x in h.rows(table, b, 0, n))
        rows = slice(start[b], start[b + 1])
        want, wl, absum, mag = attention64(q[rows].double(), k, v, n, d ** -0.5, True, window)
        (least, most), tol = bounds(want, absum, mag, n, d, float(cache.v_scale[table[b][table[b] >= 0]].max()), BF)
        assert ((out[rows] >= least) & (out[rows] <= most)).all(), b
        seen = ~torch.isinf(wl)
        assert ((lse[rows].double() - wl).abs()[seen] <= tol[seen]).all(), b
        # and, tighter than the worst case, the whole sequence's root mean square (2^-8: bf16, and f16 probabilities)
        assert (out[rows].double() - want).square().mean().sqrt() <= 2.0 ** -8 * want.square().mean().sqrt(), b
    return used


NEWS = [700, 1, 0, 300, 128, 129, 100, 42]


@pytest.mark.parametrize("stated", [False, True])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 128, 64), (32, 8, 64, 16), (8, 1, 256, 32)])
def test_rows_in_two_chunks(hq, hkv, d, bs, stated):
    news = NEWS if d < 256 else NEWS + [900, 3, 0, 0, 1, 65, 17, 14]
    lengths = [4700, 900, 4096, 5000, 128, 3000, 2111, 4200] if d < 256 else [4700, 900, 4096, 5000, 128, 3000, 2111, 4200] * 2
    used = check(lengths, news, hq, hkv, d, bs, max(news) if stated else None)
    # two chunks of the rows, each sequence's last tile in part empty, beside out, lse and small tensors
    rows = sum(news) * hq // hkv + 2 * 256 * len(news)
    assert used <= 2 * rows * hkv * (d + 2) * 4 + sum(news) * hq * (2 * d + 4) + (8 << 20)


def test_with_a_window():
    check([9000, 4100, 6000, 500, 7000], [500, 1, 300, 37, 562], 32, 8, 64, 32, None, window=4100, seed=3)


def test_single_tokens_packed():
    """Few rows over many sequences, on the plan's grid: 70 sequences of one to three tokens."""
    news = [1 + i % 3 for i in range(70)]
    check([2100 + 37 * i for i in range(70)], news, 16, 8, 128, 32, 3, seed=4)
