"""Attention of few rows where a block of threads takes more keys than its table of block constants holds (a segment: 255
blocks): long chunks, for every block size, against a float64 evaluation on the same codes.

Two bounds.  The lse's is the worst case of tests.kv8_helpers.bounds.  The output's is on the root mean square of a row's
error, since the worst case of a sum over thousands of keys is larger than the output itself.  With w_j the share that
key j's value has of an output element, and d_j the relative errors of the probabilities, the error is sum w_j d_j.  The d_j
of different keys come from roundings of different numbers: at most 2^-11 (f16) + 2 ds (scores and exponent), with no
common sign, so the sum's root mean square is at most that times sqrt(sum w_j^2); 4 times it is allowed, and the float32
sums' (n / 64 + 80) 2^-23 beside it.  Probabilities below f16's normal range are off by at most 2^-25 of a largest of 1, again
with no common sign.  The output's own rounding is half a unit of its last place.

Sixteen keys too many or too few of n change the output by sqrt(16 / n) of itself, 4 % at 9000 keys, and the lse by 16 / n.
"""
import math

import pytest
import torch

import qcom_htp_b200 as qhtp
from tests.test_kv8_gpu import BF, HF, i32, random_cache, random_table

pytestmark = pytest.mark.gpu


def check(lengths, hq, hkv, d, bs, dtype, t=1, window=0, max_len=None, seed=0):
    blocks = sum(-(-n // bs) for n in lengths) + 1
    cache = random_cache(blocks, hkv, d, bs, seed + 1)
    table = i32(random_table(lengths, bs, blocks, seed + 2))
    g = torch.Generator(device="cuda").manual_seed(seed + 3)
    q = torch.randn((len(lengths), t, hq, d), generator=g, device="cuda").to(dtype)
    out, lse = qhtp.kv8_attention(q, cache, table, i32(lengths), window=window, max_len=max_len, return_lse=True)
    group, scale, unit = hq // hkv, d ** -0.5, 2.0 ** (-9 if dtype is BF else -12)
    for b, n in enumerate(lengths):
        ids = table[b, :-(-n // bs)].long()
        pos = torch.arange(n - t, n, device="cuda")[:, None, None]
        at = torch.arange(n, device="cuda")
        see = (at <= pos) & ((at > pos - window) if window else True)  # [t, 1, n]
        for h in range(hkv):
            k, v = ((code[ids, h].double() * s[ids, h].double()[:, None, None]).reshape(-1, d)[:n]
                    for code, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            x = q[b, :, h * group:(h + 1) * group].double()
            s = (x @ k.T * scale).masked_fill(~see, -math.inf)
            mag = (x.abs() @ k.abs().T * scale).masked_fill(~see, 0.0).amax(-1)
            want_lse = torch.logsumexp(s, -1)
            p = torch.softmax(s, -1)
            want = p @ v
            ds = (mag * d + 16.0) * 2.0 ** -23 + 2.0 ** -20
            sums = (n / 64 + 80) * 2.0 ** -23
            share = torch.sqrt((p.square() @ v.square()).mean(-1))   # root mean square over d of sqrt(sum w_j^2)
            small = p.amax(-1) * torch.sqrt((see.double() @ v.square()).mean(-1))
            tol = 4 * ((2.0 ** -11 + 2 * ds + sums) * share + 2.0 ** -25 * small) + unit * want.square().mean(-1).sqrt()
            got = out[b, :, h * group:(h + 1) * group].double()
            error = (got - want).square().mean(-1).sqrt()
            assert (error <= tol).all(), (b, h, float((error / want.square().mean(-1).sqrt()).max()))
            off = (lse[b, :, h * group:(h + 1) * group].double() - want_lse).abs()
            assert (off <= ds + sums + 2.0 ** -18).all(), (b, h, float(off.max()))


@pytest.mark.parametrize("bs,length", [(16, 9000), (32, 17000), (64, 33000), (128, 70000)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (32, 2, 64), (48, 2, 64), (8, 2, 128), (12, 1, 128), (20, 1, 128), (4, 1, 256),
                                      (12, 1, 256)])
def test_several_segments(bs, length, hq, hkv, d):
    """One sequence whole in one chunk (max_len is far too small): two segments and the start of a third."""
    check([length], hq, hkv, d, bs, BF, max_len=1, seed=bs)


@pytest.mark.parametrize("window", [0, 9001])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_segments_that_start_inside_a_block(d, window):
    """With a window the first key is no block's first, and drafted tokens begin at unlike keys."""
    for bs in (16, 64):
        check([20011, 12345], 8, 2, d, bs, HF, t=3, window=window, max_len=1, seed=bs)


LONG = [  # sequences, keys, hq, hkv, d: chunks of more than 4080 keys that the plan makes by itself
    (2, 131072, 32, 8, 128), (16, 16000, 96, 8, 64), (8, 32768, 32, 8, 64), (64, 5000, 32, 8, 128), (50, 6000, 64, 8, 64),
]


@pytest.mark.parametrize("batch,keys,hq,hkv,d", LONG)
def test_long_chunks_of_small_blocks(batch, keys, hq, hkv, d):
    check([keys] * batch, hq, hkv, d, 16, BF)
