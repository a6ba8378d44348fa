"""Rows whose largest probability belongs to a key with a small value, as the first key of a sequence often does: the output is
then what thousands of keys of small probability add up to.

Probabilities are f16 in the product with V: off by at most 2^-11 of themselves, and those below f16's normal range by half
of its smallest step, 2^-25.  The kernels take p up to 2^7 for the row's largest key and more, so that step is 2^-32 of the largest
probability.  With P the largest probability the output is off by at most
    sum_j p_j |v_j| (2^-11 + 2 ds + (n / 64 + 80) 2^-23) + n P 2^-32 max|v|
(ds: error of a score and its exponent, tests.kv8_helpers.bounds), and then rounded."""
import math

import pytest
import torch

import qcom_htp_b200 as qhtp
from tests.test_kv8_gpu import BF, HF, i32, random_cache

pytestmark = pytest.mark.gpu


def check(n, t, hq, hkv, d, bs, dtype, gap, max_len=None):
    """gap: log2 of the first key's probability over the others'."""
    blocks = -(-n // bs)
    cache = random_cache(blocks, hkv, d, bs, 5, spread=0.0)
    cache.k[:] //= 32         # scores of the others: near 0
    cache.k[0, :, 0] = 100    # of the first key: the gap
    cache.v[0, :, 0] = 0
    cache.v[:, :, :, ::2].abs_()  # half of the columns do not average out
    table = torch.arange(blocks, dtype=torch.int32, device="cuda")[None]
    g = torch.Generator(device="cuda").manual_seed(2)
    q = (1 + 0.1 * torch.rand((1, t, hq, d), generator=g, device="cuda")).to(dtype)
    sk = float(cache.k_scale[0, 0])
    scale = gap * math.log(2) / (100 * sk * float(q[0].double().sum(-1).max()))
    out, lse = qhtp.kv8_attention(q, cache, table, i32([n]), scale=scale, causal=False, return_lse=True, max_len=max_len)
    group = hq // hkv
    for h in range(hkv):
        k, v = ((code[:, h].double() * s[:, h].double()[:, None, None]).reshape(-1, d)[:n]
                for code, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        x = q[0, :, h * group:(h + 1) * group].double()
        s = x @ k.T * scale
        mag = (x.abs() @ k.abs().T * scale).amax(-1, keepdim=True)
        p = torch.softmax(s, -1)
        want = p @ v
        ds = (mag * d + 16.0) * 2.0 ** -23 + 2.0 ** -20
        tol = (p @ v.abs()) * (2.0 ** -11 + 2 * ds + (n / 64 + 80) * 2.0 ** -23) * 1.01 + n * p.amax(-1, keepdim=True) * 2.0 ** -32 * v.abs().max()
        got = out[0, :, h * group:(h + 1) * group]
        assert ((got >= (want - tol).to(dtype)) & (got <= (want + tol).to(dtype))).all(), float((got.double() - want).abs().max() / want.abs().max())
        off = (lse[0, :, h * group:(h + 1) * group].double() - torch.logsumexp(s, -1)).abs()
        assert (off <= ds[..., 0] + (n / 64 + 80) * 2.0 ** -23 + 2.0 ** -18).all()


@pytest.mark.parametrize("gap", [20, 25, 28])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 64, HF), (8, 1, 128, BF), (32, 1, 128, HF), (8, 1, 256, HF)])
def test_single_tokens(gap, hq, hkv, d, dtype):
    check(30000, 1, hq, hkv, d, 32, dtype, gap)
    check(5000, 1, hq, hkv, d, 32, dtype, gap, max_len=1)


@pytest.mark.parametrize("gap", [20, 25, 28])
@pytest.mark.parametrize("t,d", [(40, 64), (40, 128), (40, 256), (300, 64), (300, 128), (300, 256)])
def test_prompts(gap, t, d):
    """One tile of 128 rows, and (300 tokens over many keys) two."""
    check(12000, t, 8, 4, d, 64, HF, gap)
