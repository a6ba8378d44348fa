"""The 8-bit KV cache on the GPU: writes and reads equal their float32 rule bit for bit, attention stays
within the bound of its roundings of a float64 evaluation on the same codes."""
import math

import numpy as np
import pytest
import torch

import qcom_htp_b200 as qhtp
from qcom_htp_b200 import _lib as L
from tests.kv8_helpers import HostCache, attention64, bounds

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def host(cache):
    return HostCache(*[t.cpu().numpy() for t in cache])


def same(a, b):
    a, b = np.asarray(a), np.asarray(b)
    np.testing.assert_array_equal(a, b)


def random_cache(blocks, heads, d, bs, seed, spread=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    code = lambda: torch.randint(-127, 128, (blocks, heads, bs, d), generator=g, device="cuda", dtype=torch.int8)
    scale = lambda: 0.01 * torch.exp(spread * torch.randn((blocks, heads), generator=g, device="cuda"))
    return qhtp.Kv8Cache(code(), code(), scale(), scale())


def random_table(lengths, bs, blocks, seed, extra=1):
    """Distinct blocks for every sequence; entries beyond a sequence's end map nothing."""
    ids = np.random.default_rng(seed).permutation(blocks)
    width = max(-(-n // bs) for n in lengths) + extra
    table, at = np.full((len(lengths), width), -1, np.int32), 0
    for b, n in enumerate(lengths):
        m = -(-n // bs)
        table[b, :m] = ids[at:at + m]
        at += m
    assert at <= blocks
    return table


# ------------------------------------------------------------------------------------------ write and read
WRITES = [  # heads, d, bs, dtype, [(past, new), ...] one after the other for three sequences
    (2, 64, 16, F32, [(0, 5), (5, 1), (6, 30)]),
    (1, 128, 64, BF, [(0, 64), (64, 1), (65, 1)]),
    (3, 128, 32, HF, [(0, 1), (1, 200), (201, 3)]),
    (2, 256, 128, F32, [(0, 129), (129, 127), (256, 1)]),
    (1, 256, 16, BF, [(0, 17), (17, 15), (32, 40)]),
    (5, 64, 128, HF, [(0, 300), (300, 1), (90, 70)]),
]


@pytest.mark.parametrize("heads,d,bs,dtype,steps", WRITES)
def test_write_and_read_equal_the_rule(heads, d, bs, dtype, steps):
    most = max(p + n for p, n in steps) + 40
    nseq = 3
    cache = random_cache(4 * (-(-most // bs)) + 5, heads, d, bs, 3)
    table = random_table([most] * nseq, bs, cache.k.shape[0], 4)
    want = host(cache)
    g = torch.Generator(device="cuda").manual_seed(7)
    for step, (past, new) in enumerate(steps):
        # unlike lengths: sequence b has b rows fewer, and starts b places later from the second step on
        news = [max(0, new - b) if step == 0 else new for b in range(nseq)]
        pasts = [past - (b if step else 0) if past else 0 for b in range(nseq)]
        pasts = [max(0, p) for p in pasts]
        start = np.cumsum([0] + news)
        k = (torch.randn((int(start[-1]), heads, d), generator=g, device="cuda") * 3.0 ** step).to(dtype)
        v = torch.randn((int(start[-1]), heads, d), generator=g, device="cuda").to(dtype)
        qhtp.kv8_write(cache, k, v, i32(table), i32(pasts), seq_start=i32(start), max_new=max(news))
        for b in range(nseq):
            sl = slice(start[b], start[b + 1])
            want.write((k[sl].float().cpu().numpy(), v[sl].float().cpu().numpy()), table, pasts[b], b)
    got = host(cache)
    for which in range(2):
        same(got.scale[which], want.scale[which])
        same(got.code[which], want.code[which])  # the whole cache: nothing else was touched
    for out in (BF, HF, F32):
        first = [0, 3, bs - 1]
        k, v = qhtp.kv8_read(cache, i32(table), i32(first), 2 * bs + 3, dtype=out)
        for b in range(nseq):
            wk, wv = want.rows(table, b, first[b], first[b] + 2 * bs + 3)
            for got_rows, w in ((k, wk), (v, wv)):
                w = torch.from_numpy(w).to(out)
                assert torch.equal(torch.nan_to_num(got_rows[b].cpu().float(), nan=1e30), torch.nan_to_num(w.float(), nan=1e30))


def test_write_uniform_rows_and_views():
    """[batch, tokens, heads, d] views of one fused projection, and a [batch, heads, tokens, d] order."""
    B, T, H, D, bs = 2, 37, 4, 128, 16
    fused = torch.randn((B, T, 3 * H * D), device="cuda", dtype=BF)
    k = fused[..., H * D:2 * H * D].unflatten(-1, (H, D))
    v = torch.randn((B, H, T, D), device="cuda", dtype=BF).transpose(1, 2)
    a, b = (qhtp.Kv8Cache.empty(10, H, D, bs) for _ in range(2))
    table = i32(random_table([T] * B, bs, 10, 1))
    past = i32([0, 0])
    qhtp.kv8_write(a, k, v, table, past)
    qhtp.kv8_write(b, k.reshape(-1, H, D).contiguous(), v.reshape(-1, H, D).contiguous(), table, past,
                   seq_start=i32([0, T, 2 * T]))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_write_special_values():
    """Zeros, values below the smallest scale, infinities and NaN, and the restart that clears them."""
    D, bs = 64, 16
    cache = random_cache(8, 1, D, bs, 5)
    table = np.array([[0, 1, 2, 3, 4]], np.int32)
    x = np.random.default_rng(1).standard_normal((5 * bs, 1, D)).astype(np.float32)
    x[0:bs] = 0
    x[bs:2 * bs] *= 1e-25
    x[2 * bs + 3, 0, 5] = np.inf
    x[3 * bs + 1, 0, 0] = np.nan
    x[4 * bs:, 0, 0] = 3e38
    want = host(cache)

    def write(lo, hi, y=x):
        r = torch.from_numpy(y[lo:hi]).cuda()
        qhtp.kv8_write(cache, r, r, i32(table), i32([lo]), seq_start=i32([0, hi - lo]))
        want.write((y[lo:hi], y[lo:hi]), table, lo, 0)
        got = host(cache)
        for w in range(2):
            same(got.scale[w], want.scale[w])
            same(got.code[w], want.code[w])

    write(0, 5 * bs)
    assert float(cache.k_scale[0, 0]) == 0 and float(cache.k_scale[1, 0]) == 0
    assert math.isnan(float(cache.k_scale[2, 0])) and math.isnan(float(cache.v_scale[3, 0]))
    clean = np.where(np.isfinite(x), x, np.float32(1))
    write(2 * bs + 8, 3 * bs, clean)       # continues a tile that holds a NaN: stays NaN
    assert math.isnan(float(cache.k_scale[2, 0]))
    write(2 * bs, 3 * bs + 4, clean)       # starts both anew
    assert math.isfinite(float(cache.k_scale[2, 0])) and math.isfinite(float(cache.k_scale[3, 0]))


def test_write_and_read_nothing_mapped():
    """Table entries outside the cache, positions past the table, broken starts: dropped or NaN, never touched."""
    cache = random_cache(4, 2, 64, 16, 6)
    before = [t.clone() for t in cache]
    r = torch.randn((2, 40, 2, 64), device="cuda")
    qhtp.kv8_write(cache, r, r, i32([[-1, 4], [1 << 30, -7]]), i32([0, 0]))
    qhtp.kv8_write(cache, r, r, torch.empty((2, 0), dtype=torch.int32, device="cuda"), i32([0, 0]))
    flat = r.reshape(-1, 2, 64)
    for start in ([0, 50, 81], [-1, -1, -1], [60, 20, 10], [0, 0, 0]):
        qhtp.kv8_write(cache, flat, flat, i32([[-1], [-1]]), i32([0, 0]), seq_start=i32(start))
    qhtp.kv8_write(cache, flat, flat, i32([[0], [1]]), i32([0, 0]), seq_start=i32([80, 81, 1 << 30]))
    for x, y in zip(cache, before):
        assert torch.equal(x, y)
    k, v = qhtp.kv8_read(cache, i32([[0, -1], [5, 2]]), i32([-3, 30]), 20, dtype=F32)
    want = host(cache)
    table = [[0, -1], [5, 2]]
    for b, lo in ((0, -3), (1, 30)):
        for got, w in zip((k, v), want.rows(table, b, lo, lo + 20)):
            same(got[b].cpu().numpy(), w)


def test_ragged_read():
    cache = random_cache(40, 2, 128, 32, 8)
    counts, first = [0, 77, 1, 33], [5, 10, 31, 0]
    table = random_table([120] * 4, 32, 40, 2)
    start = np.cumsum([0] + counts)
    want = host(cache)
    for most in (None, 77):
        k, v = qhtp.kv8_read(cache, i32(table), i32(first), seq_start=i32(start), total=int(start[-1]), max_tokens=most, dtype=F32)
        for b in range(4):
            wk, wv = want.rows(table, b, first[b], first[b] + counts[b])
            same(k[start[b]:start[b + 1]].cpu().numpy(), wk)
            same(v[start[b]:start[b + 1]].cpu().numpy(), wv)


# ------------------------------------------------------------------------------------------ attention
def attend(lengths, news, hq, hkv, d, bs, dtype, causal=True, window=0, ragged=False, seed=0, scale=None, spread=0.5,
           max_len=None, stream=None, q_amp=1.0, layout="bthd"):
    """Runs kv8_attention and compares every row with the float64 evaluation."""
    width = [max(n, 1) for n in lengths]
    blocks = sum(-(-n // bs) for n in width) + 2
    cache = random_cache(blocks, hkv, d, bs, seed + 1, spread)
    table = random_table(lengths, bs, blocks, seed + 2)
    # what no sequence owns holds NaN scales: nothing of it may reach an output
    owned = np.unique(table[table >= 0])
    idle = np.setdiff1d(np.arange(blocks), owned)
    cache.k_scale[idle] = math.nan
    cache.v_scale[idle] = math.nan
    B = len(lengths)
    g = torch.Generator(device="cuda").manual_seed(seed + 3)
    start = np.cumsum([0] + list(news))
    q = (torch.randn((int(start[-1]), hq, d), generator=g, device="cuda") * q_amp).to(dtype)
    kw = dict(scale=scale, causal=causal, window=window, return_lse=True, max_len=max_len, stream=stream)
    if ragged:
        out, lse = qhtp.kv8_attention(q, cache, i32(table), i32(lengths), seq_start=i32(start), max_new=max(news), **kw)
    else:
        assert len(set(news)) == 1
        shaped = q.reshape(B, news[0], hq, d)
        if layout == "bhtd":
            shaped = shaped.transpose(1, 2).contiguous().transpose(1, 2)
        out, lse = qhtp.kv8_attention(shaped, cache, i32(table), i32(lengths), **kw)
        out, lse = out.reshape(-1, hq, d), lse.reshape(-1, hq)
    torch.cuda.synchronize()
    assert out.dtype == dtype and lse.dtype == F32
    s = d ** -0.5 if scale is None else scale
    h = host(cache)
    for b, (n, t) in enumerate(zip(lengths, news)):
        if t == 0:
            continue
        k, v = (torch.from_numpy(x).cuda().double() for x in h.rows(table, b, 0, n))
        rows = q[start[b]:start[b + 1]].double()
        want, wl, absum, mag = attention64(rows, k, v, n, s, causal, window)
        sv = float(cache.v_scale[table[b][table[b] >= 0]].max()) if n else 0.0
        (least, most), tol_l = bounds(want, absum, mag, max(n, 1), d, sv, dtype)
        got, gl = out[start[b]:start[b + 1]], lse[start[b]:start[b + 1]].double()
        assert torch.isfinite(got).all()
        assert ((got >= least) & (got <= most)).all(), (b, float((got.double() - want).abs().max()))
        empty = torch.isinf(wl)
        assert torch.equal(empty, torch.isinf(gl)) and (gl[empty] < 0).all()
        assert (got[empty] == 0).all()
        assert ((gl - wl).abs()[~empty] <= tol_l[~empty]).all(), (b, float((gl - wl).abs()[~empty].max()))
    return out


STEP = [  # hq, hkv, d, bs, dtype
    (8, 2, 64, 16, BF), (8, 1, 128, 16, HF), (28, 4, 128, 64, BF), (3, 3, 128, 128, BF), (16, 1, 128, 32, HF),
    (32, 2, 64, 64, BF), (16, 2, 256, 64, BF), (5, 1, 256, 16, HF), (48, 2, 128, 32, BF), (12, 1, 256, 128, HF), (6, 2, 64, 128, HF),
]


@pytest.mark.parametrize("hq,hkv,d,bs,dtype", STEP)
def test_single_tokens(hq, hkv, d, bs, dtype):
    """Lengths around the edges of blocks, steps, segments and chunks; idle slots of length 0."""
    lengths = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700, 2047, 2049, 5000]
    attend(lengths, [1] * len(lengths), hq, hkv, d, bs, dtype)


@pytest.mark.parametrize("t", [2, 3, 5, 8, 13, 24])
@pytest.mark.parametrize("hq,hkv,d,bs,dtype", [(8, 2, 128, 64, BF), (14, 2, 64, 32, HF), (8, 1, 256, 16, BF)])
def test_few_tokens(t, hq, hkv, d, bs, dtype):
    """Drafted tokens; a sequence shorter than its query rows has rows that see nothing."""
    attend([t, t + 1, 100, 64, 1000, 0, t - 1, 333], [t] * 8, hq, hkv, d, bs, dtype, seed=t)


@pytest.mark.parametrize("window", [1, 7, 16, 100, 1000, 5000])
@pytest.mark.parametrize("t", [1, 6])
def test_window(window, t):
    attend([300, 33, t, 2000, 0, 64], [t] * 6, 12, 4, 128, 32, BF, window=window, seed=window)


@pytest.mark.parametrize("hq,hkv,d,bs,dtype", [(4, 2, 128, 16, HF), (6, 1, 64, 64, BF), (8, 1, 256, 32, HF)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 40), (True, 300), (False, 0)])
def test_prompts(hq, hkv, d, bs, dtype, causal, window):
    """Ragged prompts, with and without cached tokens, one of them longer than what is cached."""
    news = [130, 1, 257, 64, 0, 300]
    lengths = [130, 1, 400, 64, 10, 200]
    attend(lengths, news, hq, hkv, d, bs, dtype, causal=causal, window=window, ragged=True, seed=window)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_uniform_prompts_in_both_orders(d):
    for layout in ("bthd", "bhtd"):
        attend([200, 333], [200, 200], 4, 2, d, 64, BF, layout=layout)


def test_long_context_in_chunks():
    attend([40000, 12345], [1, 1], 8, 2, 128, 64, BF)
    attend([30001], [4], 8, 1, 64, 16, HF)
    attend([20000], [3], 4, 1, 256, 128, HF)


@pytest.mark.parametrize("max_len", [0, 1, 100, 1 << 20])
def test_the_bound_on_the_lengths_changes_no_result(max_len):
    a = attend([3000, 17, 1024], [1] * 3, 8, 2, 128, 64, BF, max_len=max_len)
    b = attend([3000, 17, 1024], [1] * 3, 8, 2, 128, 64, BF)
    assert (a.float() - b.float()).abs().max() < 0.05  # each is inside its own bound above


def test_scales_of_unlike_size():
    """V scales spread over many orders of magnitude, and large scores."""
    attend([700, 64], [1, 1], 8, 2, 128, 16, BF, spread=4.0)
    attend([700, 300], [130, 130], 8, 2, 128, 16, HF, spread=4.0)
    attend([500], [1], 4, 1, 128, 32, BF, q_amp=30.0)


@pytest.mark.parametrize("amp", [1e-30, 1e30])
def test_q_of_any_size(amp):
    """q is taken to f16 by a power of two per row: no overflow, no loss."""
    attend([300], [1], 8, 2, 128, 32, BF, q_amp=amp, scale=1.0 / amp / 11.0)
    attend([300], [140], 8, 2, 128, 32, BF, q_amp=amp, scale=1.0 / amp / 11.0)


def test_zero_tiles():
    """Tiles whose scale is zero are zeros, in K and in V, and where all of V is zero so is the output."""
    cache = random_cache(4, 1, 128, 16, 3)
    cache.k_scale[1] = 0
    cache.v_scale[2] = 0
    q = torch.randn((1, 1, 4, 128), device="cuda", dtype=BF)
    table = i32([[0, 1, 2, 3]])
    out, lse = qhtp.kv8_attention(q, cache, table, i32([60]), return_lse=True)
    k, v = (torch.from_numpy(x).cuda().double() for x in host(cache).rows([[0, 1, 2, 3]], 0, 0, 60))
    want, wl, absum, mag = attention64(q[0].double(), k, v, 60, 128 ** -0.5, True, 0)
    (least, most), tl = bounds(want, absum, mag, 60, 128, float(cache.v_scale.max()), BF)
    assert ((out[0] >= least) & (out[0] <= most)).all() and ((lse[0].double() - wl).abs() <= tl).all()
    cache.v_scale.zero_()
    assert (qhtp.kv8_attention(q, cache, table, i32([60])) == 0).all()


@pytest.mark.parametrize("t", [1, 200])
def test_a_bad_block_reaches_only_the_rows_that_see_it(t):
    """A NaN scale or an unmapped block: NaN for the rows that see it, the others as without it."""
    bs, n = 16, 400
    for spoil in ("k", "v", "map"):
        cache = random_cache(30, 1, 128, bs, 9)
        table = random_table([n], bs, 30, 3)
        q = torch.randn((1, t, 4, 128), device="cuda", dtype=BF)
        clean = qhtp.kv8_attention(q, cache, i32(table), i32([n]))
        at = 20  # keys 320..335
        bad = table.copy()
        if spoil == "map":
            bad[0, at] = -1
        else:
            (cache.k_scale if spoil == "k" else cache.v_scale)[table[0, at]] = math.nan
        out = qhtp.kv8_attention(q, cache, i32(bad), i32([n]))
        sees = torch.arange(n - t, n, device="cuda") >= at * bs
        assert torch.isnan(out[0][sees]).all()
        assert torch.equal(out[0][~sees], clean[0][~sees])
        # a window that ends before the bad block
        out = qhtp.kv8_attention(q, cache, i32(bad), i32([n]), window=40)
        assert torch.isfinite(out[0][-1]).all()


def test_length_beyond_the_table_counts_as_its_end():
    cache = random_cache(6, 1, 64, 16, 2)
    table = i32([[3, 1, 4]])
    q = torch.randn((1, 1, 2, 64), device="cuda", dtype=HF)
    a = qhtp.kv8_attention(q, cache, table, i32([48]))
    assert torch.equal(a, qhtp.kv8_attention(q, cache, table, i32([1 << 30])))
    assert (qhtp.kv8_attention(q, cache, table, i32([-5])) == 0).all()


def test_runs_repeat_bit_for_bit():
    cache = random_cache(600, 2, 128, 32, 2)
    table = i32(random_table([9000, 5000], 32, 600, 1))
    q = torch.randn((2, 3, 16, 128), device="cuda", dtype=BF)
    a = [qhtp.kv8_attention(q, cache, table, i32([9000, 5000]), return_lse=True) for _ in range(3)]
    for x in a[1:]:
        assert torch.equal(x[0], a[0][0]) and torch.equal(x[1], a[0][1])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths,t,hq,bs", [([200, 333], 200, 4, 64), ([2000, 1333, 1000], 150, 16, 16), ([4000] * 9, 1, 8, 32),
                                                ([4096], 4096, 32, 64)])
def test_many_runs_give_the_same_bits(d, lengths, t, hq, bs):
    """The kernels' roles hand over through barriers: none may depend on who comes first."""
    blocks = sum(-(-n // bs) for n in lengths)
    cache = random_cache(blocks, 2, d, bs, 1)
    table, n = i32(random_table(lengths, bs, blocks, 2)), i32(lengths)
    q = torch.randn((len(lengths), t, hq, d), device="cuda", dtype=BF)
    busy = torch.randn((1024, 1024), device="cuda")
    first = qhtp.kv8_attention(q, cache, table, n)
    for i in range(80):
        if i % 3 == 0:
            busy @ busy
        assert torch.equal(qhtp.kv8_attention(q, cache, table, n), first), i


def test_on_another_stream():
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    attend([3000, 100], [1, 1], 8, 2, 128, 64, BF, stream=s)
    cache = random_cache(10, 2, 64, 16, 3)
    r = torch.randn((1, 30, 2, 64), device="cuda", dtype=BF)
    table = i32(random_table([30], 16, 10, 1))
    past = i32([0])
    torch.cuda.synchronize()
    qhtp.kv8_write(cache, r, r, table, past, stream=s)
    k, _ = qhtp.kv8_read(cache, table, past, 30, dtype=BF, stream=s)
    s.synchronize()
    assert (k - r).abs().max() <= r.abs().max() * (0.5 / 127 + 2.0 ** -8)


def test_in_a_graph():
    """Lengths live on the device: one captured graph serves a growing context."""
    H, D, bs = 2, 128, 16
    cache = qhtp.Kv8Cache.empty(40, H, D, bs)
    table = i32(random_table([300, 300], bs, 40, 1))
    k, v = (torch.randn((2, 1, H, D), device="cuda", dtype=BF) for _ in range(2))
    q = torch.randn((2, 1, 8, D), device="cuda", dtype=BF)
    past, lengths = i32([0, 5]), i32([1, 6])

    def step():
        qhtp.kv8_write(cache, k, v, table, past)
        return qhtp.kv8_attention(q, cache, table, lengths)

    step()
    torch.cuda.synchronize()
    cache.k_scale.zero_(), cache.v_scale.zero_(), cache.k.zero_(), cache.v.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    other = qhtp.Kv8Cache.empty(40, H, D, bs)
    for i in range(20):
        for t in (k, v, q):
            t.copy_(torch.randn_like(t))
        graph.replay()
        qhtp.kv8_write(other, k, v, table, past)
        want = qhtp.kv8_attention(q, other, table, lengths)
        assert torch.equal(out, want)
        past += 1
        lengths += 1


def test_offsets_past_32_bits():
    """A cache of 4.3 GB per tensor: the last blocks of it."""
    H, D, bs, blocks = 8, 256, 128, 16500
    cache = qhtp.Kv8Cache(*[torch.empty((blocks, H, bs, D), dtype=torch.int8, device="cuda") for _ in range(2)],
                          *[torch.zeros((blocks, H), device="cuda") for _ in range(2)])
    table = np.array([[blocks - 1, blocks - 3, 8200, 0]], np.int32)
    r = torch.randn((1, 400, H, D), device="cuda", dtype=BF)
    qhtp.kv8_write(cache, r, r, i32(table), i32([0]))
    k, v = qhtp.kv8_read(cache, i32(table), i32([0]), 400, dtype=F32)
    assert (k - r.float()).abs().max() <= r.abs().max().float() * (0.51 / 127)
    for t in (1, 150):
        q = torch.randn((1, t, 16, D), device="cuda", dtype=BF)
        out = qhtp.kv8_attention(q, cache, i32(table), i32([400]))
        want, _, absum, mag = attention64(q[0].double(), k[0].double(), v[0].double(), 400, D ** -0.5, True, 0)
        (least, most), _ = bounds(want, absum, mag, 400, D, float(cache.v_scale.max()), BF)
        assert ((out[0] >= least) & (out[0] <= most)).all()


def test_nothing_to_do():
    cache = qhtp.Kv8Cache.empty(2, 1, 64, 16)
    for shape in ((0, 1, 1, 64), (2, 0, 1, 64)):
        r = torch.empty(shape, device="cuda", dtype=BF)
        table, n = torch.zeros((shape[0], 2), dtype=torch.int32, device="cuda"), torch.zeros(shape[0], dtype=torch.int32, device="cuda")
        qhtp.kv8_write(cache, r, r, table, n)
        assert qhtp.kv8_attention(r, cache, table, n).shape == shape
        assert qhtp.kv8_read(cache, table, n, shape[1])[0].shape == shape
    q = torch.randn((2, 3, 4, 64), device="cuda", dtype=BF)
    out, lse = qhtp.kv8_attention(q, cache, torch.empty((2, 0), dtype=torch.int32, device="cuda"), i32([0, 9]), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


# ------------------------------------------------------------------------------------------ refusals
def test_refusals():
    c = qhtp.Kv8Cache.empty(4, 2, 64, 16)
    table, n = i32([[0, 1]]), i32([5])
    q = torch.randn((1, 1, 4, 64), device="cuda", dtype=BF)
    ok = lambda **kw: qhtp.kv8_attention(q, c, table, n, **kw)
    ok()
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(window=-1), dict(window=3, causal=False),
               dict(out=torch.empty((1, 1, 4, 32), device="cuda", dtype=BF))):
        with pytest.raises(ValueError):
            ok(**kw)
    with pytest.raises(TypeError):
        ok(out=torch.empty_like(q, dtype=HF))
    with pytest.raises(TypeError):
        qhtp.kv8_attention(q.float(), c, table, n)
    for bad in (q[..., :32], q[:, :, :3], q[0], torch.randn((1, 1, 4, 128), device="cuda", dtype=BF)[..., ::2],
                torch.randn((1, 1, 4 * 64 + 8), device="cuda", dtype=BF)[..., 1:257].unflatten(-1, (4, 64)),
                torch.randn((2, 1, 4, 64), device="cuda", dtype=BF)):
        with pytest.raises(ValueError):
            qhtp.kv8_attention(bad, c, table, n)
    for t in (table.long(), table[0], table.cpu(), i32([[0, 1], [2, 3]]).t()):
        with pytest.raises(ValueError):
            qhtp.kv8_attention(q, c, t, n)
    for m in (n.long(), i32([5, 6]), n.cpu(), n[0]):
        with pytest.raises(ValueError):
            qhtp.kv8_attention(q, c, table, m)
    with pytest.raises(TypeError):
        qhtp.kv8_attention(q, (c.k.view(torch.uint8), c.v, c.k_scale, c.v_scale), table, n)
    for bad in ((c.k.cpu(), *c[1:]), (c.k[:2], *c[1:]), (c.k.transpose(1, 2), c.v.transpose(1, 2), *c[2:]), (*c[:3], c.v_scale[:, :1])):
        with pytest.raises(ValueError):
            qhtp.kv8_attention(q, bad, table, n)
    r = torch.randn((1, 3, 2, 64), device="cuda")
    for bad in (r[..., :63], r[0], r[:, :, :1], torch.randn((2, 3, 2, 64), device="cuda")):
        with pytest.raises(ValueError):
            qhtp.kv8_write(c, bad, bad, table, n)
    with pytest.raises(ValueError):
        qhtp.kv8_write(c, r, r[:, :2], table, n)
    with pytest.raises(TypeError):
        qhtp.kv8_write(c, r, r.half(), table, n)
    with pytest.raises(TypeError):
        qhtp.kv8_write(c, r.double(), r.double(), table, n)
    with pytest.raises(ValueError):
        qhtp.kv8_read(c, table, n)
    with pytest.raises(ValueError):
        qhtp.kv8_read(c, table, n, seq_start=i32([0, 3]))
    with pytest.raises(TypeError):
        qhtp.kv8_read(c, table, n, 3, dtype=torch.int8)
    odd = tuple(torch.zeros(s, device="cuda", dtype=t) for s, t in (((2, 1, 16, 96), torch.int8),) * 2 + (((2, 1), F32),) * 2)
    with pytest.raises(qhtp.QhtpError) as e:
        qhtp.kv8_attention(torch.randn((1, 1, 1, 96), device="cuda", dtype=BF), odd, table, n)
    assert e.value.status == L.UNSUPPORTED
