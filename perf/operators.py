"""The 8-bit KV cache operators as they are measured: writing new tokens into the paged cache, reading
tokens back, and attention over it.

The cache holds int8 codes [num_blocks, kv_heads, block_size, head_dim] for K and for V, and one float32
scale per (block, kv head) of each; token p of sequence b is slot p % block_size of block
block_table[b, p // block_size].  ``own`` false: the plain forms below, in float32 torch operations.
``own`` true: this package's kernels.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
SCALE_MIN = 2.0 ** -64  # a block whose scale would be smaller is stored as zeros


def _write(name, b, t, past, hkv, d, bs, dtype, ragged):
    return dict(name=name, op="write", b=b, t=t, past=past, hkv=hkv, d=d, bs=bs, dtype=dtype, ragged=ragged)


def _read(name, b, t, hkv, d, bs, dtype, ragged):
    return dict(name=name, op="read", b=b, t=t, past=0, hkv=hkv, d=d, bs=bs, dtype=dtype, ragged=ragged)


def _attn(name, b, t, past, hq, hkv, d, bs, dtype, ragged, causal=True, window=0, idle=False):
    return dict(name=name, op="attention", b=b, t=t, past=past, hq=hq, hkv=hkv, d=d, bs=bs, dtype=dtype, ragged=ragged,
                causal=causal, window=window, idle=idle)


def listed():
    return [
        # one decoding step of a batch: a token of each sequence goes into its partly filled block
        _write("write_step", 64, 1, 4000, 8, 128, 64, "bf16", True),
        # prompts of several requests are written after their prefill
        _write("write_prompts", 8, 4096, 700, 8, 128, 64, "f16", True),
        # a short context handed to code that wants plain rows
        _read("read_short", 4, 333, 4, 64, 16, "f32", True),
        # a long context read back, for export or for another attention
        _read("read_long", 2, 40000, 8, 128, 64, "bf16", False),
        # one user, a short conversation: latency
        _attn("step_one_short", 1, 1, 500, 32, 8, 128, 64, "bf16", False),
        # a serving batch of mixed lengths, with idle slots of length zero as a fixed-size graph has them
        _attn("step_batch", 64, 1, 8000, 32, 8, 128, 64, "bf16", True, idle=True),
        # two users with very long contexts
        _attn("step_long", 2, 1, 131071, 32, 8, 128, 128, "f16", False),
        # wide heads, few kv heads
        _attn("step_wide_heads", 16, 1, 16000, 16, 2, 256, 32, "bf16", True),
        # a few drafted tokens per sequence checked at once
        _attn("verify_drafts", 16, 6, 4100, 28, 4, 128, 64, "bf16", True),
        # a piece of a long prompt after what is cached, narrow heads, sliding window
        _attn("piece_window", 3, 1000, 20000, 24, 8, 64, 32, "f16", True, window=4096),
        # a whole prompt with wide heads
        _attn("prompt_wide_heads", 2, 2500, 0, 16, 2, 256, 64, "bf16", True),
        # the largest: one long prompt
        _attn("prompt_long", 1, 8192, 0, 32, 8, 128, 64, "bf16", False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _plain_bytes(c):
    """What the plain forms hold: dense rows of the context, and the scores."""
    return 8 * c["b"] * (c["past"] + c["t"]) * (c["hkv"] * c["d"] + c.get("hq", 0) * c["t"])


def draw(rng):
    """A case of the ranges above, of at most the largest listed one's cost."""
    top = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    room = max(_plain_bytes(c) for c in listed())
    while True:
        op = rng.choice(["write", "read", "attention", "attention", "attention"])
        d, bs = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
        hkv, ragged = rng.choice([1, 2, 4, 8]), rng.random() < 0.6
        if op == "write":
            c = _write("", _log(rng, 1, 128), rng.choice([1, _log(rng, 2, 8192)]), rng.choice([0, _log(rng, 1, 8000)]), hkv, d, bs,
                       rng.choice(["bf16", "f16", "f32"]), ragged)
        elif op == "read":
            c = _read("", _log(rng, 1, 64), _log(rng, 1, 60000), hkv, d, bs, rng.choice(["bf16", "f16", "f32"]), ragged)
        else:
            shape = rng.choice(["step", "step", "few", "prompt"])
            group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
            t = {"step": 1, "few": rng.randint(2, 24), "prompt": _log(rng, 25, 8192)}[shape]
            past = rng.choice([0, _log(rng, 1, 30000)]) if shape == "prompt" else _log(rng, 1, 131072)
            b = _log(rng, 1, 128) if shape != "prompt" else _log(rng, 1, 8)
            causal = rng.random() < 0.9
            window = _log(rng, 16, 8192) if causal and rng.random() < 0.25 else 0
            c = _attn("", b, t, past, hkv * group, hkv, d, bs, rng.choice(["bf16", "f16"]), ragged, causal, window, rng.random() < 0.2)
        w = work(c)
        if w["flops"] <= top["flops"] and w["bytes"] <= top["bytes"] and _plain_bytes(c) <= room:
            del c["name"]
            return c


# ------------------------------------------------------------------------------------------ lengths
def _fractions(n, ragged):
    """Shares of the nominal length for the n sequences: 1 for all, or spread over [1/8, 1]."""
    if not ragged:
        return [1.0] * n
    return [0.125 + 0.875 * ((0.61803398875 * i + 0.9) % 1.0) for i in range(n)]


def _lengths(c):
    """Per sequence: new tokens, and tokens cached before them."""
    f = _fractions(c["b"], c["ragged"])
    new = [max(1, round(c["t"] * x)) if c["t"] > 24 else c["t"] for x in f]
    past = [round(c["past"] * x) for x in f]
    return new, past


def _idle(c, i):
    """Whether sequence i is an idle slot of a batch: nothing of it is visible."""
    return c["op"] == "attention" and c["idle"] and i % 8 == 7


def _rows(c):
    """(new, past, total length seen) per sequence, as attention sees them."""
    new, past = _lengths(c)
    return new, past, [0 if _idle(c, i) else p + n for i, (n, p) in enumerate(zip(new, past))]


def _pairs(c, n, length):
    """Visible (query token, key) pairs of one sequence, and the keys that any of them sees."""
    if length == 0:
        return 0, 0
    if not c["causal"]:
        return n * length, length
    w = c["window"] or length
    first, last = length - n + 1, length  # keys up to the first and the last token
    full = max(0, last - max(first, w) + 1) * w  # tokens that see a whole window
    hi = min(last, w - 1)
    part = (first + hi) * (hi - first + 1) // 2 if hi >= first else 0
    return full + part, min(length, n + w - 1)


def work(case):
    c = case
    new, past, length = _rows(c)
    row = c["hkv"] * c["d"]
    if c["op"] == "attention":
        seen = [_pairs(c, n, x) for n, x in zip(new, length)]
        keys = sum(k for _, k in seen)
        tokens = sum(new)
        blocks = sum(-(-k // c["bs"]) for _, k in seen)
        return {"bytes": 2 * keys * row + 8 * blocks * c["hkv"] + 4 * blocks + tokens * c["hq"] * (2 * c["d"] * SIZE[c["dtype"]] + 4),
                "flops": 4 * c["d"] * c["hq"] * sum(p for p, _ in seen)}
    if c["op"] == "read":
        return {"bytes": 2 * sum(new) * row * (1 + SIZE[c["dtype"]]), "flops": 2 * sum(new) * row}
    # write: the new rows in, their codes out; then the touched blocks back, as float32 rows
    back = sum(n + p % c["bs"] for n, p in zip(new, past))
    return {"bytes": 2 * sum(new) * row * (SIZE[c["dtype"]] + 1) + 2 * back * row * 5, "flops": 8 * sum(new) * row}


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = case
    dev, g = "cuda", torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    new, past, length = _rows(c)
    b, hkv, d, bs = c["b"], c["hkv"], c["d"], c["bs"]
    full = [n + p for n, p in zip(new, past)]
    per = [-(-x // bs) for x in full]
    pool, width = sum(per) + 3, max(per)
    ids = torch.randperm(pool, device=dev, generator=g).to(torch.int32)
    slot = torch.stack([torch.arange(width, device=dev).clamp(max=per[i] - 1) + sum(per[:i]) for i in range(b)])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    codes = lambda: (torch.randn((pool, hkv, bs, d), device=dev, generator=g) * 32).round_().clamp_(-127, 127).to(torch.int8)
    scales = lambda: 0.03 * torch.exp(0.3 * torch.randn((pool, hkv), device=dev, generator=g))
    s = {"case": c, "cache": (codes(), codes(), scales(), scales()), "table": ids[slot], "dtype": DTYPES[c["dtype"]]}
    starts = [sum(new[:i]) for i in range(b + 1)]
    if c["op"] == "attention":
        s["scale"] = d ** -0.5
        s["max_len"], s["max_new"] = max(max(length), 1), max(new)
        s["lengths"] = i32(length)
        if c["t"] > 24 and c["ragged"]:  # prompts of several lengths, one after the other
            s["start"] = i32(starts)
            shape = (starts[-1], c["hq"], d)
        else:
            s["start"] = None
            shape = (b, c["t"], c["hq"], d)
        s["q"] = torch.randn(shape, device=dev, generator=g).to(s["dtype"])
    elif c["op"] == "write":
        loud = 1 + 5 * (torch.rand((hkv, d), device=dev, generator=g) < 0.03)  # a few channels are larger
        rows = lambda: (torch.randn((starts[-1], hkv, d), device=dev, generator=g) * loud).to(s["dtype"])
        s["k"], s["v"] = rows(), rows()
        s["start"], s["max_new"], s["past"] = i32(starts), max(new), i32(past)
        first = [p - p % bs for p in past]
        back = [x - f for x, f in zip(full, first)]
        s["first"], s["back_start"] = i32(first), i32([sum(back[:i]) for i in range(b + 1)])
        s["back"], s["back_max"] = sum(back), max(back)
    else:
        s["start"], s["max_new"], s["first"], s["total"] = i32(starts), max(new), i32([0] * b), starts[-1]
    return s


# ------------------------------------------------------------------------------------------ the plain forms
def _places(start, total, first, table, bs):
    """Block and slot of each of `total` tokens: token i of sequence b is the cache's token first[b] + i."""
    i = torch.arange(total, device=start.device)
    b = torch.searchsorted(start.long(), i, right=True) - 1
    p = first.long()[b] + i - start.long()[b]
    return table.long()[b, p // bs], p % bs, b, p


def _plain_read(cache, start, total, first, table, dtype):
    block, slot, _, _ = _places(start, total, first, table, cache[0].shape[2])
    one = lambda code, scale: (code[block, :, slot].float() * scale[block][:, :, None]).to(dtype)
    return one(cache[0], cache[2]), one(cache[1], cache[3])


def _plain_store(x, code, scale, block, slot, fresh):
    """Quantises the rows x into their blocks of one cache tensor; `fresh`: blocks that start anew."""
    x = x.float()
    a = torch.zeros_like(scale).index_reduce_(0, block, x.abs().amax(-1), "amax")
    s = a / torch.full_like(a, 127.0)
    s = torch.where(s < SCALE_MIN, torch.zeros_like(s), s)
    touched = torch.zeros_like(fresh).index_fill_(0, block, True)
    old = torch.where(fresh[:, None], torch.zeros_like(scale), scale)
    s = torch.where(touched[:, None], torch.maximum(old, s), scale)
    ratio = torch.where(s > 0, old / s, torch.ones_like(s))
    # what a partly filled block held before, in the block's new scale
    part = torch.nonzero(touched & ~fresh)[:, 0]
    code[part] = (code[part].float() * ratio[part][:, :, None, None]).round().to(torch.int8)
    inv = torch.where(s > 0, torch.reciprocal(s), torch.zeros_like(s))[block]
    code[block, :, slot] = (x * inv[:, :, None]).round().clamp(-127, 127).to(torch.int8)
    scale.copy_(s)


def _plain_write(s):
    k, v, ks, vs = s["cache"]
    block, slot, _, _ = _places(s["start"], s["k"].shape[0], s["past"], s["table"], k.shape[2])
    fresh = torch.zeros(k.shape[0], dtype=torch.bool, device=k.device)
    fresh[block[slot == 0]] = True
    _plain_store(s["k"], k, ks, block, slot, fresh)
    _plain_store(s["v"], v, vs, block, slot, fresh)


def _plain_attention(s):
    c, q, table, length = s["case"], s["q"], s["table"], s["lengths"].long()
    k, v, ks, vs = s["cache"]
    bs, hkv, d, hq = c["bs"], c["hkv"], c["d"], c["hq"]
    b, n = length.shape[0], s["max_len"]
    if s["start"] is None:
        t = torch.full_like(length, q.shape[1])
        dense = q
    else:  # prompts of several lengths, padded
        t = s["start"].long().diff()
        at = torch.arange(s["max_new"], device=q.device)
        row = (s["start"].long()[:-1, None] + at).clamp(max=q.shape[0] - 1)
        dense = q[row]
    tq = dense.shape[1]
    blocks = table.long()[:, : -(-n // bs)]
    rows = lambda code, scale: (code[blocks].float() * scale[blocks][..., None, None]).transpose(2, 3).reshape(b, -1, hkv, d)[:, :n]
    valid = torch.arange(n, device=q.device) < length[:, None]
    values = torch.where(valid[..., None, None], rows(v, vs), 0.0).permute(0, 2, 1, 3)
    keys = torch.where(valid[..., None, None], rows(k, ks), 0.0).permute(0, 2, 3, 1)
    x = dense.float().reshape(b, tq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    score = torch.matmul(x, keys).mul_(s["scale"]).reshape(b, hq, tq, n)
    at = torch.arange(n, device=q.device)
    place = (length - t)[:, None] + torch.arange(tq, device=q.device)
    see = valid[:, None, :].expand(b, tq, n)
    if c["causal"]:
        see = see & (at <= place[..., None])
    if c["window"]:
        see = see & (at > place[..., None] - c["window"])
    score.masked_fill_(~see[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(b, hkv, -1, n), values).reshape(b, hq, tq, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total))[..., 0]
    out, lse = out.permute(0, 2, 1, 3), lse.permute(0, 2, 1)
    if s["start"] is not None:
        i = torch.arange(q.shape[0], device=q.device)
        seq = torch.searchsorted(s["start"].long(), i, right=True) - 1
        out, lse = out[seq, i - s["start"].long()[seq]], lse[seq, i - s["start"].long()[seq]]
    return out.to(q.dtype).contiguous(), lse.contiguous()


def run(state):
    s, c = state, state["case"]
    if own:
        import qcom_htp_b200 as qhtp
        if c["op"] == "attention":
            out, lse = qhtp.kv8_attention(s["q"], s["cache"], s["table"], s["lengths"], scale=s["scale"], causal=c["causal"], window=c["window"],
                                          seq_start=s["start"], max_new=s["max_new"], max_len=s["max_len"], return_lse=True)
            return {"out": out, "lse": lse}
        if c["op"] == "read":
            k, v = qhtp.kv8_read(s["cache"], s["table"], s["first"], seq_start=s["start"], total=s["total"], max_tokens=s["max_new"], dtype=s["dtype"])
            return {"k": k, "v": v}
        qhtp.kv8_write(s["cache"], s["k"], s["v"], s["table"], s["past"], seq_start=s["start"], max_new=s["max_new"])
        k, v = qhtp.kv8_read(s["cache"], s["table"], s["first"], seq_start=s["back_start"], total=s["back"], max_tokens=s["back_max"], dtype=torch.float32)
        return {"k": k, "v": v, "k_scale": s["cache"][2], "v_scale": s["cache"][3]}
    if c["op"] == "attention":
        out, lse = _plain_attention(s)
        return {"out": out, "lse": lse}
    if c["op"] == "read":
        k, v = _plain_read(s["cache"], s["start"], s["total"], s["first"], s["table"], s["dtype"])
        return {"k": k, "v": v}
    _plain_write(s)
    k, v = _plain_read(s["cache"], s["back_start"], s["back"], s["first"], s["table"], torch.float32)
    return {"k": k, "v": v, "k_scale": s["cache"][2], "v_scale": s["cache"][3]}


# ------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    w = work(c)
    if w["flops"] > 3e12 or w["bytes"] > 4e9:
        return None
    new, past, length = _rows(c)
    bs = c["bs"]
    k, v, ks, vs = s["cache"]
    table = s["table"].cpu().tolist()

    def rows(code, scale, b, lo, hi):
        ids = torch.tensor(table[b][lo // bs: -(-hi // bs)], device=code.device)
        x = code[ids].double() * scale[ids].double()[:, :, None, None]
        return x.permute(0, 2, 1, 3).reshape(-1, c["hkv"], c["d"])[lo % bs: lo % bs + hi - lo]

    if c["op"] == "read":
        one = lambda code, scale: torch.cat([rows(code, scale, b, 0, n) for b, n in enumerate(new)])
        return {"k": one(k, ks), "v": one(v, vs)}

    if c["op"] == "write":
        def store(x, code, scale):
            outs, scale = [], scale.double()
            for b, (n, p) in enumerate(zip(new, past)):
                x0 = sum(new[:b])
                for j in range(p // bs, -(-(p + n) // bs)):
                    lo, hi = max(p, j * bs), min(p + n, (j + 1) * bs)
                    z = x[x0 + lo - p: x0 + hi - p].double().transpose(0, 1)
                    sc = z.abs().amax((1, 2)) / 127
                    sc = torch.where(sc < SCALE_MIN, 0.0, sc)
                    held = code[table[b][j]][:, : lo - j * bs].double()
                    if lo > j * bs:
                        old = scale[table[b][j]].clone()
                        sc = torch.maximum(sc, old)
                        held = torch.round(held * (old / sc)[:, None, None])
                    fresh = torch.round(z / torch.where(sc > 0, sc, 1.0)[:, None, None]).clamp(-127, 127)
                    scale[table[b][j]] = sc
                    outs.append((torch.cat([held, fresh], 1) * sc[:, None, None]).transpose(0, 1))
            return torch.cat(outs), scale
        (ek, eks), (ev, evs) = store(s["k"], k, ks), store(s["v"], v, vs)
        return {"k": ek, "v": ev, "k_scale": eks, "v_scale": evs}

    group = c["hq"] // c["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda").reshape(-1, c["hq"], c["d"])
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    q = s["q"].reshape(-1, c["hq"], c["d"])
    for b, (n, length_b) in enumerate(zip(new, length)):
        x0 = sum(new[:b])
        if length_b == 0:
            continue
        kk, vv = rows(k, ks, b, 0, length_b), rows(v, vs, b, 0, length_b)
        step = max(1, int(2e8 // (length_b * group)))
        for h in range(c["hkv"]):
            for t0 in range(0, n, step):
                t1 = min(n, t0 + step)
                place = torch.arange(length_b - n + t0, length_b - n + t1, device="cuda")[:, None]
                at = torch.arange(length_b, device="cuda")
                hide = torch.zeros((t1 - t0, length_b), dtype=torch.bool, device="cuda")
                if c["causal"]:
                    hide |= at > place
                if c["window"]:
                    hide |= at <= place - c["window"]
                x = q[x0 + t0: x0 + t1, h * group: (h + 1) * group].double()
                z = torch.einsum("tgd,ld->tgl", x, kk[:, h]) * s["scale"]
                z = z.masked_fill(hide[:, None], -math.inf)
                lse[x0 + t0: x0 + t1, h * group: (h + 1) * group] = torch.logsumexp(z, -1)
                out[x0 + t0: x0 + t1, h * group: (h + 1) * group] = torch.einsum("tgl,ld->tgd", torch.softmax(z, -1), vv[:, h])
    return {"out": out.reshape(s["q"].shape), "lse": lse.reshape(s["q"].shape[:-1])}
