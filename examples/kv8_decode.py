"""One attention layer served with quantized projections and the 8-bit paged KV cache.

    python examples/kv8_decode.py [--batch 16] [--hidden 4096] [--steps 64]

The layer's projections are W4A16 ``QuantMatMul`` ops on 16-bit activation codes; between them its K and V rows go into
the cache (``kv8_write``) and its queries attend over it (``kv8_attention``):

    prefill   the prompts of all sequences at once, of unlike lengths, packed row after row (``seq_start``)
    decoding  one token of every sequence a step, in a CUDA graph: positions and lengths live on the device, so one
              captured graph serves the growing contexts
    export    a finished sequence's K and V as plain rows (``kv8_read``)

At the end the last step is compared with plain float32 attention over the K and V rows that the projections gave
(never quantized), and the time of a step is printed.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from qcom_htp_b200 import Kv8Cache, QuantMatMul, kv8_attention, kv8_check, kv8_read, kv8_write  # noqa: E402

ZERO = 32768
STEP = 8.0 / 32768  # 16-bit codes of values in [-8, 8)


def codes(x: torch.Tensor) -> torch.Tensor:
    return (torch.round(x.float() / STEP) + ZERO).clamp(0, 65535).to(torch.int32).to(torch.uint16)


def values(c: torch.Tensor) -> torch.Tensor:
    return ((c.to(torch.int32) - ZERO).float() * STEP).to(torch.bfloat16)


def projection(k: int, n: int, seed: int) -> QuantMatMul:
    """Random int4 weights that keep the variance of their input, one scale per output channel."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    weight = torch.randint(0, 256, (k // 2, n), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.full((n,), 1.0 / (4.64 * k ** 0.5), device="cuda")  # 4.64: root mean square of an int4 code
    return QuantMatMul("w4a16", weight, scale, torch.zeros(n, dtype=torch.int32, device="cuda"), act_scale=STEP, out_scale=STEP)


class AttentionLayer:
    def __init__(self, hidden: int, q_heads: int, kv_heads: int, head_dim: int, blocks: int, block_size: int):
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.qkv = projection(hidden, (q_heads + 2 * kv_heads) * head_dim, 1)
        self.out = projection(q_heads * head_dim, hidden, 2)
        self.cache = Kv8Cache.empty(blocks, kv_heads, head_dim, block_size)

    def split(self, x: torch.Tensor):
        """q, k and v of hidden codes [rows, hidden], as views of the fused projection [rows, heads, head_dim]."""
        heads = values(self.qkv(x)).view(x.shape[0], -1, self.head_dim)
        return heads.split([self.q_heads, self.kv_heads, self.kv_heads], 1)

    def prefill(self, x, table, past, lengths, start, max_new):
        q, k, v = self.split(x)
        kv8_write(self.cache, k, v, table, past, seq_start=start, max_new=max_new)
        o = kv8_attention(q, self.cache, table, lengths, seq_start=start, max_new=max_new, max_len=max_new)
        return self.out(codes(o.reshape(x.shape[0], -1))), k, v

    def step(self, x, table, past, lengths):
        q, k, v = (t.unsqueeze(1) for t in self.split(x))
        kv8_write(self.cache, k, v, table, past)
        o = kv8_attention(q, self.cache, table, lengths)
        return self.out(codes(o.reshape(x.shape[0], -1))), q, k, v, o


def run(batch: int = 16, hidden: int = 4096, q_heads: int = 32, kv_heads: int = 8, head_dim: int = 128, prompt: int = 1500,
        steps: int = 64, block_size: int = 64) -> dict:
    dev, i32 = "cuda", lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(0)
    news = torch.randint(max(1, prompt // 4), prompt + 1, (batch,), generator=g).tolist()
    # every sequence gets the blocks that it will need, in no order
    need = [-(-(n + steps) // block_size) for n in news]
    ids, table, at = torch.randperm(sum(need), generator=g).tolist(), torch.full((batch, max(need)), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[at:at + n])
        at += n
    table = table.to(dev)
    layer = AttentionLayer(hidden, q_heads, kv_heads, head_dim, sum(need), block_size)

    start = [0]
    for n in news:
        start.append(start[-1] + n)
    gd = torch.Generator(device=dev).manual_seed(1)
    x = codes(torch.randn((start[-1], hidden), generator=gd, device=dev))
    _, k, v = layer.prefill(x, table, i32([0] * batch), i32(news), i32(start), max(news))
    seen = [(k[start[b]:start[b + 1]], v[start[b]:start[b + 1]]) for b in range(batch)]  # for the comparison

    past, lengths = i32(news), i32([n + 1 for n in news])
    x = codes(torch.randn((batch, hidden), generator=gd, device=dev))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a first step outside the graph; the same token is written again below
        layer.step(x, table, past, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, q, k, v, o = layer.step(x, table, past, lengths)
        h = values(x).float() + values(y).float()  # what comes out, added and normalised, is the next token's input
        x.copy_(codes(h * torch.rsqrt(h.square().mean(-1, keepdim=True))))
        past += 1
        lengths += 1
    later = []
    times = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    times[0].record()
    for _ in range(steps):
        graph.replay()
        later.append((k.clone(), v.clone()))
    times[1].record()
    kv8_check()  # waits for the GPU, and raises if a kernel reported an error
    ms = times[0].elapsed_time(times[1]) / steps

    # the last step against attention over the rows that were never quantized
    worst = 0.0
    for b in range(batch):
        kk, vv = (torch.cat([seen[b][i]] + [t[i][b] for t in later]).float().repeat_interleave(q_heads // kv_heads, 1) for i in range(2))
        p = torch.softmax(torch.einsum("hd,lhd->hl", q[b, 0].float(), kk) * head_dim ** -0.5, -1)
        want = torch.einsum("hl,lhd->hd", p, vv)
        worst = max(worst, float((o[b, 0].float() - want).norm() / want.norm()))
    # a sequence leaves the cache
    n = news[0] + steps
    rk, rv = kv8_read(layer.cache, table[:1], i32([0]), n)
    held = torch.cat([seen[0][0]] + [t[0][0] for t in later]).float()
    export = float((rk[0].float() - held).norm() / held.norm())
    return {"step_ms": ms, "attention_error": worst, "export_error": export, "tokens": n, "out": o}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--prompt", type=int, default=1500)
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args()
    r = run(batch=a.batch, hidden=a.hidden, prompt=a.prompt, steps=a.steps)
    print(f"{a.batch} sequences, {a.steps} steps: {r['step_ms'] * 1e3:.0f} us a step (projections, cache and attention, one layer)")
    print(f"last step against unquantized K and V: relative error {r['attention_error']:.4f}; "
          f"{r['tokens']} exported K rows: {r['export_error']:.4f}")


if __name__ == "__main__":
    main()
