"""8-bit paged KV cache: quantizing K and V rows as they are written, reading them back, and attention
over the cache (single tokens, a few tokens, prompts).

The reference has no counterpart: its attention stays with the QNN runtime.  A model that uses the
quantized MatMuls and the GDN inverse of this package also has attention layers, and their cache is held
here like everything else, as integer codes with a scale.

    cache = Kv8Cache.empty(num_blocks, kv_heads, head_dim, block_size)
    kv8_write(cache, k, v, block_table, past)                    # this step's rows
    out = kv8_attention(q, cache, block_table, past + q.shape[1])

Token p of sequence b is slot ``p % block_size`` of block ``block_table[b, p // block_size]``.  Each (block,
kv head) of K and of V has one float32 scale; value = code * scale.  include/qhtp.h has the arithmetic.

Rows come as [batch, tokens, heads, head_dim], the same number for every sequence, or, with ``seq_start``
int32 [batch + 1], as [rows, heads, head_dim] with the rows ``seq_start[b]:seq_start[b + 1]`` of sequence b.
They may be views (a slice of a fused projection, a transposed tensor) as long as head_dim is contiguous and
every head starts on a multiple of 16 bytes.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from . import _lib as L

HEAD_DIMS = (64, 128, 256)
BLOCK_SIZES = (16, 32, 64, 128)
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_SCALE_MOST = 2.35e38  # times log2(e) still a float32
# QhtpKv8Move and QhtpKv8Attention, packed in one call (native sizes and alignment)
_MOVE = struct.Struct("@4Pq4I 2P2q4I P P3q P3q 2I P")
_ATTENTION = struct.Struct("@4Pq4I 2P2q4I P P3q P3q P 4I f I P N P")
_TAIL = struct.Struct("@P N P")  # workspace, its size, stream


class Kv8Cache(NamedTuple):
    """The cache's four tensors: codes int8 [num_blocks, kv_heads, block_size, head_dim], contiguous, and
    scales float32 [num_blocks, kv_heads], of K and of V.  Any 4-tuple of such tensors is as good."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, num_blocks: int, kv_heads: int, head_dim: int, block_size: int = 64, device="cuda") -> "Kv8Cache":
        """A cache that holds zeros."""
        if head_dim not in HEAD_DIMS or block_size not in BLOCK_SIZES:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS} and block_size one of {BLOCK_SIZES}")
        if num_blocks <= 0 or kv_heads <= 0:
            raise ValueError("num_blocks and kv_heads must be positive")
        codes = [torch.zeros((num_blocks, kv_heads, block_size, head_dim), dtype=torch.int8, device=device) for _ in range(2)]
        return cls(*codes, *[torch.zeros((num_blocks, kv_heads), dtype=torch.float32, device=device) for _ in range(2)])


def _cache_fields(cache):
    """The cache's fields of the packed structures, and its device."""
    k, v, ks, vs = cache
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or ks.shape != shape[:2] or vs.shape != ks.shape:
        raise ValueError("the cache is int8 [num_blocks, kv_heads, block_size, head_dim] twice and float32 [num_blocks, kv_heads] twice")
    if 0 in shape:
        raise ValueError("the cache needs blocks and heads")
    if not (k.dtype is v.dtype is torch.int8 and ks.dtype is vs.dtype is torch.float32):
        raise TypeError("the cache's codes must be int8 and its scales float32")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("the cache's tensors must be contiguous")
    dev = k.device
    if not k.is_cuda or v.device != dev or ks.device != dev or vs.device != dev:
        raise ValueError("the cache's tensors must be on one CUDA device")
    return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), shape[0], shape[1], shape[3], shape[2], 0), dev


def _ints(name, t, n, dev):
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} elements on the cache's device")
    return t.data_ptr()


def _seqs_fields(table, seq_start, tokens, total, dev):
    shape = table.shape
    if table.dtype is not torch.int32 or len(shape) != 2 or table.device != dev:
        raise ValueError("block_table must be an int32 [batch, blocks] tensor on the cache's device")
    b, width = shape
    row, col = table.stride()
    if col != 1 and width > 1:
        raise ValueError("block_table's rows must be contiguous")
    return table.data_ptr(), 0 if seq_start is None else _ints("seq_start", seq_start, b + 1, dev), row, total, width, b, tokens, 0


def _rows_fields(name, t, heads, head_dim, dtype, dev, ragged):
    """Pointer and strides (batch, token, head) of rows; they may be views."""
    shape = t.shape
    if len(shape) != (3 if ragged else 4) or shape[-2] != heads or shape[-1] != head_dim:
        raise ValueError(f"{name} must be [{'rows' if ragged else 'batch, tokens'}, {heads}, {head_dim}]")
    if t.dtype is not dtype or t.device != dev:
        raise TypeError(f"{name} must be {dtype} on the cache's device")
    s = t.stride()
    if s[-1] != 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    ptr = t.data_ptr()
    if ragged:
        bs, ts, hs = 0, s[0], s[1]
    else:
        bs, ts, hs, _ = s
    size = 4 if dtype is torch.float32 else 2
    if (ptr | (bs | ts | hs) * size) & 15:
        # the stride of an axis of extent 1 moves nothing, and may be anything
        bs, ts, hs = (stride if n > 1 else 0 for stride, n in zip((bs, ts, hs), shape if not ragged else (1, *shape)))
        if (ptr | (bs | ts | hs) * size) & 15:
            raise ValueError(f"{name}: every head must start on a multiple of 16 bytes")
    return ptr, bs, ts, hs


def _counts(t, seq_start, most, what):
    """(most rows of a sequence, rows in all) of the rows t."""
    if seq_start is None:
        if t.dim() != 4:
            raise ValueError(f"{what} must be [batch, tokens, heads, head_dim], or come with seq_start")
        return t.shape[1], 0
    if t.dim() != 3:
        raise ValueError(f"{what} must be [rows, heads, head_dim] with seq_start")
    total = t.shape[0]
    return total if most is None else max(0, min(int(most), total)), total


# the current stream's handle without making a Stream object (a tenth of the time), where torch has it
_current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _on(stream, dev):
    """The stream to launch on, as a handle."""
    if stream is None:
        return _current(dev.index)
    if stream.device != dev:
        raise ValueError("the stream must be on the cache's device")
    return stream.cuda_stream


def _call(fn, name, dev, arg):
    if dev.index != _device():
        with torch.cuda.device(dev):
            st = fn(arg)
    else:
        st = fn(arg)
    if st:
        L.check(name, st)


def _empty(like, shape, dtype, stream):
    """A tensor of the allocator's on the device of `like`, to be used on `stream`."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _like(t, stream):
    """_empty of a tensor's own shape and type, in half the time; contiguous."""
    if stream is None:
        return torch.empty_like(t, memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        return torch.empty_like(t, memory_format=torch.contiguous_format)


def kv8_write(cache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, past: torch.Tensor, *,
              seq_start: torch.Tensor | None = None, max_new: int | None = None, stream=None) -> None:
    """Quantize the rows k and v (bf16, f16 or f32) into the cache (qhtp_kv8_write), in place.

    Row i of sequence b becomes its token ``past[b] + i`` (past int32 [batch]).  A block that is written from
    its first slot starts anew; one that is continued keeps the larger of its scale and the new rows', and
    its old codes are rounded to that scale where it grew.  ``max_new``: with ``seq_start``, at least the largest
    number of rows of a sequence (default: all of the rows; a smaller number launches fewer blocks)."""
    cf, dev = _cache_fields(cache)
    dtype = k.dtype
    if dtype not in _DTYPE:
        raise TypeError("k and v must be bfloat16, float16 or float32")
    tokens, total = _counts(k, seq_start, max_new, "k")
    if v.shape != k.shape:
        raise ValueError("k and v must have one shape")
    sf = _seqs_fields(block_table, seq_start, tokens, total, dev)
    if seq_start is None and k.shape[0] != sf[5]:
        raise ValueError("k and block_table must have one batch size")
    heads, d, ragged = cf[5], cf[6], seq_start is not None
    rk = _rows_fields("k", k, heads, d, dtype, dev, ragged)
    rv = _rows_fields("v", v, heads, d, dtype, dev, ragged)
    arg = _MOVE.pack(*cf, *sf, _ints("past", past, sf[5], dev), *rk, *rv, _DTYPE[dtype], 0, _on(stream, dev))
    _call(L.lib.qhtp_kv8_write, "qhtp_kv8_write", dev, arg)


def kv8_read(cache, block_table: torch.Tensor, first: torch.Tensor, tokens: int | None = None, *,
             seq_start: torch.Tensor | None = None, total: int | None = None, max_tokens: int | None = None,
             dtype: torch.dtype = torch.bfloat16, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V rows of the cache (qhtp_kv8_read): code * scale in float32, rounded once to ``dtype``.

    ``tokens`` of every sequence from position ``first[b]`` on, as [batch, tokens, kv_heads, head_dim]; or, with
    ``seq_start``, ``seq_start[b + 1] - seq_start[b]`` of sequence b, as [total, kv_heads, head_dim] (``total``: the
    rows in all; ``max_tokens``: at least the largest count, default total).  Positions that the block table
    does not map come back as NaN; rows of a ragged read that no sequence has are not written."""
    cf, dev = _cache_fields(cache)
    if dtype not in _DTYPE:
        raise TypeError("dtype must be bfloat16, float16 or float32")
    heads, d, ragged = cf[5], cf[6], seq_start is not None
    if ragged:
        if total is None or tokens is not None or total < 0:
            raise ValueError("a read with seq_start takes total (the rows in all) instead of tokens")
        shape = (total, heads, d)
        tokens = total if max_tokens is None else max(0, min(int(max_tokens), total))
    else:
        if tokens is None or tokens < 0:
            raise ValueError("tokens must be given, or seq_start and total")
        total = 0
    sf = _seqs_fields(block_table, seq_start, tokens, total, dev)
    if not ragged:
        shape = (sf[5], tokens, heads, d)
    pf = _ints("first", first, sf[5], dev)
    k = _empty(first, shape, dtype, stream)
    v = _like(k, stream)
    ts = heads * d
    arg = _MOVE.pack(*cf, *sf, pf, k.data_ptr(), 0 if ragged else tokens * ts, ts, d,
                     v.data_ptr(), 0 if ragged else tokens * ts, ts, d, _DTYPE[dtype], 0, _on(stream, dev))
    _call(L.lib.qhtp_kv8_read, "qhtp_kv8_read", dev, arg)
    return k, v


def kv8_attention(q: torch.Tensor, cache, block_table: torch.Tensor, lengths: torch.Tensor, *, scale: float | None = None,
                  causal: bool = True, window: int = 0, seq_start: torch.Tensor | None = None, max_new: int | None = None,
                  max_len: int | None = None, out: torch.Tensor | None = None, return_lse: bool = False, stream=None):
    """softmax(scale * q K^T) V over the cache (qhtp_kv8_attention); q bf16 or f16, q_heads a multiple of
    the cache's kv_heads (query head h reads kv head ``h // (q_heads // kv_heads)``).

    ``lengths`` int32 [batch]: tokens of the cache that belong to the sequence, of which its T query tokens are the
    last.  Query token t stands at position ``lengths[b] - T + t``; with ``causal`` it sees the keys up to that
    position, with ``window`` > 0 only the last ``window`` of those.  A row that sees no key is zero, its lse -inf.

    ``scale``: default head_dim ** -0.5.  ``max_new``: with ``seq_start``, at least the largest number of query tokens
    of a sequence (rows beyond it may be left out; default all).  ``max_len``: about the largest length (default: the
    block table's reach); it sizes the launch, and any value gives a right result.  How the keys are cut, and so the last bits,
    depends on the call's lengths and shapes: the same call gives the same bits.  Returns out (q's shape and dtype), or
    (out, lse) with lse float32 of q's shape without head_dim."""
    cf, dev = _cache_fields(cache)
    dtype = q.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError("q must be bfloat16 or float16")
    tokens, total = _counts(q, seq_start, max_new, "q")
    sf = _seqs_fields(block_table, seq_start, tokens, total, dev)
    b, d, ragged, shape = sf[5], cf[6], seq_start is not None, q.shape
    if not ragged and shape[0] != b:
        raise ValueError("q and block_table must have one batch size")
    heads = shape[-2]
    if heads == 0 or heads % cf[5]:
        raise ValueError("q's heads must be a multiple of the cache's")
    rq = _rows_fields("q", q, heads, d, dtype, dev, ragged)
    lf = _ints("lengths", lengths, b, dev)
    if not 0 <= window <= 1 << 30 or (window and not causal):
        raise ValueError("window must be 0, or positive (up to 2^30) and causal")
    if scale is None:
        scale = d ** -0.5
    if not 2.0 ** -149 <= scale <= _SCALE_MOST:
        raise ValueError("scale must be above 0 and no more than 2.35e38, in float32")
    if out is None:  # contiguous
        out, ts = _like(q, stream), heads * d
        ro = out.data_ptr(), 0 if ragged else tokens * ts, ts, d
    elif out.shape != shape:
        raise ValueError("out must have q's shape")
    else:
        ro = _rows_fields("out", out, heads, d, dtype, dev, ragged)
    lse = _empty(q, shape[:-1], torch.float32, stream) if return_lse else None
    reach = sf[4] * cf[7]
    if max_len is not None:
        reach = max(0, min(int(max_len), reach))
    handle = _on(stream, dev)
    arg = _ATTENTION.pack(*cf, *sf, lf, *rq, *ro, lse.data_ptr() if return_lse else 0, _DTYPE[dtype], heads, 1 if causal else 0,
                          window, scale, reach, 0, 0, handle)

    def launch(arg):  # both on the cache's device: the plan depends on its number of SMs
        need = L.lib.qhtp_kv8_attention_workspace_bytes(arg)
        if need:
            ws = _empty(q, (need,), torch.uint8, stream)
            arg = arg[:-_TAIL.size] + _TAIL.pack(ws.data_ptr(), need, handle)
        return L.lib.qhtp_kv8_attention(arg)

    _call(launch, "qhtp_kv8_attention", dev, arg)
    return (out, lse) if return_lse else out


def kv8_check(device=None, stream=None) -> None:
    """Synchronize ``stream`` (default: the current one) and raise if a kernel of kv8_attention on ``device`` (default: the
    stream's, or the current one) has recorded a wait that gave up since the last check (qhtp_kv8_check), which leaves
    the outputs of that call undefined.  No call does this by itself: it would wait for the GPU."""
    if device is None:
        device = _device() if stream is None else stream.device
    with torch.cuda.device(device):
        code = C.c_int(0)
        handle = _current(_device()) if stream is None else stream.cuda_stream
        st = L.lib.qhtp_kv8_check(C.byref(code), handle)
    if st:
        raise L.QhtpError(f"qhtp_kv8_check (device code {code.value})", st)
