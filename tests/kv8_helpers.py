"""Plain restatements of the 8-bit KV cache operators for the tests: the write rule tile by tile in
float32 (numpy, every operation correctly rounded), attention row by row in float64, and the bound that the
kernels' roundings allow."""
import numpy as np
import torch

SCALE_MIN = np.float32(2.0 ** -64)


class HostCache:
    """The cache as numpy arrays."""

    def __init__(self, k, v, ks, vs):
        self.code, self.scale = [k.copy(), v.copy()], [ks.copy(), vs.copy()]

    @property
    def block_size(self):
        return self.code[0].shape[2]

    def write(self, rows, table, past, b):
        """rows: (k, v) float32 [n, heads, d] of sequence b at positions past, past + 1, ..."""
        bs = self.block_size
        n = rows[0].shape[0]
        for which in range(2):
            code, scale, x = self.code[which], self.scale[which], rows[which]
            for j in range(past // bs, -(-(past + n) // bs)):
                block = table[b][j] if j < len(table[b]) else -1
                if not 0 <= block < code.shape[0]:
                    continue
                lo, hi = max(past, j * bs), min(past + n, (j + 1) * bs)
                for h in range(code.shape[1]):
                    z = x[lo - past:hi - past, h]
                    old = scale[block, h] if lo > j * bs else np.float32(0)
                    fine = bool(np.isfinite(z).all() and np.isfinite(old))
                    if not fine:
                        scale[block, h] = np.nan
                        code[block, h, lo - j * bs:hi - j * bs] = 0
                        continue
                    s = np.float32(np.abs(z).max()) / np.float32(127)
                    if s < SCALE_MIN:
                        s = np.float32(0)
                    if lo > j * bs:
                        s = max(s, old)
                        if s != old:
                            held = code[block, h, :lo - j * bs].astype(np.float32) * (old / s)
                            code[block, h, :lo - j * bs] = np.rint(held).astype(np.int8)
                    inv = np.float32(1) / s if s > 0 else np.float32(0)
                    code[block, h, lo - j * bs:hi - j * bs] = np.clip(np.rint(z * inv), -127, 127).astype(np.int8)
                    scale[block, h] = s

    def rows(self, table, b, lo, hi):
        """float32 values [hi - lo, heads, d] of K and of V; NaN where the table maps nothing."""
        bs = self.block_size
        out = [np.full((hi - lo, c.shape[1], c.shape[3]), np.nan, np.float32) for c in self.code]
        for p in range(lo, hi):
            block = table[b][p // bs] if 0 <= p // bs < len(table[b]) else -1
            if 0 <= block < self.code[0].shape[0]:
                for which in range(2):
                    out[which][p - lo] = self.code[which][block, :, p % bs].astype(np.float32) * self.scale[which][block][:, None]
        return out


def attention64(q, k, v, length, scale, causal, window):
    """q [T, hq, d], k and v [length, hkv, d] float64 -> out, lse, and A = sum p |v| (for the bound), all float64."""
    T, hq, d = q.shape
    group = hq // k.shape[1]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("thd,lhd->htl", q, kk) * scale
    mag = torch.einsum("thd,lhd->htl", q.abs(), kk.abs()) * scale
    pos = torch.arange(length - T, length, device=q.device)[:, None]
    at = torch.arange(length, device=q.device)[None]
    see = torch.ones((T, length), dtype=torch.bool, device=q.device)
    if causal:
        see &= at <= pos
    if window:
        see &= at > pos - window
    s = s.masked_fill(~see, -torch.inf)
    top = s.amax(-1, keepdim=True) if length else torch.full((hq, T, 1), -torch.inf, dtype=q.dtype, device=q.device)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(s - top)
    tot = p.sum(-1)
    norm = torch.where(tot > 0, tot, 1.0)
    p = p / norm[..., None]
    out = torch.einsum("htl,lhd->thd", p, vv)
    absum = torch.einsum("htl,lhd->thd", p, vv.abs())
    lse = (top[..., 0] + torch.log(tot)).transpose(0, 1)
    mag = mag.masked_fill(~see, 0.0)
    mag = mag.amax(-1).transpose(0, 1) if length else torch.zeros((T, hq), dtype=q.dtype, device=q.device)
    return out, lse, absum, mag


def bounds(want, absum, mag, n, d, sv_max, dtype):
    """The least and the largest output, and the bound of the lse's error, that the kernels' roundings allow:
    the scores' float32 sums of d products and the exponent (ds), probabilities to f16 (2^-11 relative, 2^-25 absolute
    against a largest one of 1), the float32 sum over n keys (in parts of at least 64).  The output's own rounding is
    applied to both ends: rounding keeps the order, so nothing has to be allowed for it."""
    ds = (mag * d + 16.0) * 2.0 ** -23 + 2.0 ** -20
    rel = 2.0 ** -11 + 2 * ds + (n / 64 + 80) * 2.0 ** -23
    tol = absum * rel[..., None] * 1.01 + n * 2.0 ** -25 * 127 * sv_max + 2.0 ** -24
    return ((want - tol).to(dtype), (want + tol).to(dtype)), ds + (n / 64 + 80) * 2.0 ** -23 + 2.0 ** -18
