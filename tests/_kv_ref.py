"""The cache operators in 64 bits, from their definitions, on the CPU."""
from __future__ import annotations

import math

import torch

BLOCK = 64


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def see(p: int, end: int, window: int | None, sinks: int) -> torch.Tensor:
    """The positions of [0, end) that a query at position p attends."""
    j = torch.arange(end)
    ok = j <= p
    if window is not None:
        ok &= (j > p - window) | (j < sinks)
    return ok


def attention(q, k, v, pos, counts, window, sinks, scale=None):
    """q [B, T, nh, d], k and v [B, nkv, rows, d] (any dtype) -> (out, tol) in fp64: the
    output and how far a kernel may be off (tolerance()).  Rows past counts are NaN."""
    dtype = q.dtype
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    B, T, nh, d = q.shape
    G = nh // k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.full((B, T, nh, d), math.nan, dtype=torch.float64)
    tol = out.clone()
    for b in range(B):
        for t in range(counts[b]):
            p = pos[b] + t
            j = see(p, p + 1, window, sinks).nonzero()[:, 0]
            kk = k[b][:, j].repeat_interleave(G, 0)
            vv = v[b][:, j].repeat_interleave(G, 0)
            w = torch.softmax((kk @ q[b, t][:, :, None])[..., 0] * scale, -1)
            out[b, t] = (w[:, None] @ vv)[:, 0]
            mass = (w[:, None] @ vv.abs())[:, 0]
            size = (kk.abs() @ q[b, t].abs()[:, :, None])[..., 0].amax(-1, keepdim=True) * scale
            tol[b, t] = tolerance(out[b, t], mass, dtype, size)
    return out, tol


def tolerance(out, mass, dtype, size):
    """What an attention with 16-bit products and fp32 sums may be off by.  u is half a step.

    Each softmax weight is rounded to dtype once, which moves the output by up to u times
    mass = sum p |v| / sum p.  A score's 128 products are summed in fp32: off by up to 2^-17 of
    size, the sum of their magnitudes (times scale), twice (the maximum's too); exp, the
    running sums and the products are off by 2^-18.  The output is rounded once: u of it, or
    half the smallest subnormal's step where it is below the normal numbers."""
    u, f = half_step(dtype), torch.finfo(dtype)
    off = (u + 2.0 ** -16 * size + 2.0 ** -18) * mass
    return off + u * (out.abs() + off) + f.tiny * f.eps / 2


def rope(x, w, p, inv_freq, eps):
    """x [..., 128] at position p (a tensor that broadcasts to x[..., 0])."""
    y = x.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    a = p.double()[..., None] * inv_freq.double()
    lo, hi = y[..., :64], y[..., 64:]
    out = torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)
    size = torch.cat([lo.abs() + hi.abs()] * 2, -1)
    return out, size


E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def quantise(x, kind):
    """One block -> (values that the elements stand for before the scale, scale)."""
    x = x.double().cpu()
    if not torch.isfinite(x).all():
        return torch.zeros_like(x), math.nan
    big = max(x.abs().max().item(), 2.0 ** -100)
    scale = torch.tensor(big / (127 if kind == torch.int8 else 448)).float().double().item()
    y = x / scale
    if kind == torch.int8:
        return torch.round(y), scale
    m, mid = y.abs(), (E4M3[1:] + E4M3[:-1]) / 2
    i = torch.bucketize(m, mid)
    tie = torch.bucketize(m, mid, right=True) - i
    return torch.sign(y) * E4M3[i + tie * (i & 1)], scale


class Cache8:
    """What a KV8Cache holds after a history of appends, per sequence and head."""

    def __init__(self, B, n, blocks, kind, dtype):
        self.kind, self.B, self.n, self.blocks = kind, B, n, blocks
        self.elem = torch.zeros(2, B, n, blocks, BLOCK, 128, dtype=torch.float64)
        self.scale = torch.zeros(2, B, n, blocks, dtype=torch.float64)
        self.tail = torch.zeros(2, B, n, BLOCK, 128, dtype=dtype)

    def append(self, kv, pos, counts):
        """kv [2, B, T, n, 128]"""
        kv = kv.cpu()
        for b in range(self.B):
            if not 0 <= pos[b] < self.blocks * BLOCK:
                continue
            c = min(counts[b], self.blocks * BLOCK - pos[b])
            r, first = pos[b] % BLOCK, pos[b] // BLOCK
            for s in range(2):
                for g in range(self.n):
                    seq = torch.cat([self.tail[s, b, g, :r], kv[s, b, :c, g]])
                    done = len(seq) // BLOCK
                    for i in range(done):
                        e, sc = quantise(seq[i * BLOCK:(i + 1) * BLOCK], self.kind)
                        self.elem[s, b, g, first + i] = e
                        self.scale[s, b, g, first + i] = sc
                    self.tail[s, b, g, :len(seq) - done * BLOCK] = seq[done * BLOCK:]

    def rows(self, end):
        """k and v [B, n, rows, 128] in fp64 as attended after end[b] tokens."""
        x = self.elem * self.scale[..., None, None]
        for b in range(self.B):
            if end[b] % BLOCK:
                x[:, b, :, end[b] // BLOCK] = self.tail[:, b].double()
        return x.reshape(2, self.B, self.n, self.blocks * BLOCK, 128)
