"""Rotary embeddings and a paged cache in 64 bits, from their definitions, on the CPU."""
from __future__ import annotations

import torch

from tests import _kv_ref as ref


def turned(x, inv_freq, positions, layout="half", factor=1.0, axes=None):
    """x [B, T, heads, d] turned by positions [B, T] or [axes, B, T] -> (out, size): size bounds
    the magnitude of each output's terms."""
    x = x.double().cpu()
    f, p = inv_freq.double().cpu(), positions.cpu().double()
    n = f.numel()
    if p.dim() == 3:
        p = torch.stack([p[a] for a in (axes or [0] * n)], -1)  # [B, T, pairs]
    else:
        p = p[..., None].expand(*p.shape, n)
    a = (p * f)[:, :, None]
    c, s = a.cos() * factor, a.sin() * factor
    lo, hi = ((slice(0, n), slice(n, 2 * n)) if layout == "half" else
              (slice(0, 2 * n, 2), slice(1, 2 * n, 2)))
    u, v = x[..., lo], x[..., hi]
    out, size = x.clone(), x.abs()
    out[..., lo], out[..., hi] = u * c - v * s, v * c + u * s
    size[..., lo] = size[..., hi] = (u.abs() + v.abs()) * abs(factor)
    return out, size


def normed(x, w, eps=1e-6):
    x = x.double().cpu()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double().cpu()


def rounded(out, size, dtype, lead):
    """What a rotation in fp32 that is rounded once may be off by: lead times size before the
    rounding, then half a step (of the smallest normal number for smaller ones)."""
    f = torch.finfo(dtype)
    return lead * size + ref.half_step(dtype) * (out.abs() + lead * size) + f.tiny * f.eps / 2


def gathered(pool, table):
    """The rows [B, n_kv, positions, d] of a table's pages; entries outside the pool are NaN."""
    pool, table = pool.cpu(), table.cpu().long()
    pages, n, page, d = pool.shape
    ok = (table >= 0) & (table < pages)
    x = pool[table.clamp(0, pages - 1)]  # [B, entries, n, page, d]
    x = torch.where(ok[:, :, None, None, None], x, torch.full_like(x, float("nan")))
    return x.permute(0, 2, 1, 3, 4).reshape(table.shape[0], n, -1, d)
