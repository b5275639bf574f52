"""Many sessions' KV caches in one pool of pages.

    PagedCache     a pool of pages of 16 to 1024 positions, for keys and for values
    paged_append   q/k RMSNorm + rotary embedding of many tokens, k and v into the pages
    attn_paged     attn_window over the pages

attn_window's caches (kv.py) hold one run of rows a sequence, whatever its length will be.  Here
a sequence has a table: int32 [B, n] on the device, whose entry i is the page of positions
i * page .. (i + 1) * page - 1.  Pages are handed out as a context grows, given back (an entry
that nothing visible needs may hold anything, such as -1) behind a window, and shared: sequences
that begin alike may hold the same pages, as long as who appends to one holds it alone.  An entry
outside the pool where one is needed is never followed: nothing is written there, and the rows
that needed it are NaN.

Tokens, positions and counts are those of kv.py: [T, ...] of one sequence (a table [n]) or
[B, T, ...] of B, token t of sequence b at position pos + t, pos an int or int32 [B] on the
device.  The padding's rows are zeros in a new output and left as they are in a given one.
Every op enqueues on torch's current stream of the tensors' device and does not synchronise.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .kv import _attend, _batched, _call, _host_pos, _int32, _out
from .ops import Workspace
from .rotary import Rotary, _turn_c, overlaps


class PagedCache:
    """The pool: k and v [pages, n_kv_heads, page, head_dim] in 16 bits, views of any strides
    whose pages' rows are dense (a head's page is page * head_dim adjacent values).  The kernels
    write the tensors in place and the object holds their addresses, so they cannot be
    replaced."""

    __slots__ = ("k", "v", "_c")

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _lib.require_device(k, v)
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise RuntimeError("k and v are [pages, n_kv_heads, page, head_dim] and agree in "
                               "shape, strides and dtype")
        pages, n, page, hd = k.shape
        if k.stride(3) != 1 or k.stride(2) != hd:
            raise RuntimeError("the rows of a head's page must be dense")
        if k.data_ptr() == v.data_ptr():
            raise RuntimeError("k and v must be pools of their own")
        if page < 16 or page > 1024 or page & (page - 1):
            raise RuntimeError(f"a page holds 16 to 1024 positions, a power of two, got {page}")
        self.k, self.v = k, v
        self._c = (pages, page, n, hd, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
                   _lib.half_code(k.dtype))

    @classmethod
    def empty(cls, n_kv_heads: int, pages: int, page: int = 64, head_dim: int = 128, *,
              dtype: torch.dtype = torch.bfloat16,
              device: torch.device | str = "cuda") -> "PagedCache":
        """A pool of zeros."""
        return cls(*(torch.zeros(pages, n_kv_heads, page, head_dim, dtype=dtype, device=device)
                     for _ in range(2)))

    def __reduce__(self):  # a copy holds its own tensors' addresses
        return PagedCache, (self.k, self.v)

    pages = property(lambda self: self._c[0])
    page = property(lambda self: self._c[1])
    n_kv_heads = property(lambda self: self._c[2])
    head_dim = property(lambda self: self._c[3])

    def _with(self, table: torch.Tensor, B: int, dev: torch.device) -> _lib.PagedCacheC:
        """struct i4_pagedcache of this pool under a call's table."""
        shape, stride = table.shape, table.stride()
        if len(shape) not in (1, 2) or (shape[0] if len(shape) == 2 else 1) != B \
                or table.dtype != torch.int32 or table.device != dev or shape[-1] < 1 \
                or stride[-1] != 1 and shape[-1] > 1:
            raise RuntimeError(f"the table is int32 [{B}, n] on the tensors' device, a sequence's "
                               f"entries adjacent")
        pages, page, n, hd, k, v, ps, hs, dt = self._c
        return _lib.PagedCacheC(k, v, table.data_ptr(), ps, hs, stride[0] if B > 1 else 0, B, n,
                                pages, page, shape[-1], hd, dt)


def paged_append(qkv: torch.Tensor, n_heads: int, q_norm_w: torch.Tensor | None,
                 k_norm_w: torch.Tensor | None, eps: float, rotary: Rotary,
                 pos: int | torch.Tensor, cache: PagedCache, table: torch.Tensor, *,
                 turn: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """The fused projection rows qkv [T, (n_heads + 2 n_kv_heads) * 128] (or [B, T, ...]):
    RMSNorm of the queries and keys over head_dim where a weight is given (None: none), their
    rotary embedding, each token's rotated key and its value to the row of its position pos + t
    in the sequence's pages; returns the rotated queries [T, n_heads, 128] (or [B, T, ...]).

    turn: the positions that the angles take where they are not the tokens' own, as rope takes
    them ([B, T] or [axes, B, T]).  "half" embeddings turn a multiple of 16 dims here.  fp32
    inside, rounded once (i4_paged_append)."""
    dev = _lib.require_device(qkv, q_norm_w, k_norm_w, cache.k, turn, counts, out)
    x = _batched(qkv, 3, "qkv")
    B, T, width = x.shape
    cc = cache._with(table, B, dev)
    hd = cc.head_dim
    if cc.dtype != _lib.half_code(x.dtype):
        raise RuntimeError("the pages must have the activation dtype")
    if width != (n_heads + 2 * cc.n_kv_heads) * hd:
        raise RuntimeError("qkv's width does not match the head counts")
    for w in (q_norm_w, k_norm_w):
        if w is not None and (w.dtype != x.dtype or w.shape != (hd,) or w.stride(0) != 1):
            raise RuntimeError(f"a norm weight is {hd} adjacent values of the activation dtype")
    if rotary.dims > hd or rotary.layout == "half" and rotary.dims % 16:
        raise RuntimeError(f"{rotary.dims} of {hd} dims turn: at most all, and with the layout "
                           "'half' a multiple of 16")
    if x.stride(2) != 1:
        x = x.contiguous()
    shape = (B, T, n_heads, hd)
    q = _out(out, x, shape if qkv.dim() == 3 else shape[1:], False)
    if out is not None and overlaps(q.view(B, T, n_heads, hd), x.unflatten(2, (-1, hd))):
        raise RuntimeError("out must not overlap qkv")
    on_dev = isinstance(pos, torch.Tensor)
    tc = None if turn is None else _turn_c(turn, rotary, qkv.dim() == 3, B, T, dev)
    _call(dev, _lib.lib().i4_paged_append, x.data_ptr(), cc.dtype, T, x.stride(0), x.stride(1),
          n_heads, _lib.ptr(q_norm_w), _lib.ptr(k_norm_w), eps, rotary._c,
          _int32(pos, B, dev, "pos") if on_dev else None,
          0 if on_dev else _host_pos(pos, T, cc.table_len * cc.page), tc,
          _int32(counts, B, dev, "counts"), out is None, q.data_ptr(), ctypes.byref(cc))
    return q


def attn_paged(q: torch.Tensor, cache: PagedCache, table: torch.Tensor,
               pos: int | torch.Tensor, *, window: int | None = None, sinks: int = 0,
               scale: float | None = None, counts: torch.Tensor | None = None,
               out: torch.Tensor | None = None,
               workspace: Workspace | None = None) -> torch.Tensor:
    """attn_window over pages: rotated queries q [T, n_heads, 128] (or [B, T, ...]) at positions
    pos + t, over the positions of their sequence's table up to and including theirs
    (paged_append), and with a window those j > p - window or j < sinks.  The same roundings
    as attn_window (i4_attn_paged)."""
    dev = _lib.require_device(q, cache.k, counts, out)
    cc = cache._with(table, q.shape[0] if q.dim() == 4 else 1, dev)
    if out is not None and out.dim() == q.dim() and overlaps(
            *(_batched(t, 4, "q") for t in (out, q))):
        raise RuntimeError("out must not overlap q")
    lib = _lib.lib()
    return _attend(lib.i4_attn_paged, cc, cc.table_len * cc.page, q, dev, pos, window, sinks, scale,
                   counts, out, workspace, lib.i4_attn_paged_workspace_bytes, (out is None,))
