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

import struct

import torch

from . import _lib, kv
from .kv import _batched, _call, _host_pos, _int32, _out
from .ops import Workspace
from .rotary import Rotary, _turn_c, distinct, overlaps

_paged = struct.Struct("<3Q3q7i4x").pack  # struct i4_pagedcache
HEAD_DIM = 128


class PagedCache(_lib.Handle):
    """The pool: k and v [pages, n_kv_heads, page, 128] in 16 bits, views of any strides that
    keep pages and heads apart and whose pages' rows are dense (a head's page is page * 128
    adjacent values).  The kernels write the tensors in place and the object holds their
    addresses, so they cannot be replaced (AttributeError)."""

    __slots__ = ("k", "v", "device", "dtype", "_c", "_index")

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        self.device = _lib.require_device(k, v)
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise RuntimeError("k and v are [pages, n_kv_heads, page, head_dim] and agree in "
                               "shape, strides and dtype")
        pages, n, page, hd = k.shape
        if hd != HEAD_DIM:
            raise RuntimeError(f"the kernels take heads of {HEAD_DIM} dims, got {hd}")
        if k.stride(3) != 1 or k.stride(2) != hd:
            raise RuntimeError("the rows of a head's page must be dense")
        if not distinct(page * hd, (pages, k.stride(0)), (n, k.stride(1))):
            raise RuntimeError("pages or heads of the pool overlap")
        if k.numel() and overlaps(k, v):
            raise RuntimeError("k and v must be pools of their own")
        if page < 16 or page > 1024 or page & (page - 1):
            raise RuntimeError(f"a page holds 16 to 1024 positions, a power of two, got {page}")
        self.k, self.v, self.dtype = k, v, k.dtype
        self._index = k.get_device()
        self._c = (pages, page, n, hd, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
                   _lib.half_code(k.dtype))

    @classmethod
    def empty(cls, n_kv_heads: int, pages: int, page: int = 64, head_dim: int = HEAD_DIM, *,
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

    def _beside(self, *ts: torch.Tensor | None) -> torch.device:
        """The device of the pool and of the given tensors."""
        for t in ts:
            if t is not None and t.get_device() != self._index:
                _lib.require_device(self.k, t)  # which says what is wrong
        return self.device

    def _beyond(self, out: torch.Tensor) -> None:
        """A given output lies outside the pool, which a call reads or writes as it writes it."""
        rows = out.view(1, 1, -1, out.shape[-1])
        if overlaps(rows, self.k) or overlaps(rows, self.v):
            raise RuntimeError("out must not overlap the pool")

    def _with(self, table: torch.Tensor, B: int) -> tuple[bytes, int]:
        """struct i4_pagedcache of this pool under a call's table, and its positions."""
        shape, stride = table.shape, table.stride()
        if len(shape) == 2 and shape[0] == B:
            step, n, last = stride[0], shape[1], stride[1]
        elif len(shape) == 1 and B == 1:
            step, n, last = 0, shape[0], stride[0]
        else:
            n = 0
        if n < 1 or last != 1 and n > 1 or table.dtype != torch.int32 \
                or table.get_device() != self._index:
            raise RuntimeError(f"the table is int32 [{B}, n] on the tensors' device, a sequence's "
                               f"entries adjacent")
        pages, page, heads, hd, k, v, ps, hs, dt = self._c
        return _paged(k, v, table.data_ptr(), ps, hs, step, B, heads, pages, page, n, hd,
                      dt), n * page


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
    dev = cache._beside(qkv, q_norm_w, k_norm_w, turn, counts, out)
    batched = qkv.dim() == 3
    x = qkv if batched else _batched(qkv, 3, "qkv")
    B, T, width = x.shape
    cc, keys = cache._with(table, B)
    _, _, n_kv, hd, _, _, _, _, dtype = cache._c
    if x.dtype != cache.dtype:
        raise RuntimeError("the pages must have the activation dtype")
    if width != (n_heads + 2 * n_kv) * hd:
        raise RuntimeError("qkv's width does not match the head counts")
    for w in (q_norm_w, k_norm_w):
        if w is not None and (w.dtype != x.dtype or w.shape != (hd,) or w.stride(0) != 1):
            raise RuntimeError(f"a norm weight is {hd} adjacent values of the activation dtype")
    if rotary.dims > hd or rotary.layout == "half" and rotary.dims % 16:
        raise RuntimeError(f"{rotary.dims} of {hd} dims turn: at most all, and with the layout "
                           "'half' a multiple of 16")
    b, t, e = x.stride()
    if e != 1:
        x = x.contiguous()
        b, t, _ = x.stride()
    shape = (B, T, n_heads, hd) if batched else (T, n_heads, hd)
    if out is None:
        q = x.new_empty(shape)
    else:
        q = _out(out, x, shape, False)
        y = q.view(B, T, n_heads, hd)
        if overlaps(y, x.unflatten(2, (-1, hd))):
            raise RuntimeError("out must not overlap qkv")
        cache._beyond(y)
    pd, ph = (_int32(pos, B, dev, "pos"), 0) if isinstance(pos, torch.Tensor) \
        else (None, _host_pos(pos, T, keys))
    tc = None if turn is None else _turn_c(turn, rotary, batched, B, T, dev)
    _call(dev, _lib.lib().i4_paged_append, x.data_ptr(), dtype, T, b, t, n_heads,
          None if q_norm_w is None else q_norm_w.data_ptr(),
          None if k_norm_w is None else k_norm_w.data_ptr(), eps, rotary._at, pd, ph, tc,
          None if counts is None else _int32(counts, B, dev, "counts"), out is None,
          q.data_ptr(), cc)
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
    dev = cache._beside(q, counts, out)
    x = q if q.dim() == 4 else _batched(q, 4, "q")
    B, T, nh, hd = x.shape
    cc, keys = cache._with(table, B)
    _, _, n_kv, head_dim, _, _, _, _, dtype = cache._c
    if hd != head_dim:
        raise RuntimeError(f"q {tuple(q.shape)} does not match the cache's head_dim {head_dim}")
    if q.dtype != cache.dtype:
        raise RuntimeError("the pages must have the activation dtype")
    w, sinks = kv._bounds(window, sinks)
    b, t, h, e = x.stride()
    if e != 1:
        x = x.contiguous()
        b, t, h, _ = x.stride()
    if out is None:
        y = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    else:
        y = _out(out, x, tuple(q.shape), False)
        if overlaps(out, q):
            raise RuntimeError("out must not overlap q")
        cache._beyond(out)
    pd, ph = (_int32(pos, B, dev, "pos"), 0) if isinstance(pos, torch.Tensor) \
        else (None, _host_pos(pos, T, keys))
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return attn_paged(q, cache, table, pos, window=window, sinks=sinks, scale=scale,
                              counts=counts, out=out, workspace=workspace)
    lib = _lib.lib()
    args = (x.data_ptr(), dtype, T, b, t, h, nh, cc, pd, ph,
            None if counts is None else _int32(counts, B, dev, "counts"), out is None, w, sinks,
            hd ** -0.5 if scale is None else scale, y.data_ptr())
    # the workspace that is there, and only if it does not do what the call needs
    stream = _lib.stream(dev)
    ws, counters = kv._held(workspace, dev, stream)
    rc = lib.i4_attn_paged(*args, None, 0, None, stream) if ws is None else lib.i4_attn_paged(
        *args, ws.data_ptr(), ws.numel(), counters.data_ptr(), stream)
    if rc == _lib.ERR_WORKSPACE:
        need = lib.i4_attn_paged_call_bytes(B, T, nh, n_kv, keys if pd else ph + T, w, sinks,
                                            pd is not None or counts is not None)
        ws, counters = kv._scratch(workspace, need, dev, True)
        rc = lib.i4_attn_paged(*args, ws.data_ptr(), need, _lib.ptr(counters), stream)
    if rc:
        _lib.check(rc)
    return y
