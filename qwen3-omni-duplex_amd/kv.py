"""A long conversation's KV cache: rotary append, bounded attention, 8-bit blocks.

    rope_append   q/k RMSNorm + rotary embedding of many tokens, k and v into the cache
                  (Qwen3OmniMoeThinkerTextAttention.forward between the q|k|v projection and
                  the attention, modeling_qwen3_omni_moe.py:1473-1500 in transformers 5.15)
    attn_window   attention of many tokens over a 16-bit cache, under a sliding window whose
                  first tokens stay visible, or over everything
    KV8Cache      a cache in 8 bits with a scale for each block of 64 tokens and head
    kv8_append    tokens into it
    attn_kv8      attn_window over it

The clock path attends every cached position of one session one token at a time
(src/duplex/streaming/clock.py:164-172; ops.attn_decode); these take prompt chunks and
several sessions, bound what a token attends, and halve the cache.

Tokens: [T, ...] of one sequence or [B, T, ...] of B, token t of sequence b at position
pos + t.  pos is an int (every sequence), or an int32 device tensor of B elements that the
kernels read, so that a captured graph serves every position.  counts (int32 device tensor of
B elements, optional) says how many of the T tokens each sequence has; the rest is padding,
whose output rows are left as they are.  A device position outside the cache writes nothing
to it and NaN to the token's output row; an int is refused.

Every op enqueues on torch's current stream of the tensors' device and does not synchronise,
with one exception: an inv_freq that is on the device is copied to the host, which waits.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import Workspace, _capturing

KV8_BLOCK = 64
_FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}


def _int32(t: torch.Tensor | None, B: int, dev: torch.device, name: str) -> int | None:
    """The address of B int32 on the device (None: not given)."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.numel() != B or t.device != dev or not t.is_contiguous():
        raise RuntimeError(f"{name} on the device: {B} contiguous int32 on the tensors' device")
    return t.data_ptr()


def _host_pos(pos: int, T: int, limit: int) -> int:
    """A host position whose T tokens fit below limit (ctypes would wrap a larger int)."""
    if not 0 <= pos <= limit - T:
        raise RuntimeError(f"positions {pos} to {pos + T - 1} outside [0, {limit})")
    return int(pos)


def _batched(x: torch.Tensor, dims: int, name: str) -> torch.Tensor:
    """x with its batch dimension (one sequence may come without)."""
    if x.dim() == dims:
        return x
    if x.dim() == dims - 1:
        return x.unsqueeze(0)
    raise RuntimeError(f"{name} has {x.dim()} dimensions, expected {dims - 1} or {dims}")


def _cache_c(k: torch.Tensor, v: torch.Tensor) -> _lib.KVCacheC:
    """struct i4_kvcache of [n_kv_heads, max_len, head_dim] or [B, n_kv_heads, max_len,
    head_dim] caches (views with any strides above a dense last dimension)."""
    if k.dim() != 4 or v.dim() != 4:
        k, v = _batched(k, 4, "k_cache"), _batched(v, 4, "v_cache")
    shape, strides, dtype = k.shape, k.stride(), k.dtype
    if shape != v.shape or dtype != v.dtype or strides != v.stride():
        raise RuntimeError("k_cache and v_cache must agree in shape, strides and dtype")
    if strides[3] != 1:
        raise RuntimeError("the caches' last dimension must be contiguous")
    return _lib.KVCacheC(k.data_ptr(), v.data_ptr(), strides[0], strides[1], strides[2], *shape,
                         _lib.half_code(dtype))


def _out(out: torch.Tensor | None, like: torch.Tensor, shape: tuple[int, ...],
         padded: bool) -> torch.Tensor:
    """The given output, checked, or a new one (zeros where padding will stay unwritten)."""
    if out is None:
        if padded:
            return torch.zeros(shape, dtype=like.dtype, device=like.device)
        if like.shape == shape and like.is_contiguous():
            return torch.empty_like(like)  # 0.5 us less than spelling it out
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if tuple(out.shape) != shape or out.dtype != like.dtype or not out.is_contiguous():
        raise RuntimeError(f"out must be a contiguous {shape} tensor of {like.dtype}")
    return out


def _call(dev: torch.device, entry, *args) -> None:
    """entry(*args, stream) with the tensors' device current: a launch on the default stream
    goes to the current one."""
    if torch.cuda.current_device() == dev.index:
        rc = entry(*args, _lib.stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = entry(*args, _lib.stream(dev))
    if rc:
        _lib.check(rc)


_STREAM_WS: dict = {}

# Scratch up to which a workspace keeps it from call to call.  Calls of few query rows need at
# most 17 MB; the parts of a long chunk's rows (30 MB for 300 tokens at 32000 positions and the
# Thinker's heads, 339 MB for 2912 at 65536) are memory of that call.
KEPT_BYTES = 1 << 25


def _scratch(workspace: Workspace | None, need: int, dev: torch.device,
             current: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """`need` bytes and the counters: of the caller's workspace, else of one per stream, whose
    calls run in order; under capture one of the call's own, which the graph then owns.  More
    than KEPT_BYTES are the call's own throughout (stream ordered, without counters: only calls
    of few rows count).  The caller holds them until its call is queued (another thread's may
    grow the workspace).  current: dev is the current device, which need not be asked again."""
    if need > KEPT_BYTES:
        return torch.empty(need, dtype=torch.uint8, device=dev), None
    if workspace is None:
        if torch.cuda.is_current_stream_capturing() if current else _capturing(dev):
            workspace = Workspace()
        else:
            key = (dev.index, _lib.stream(dev))
            workspace = _STREAM_WS.get(key) or _STREAM_WS.setdefault(key, Workspace())
            buf, counters = workspace.buf, workspace._counters
            if buf is not None and buf.numel() >= need and counters is not None:
                return buf, counters
    return workspace.get(need, dev), workspace.counters(dev)


def rope_append(qkv: torch.Tensor, n_heads: int, n_kv_heads: int, q_norm_w: torch.Tensor,
                k_norm_w: torch.Tensor, eps: float, inv_freq: torch.Tensor,
                pos: int | torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                first_row: int | None = None, counts: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """RMSNorm over head_dim and rotary embedding of the queries and keys in the fused
    projection rows qkv [T, (n_heads + 2 n_kv_heads) * head_dim] (or [B, T, ...]); returns
    the rotated queries [T, n_heads, head_dim] (or [B, T, ...]) and writes each token's
    rotated key and its value to the caches ([n_kv_heads, max_len, head_dim] or [B, ...]):
    at the row of its position, or at first_row + t when first_row is given.  inv_freq is the
    host fp32 table [head_dim / 2].  fp32 inside, rounded once (i4_rope_append); attn_decode
    and the other one-token entries round the norm, the sines and each product to the dtype, as
    the model's own code does, so their keys differ from these by several half steps."""
    dev = _lib.require_device(qkv, q_norm_w, k_norm_w, k_cache, v_cache, counts, out)
    x = _batched(qkv, 3, "qkv")
    cc = _cache_c(k_cache, v_cache)
    B, T, width = x.shape
    hd = cc.head_dim
    if cc.dtype != _lib.half_code(x.dtype):
        raise RuntimeError("the caches must have the activation dtype")
    if q_norm_w.dtype != x.dtype or k_norm_w.dtype != x.dtype:
        raise RuntimeError("the norm weights must have the activation dtype")
    if q_norm_w.numel() != hd or k_norm_w.numel() != hd:
        raise RuntimeError(f"the norm weights hold head_dim = {hd} values")
    if cc.batch != B or cc.n_kv_heads != n_kv_heads or width != (n_heads + 2 * n_kv_heads) * hd:
        raise RuntimeError("qkv / cache shapes do not match the head counts")
    if inv_freq.numel() != hd // 2:
        raise RuntimeError("inv_freq must hold head_dim / 2 values")
    if x.stride(2) != 1:
        x = x.contiguous()
    if inv_freq.dtype != torch.float32 or inv_freq.device.type != "cpu" \
            or not inv_freq.is_contiguous():
        inv_freq = inv_freq.detach().to("cpu", torch.float32).contiguous()
    q_norm_w, k_norm_w = q_norm_w.contiguous(), k_norm_w.contiguous()
    if first_row is not None:
        if not 0 <= first_row <= cc.max_len - T:
            raise RuntimeError(f"first_row {first_row}: {T} rows do not fit the cache")
    shape = (B, T, n_heads, hd)
    q = _out(out, x, shape if qkv.dim() == 3 else shape[1:], counts is not None)
    on_dev = isinstance(pos, torch.Tensor)
    _call(dev, _lib.lib().i4_rope_append, x.data_ptr(), cc.dtype, T, x.stride(0), x.stride(1),
          n_heads, q_norm_w.data_ptr(), k_norm_w.data_ptr(), eps, inv_freq.data_ptr(),
          _int32(pos, B, dev, "pos") if on_dev else None,
          0 if on_dev else _host_pos(pos, T, cc.max_len if first_row is None else 1 << 24),
          -1 if first_row is None else int(first_row), _int32(counts, B, dev, "counts"),
          q.data_ptr(), ctypes.byref(cc))
    return q


def _attend(entry, cc, keys: int, q: torch.Tensor, dev: torch.device,
            pos: int | torch.Tensor, window: int | None, sinks: int, scale: float | None,
            counts: torch.Tensor | None, out: torch.Tensor | None,
            workspace: Workspace | None) -> torch.Tensor:
    """The call that attn_window and attn_kv8 share; keys: the positions of the cache."""
    x = _batched(q, 4, "q")
    B, T, nh, hd = x.shape
    if B != cc.batch or hd != cc.head_dim:
        raise RuntimeError(f"q {tuple(q.shape)} does not match the cache's batch {cc.batch} and "
                           f"head_dim {cc.head_dim}")
    if window is not None and window < 1:
        raise RuntimeError("window must be at least 1 (None: no bound)")
    sinks = min(sinks, 2**31 - 1)
    if window is None and sinks:
        raise RuntimeError("sinks are the first tokens outside a window: give the window too")
    if x.stride(3) != 1:
        x = x.contiguous()
    y = _out(out, x, (B, T, nh, hd) if q.dim() == 4 else (T, nh, hd), counts is not None)
    on_dev = isinstance(pos, torch.Tensor)
    pd, ph = (_int32(pos, B, dev, "pos"), 0) if on_dev else (None, _host_pos(pos, T, keys))
    w = 0 if window is None else min(window, 2**31 - 1)
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _attend(entry, cc, keys, q, dev, pos, window, sinks, scale, counts, y, workspace)
    need = _lib.lib().i4_attn_window_workspace_bytes(
        B, T, nh, cc.n_kv_heads, keys if on_dev else ph + T, w, sinks)
    ws, counters = _scratch(workspace, need, dev, True) if need else (None, None)
    s0, s1, s2, _ = x.stride()
    rc = entry(x.data_ptr(), _lib.half_code(x.dtype), T, s0, s1, s2, nh, ctypes.byref(cc),
               pd, ph, _int32(counts, B, dev, "counts"), w, sinks,
               hd ** -0.5 if scale is None else scale, y.data_ptr(), _lib.ptr(ws), need,
               _lib.ptr(counters), _lib.stream(dev))
    if rc:
        _lib.check(rc)
    return y


def attn_window(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                pos: int | torch.Tensor, *, window: int | None = None, sinks: int = 0,
                scale: float | None = None, counts: torch.Tensor | None = None,
                out: torch.Tensor | None = None,
                workspace: Workspace | None = None) -> torch.Tensor:
    """Attention of rotated queries q [T, n_heads, head_dim] (or [B, T, ...]) at positions
    pos + t over caches [n_kv_heads, max_len, head_dim] (or [B, ...]) that hold the tokens up
    to and including theirs (rope_append): softmax(scale q k^T) v over the positions j <= p
    and, with a window, j > p - window or j < sinks.  scale defaults to head_dim ** -0.5.
    Scores, maxima and sums are fp32 and the output is rounded once; the weights are rounded
    on their way into the second product: to a sum of two numbers of the activation dtype for
    up to 16 rows of a kv head (T n_heads / n_kv_heads), to one for more (i4_attn_window)."""
    dev = _lib.require_device(q, k_cache, v_cache, counts, out)
    cc = _cache_c(k_cache, v_cache)
    return _attend(_lib.lib().i4_attn_window, cc, cc.max_len, q, dev, pos, window, sinks, scale,
                   counts, out, workspace)


class KV8Cache:
    """A KV cache in 8 bits with one fp32 scale for each block of 64 tokens and head:

    k [B, n_kv_heads, blocks, 64, head_dim] and v [B, n_kv_heads, blocks, head_dim, 64]
    (value blocks are kept transposed), int8 or float8_e4m3fn; k_scale, v_scale
    [B, n_kv_heads, blocks] fp32; k_tail, v_tail [B, n_kv_heads, 64, head_dim] in 16 bits, the
    tokens of the unfinished block.  The kernels write the tensors in place and the object
    holds their addresses, so they cannot be replaced."""

    __slots__ = ("_t", "_c")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor, k_tail: torch.Tensor, v_tail: torch.Tensor):
        _lib.require_device(k, v, k_scale, v_scale, k_tail, v_tail)
        if k.dtype not in _FORMATS or v.dtype != k.dtype:
            raise RuntimeError(f"k and v are int8 or float8_e4m3fn, got {k.dtype}, {v.dtype}")
        if k.dim() != 5 or k.shape[3] != KV8_BLOCK:
            raise RuntimeError("k is [B, n_kv_heads, blocks, 64, head_dim]")
        B, n, blocks, _, hd = k.shape
        want = {"v": (v, (B, n, blocks, hd, KV8_BLOCK)), "k_scale": (k_scale, (B, n, blocks)),
                "v_scale": (v_scale, (B, n, blocks)), "k_tail": (k_tail, (B, n, KV8_BLOCK, hd)),
                "v_tail": (v_tail, (B, n, KV8_BLOCK, hd)), "k": (k, tuple(k.shape))}
        for name, (t, shape) in want.items():
            if tuple(t.shape) != shape or not t.is_contiguous():
                raise RuntimeError(f"{name} must be a contiguous {shape} tensor")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise RuntimeError("the scales are float32")
        if k_tail.dtype != v_tail.dtype:
            raise RuntimeError("k_tail and v_tail must have one dtype")
        self._t = (k, v, k_scale, v_scale, k_tail, v_tail)
        self._c = _lib.KV8CacheC(*(t.data_ptr() for t in self._t), B, n, blocks, hd,
                                 _lib.half_code(k_tail.dtype), _FORMATS[k.dtype])

    @classmethod
    def empty(cls, n_kv_heads: int, max_len: int, head_dim: int = 128, *, batch: int = 1,
              dtype: torch.dtype = torch.bfloat16, kind: torch.dtype = torch.int8,
              device: torch.device | str = "cuda") -> "KV8Cache":
        """A cache of zeros for max_len tokens (rounded up to whole blocks)."""
        blocks = -(-max_len // KV8_BLOCK)
        shape = (batch, n_kv_heads, blocks)
        bits = [torch.zeros(*shape, *s, dtype=torch.int8, device=device).view(kind)
                for s in ((KV8_BLOCK, head_dim), (head_dim, KV8_BLOCK))]
        scales = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)]
        tails = [torch.zeros(batch, n_kv_heads, KV8_BLOCK, head_dim, dtype=dtype, device=device)
                 for _ in range(2)]
        return cls(*bits, *scales, *tails)

    @property
    def tensors(self) -> tuple[torch.Tensor, ...]:
        """k, v, k_scale, v_scale, k_tail, v_tail: what the constructor takes."""
        return self._t

    k = property(lambda self: self._t[0])
    v = property(lambda self: self._t[1])
    k_scale = property(lambda self: self._t[2])
    v_scale = property(lambda self: self._t[3])
    k_tail = property(lambda self: self._t[4])
    v_tail = property(lambda self: self._t[5])

    @property
    def max_len(self) -> int:
        return self._c.blocks * KV8_BLOCK

    def reset(self) -> None:
        """Empty the cache in place (a new conversation)."""
        for t in self._t:
            (t.view(torch.int8) if t.element_size() == 1 else t).zero_()

    def values(self) -> tuple[torch.Tensor, torch.Tensor]:
        """What the finished blocks stand for: k and v [B, n_kv_heads, max_len, head_dim]
        fp32 (i4_kv8_values; the tail's tokens are not among them)."""
        c, dev = self._c, self._t[0].device
        out = torch.empty(2, c.batch, c.n_kv_heads, self.max_len, c.head_dim, dtype=torch.float32,
                          device=dev)
        k, v = out.unbind(0)
        _call(dev, _lib.lib().i4_kv8_values, ctypes.byref(c), k.data_ptr(), v.data_ptr())
        return k, v


def kv8_append(k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, pos: int | torch.Tensor, *,
               counts: torch.Tensor | None = None) -> None:
    """The rotated keys and the values of T tokens, k and v [T, n_kv_heads, head_dim] (or
    [B, T, ...], any strides above a dense last dimension), into the cache behind the pos
    tokens it holds (i4_kv8_append).  The blocks that they finish are rounded from 16 bits;
    the rest goes to the tail.  Tokens arrive in order: pos is what the cache holds, or lies
    in its unfinished block."""
    c = cache._c
    dev = _lib.require_device(k, v, cache._t[0], counts)
    k, v = _batched(k, 4, "k"), _batched(v, 4, "v")
    if k.shape != v.shape or k.dtype != v.dtype:
        raise RuntimeError("k and v must agree in shape and dtype")
    if k.stride() != v.stride() or k.stride(3) != 1:
        k, v = k.contiguous(), v.contiguous()
    B, T, n, hd = k.shape
    if (B, n, hd) != (c.batch, c.n_kv_heads, c.head_dim):
        raise RuntimeError(f"k {tuple(k.shape)} does not match the cache")
    on_dev = isinstance(pos, torch.Tensor)
    _call(dev, _lib.lib().i4_kv8_append, k.data_ptr(), v.data_ptr(), _lib.half_code(k.dtype), T,
          *k.stride()[:3], ctypes.byref(c), _int32(pos, B, dev, "pos") if on_dev else None,
          0 if on_dev else _host_pos(pos, T, cache.max_len), _int32(counts, B, dev, "counts"))


def attn_kv8(q: torch.Tensor, cache: KV8Cache, pos: int | torch.Tensor, *,
             window: int | None = None, sinks: int = 0, scale: float | None = None,
             counts: torch.Tensor | None = None, out: torch.Tensor | None = None,
             workspace: Workspace | None = None) -> torch.Tensor:
    """attn_window over an 8-bit cache whose last tokens are the queries' own (kv8_append):
    positions in the finished blocks of the pos + T (or counts) tokens are read in 8 bits, the
    unfinished block from the tail (i4_attn_kv8).  A query of several therefore reads its own
    block, if the call finished it, in 8 bits with a scale that later tokens have a part in
    (one that is not finite makes the block NaN); token by token it is read in 16 bits."""
    dev = _lib.require_device(q, cache._t[0], counts, out)
    return _attend(_lib.lib().i4_attn_kv8, cache._c, cache.max_len, q, dev, pos, window, sinks,
                   scale, counts, out, workspace)
