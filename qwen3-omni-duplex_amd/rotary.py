"""Rotary embeddings of any model's queries and keys.

    Rotary   a rotation as the kernels take it: which dims pair, how fast each pair turns
    rope     queries and keys turned by their positions

rope_append (kv.py) turns the Thinker's heads by a plain table on their way into a cache; these
take neighbouring pairs, part of a head, tables scaled for long contexts, positions given for
each token, and the several positions of an image's or a video's tokens (the reference's model
turns its pairs by three axes then: Qwen3OmniMoeThinkerTextRotaryEmbedding, transformers 5.15).
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Sequence

import torch

from . import _lib
from .kv import _batched, _call, _int32

_heads = struct.Struct("<2Q6qi4x").pack  # struct i4_heads
_turn = struct.Struct("<Q2qi4x").pack    # struct i4_turn
_empty = torch.empty_like
_DENSE = torch.contiguous_format
LAYOUTS = {"half": 0, "interleaved": 1}
MAX_PAIRS = 128
MAX_POS = 1 << 24


class Rotary(_lib.Handle):
    """Pair i of a head's first 2 len(inv_freq) dims turns by the angle position * inv_freq[i]:
    dims i and i + len(inv_freq) (layout "half") or 2 i and 2 i + 1 ("interleaved").  factor
    multiplies cos and sin (the attention factor of a scaled table).  axes: for tokens that are
    given several positions, which of them each pair turns by.  The table is copied to the host;
    the kernels take it from there, so none of this can be replaced (AttributeError)."""

    __slots__ = ("inv_freq", "layout", "factor", "axes", "dims", "_bytes", "_c", "_at")

    def __init__(self, inv_freq: torch.Tensor, *, layout: str = "half", factor: float = 1.0,
                 axes: Sequence[int] | None = None):
        f = inv_freq.detach().to("cpu", torch.float32).clone().contiguous()
        n = f.numel()
        if f.dim() != 1 or not 1 <= n <= MAX_PAIRS:
            raise RuntimeError(f"inv_freq holds 1 to {MAX_PAIRS} values, got {tuple(f.shape)}")
        if not bool((f.abs() <= 16).all()):
            raise RuntimeError("inverse frequencies are finite and at most 16")
        if layout not in LAYOUTS:
            raise RuntimeError(f"layout is one of {sorted(LAYOUTS)}, got {layout!r}")
        if not math.isfinite(factor):
            raise RuntimeError(f"factor is {factor}")
        if axes is not None and (len(axes) != n or not all(0 <= a < 4 for a in axes)):
            raise RuntimeError(f"axes: {n} numbers from 0 to 3")
        self.inv_freq, self.layout, self.factor = f, layout, float(factor)
        self.dims = 2 * n  # of a head that turn
        self.axes = None if axes is None else tuple(int(a) for a in axes)
        self._bytes = None if axes is None else (ctypes.c_uint8 * n)(*self.axes)
        self._c = _lib.RotaryC(f.data_ptr(), None if axes is None else
                               ctypes.addressof(self._bytes), self.factor, n, LAYOUTS[layout])
        self._at = ctypes.addressof(self._c)

    @classmethod
    def plain(cls, dims: int, theta: float, **kw) -> "Rotary":
        """The default table of `dims` turning dims: theta ** (-2 i / dims)."""
        return cls(1.0 / theta ** (torch.arange(0, dims, 2, dtype=torch.float) / dims), **kw)

    @classmethod
    def scaled(cls, dims: int, theta: float, scale: float, trained: int | None = None, *,
               slow: float = 1.0, fast: float = 32.0, blend: str = "turns", whole: bool = True,
               factor: float | None = None, **kw) -> "Rotary":
        """A table for contexts `scale` times as long as the model was trained for.

        trained None: every position is divided by scale.  Else by parts (arXiv 2309.00071): a
        pair that turns more than `fast` times within `trained` positions keeps its frequency,
        one that turns less than `slow` times has it divided by scale, and those between are
        blended; factor defaults to 0.1 ln(scale) + 1.  blend says by what:

        "turns"  by their number of turns, as that paper's text has it
        "pairs"  by their number, linearly between the two bounds, each a pair's number (whole:
                 the next whole one outwards).  That is the table of published checkpoints whose
                 config says "yarn"; the frequencies in between differ from the other rule's by
                 up to half."""
        if not scale >= 1 or not fast > slow or not slow > 0:
            raise RuntimeError("scale is at least 1, and fast above slow above 0")
        if blend not in ("turns", "pairs"):
            raise RuntimeError(f"blend is 'turns' or 'pairs', got {blend!r}")
        i = torch.arange(0, dims, 2, dtype=torch.double)
        f = theta ** (-i / dims)
        if trained is None:
            f = f / scale
        else:
            if blend == "turns":
                keep = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
            else:
                # pair n turns trained theta ** (-2 n / dims) / (2 pi) times
                lo, hi = (dims * math.log(trained / (2 * math.pi * n)) / (2 * math.log(theta))
                          for n in (fast, slow))
                if whole:
                    lo, hi = math.floor(lo), math.ceil(hi)
                lo, hi = max(lo, 0), min(hi, dims - 1)
                if lo > hi:
                    raise RuntimeError(f"no pair turns between {slow} and {fast} times within "
                                       f"{trained} positions")
                # (bounds at one pair: a step behind it)
                keep = 1 - ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            f = f * keep + f / scale * (1 - keep)
            factor = 0.1 * math.log(scale) + 1 if factor is None else factor
        return cls(f.float(), factor=1.0 if factor is None else factor, **kw)

    def __reduce__(self):
        return _rebuilt, (self.inv_freq, self.layout, self.factor, self.axes)

    def __repr__(self) -> str:
        return (f"Rotary(dims={self.dims}, layout={self.layout!r}, factor={self.factor}"
                + (f", axes={self.axes}" if self.axes else "") + ")")


def _rebuilt(inv_freq, layout, factor, axes) -> Rotary:
    return Rotary(inv_freq, layout=layout, factor=factor, axes=axes)


def interleaved_axes(sections: Sequence[int]) -> tuple[int, ...]:
    """The axes of a multimodal rotary embedding whose sections are interleaved: the pairs take
    the axes in turn, axis a > 0 for its sections[a] first turns, and axis 0 otherwise."""
    axes = [0] * sum(sections)
    for a in range(1, len(sections)):
        for i in range(a, min(len(axes), len(sections) * sections[a]), len(sections)):
            axes[i] = a
    return tuple(axes)


def _turn_c(turn: torch.Tensor, rotary: Rotary, batched: bool, B: int, T: int,
            dev: torch.device) -> bytes:
    """struct i4_turn of given positions [B, T] or [axes, B, T] ([T] or [axes, T] for tokens
    without a batch)."""
    t = turn if batched else turn.unsqueeze(-2) if turn.dim() else turn
    shape = tuple(t.shape)
    if shape[-2:] != (B, T) or len(shape) > 3:
        raise RuntimeError(f"given positions {tuple(turn.shape)} for {B} x {T} tokens")
    axes = shape[0] if len(shape) == 3 else 1
    if axes > 1 and (axes > 4 or rotary.axes is None or max(rotary.axes) >= axes):
        raise RuntimeError(f"positions on {axes} axes for a rotary embedding with "
                           f"{'none' if rotary.axes is None else max(rotary.axes) + 1}")
    if turn.dtype != torch.int32 or turn.device != dev or (T > 1 and t.stride(-1) != 1):
        raise RuntimeError("given positions are int32 on the tensors' device, tokens adjacent")
    return _turn(turn.data_ptr(), t.stride(0) if axes > 1 else 0, t.stride(-2) if B > 1 else 0,
                 axes)


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The first byte that a tensor covers, and the one behind its last."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def overlaps(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether elements of x may be elements of y (of as many dimensions): their memory meets, and
    they are not separate parts of one strided tensor, as q and k of a fused projection are."""
    (a, b), (c, d) = _span(x), _span(y)
    if b <= c or d <= a:
        return False
    if a > c:
        x, y, a, c = y, x, c, a
    if x.element_size() != y.element_size() or (c - a) % x.element_size():
        return True
    dims = []  # (stride, x's size, y's size) where one of them has several
    for n, s, m, t in zip(x.shape, x.stride(), y.shape, y.stride()):
        if n > 1 and m > 1 and s != t:
            return True
        if n > 1 or m > 1:
            dims.append((s if n > 1 else t, n, m))
    # where y begins in x's steps, from the largest; x lies at [0, n) and y at [q, q + m) of each
    off, apart, inner = (c - a) // x.element_size(), False, []
    for s, n, m in sorted(dims, reverse=True):
        q = off // s if s else 0
        off -= q * s
        apart |= q >= n
        inner.append((s, max(n, q + m)))
    # what the smaller steps reach must stay below a step, or places are not unique
    reach = off
    for s, n in reversed(inner):
        if reach >= s:
            return True
        reach += (n - 1) * s
    return not apart and off == 0


def distinct(size: int, *dims: tuple[int, int]) -> bool:
    """Whether blocks of `size` adjacent elements, dims of (count, stride) of them, are distinct:
    each dimension steps over all that the smaller strides reach."""
    for n, s in sorted(dims, key=lambda d: d[1]):
        if n > 1:
            if s < size:
                return False
            size += (n - 1) * s
    return True


def _dense(shape: tuple[int, ...], stride: tuple[int, ...]) -> bool:
    """Whether the rows [B, T, heads, head_dim] are as the entry reads them."""
    hd = shape[3]
    return stride[3] == 1 and (shape[2] == 1 or stride[2] >= hd) and (
        shape[1] == 1 or stride[1] >= hd) and (shape[0] == 1 or stride[0] >= hd)


def _new(x: torch.Tensor, T: int, hd: int, held: list[torch.Tensor]) -> bytes:
    """A dense output for x [B, T, heads, hd], appended to held, and struct i4_heads of both.
    What the struct points at is held until the call is queued."""
    B, _, n, _ = x.shape
    a, b, c, d = x.stride()
    if d != 1 or c < hd and n > 1 or b < hd and T > 1 or a < hd and B > 1:
        x = x.contiguous()
        a, b, c, _ = x.stride()
        held.insert(0, x)
    y = _empty(x, memory_format=_DENSE)
    held.append(y)
    return _heads(x.data_ptr(), y.data_ptr(), a, b, c, T * n * hd, n * hd, hd, n)


def _into(xs: list[torch.Tensor], out: tuple[torch.Tensor | None, ...],
          held: list[torch.Tensor]) -> list[bytes | None]:
    """struct i4_heads of the inputs and the given outputs, checked."""
    outs = list(out)
    if len(outs) == 2 and len(xs) == 1 and outs[1] is None:
        outs.pop()
    if len(outs) != len(xs) or any(t is None for t in outs):
        raise RuntimeError("out holds a tensor for each input")
    _lib.require_device(*xs, *outs)
    cs, ys = [], [_batched(t, 4, "out") for t in outs]
    if len(ys) > 1 and (overlaps(ys[0], ys[1]) or overlaps(ys[0], xs[1])
                        or overlaps(ys[1], xs[0])):
        raise RuntimeError("an output overlaps the other one or the other input")
    for y, x in zip(ys, xs):
        if y.shape != x.shape or y.dtype != x.dtype:
            raise RuntimeError(f"out must be a {tuple(x.shape)} tensor of {x.dtype}")
        if not _dense(y.shape, y.stride()) \
                or not distinct(y.shape[3], *zip(y.shape[:3], y.stride()[:3])):
            raise RuntimeError("out's rows must be dense and lie apart")
        if y.data_ptr() != x.data_ptr() or y.stride() != x.stride():  # not in place
            if overlaps(y, x):
                raise RuntimeError("out is its input itself or does not overlap it")
            if not _dense(x.shape, x.stride()):
                x = x.contiguous()
                held.append(x)
        cs.append(_heads(x.data_ptr(), y.data_ptr(), *x.stride()[:3], *y.stride()[:3],
                         x.shape[2]))
    return cs if len(cs) > 1 else [cs[0], None]


def rope(q: torch.Tensor, k: torch.Tensor | None, pos: int | torch.Tensor, rotary: Rotary, *,
         counts: torch.Tensor | None = None,
         out: tuple[torch.Tensor, torch.Tensor | None] | None = None):
    """The rotary embedding of queries q [T, heads, head_dim] (or [B, T, ...]) and, if given, of
    keys k with heads of their own: (q, k) turned, or q alone where k is None.  fp32 inside (the
    angles as good as exact for every position within 2^24), rounded once (i4_rope).

    pos: an int or int32 [B] on the device, the position of each sequence's first token; or the
    positions of the tokens themselves, int32 [B, T] on the device, or [axes, B, T] for a rotary
    embedding with axes ([T] or [axes, T] for tokens without a batch); with one position a token
    every pair turns by it, as text tokens do.  A position at or behind +-2^24 gives NaN, an int
    is refused.

    Negative positions turn back: with p the tokens' own positions ([B, T] or [axes, B, T]; T
    tokens behind a start take theirs, since -start is a start again) rope(rope(x, p), -p) is
    factor ** 2 x to rounding, and rope(dy, -p) the gradient of rope(x, p).  No autograd graph is
    recorded.

    q and k may have any strides above a dense last dimension, and so may out, a pair of tensors
    that are q and k themselves (in place) or do not overlap them, each other or themselves.
    Padding (counts, int32 [B] on the device) is zeros in new outputs and left as it is in given
    ones."""
    dev = _lib.require_device(q, k, counts)
    code = _lib.half_code(q.dtype)
    batched = q.dim() == 4
    x = q if batched else _batched(q, 4, "q")
    B, T, _, hd = x.shape
    xs = [x]
    if k is not None:
        z = k if batched else k.unsqueeze(0)
        if z.dim() != 4 or z.shape[0] != B or z.shape[1] != T or z.shape[3] != hd:
            raise RuntimeError(f"q {tuple(q.shape)} and k {tuple(k.shape)} do not match")
        if k.dtype != q.dtype:
            raise RuntimeError("q and k must have one dtype")
        xs.append(z)
    if rotary.dims > hd:
        raise RuntimeError(f"{rotary.dims} dims turn, the heads have {hd}")
    turn = pd = None
    ph = 0
    if not isinstance(pos, torch.Tensor):
        ph = int(pos)
        if not -MAX_POS < ph <= MAX_POS - T:
            raise RuntimeError(f"positions {ph} to {ph + T - 1} outside (-2^24, 2^24)")
    elif pos.dim() == 1 and (batched or pos.numel() == 1):
        pd = _int32(pos, B, dev, "pos")
    else:
        turn = _turn_c(pos, rotary, batched, B, T, dev)
    held: list[torch.Tensor] = []  # the new outputs are its last elements
    if out is None:
        qc = _new(x, T, hd, held)
        kc = None if k is None else _new(xs[1], T, hd, held)
    else:
        qc, kc = _into(xs, out, held)
    _call(dev, _lib.lib().i4_rope, qc, kc, code, B, T, hd, rotary._at, pd, ph, turn,
          None if counts is None else _int32(counts, B, dev, "counts"), out is None)
    if out is not None:
        return out[0] if k is None else (out[0], out[1])
    if not batched:
        held = [y[0] for y in held]
    return held[-1] if k is None else (held[-2], held[-1])
