"""What the handles and calls of the paged cache and the rotary embeddings promise beyond their
results: on the host, before any launch."""
from __future__ import annotations

import copy

import pytest
import torch

from tests.test_kv import ALIGN, STRIDE, WORKSPACE, P
from tests.test_paged import cache, call_append, call_attn, call_rope, heads
from tests.test_paged import lb  # noqa: F401 (a fixture)
from tests.test_paged import rotary as rot

BF = torch.bfloat16


@pytest.fixture
def on_cpu(pkg, monkeypatch):
    """Tensors of the CPU pass for the device's: checks that come before any address is used."""
    from qwen3_omni_duplex_amd import _lib

    monkeypatch.setattr(_lib, "require_device", lambda *ts: torch.device("cpu"))
    return pkg


def pool(pkg, shape=(4, 2, 16, 128)):
    return pkg.PagedCache(torch.zeros(shape, dtype=BF), torch.zeros(shape, dtype=BF))


def test_a_pool_keeps_its_tensors(on_cpu):
    """The kernels hold the tensors' addresses: nothing can be put in their place, and what the
    object says of itself stays what they read."""
    c = pool(on_cpu)
    k, other = c.k, torch.zeros_like(c.k)
    for name, value in (("k", other), ("v", other), ("device", "cpu"), ("dtype", torch.float16),
                        ("page", 32), ("pages", 9), ("_c", ()), ("k", c.k)):
        with pytest.raises(AttributeError):
            setattr(c, name, value)
    for name in ("k", "v", "_c"):
        with pytest.raises(AttributeError):
            delattr(c, name)
    assert c.k is k and c._c[4] == k.data_ptr() and c.page == 16
    d = copy.deepcopy(c)
    assert d.k.data_ptr() == d._c[4] != c._c[4]


def test_a_rotary_embedding_keeps_its_table(pkg):
    """The struct that the kernels read holds the table's address, the layout and the factor."""
    r = pkg.Rotary.plain(32, 1e4, factor=1.5, axes=[0, 1] * 8)
    f = r.inv_freq
    for name, value in (("factor", 3.0), ("inv_freq", torch.ones(16)), ("layout", "interleaved"),
                        ("axes", None), ("dims", 16), ("_c", None), ("_bytes", None), ("_at", 0)):
        with pytest.raises(AttributeError):
            setattr(r, name, value)
    with pytest.raises(AttributeError):
        del r.inv_freq
    assert r.inv_freq is f and r._c.inv_freq == f.data_ptr()
    assert (r.factor, r._c.factor, r.layout, r._c.layout, r.dims) == (1.5, 1.5, "half", 0, 32)
    assert copy.deepcopy(r).factor == 1.5


def distinct_elements(x):
    """Whether no two places of a view are one element (by counting them)."""
    at = torch.zeros(1, dtype=torch.long)
    for n, s in zip(x.shape, x.stride()):
        at = (at[:, None] + torch.arange(n) * s).flatten()
    return at.unique().numel() == at.numel()


POOLS = [  # pages, heads, strides of pages and heads in pages' rows (16 x 128 values), distinct
    (4, 4, 1, 1, False), (4, 4, 4, 1, True), (4, 4, 1, 4, True), (4, 4, 3, 1, False),
    (4, 4, 1, 3, False), (5, 3, 3, 1, True), (5, 3, 1, 5, True), (5, 3, 1, 4, False),
    (3, 4, 9, 2, True), (3, 4, 2, 6, True), (1, 4, 1, 1, True), (4, 1, 1, 1, True),
    (1, 4, 0, 1, True), (4, 1, 1, 0, True), (2, 2, 0, 1, False)]


@pytest.mark.parametrize("pages,heads,ps,hs,good", POOLS)
def test_pages_of_a_pool_are_distinct(lb, on_cpu, pages, heads, ps, hs, good):  # noqa: F811
    """Pages or heads that lie on each other would be written by several sessions or heads."""
    rows = 16 * 128
    k, v = (torch.zeros(40 * rows, dtype=BF).as_strided(
        (pages, heads, 16, 128), (ps * rows, hs * rows, 128, 1)) for _ in range(2))
    assert distinct_elements(k) == good
    bad = dict(pages=pages, n_kv_heads=heads, page=16, page_stride=ps * rows, head_stride=hs * rows)
    if good:
        assert on_cpu.PagedCache(k, v).pages == pages
        # the C entries come as far as the checks behind it, and are stopped there
        assert call_append(lb, on_cpu.lib(), cache(lb, **bad), nh=heads, qkv=P + 2) == ALIGN
        assert call_attn(lb, on_cpu.lib(), cache(lb, **bad), nh=heads, q=P + 2) == ALIGN
    else:
        with pytest.raises(RuntimeError, match="overlap"):
            on_cpu.PagedCache(k, v)
        assert call_append(lb, on_cpu.lib(), cache(lb, **bad), nh=heads, qkv=P + 2) == STRIDE
        assert call_attn(lb, on_cpu.lib(), cache(lb, **bad), nh=heads, q=P + 2) == STRIDE


OUTPUTS = [  # strides of sequences, tokens and heads in rows (2 x 3 x 4 of 16 dims), distinct
    ((12, 4, 1), True), ((12, 1, 3), True), ((4, 8, 1), True), ((1, 8, 2), True),
    ((40, 9, 2), True), ((12, 1, 1), False), ((12, 4, 4), False), ((12, 3, 1), False),
    ((12, 1, 2), False), ((9, 4, 1), False), ((1, 1, 1), False), ((4, 4, 1), False)]


@pytest.mark.parametrize("strides,good", OUTPUTS)
def test_rows_of_an_output_are_distinct(lb, on_cpu, strides, good):  # noqa: F811
    """Rows that lie on each other are written by several workgroups at once."""
    (b, t, h), hd = strides, 16
    y = torch.zeros(100 * hd, dtype=BF).as_strided((2, 3, 4, hd), (b * hd, t * hd, h * hd, 1))
    x = torch.zeros(2, 3, 4, hd, dtype=BF)
    r = on_cpu.Rotary.plain(hd, 1e4)
    assert distinct_elements(y) == good
    c = dict(xb=192, xt=64, xh=16, yb=b * hd, yt=t * hd, yh=h * hd, heads=4)
    one = dict(pairs=8)
    if good:  # as far as the next check, in place too
        assert call_rope(lb, on_cpu.lib(), heads(lb, **c), r=rot(lb, **one), hd=hd, T=3,
                         pos_dev=P + 2) == ALIGN
    else:
        for out in ((y, None), (x, y)):
            with pytest.raises(RuntimeError, match="apart"):
                on_cpu.rope(x, None if out[1] is None else x.clone(), 0, r, out=out)
        with pytest.raises(RuntimeError, match="apart"):
            on_cpu.rope(y, None, 0, r, out=(y, None))
        for q, k in ((c, None), ({}, c)):
            base = dict(xb=192, xt=64, xh=16, yb=192, yt=64, yh=16, heads=4)
            assert call_rope(lb, on_cpu.lib(), heads(lb, **{**base, **q}),
                             k and heads(lb, **k), r=rot(lb, **one), hd=hd, T=3,
                             pos_dev=P + 2) == STRIDE


def test_outputs_lie_outside_the_pool(on_cpu, monkeypatch):
    """A call reads or writes the pool while it writes its output."""
    room = torch.zeros(3, 4, 2, 16, 128, dtype=BF)  # two pools, and rows behind them
    c = on_cpu.PagedCache(room[0], room[1])
    t = torch.zeros(1, 2, dtype=torch.int32)
    q, x = torch.zeros(1, 3, 4, 128, dtype=BF), torch.zeros(1, 3, 8 * 128, dtype=BF)
    r = on_cpu.Rotary.plain(128, 1e4)
    flat = room.view(-1, 128)
    edge = 2 * 4 * 2 * 16  # the first row behind the pools
    for row in (0, 100, 128, edge - 12, edge - 1):
        out = flat[row:row + 12].view(1, 3, 4, 128)
        with pytest.raises(RuntimeError, match="overlap the pool"):
            on_cpu.attn_paged(q, c, t, 0, out=out)
        with pytest.raises(RuntimeError, match="overlap the pool"):
            on_cpu.paged_append(x, 4, None, None, 1e-6, r, 0, c, t, out=out)
        with pytest.raises(RuntimeError, match="overlap the pool"):
            on_cpu.attn_paged(q[0], c, t[0], 0, out=out[0])
    behind = flat[edge:edge + 12].view(1, 3, 4, 128)
    for call in (lambda: on_cpu.attn_paged(q, c, t, 40, out=behind),
                 lambda: on_cpu.paged_append(x, 4, None, None, 1e-6, r, 40, c, t, out=behind)):
        with pytest.raises(RuntimeError, match="outside"):  # the check behind this one
            call()


@pytest.mark.parametrize("B,T,nh,nkv,pos,window", [
    (2, 100, 32, 4, 8000, 0), (4, 400, 32, 4, 9000, 0), (2, 100, 32, 4, 8000, 3000),
    (1, 64, 32, 4, 30000, 0), (3, 17, 8, 1, 16000, 0), (24, 1, 32, 4, 20000, 0),
    (1, 1, 8, 2, 5000, 0), (2, 300, 8, 2, 100, 0)])
@pytest.mark.parametrize("form", ["host", "counts", "device"])
def test_a_call_needs_the_scratch_that_it_uses(lb, pkg, B, T, nh, nkv, pos, window,  # noqa: F811
                                               form):
    """One byte less than i4_attn_paged_call_bytes is refused, that many are not.  A call whose
    lengths the host knows is split as attn_window's of many rows are, and needs no more."""
    lib = pkg.lib()
    n = -(-(pos + T) // 64)
    keys = n * 64 if form == "device" else pos + T
    size = (B, T, nh, nkv, keys, window, 0)
    need = lib.i4_attn_paged_call_bytes(*size, form != "host")
    assert need <= lib.i4_attn_paged_workspace_bytes(*size) \
        == max(lib.i4_attn_paged_call_bytes(*size, d) for d in (0, 1))
    if form == "host" and T * nh // nkv > 16:
        assert need == lib.i4_attn_window_workspace_bytes(*size)
    c = cache(lb, batch=B, n_kv_heads=nkv, table_len=n, table_stride=n, pages=5)
    a = dict(T=T, nh=nh, ts=nh * 128, bs=T * nh * 128, window=window,
             pos=0 if form == "device" else pos, pos_dev=P if form == "device" else None,
             counts=P if form == "counts" else None)
    if need:
        assert call_attn(lb, lib, c, **a, wsb=need - 1) == WORKSPACE
        assert call_attn(lb, lib, c, **a, wsb=need, ws=P + 128) == ALIGN  # the check behind it


@pytest.mark.parametrize("hd", [64, 96, 256])
def test_a_pool_of_other_heads_is_refused(on_cpu, hd):
    """No call takes it."""
    with pytest.raises(RuntimeError, match="128 dims"):
        pool(on_cpu, (4, 2, 16, hd))
    with pytest.raises(RuntimeError, match="128 dims"):
        on_cpu.PagedCache.empty(2, 4, 16, hd, device="cpu")
