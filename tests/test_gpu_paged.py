"""paged_append and attn_paged on the GPU against 64 bits, and against the same calls over one
run of rows."""
from __future__ import annotations

import math

import pytest
import torch

from tests import _kv_ref as kvref
from tests import _paged_ref as ref
from tests.test_gpu_kv import DTS, HD, check, i32, rand, same, starts

pytestmark = pytest.mark.gpu
QNAN = float("nan")


def pool_of(pkg, dev, rows, need, page, seed=0, spare=3, width=None, fill=QNAN):
    """rows [2, B, nkv, n, HD] (k and v of every position) in a pool in no order: the cache and
    its table.  need: a sequence's first positions that have a page.  Everything else in the
    pool is `fill`, entries without a page are alternately -1 and beyond the pool."""
    _, B, nkv, n, _ = rows.shape
    g = torch.Generator().manual_seed(seed)
    entries = [-(-x // page) for x in need]
    ids = torch.randperm(sum(entries) + spare, generator=g).tolist()
    width = max(max(entries), 1) if width is None else width
    table = torch.tensor([[-1, 2**31 - 1][i % 2] for i in range(B * width)],
                         dtype=torch.int32).view(B, width)
    kv = torch.full((2, len(ids), nkv, page, HD), fill, dtype=rows.dtype, device=dev)
    for b in range(B):
        for i in range(entries[b]):
            table[b, i] = ids.pop()
            part = rows[:, b, :, i * page:min((i + 1) * page, need[b])]
            kv[:, table[b, i], :, :part.shape[2]] = part
    return pkg.PagedCache(kv[0], kv[1]), table.to(dev)


def case(dev, B, T, nh, nkv, n, dtype, seed=0):
    q = rand(dev, B, T, nh, HD, seed=seed, dtype=dtype, gain=1.5)
    rows = rand(dev, 2, B, nkv, n, HD, seed=seed + 1, dtype=dtype)
    rows[1] += 0.25
    return q, rows


def dirty(x):
    """Leaves memory of x's size, not zeros, to the next allocation."""
    torch.full_like(x, 5.0, memory_format=torch.contiguous_format)


@pytest.mark.parametrize("T,nh,pos", [(1, 8, 100), (1, 8, 9000), (2, 8, 500), (40, 8, 100),
                                      (40, 8, 9000)])
def test_padding_of_a_new_output_is_zeros(pkg, dev, T, nh, pos):
    """On every path: one part and several, few rows and many, one sequence (split by its cost)
    and two (shared out); appended rows too."""
    for B in (1, 2):
        q, rows = case(dev, B, T, nh, 2, pos + T, torch.bfloat16)
        cache, table = pool_of(pkg, dev, rows, [pos + T] * B, 64)
        for counts in ([T, 0][:B], [0, T - 1][:B], [T // 2, T][:B]):
            dirty(q)
            got = pkg.attn_paged(q, cache, table, i32(dev, [pos] * B), counts=i32(dev, counts))
            want = pkg.attn_paged(q, cache, table, i32(dev, [pos] * B), counts=i32(dev, counts),
                                  out=torch.full_like(q, 5.0))
            qkv = rand(dev, B, T, (nh + 4) * HD, seed=3)
            dirty(q)
            new = pkg.paged_append(qkv, nh, None, None, 1e-6, pkg.Rotary.plain(HD, 1e4),
                                   i32(dev, [pos] * B), cache, table, counts=i32(dev, counts))
            for b, n in enumerate(counts):
                assert same(got[b, :n], want[b, :n]) and not got[b, n:].any()
                assert (want[b, n:] == 5.0).all() and not new[b, n:].any() and new[b, :n].any() == (n > 0)


# ------------------------------------------------------------------- attention

SHAPES = [
    (1, 1, 32, 4, 0, None, 0),        # the first token
    (1, 1, 32, 4, 64, None, 0),
    (1, 1, 1, 1, 700, None, 0),
    (1, 1, 7, 1, 1000, 100, 3),
    (1, 1, 32, 4, 4000, 1, 0),        # itself alone
    (1, 1, 32, 4, 4000, 1, 1),
    (2, 1, 40, 2, 900, 333, 400),     # more sinks than the window
    (3, 1, 16, 16, 2100, 2000, 64),
    (1, 2, 32, 4, 511, 128, 4),
    (5, 3, 28, 4, 130, None, 0),
    (2, 8, 32, 4, 64, 5000, 4),       # a window longer than the context
    (1, 17, 32, 4, 0, None, 0),
    (1, 33, 6, 2, 31, 16, 5),
    (1, 63, 4, 4, 1, 64, 0),
    (2, 64, 8, 2, 0, 65, 1),
    (1, 130, 8, 1, 300, 100, 20),
    (3, 40, 8, 4, 500, None, 0),
    (1, 257, 4, 2, 15, 300, 33)]


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("B,T,nh,nkv,pos,window,sinks", SHAPES)
def test_attention_matches_64_bits(pkg, dev, dtype, page, B, T, nh, nkv, pos, window, sinks):
    """Pages in no order, NaN in every row behind the last one and in every other page."""
    at = starts(pos, B)
    n = pos + T
    q, rows = case(dev, B, T, nh, nkv, n, dtype)
    cache, table = pool_of(pkg, dev, rows, [p + T for p in at], page)
    got = pkg.attn_paged(q, cache, table, i32(dev, at), window=window, sinks=sinks)
    want, tol = kvref.attention(q, rows[0], rows[1], at, [T] * B, window, sinks)
    check(got, want, tol)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("B,T,nh,nkv,pos,window,sinks", [
    (1, 1, 32, 4, 8191, None, 0), (4, 1, 32, 4, 3000, None, 0), (2, 2, 16, 2, 777, 256, 20),
    (1, 4110, 32, 4, 100, 300, 5), (2, 2100, 64, 8, 77, None, 0)])
def test_attention_is_that_over_rows(pkg, dev, dtype, page, B, T, nh, nkv, pos, window, sinks):
    """The bits of attn_window over the same rows, for host and device positions: for few rows,
    and for so many that their context tiles are not shared out."""
    n = -(-(pos + T) // page) * page
    q, rows = case(dev, B, T, nh, nkv, n, dtype)
    cache, table = pool_of(pkg, dev, rows, [n] * B, page, seed=1)
    bounds = dict(window=window, sinks=sinks)
    for p in (pos, i32(dev, starts(pos, B))):
        want = pkg.attn_window(q, rows[0], rows[1], p, **bounds)
        assert same(pkg.attn_paged(q, cache, table, p, **bounds), want)
    # another table of the same pages, wider: the same rows, and the same bits where the splits
    # do not go by the table's width (a host position)
    wide = torch.cat([table, torch.full((B, 5), -7, dtype=torch.int32, device=dev)], 1)[:, :-2]
    assert same(pkg.attn_paged(q, cache, wide, pos, **bounds),
                pkg.attn_window(q, rows[0], rows[1], pos, **bounds))


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("B,T,nh,nkv,pos,window,sinks", [
    (1, 1, 32, 4, 8192, None, 0),     # one context tile more than 128
    (1, 1, 32, 4, 20011, None, 0),    # 32 parts a kv head
    (1, 2, 8, 1, 20011, None, 0),     # 64
    (1, 3, 4, 2, 33000, 17000, 70),
    (2, 1, 32, 4, 17000, None, 0),    # ages apart: most of the parts are the older's
    (4, 4, 12, 3, 9999, 9000, 1),
    (3, 2, 4, 2, 26000, None, 0),     # more parts of few heads
    (3, 1, 11, 11, 8500, None, 0)])   # one head too many for few
def test_long_contexts_of_few_rows(pkg, dev, dtype, B, T, nh, nkv, pos, window, sinks):
    """Contexts so long that the splits differ from those over rows, against 64 bits: ages that
    the host knows and the device's, the first sequence the oldest, the last one young."""
    q, rows = case(dev, B, T, nh, nkv, pos + T, dtype)
    at = [pos // (5 * b + 1) for b in range(B)]
    cache, table = pool_of(pkg, dev, rows, [p + T for p in at], 64, width=-(-(pos + T) // 64))
    bounds = dict(window=window, sinks=sinks)
    want, tol = kvref.attention(q, rows[0], rows[1], at, [T] * B, window, sinks)
    got = pkg.attn_paged(q, cache, table, i32(dev, at), **bounds)
    check(got, want, tol)
    assert same(pkg.attn_paged(q, cache, table, i32(dev, at), **bounds), got)
    if B == 1:
        check(pkg.attn_paged(q, cache, table, pos, **bounds), want, tol)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_padding_and_positions_outside(pkg, dev, T):
    """Counts, a given output whose padding stays, and device positions outside the table."""
    B, page = 7, 16
    pos = [40, 7, 20, 95, -1, 96, 2**31 - 1]
    counts = [T, 0, max(T - 1, 0), T, T, T, T + 5]
    q, rows = case(dev, B, T, 8, 2, 96, torch.bfloat16)
    cache, table = pool_of(pkg, dev, rows, [96] * B, page)
    out = torch.full_like(q, 5.0)
    got = pkg.attn_paged(q, cache, table, i32(dev, pos), counts=i32(dev, counts), out=out)
    assert got is out
    have = [min(c, T) for c in counts]
    fit = [min(c, max(0, 96 - p)) if 0 <= p < 96 else 0 for c, p in zip(have, pos)]
    want, tol = kvref.attention(q, rows[0], rows[1], pos, fit, None, 0)
    for b in range(B):
        check(got[b:b + 1, :fit[b]], want[b:b + 1, :fit[b]], tol[b:b + 1, :fit[b]])
        assert torch.isnan(got[b, fit[b]:have[b]]).all() and (got[b, have[b]:] == 5.0).all()
    dirty(q)
    fresh = pkg.attn_paged(q, cache, table, i32(dev, pos), counts=i32(dev, counts))
    assert all(same(fresh[b, :have[b]], got[b, :have[b]]) and not fresh[b, have[b]:].any()
               for b in range(B))


@pytest.mark.parametrize("bad", [-1, -2**31, 2**31 - 1, "pages"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("T,pos,window,sinks", [(1, 500, None, 0), (1, 500, 64, 20), (2, 300, 40, 0),
                                                (60, 400, None, 0), (40, 400, 50, 30)])
def test_a_missing_page_is_nan_for_the_rows_that_see_it(pkg, dev, page, bad, T, pos, window, sinks):
    """Every entry in turn: NaN in exactly the rows that see one of its positions, the other
    rows as they were."""
    q, rows = case(dev, 1, T, 8, 2, pos + T, torch.bfloat16)
    cache, table = pool_of(pkg, dev, rows, [pos + T], page, fill=0.5)
    bounds = dict(window=window, sinks=sinks)
    clean = pkg.attn_paged(q, cache, table, pos, **bounds)
    entries = table.shape[1]
    for i in (x for x in range(entries) if entries <= 10 or x % 3 == 0 or x > entries - 3):
        broken = table.clone()
        broken[0, i] = cache.pages if bad == "pages" else bad
        got = pkg.attn_paged(q, cache, broken, pos, **bounds)
        for t in range(T):
            see = kvref.see(pos + t, pos + T, window, sinks)
            if see[i * page:(i + 1) * page].any():
                assert torch.isnan(got[0, t]).all()
            else:
                assert same(got[0, t], clean[0, t])


@pytest.mark.parametrize("T", [1, 40])
def test_pages_behind_the_window_may_be_gone(pkg, dev, T):
    """Entries between the first tokens and the window are given back: the bits stay."""
    pos, window, sinks, page = 900, 200, 20, 16
    q, rows = case(dev, 1, T, 8, 2, pos + T, torch.float16)
    cache, table = pool_of(pkg, dev, rows, [pos + T], page)
    want = pkg.attn_paged(q, cache, table, pos, window=window, sinks=sinks)
    gone = table.clone()
    gone[0, -(-sinks // page):(pos - window + 1) // page] = -1
    assert same(pkg.attn_paged(q, cache, gone, pos, window=window, sinks=sinks), want)


@pytest.mark.parametrize("T", [1, 2, 40])
def test_shared_pages(pkg, dev, T):
    """Sequences whose first pages are the same, with tails of their own; the same sequence
    twice in one call (with the same bits where a context is not cut for the whole batch)."""
    page, common, pos, B = 32, 160, 300, 3
    q, rows = case(dev, B, T, 8, 2, pos + T, torch.bfloat16)
    rows[:, 1:, :, :common] = rows[:, :1, :, :common]
    cache, table = pool_of(pkg, dev, rows, [pos + T] * B, page)
    one = table.clone()
    one[1:, :common // page] = table[0, :common // page]
    want = pkg.attn_paged(q, cache, table, pos)
    assert same(pkg.attn_paged(q, cache, one, pos), want)
    twice = table[[0, 0, 2]]
    got = pkg.attn_paged(q[[0, 0, 2]], cache, twice, pos)
    assert same(got[0], want[0]) and same(got[2], want[2])
    assert T == 40 or same(got[0], got[1])
    check(got, *(x[[0, 0, 2]] for x in kvref.attention(q, rows[0], rows[1], [pos] * B, [T] * B,
                                                       None, 0)))


@pytest.mark.parametrize("T,pos,window", [(1, 100, None), (2, 90, 33), (5, 60, None), (50, 70, 40)])
def test_values_that_are_not_finite(pkg, dev, T, pos, window):
    """An infinity or a NaN among the values reaches the rows that see it and no other."""
    page = 16
    q, rows = case(dev, 1, T, 8, 2, pos + T, torch.bfloat16)
    for j in (0, 3, pos - 35, pos - 1, pos, pos + T - 1):
        bad = rows.clone()
        bad[1, 0, 1, j, 5] = math.inf
        bad[1, 0, 1, j, 77] = QNAN
        cache, table = pool_of(pkg, dev, bad, [pos + T], page)
        got = pkg.attn_paged(q, cache, table, pos, window=window)
        want, tol = kvref.attention(q, rows[0], rows[1], [pos], [T], window, 0)
        for t in range(T):
            saw = bool(kvref.see(pos + t, pos + T, window, 0)[j])
            y = got[0, t].double().cpu()
            # infinite or NaN, as attn_window: a weight's second number may be negative, and an
            # infinity times both is then a NaN
            assert torch.equal(~torch.isfinite(y[4:, [5, 77]]), torch.full((4, 2), saw))
            rest = torch.ones_like(y, dtype=torch.bool)
            if saw:
                rest[4:, [5, 77]] = False
            assert ((y - want[0, t]).abs() <= tol[0, t])[rest].all()


@pytest.mark.parametrize("page", [16, 64])
def test_far_pages(pkg, dev, page):
    """Pages that lie past 2^32 bytes of the pool."""
    nkv, B, pos = 4, 2, 200
    per = nkv * page * HD * 2
    pages = (2**32 + 2**28) // per
    kv = [torch.empty(pages, nkv, page, HD, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    cache = pkg.PagedCache(*kv)
    for T in (1, 30):
        q, rows = case(dev, B, T, 8, nkv, pos + T, torch.bfloat16)
        small, table = pool_of(pkg, dev, rows, [pos + T] * B, page)
        far = (pages - 1 - table).clamp(min=-1)
        far[:, 0] = table[:, 0]  # and some near
        used = (table >= 0) & (table < small.pages)
        for a, b in zip(kv, (small.k, small.v)):
            a[far[used].long()] = b[table[used].long()]
        assert same(pkg.attn_paged(q, cache, far, pos), pkg.attn_paged(q, small, table, pos))
    x = rand(dev, B, 3, (8 + 2 * nkv) * HD, seed=3)
    r, tab = pkg.Rotary.plain(HD, 1e6), i32(dev, [[pages - 1], [pages - 2]])
    q1 = pkg.paged_append(x, 8, None, None, 1e-6, r, 5, cache, tab)
    few = pkg.PagedCache.empty(nkv, 2, page)
    assert same(q1, pkg.paged_append(x, 8, None, None, 1e-6, r, 5, few, i32(dev, [[1], [0]])))
    for a, b in ((cache.k, few.k), (cache.v, few.v)):
        assert same(a[-2:, :, 5:8].contiguous(), b[:, :, 5:8].contiguous())


def test_pool_views(pkg, dev):
    """k and v interleaved in one tensor, and heads before pages."""
    q, rows = case(dev, 2, 3, 8, 2, 100, torch.bfloat16)
    cache, table = pool_of(pkg, dev, rows, [100, 100], 32)
    want = pkg.attn_paged(q, cache, table, 60)
    both = torch.stack([cache.k, cache.v], 1)
    assert same(pkg.attn_paged(q, pkg.PagedCache(both[:, 0], both[:, 1]), table, 60), want)
    k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (cache.k, cache.v))
    turned = pkg.PagedCache(k, v)
    assert turned.k.stride(1) > turned.k.stride(0)
    assert same(pkg.attn_paged(q, turned, table, 60), want)
    wide = torch.zeros(2, 9, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    assert same(pkg.attn_paged(q, cache, wide[:, :table.shape[1]], 60), want)
    # queries as a view of wider rows, heads before tokens
    view = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert same(pkg.attn_paged(view, cache, table, 60), want)
    # one sequence without a batch
    assert same(pkg.attn_paged(q[1], cache, table[1], 60), want[1])


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("B,T,nh,nkv,pos,window,sinks", [
    (2, 33, 32, 4, 3000, None, 0),    # many runs for each row tile
    (3, 90, 16, 2, 700, None, 0),     # row tiles that runs cut
    (9, 50, 8, 8, 260, 100, 3),       # runs of several row tiles, under a window
    (9, 50, 8, 8, 260, 5000, 3),
    (2, 18, 8, 1, 0, None, 0),        # fewer tiles than a run of four for each XCD
    (2, 18, 8, 1, 300, None, 0),
    (40, 24, 8, 2, 90, None, 0)])
def test_shared_out_tiles(pkg, dev, dtype, B, T, nh, nkv, pos, window, sinks):
    """Padded batches of several rows whose context tiles are shared out (a wide table: it goes by
    what the table could hold), against 64 bits: ages and counts that differ, none among them;
    the same bits again and from a larger workspace."""
    at = starts(pos, B)
    counts = [T if b == 0 else (T - 7 * b) % (T + 1) for b in range(B)]
    q, rows = case(dev, B, T, nh, nkv, pos + T, dtype)
    cache, table = pool_of(pkg, dev, rows, [p + n for p, n in zip(at, counts)], 16,
                           width=max(130, -(-(pos + T) // 16)))
    bounds = dict(window=window, sinks=sinks, counts=i32(dev, counts))
    out = torch.full_like(q, 5.0)
    got = pkg.attn_paged(q, cache, table, i32(dev, at), out=out, **bounds)
    want, tol = kvref.attention(q, rows[0], rows[1], at, counts, window, sinks)
    check(got, want, tol)
    for b, n in enumerate(counts):
        assert (out[b, n:] == 5.0).all()
    ws = pkg.Workspace()
    ws.get(1 << 25, dev).fill_(0xFF)
    dirty(q)
    again = pkg.attn_paged(q, cache, table, i32(dev, at), workspace=ws, **bounds)
    for b, n in enumerate(counts):
        assert same(again[b, :n], got[b, :n]) and not again[b, n:].any()


@pytest.mark.parametrize("window,sinks", [(None, 0), (90, 20)])
def test_shared_out_missing_pages(pkg, dev, window, sinks):
    """As above where the context tiles are shared out: NaN in exactly the rows that see one of
    the missing page's positions; the other sequence as it was."""
    T, pos, page = 40, 400, 16
    q, rows = case(dev, 2, T, 8, 2, pos + T, torch.bfloat16)
    cache, table = pool_of(pkg, dev, rows, [pos + T] * 2, page, width=130, fill=0.5)
    at, bounds = i32(dev, [pos, pos]), dict(window=window, sinks=sinks)
    clean = pkg.attn_paged(q, cache, table, at, **bounds)
    for i in (0, 1, 5, 19, 20, 24, 25, 26, 27):
        broken = table.clone()
        broken[1, i] = [-1, cache.pages, 2**31 - 1][i % 3]
        got = pkg.attn_paged(q, cache, broken, at, **bounds)
        assert same(got[0], clean[0])
        for t in range(T):
            if kvref.see(pos + t, pos + T, window, sinks)[i * page:(i + 1) * page].any():
                assert torch.isnan(got[1, t]).all()
            else:
                assert same(got[1, t], clean[1, t])


@pytest.mark.parametrize("window", [None, 70])
def test_shared_out_values_that_are_not_finite(pkg, dev, window):
    T, pos = 40, 300
    q, rows = case(dev, 2, T, 8, 2, pos + T, torch.bfloat16)
    want, tol = kvref.attention(q, rows[0], rows[1], [pos] * 2, [T] * 2, window, 0)
    for j in (0, 250, pos, pos + 17, pos + T - 1):
        bad = rows.clone()
        bad[1, 1, 1, j, 5] = math.inf
        bad[1, 1, 1, j, 77] = QNAN
        cache, table = pool_of(pkg, dev, bad, [pos + T] * 2, 16, width=130)
        got = pkg.attn_paged(q, cache, table, i32(dev, [pos, pos]), window=window).double().cpu()
        rest = torch.ones_like(got, dtype=torch.bool)
        for t in range(T):
            if kvref.see(pos + t, pos + T, window, 0)[j]:
                rest[1, t, 4:, [5, 77]] = False
        assert torch.equal(torch.isfinite(got), rest)
        assert ((got - want).abs() <= tol)[rest].all()


def test_shared_out_positions_outside(pkg, dev):
    """Rows past the table are NaN, padding stays, where the context tiles are shared out; also
    when no sequence has a token inside."""
    B, T, page, width = 5, 40, 16, 130
    end = page * width
    pos, counts = [end - 20, -1, end, 100, 2**31 - 1], [40, 40, 7, 33, 40]
    q, rows = case(dev, B, T, 8, 2, end, torch.float16)
    cache, table = pool_of(pkg, dev, rows, [end] * B, page)
    out = torch.full_like(q, 5.0)
    pkg.attn_paged(q, cache, table, i32(dev, pos), counts=i32(dev, counts), out=out)
    fit = [20, 0, 0, 33, 0]
    want, tol = kvref.attention(q, rows[0], rows[1], pos, fit, None, 0)
    for b in range(B):
        check(out[b:b + 1, :fit[b]], want[b:b + 1, :fit[b]], tol[b:b + 1, :fit[b]])
        assert torch.isnan(out[b, fit[b]:counts[b]]).all() and (out[b, counts[b]:] == 5.0).all()
    out.fill_(5.0)
    pkg.attn_paged(q, cache, table, i32(dev, [-1] * B), counts=i32(dev, [0, 1, 2, 40, 9]), out=out)
    for b, n in enumerate([0, 1, 2, 40, 9]):
        assert torch.isnan(out[b, :n]).all() and (out[b, n:] == 5.0).all()


# ------------------------------------------------------------------- append

@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("layout,dims", [("half", 128), ("half", 64), ("half", 16), ("half", 112),
                                         ("interleaved", 128), ("interleaved", 20),
                                         ("interleaved", 2)])
@pytest.mark.parametrize("B,T,nh,nkv,pos,page,norm,form", [
    (1, 1, 32, 4, 0, 16, "both", "int"), (3, 5, 8, 8, 13, 16, "none", "start"),
    (2, 70, 6, 2, 100, 32, "q", "axes"), (1, 300, 4, 4, 1, 256, "k", "tokens")])
def test_append_matches_64_bits(pkg, dev, dtype, layout, dims, B, T, nh, nkv, pos, page, norm,
                                form):
    width, n = (nh + 2 * nkv) * HD, dims // 2
    qkv = rand(dev, B, T, width + 64, dtype=dtype, seed=1)[..., :width]
    qw, kw = ((1 + 0.2 * rand(dev, HD, seed=s).float()).to(dtype) for s in (2, 3))
    qw, kw = qw if norm in ("both", "q") else None, kw if norm in ("both", "k") else None
    axes = [i % 3 for i in range(n)] if form == "axes" else None
    r = pkg.Rotary.plain(dims, 1e4, layout=layout, factor=1.1, axes=axes)
    at = [pos] * B if form == "int" else starts(pos, B)
    p = torch.tensor(at, dtype=torch.int32)[:, None] + torch.arange(T, dtype=torch.int32)
    turn = None
    if form in ("axes", "tokens"):
        g = torch.Generator().manual_seed(5)
        turn = torch.randint(-9, 70000, ((3, B, T) if axes else (B, T)), generator=g,
                             dtype=torch.int32)
        p = turn
    rows = rand(dev, 2, B, nkv, pos + T + 5, HD, seed=4, dtype=dtype)
    cache, table = pool_of(pkg, dev, rows, [pos + T + 5] * B, page, fill=7.0)
    before = cache.k.clone(), cache.v.clone()
    q = pkg.paged_append(qkv, nh, qw, kw, 1e-6, r, pos if form == "int" else i32(dev, at), cache,
                         table, turn=None if turn is None else turn.to(dev))
    x = qkv.cpu().reshape(B, T, nh + 2 * nkv, HD)
    new = ref.gathered(cache.k, table), ref.gathered(cache.v, table)
    put = lambda c: torch.stack([c[b, :, at[b]:at[b] + T].transpose(0, 1) for b in range(B)])
    for lo, m, w, got in ((0, nh, qw, q.cpu()), (nh, nkv, kw, put(new[0]))):
        y = x[:, :, lo:lo + m]
        y = y.double() if w is None else ref.normed(y, w)
        want, size = ref.turned(y, r.inv_freq, p, layout, r.factor, axes)
        # the norm's sum, root, quotient and products: 2^-20 together; the rotation: 2^-21
        tol = ref.rounded(want, size, dtype, 2.0 ** -19)
        assert ((got.double() - want).abs() <= tol).all()
    assert same(put(new[1]).contiguous(), x[:, :, nh + nkv:].contiguous())
    # the other rows of the pool as they were
    for c, c0 in zip((cache.k, cache.v), before):
        c = c.clone()
        for b in range(B):
            for t in range(T):
                e = int(table[b, (at[b] + t) // page])
                c[e, :, (at[b] + t) % page] = c0[e, :, (at[b] + t) % page]
        assert same(c, c0)


def test_append_is_rope_append(pkg, dev):
    """The plain case against rope_append: the same norm, another way to the cosines."""
    T, nh, nkv = 40, 8, 2
    qkv = rand(dev, T, (nh + 2 * nkv) * HD, seed=1)
    w = (1 + 0.2 * rand(dev, HD, seed=2).float()).to(torch.bfloat16)
    k, v = (torch.zeros(nkv, 64, HD, dtype=torch.bfloat16, device=dev) for _ in range(2))
    inv = pkg.rope_inv_freq(HD, 1e6)
    a = pkg.rope_append(qkv, nh, nkv, w, w, 1e-6, inv, 20, k, v)
    cache = pkg.PagedCache.empty(nkv, 4, 16)
    table = i32(dev, [2, 0, 3, 1])
    b = pkg.paged_append(qkv, nh, w, w, 1e-6, pkg.Rotary(inv), 20, cache, table)
    u = 2 * kvref.half_step(torch.bfloat16)
    for x, y in ((b, a), (ref.gathered(cache.k, table[None])[0], k.cpu())):
        x, y = x.double().cpu(), y.double().cpu()
        assert ((x - y).abs() <= 1.01 * u * y.abs() + 1e-5).all()  # one step where they differ
        assert (x != y).double().mean() < 0.01
    assert same(ref.gathered(cache.v, table[None])[0].contiguous(), v.cpu())


def test_append_padding_and_missing_pages(pkg, dev):
    """Counts, a given output whose padding stays, positions outside the table, and entries
    outside the pool: nothing is written for them, and their rows are NaN."""
    B, T, nh, nkv, page = 6, 6, 4, 2, 16
    qkv = rand(dev, B, T, (nh + 2 * nkv) * HD, seed=1)
    r = pkg.Rotary.plain(HD, 1e4)
    whole = pkg.PagedCache.empty(nkv, 2 * B, page)
    full = torch.arange(2 * B, dtype=torch.int32, device=dev).view(B, 2)
    pos = [13, 5, 30, -1, 32, 12]
    counts = [6, 0, 9, 6, 6, 4]
    want = pkg.paged_append(qkv, nh, None, None, 1e-6, r, i32(dev, [13, 5, 26, 0, 0, 12]), whole,
                            full)
    cache = pkg.PagedCache(*(torch.full_like(whole.k, 7.0) for _ in range(2)))
    table = full.clone()
    table[0, 1], table[5, 0] = 2 * B, -2**31
    out = torch.full((B, T, nh, HD), 5.0, dtype=qkv.dtype, device=dev)
    q = pkg.paged_append(qkv, nh, None, None, 1e-6, r, i32(dev, pos), cache, table,
                         counts=i32(dev, counts), out=out)
    written = torch.zeros(2 * B, page, dtype=torch.bool)
    for b in range(B):
        for t in range(T):
            p = pos[b] + t
            row = q[b, t]
            if t >= min(counts[b], T):
                assert (row == 5.0).all()
            elif not 0 <= pos[b] <= p < 32 or not 0 <= int(table[b, p // page]) < 2 * B:
                assert torch.isnan(row).all()
            else:
                assert torch.isfinite(row).all()
                written[int(table[b, p // page]), p % page] = True
                if pos[b] == [13, 5, 26, 0, 0, 12][b]:
                    assert same(row, want[b, t])
    for c in (cache.k, cache.v):
        assert ((c == 7.0).all(-1).all(1).cpu() == ~written).all()
    # an angle's position out of range: as a position outside
    turn = torch.zeros(B, T, dtype=torch.int32, device=dev)
    turn[2, 3], turn[4, 0] = 2**24, -2**31
    cache.k.fill_(7.0)
    q = pkg.paged_append(qkv, nh, None, None, 1e-6, r, 3, cache, full, turn=turn)
    bad = torch.isnan(q).flatten(2).any(-1).cpu()
    assert bad[2, 3] and bad[4, 0] and int(bad.sum()) == 2
    assert (cache.k[4, :, 6] == 7.0).all() and (cache.k[8, :, 3] == 7.0).all()


# ------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", DTS)
def test_sessions_of_different_ages(pkg, dev, dtype):
    """Prompts, padded chunks and tokens of three sessions on one pool whose pages are handed out
    as they grow and given back behind the window, against 64 bits over the rows appended."""
    B, nh, nkv, page, window, sinks = 3, 8, 2, 16, 60, 5
    r = pkg.Rotary.scaled(HD, 1e4, 4.0, 64)
    w = (1 + 0.2 * rand(dev, HD, seed=2).float()).to(dtype)
    cache = pkg.PagedCache(*(torch.full((26, nkv, page, HD), QNAN, dtype=dtype, device=dev)
                             for _ in range(2)))
    table = torch.full((B, 16), -1, dtype=torch.int32)
    free = torch.randperm(26, generator=torch.Generator().manual_seed(1)).tolist()
    kept = torch.full((2, B, nkv, 256, HD), QNAN, dtype=dtype)
    pos = [0] * B
    for step, counts in enumerate(([70, 33, 1], [1, 1, 1], [0, 40, 17], [1, 0, 1], [9, 2, 30],
                                   [1, 1, 1], [40, 20, 3], [1, 1, 1])):
        T = max(counts)
        for b, c in enumerate(counts):
            for e in range(-(-(pos[b] + c) // page)):  # the pages that the call needs
                if table[b, e] < 0 and e * page >= pos[b] - page:
                    table[b, e] = free.pop()
        tab, at, n = table.to(dev), i32(dev, pos), i32(dev, counts)
        qkv = rand(dev, B, T, (nh + 2 * nkv) * HD, seed=10 + step, dtype=dtype)
        q = pkg.paged_append(qkv, nh, w, w, 1e-6, r, at, cache, tab, counts=n)
        got = pkg.attn_paged(q, cache, tab, at, window=window, sinks=sinks, counts=n)
        for i, pool in enumerate((cache.k, cache.v)):
            x = ref.gathered(pool, tab)
            for b, c in enumerate(counts):
                kept[i, b, :, pos[b]:pos[b] + c] = x[b, :, pos[b]:pos[b] + c]
        want, tol = kvref.attention(q, kept[0], kept[1], pos, counts, window, sinks)
        check(got, want, tol)
        for b, c in enumerate(counts):
            pos[b] += c
            for e in range(1, max(0, pos[b] - window + 1) // page):  # behind the window
                if table[b, e] >= 0:
                    free.insert(0, int(table[b, e]))
                    table[b, e] = -1
    assert max(pos) > 100 and (table[:, 1:3] < 0).any()


@pytest.mark.parametrize("T", [1, 24])
def test_graphs_and_streams(pkg, dev, T):
    """Append and attention captured as one graph, replayed with other positions and pages and
    with eager work between; two graphs share one workspace."""
    B, nh, nkv, page, n = 2, 16, 2, 16, 2048
    r = pkg.Rotary.plain(HD, 1e6)
    rows = rand(dev, 2, B, nkv, n, HD, seed=4)
    cache, table = pool_of(pkg, dev, rows, [n] * B, page, fill=0.0)
    qkv = rand(dev, B, T, (nh + 2 * nkv) * HD, seed=1)
    ws = pkg.Workspace()

    def call(x, at, tab, workspace=None):
        q = pkg.paged_append(x, nh, None, None, 1e-6, r, at, cache, tab)
        return pkg.attn_paged(q, cache, tab, at, workspace=workspace)

    places = [i32(dev, p) for p in ([1500, 900], [0, 31], [2000, 64])]
    tables = [table, table.flip(0), table]
    for p, t in zip(places, tables):  # what each call appends stays from here on
        call(qkv, p, t)
    want = [call(qkv, p, t).clone() for p, t in zip(places, tables)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert same(call(qkv, places[0], table), want[0])
    torch.cuda.current_stream().wait_stream(side)
    at, tab = places[0].clone(), table.clone()
    graphs, outs = [], []
    for _ in range(2):
        call(qkv, at, tab, ws)  # the workspace and its counters are there before the capture
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(qkv, at, tab, ws))
    alone = torch.cuda.CUDAGraph()
    with torch.cuda.graph(alone):
        outs.append(call(qkv, at, tab))
    for i in (2, 0, 1, 1, 0):
        at.copy_(places[i])
        tab.copy_(tables[i])
        for g, o in zip((*graphs, alone), outs):
            g.replay()
            torch.cuda.synchronize()
            assert same(o, want[i])
            assert same(call(qkv, at, tab), want[i])


def test_many_sequences(pkg, dev):
    """More kv heads than the shared-out contexts count (a workgroup each), and repeated calls
    give the same bits."""
    B, nkv = 300, 4
    at = [(37 * b) % 200 for b in range(B)]
    q, rows = case(dev, B, 1, 8, nkv, 201, torch.bfloat16)
    cache, table = pool_of(pkg, dev, rows, [a + 1 for a in at], 16)
    got = pkg.attn_paged(q, cache, table, i32(dev, at))
    want, tol = kvref.attention(q, rows[0], rows[1], at, [1] * B, None, 0)
    check(got, want, tol)
    for _ in range(3):
        assert same(pkg.attn_paged(q, cache, table, i32(dev, at)), got)
