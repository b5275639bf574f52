"""What the documents promise of the paged cache and the rotary embeddings beyond single calls."""
from __future__ import annotations

import pytest
import torch

from tests import _kv_ref as kvref
from tests import _paged_ref as ref
from tests.test_gpu_kv import i32, rand, same
from tests.test_gpu_kv_module import build, near, tokens

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("start", [30, [30, 4000]])
def test_turning_back_of_tokens_behind_a_start(pkg, dev, layout, start):
    """Minus each token's own position turns back, to the square of the factor; minus the start
    is a start, whose tokens turn by -start + t."""
    B, T, hd, f = 2, 5, 64, 1.5
    r = pkg.Rotary.plain(48, 1e4, layout=layout, factor=f)
    x = rand(dev, B, T, 3, hd, seed=1)
    first = torch.tensor(start if isinstance(start, list) else [start] * B)
    p = (first[:, None] + torch.arange(T)).int()
    y = pkg.rope(x, None, i32(dev, start) if isinstance(start, list) else start, r)
    back = pkg.rope(y, None, -p.to(dev), r)
    # y is off by half a step of up to factor (|a| + |b|), of which two enter each dim of back,
    # times up to factor; then back is rounded: at most 3 halves, with room for fp32's own errors
    xs = x.double().cpu()
    _, size = ref.turned(x, r.inv_freq, p, layout, f)
    want = xs.clone()
    want[..., :48] *= f * f
    tol = 3.1 * kvref.half_step(BF) * f * size
    assert ((back.double().cpu() - want).abs() <= tol)[..., :48].all()
    assert torch.equal(back[..., 48:], x[..., 48:])
    again = pkg.rope(y, None, i32(dev, [-s for s in start]) if isinstance(start, list) else -start,
                     r)
    out, size = ref.turned(y, r.inv_freq, (torch.arange(T) - first[:, None]).int(), layout, f)
    assert ((again.double().cpu() - out).abs() <= ref.rounded(out, size, BF, 2.0 ** -20)).all()


def test_scratch_of_a_call_with_host_positions(pkg, dev):
    """Two chunks at a host position keep their scratch in the workspace; the same chunks at
    device positions, which are shared out, take more."""
    B, T, nh, nkv, pos, page = 2, 20, 32, 4, 2500, 64
    n = -(-(pos + T) // page)
    cache = pkg.PagedCache(*(rand(dev, B * n, nkv, page, 128, seed=s) for s in (1, 2)))
    table = torch.arange(B * n, dtype=torch.int32, device=dev).view(B, n)
    q = rand(dev, B, T, nh, 128, seed=3)
    need = [pkg.lib().i4_attn_paged_call_bytes(B, T, nh, nkv, k, 0, 0, d)
            for d, k in ((0, pos + T), (1, n * page))]
    assert 0 < need[0] < need[1]
    ws = pkg.Workspace()
    a = pkg.attn_paged(q, cache, table, pos, workspace=ws)
    assert need[0] <= ws.buf.numel() < need[1]
    b = pkg.attn_paged(q, cache, table, i32(dev, [pos] * B))
    # Split in another way the weights have other maxima and round elsewhere: each is off by half a
    # step, a weighted mean by at most twice that of |v| + |mean|, on both sides; then one rounding.
    h, top = kvref.half_step(BF), a.double().abs().max()
    most = 4 * h * (cache.v.double().abs().max() + top) + 2.1 * h * top
    assert (a.double() - b.double()).abs().max() <= most
    assert same(pkg.attn_paged(q, cache, table, pos, workspace=ws), a)


@pytest.mark.parametrize("T", [1, 4, 30])
def test_a_session_without_its_page_stays_alone(pkg, dev, T):
    """Sessions that lack a page, are past their table's end or padded with NaN give NaN rows of
    their own; the others' rows and pages are what they are without them."""
    page, layers, H = 16, 2, 1024
    dec, twin = (build(pkg, dev, layers=layers, pages=40, page=page) for _ in range(2))
    table = torch.arange(30, dtype=torch.int32, device=dev).view(5, 6)
    h = torch.stack([tokens(dev, 80, seed=s) for s in range(5)])
    for d in (dec, twin):
        d.step(h[:, :40], 0, table=table)
    pools = [c for l in dec.layers for c in (l.attn.paged.k, l.attn.paged.v)]
    before = [c.clone() for c in pools]
    x, tab = h[:, 40:40 + T].clone(), table.clone()
    tab[1, 0] = -1           # lacks a page of its past
    tab[2, 40 // page:] = 99  # and one of its own tokens': not a page of the pool
    pos = i32(dev, [40, 40, 40, 6 * page, 40])
    counts = i32(dev, [T, T, T, T, T - 1])
    if T > 1:
        x[4, T - 1:] = float("nan")
    got = dec.step(x, pos, table=tab, counts=counts)
    good = [0, 4]
    want = twin.step(x[good], 40, table=table[good], counts=counts[good])
    assert torch.isnan(got[1:4]).all()
    for i, b in enumerate(good):
        n = int(counts[b])
        if n:
            assert near(got[b, :n], want[i, :n])
    other = [c for l in twin.layers for c in (l.attn.paged.k, l.attn.paged.v)]
    for c, old, o in zip(pools, before, other):
        assert near(c[table[good].long()], o[table[good].long()])
        # of the others, the first layer's own rows are finite and in their pages alone; nothing
        # of a session without its page or place is written
        assert same(c[table[2].long()], old[table[2].long()])
        assert same(c[table[3].long()], old[table[3].long()])
        assert same(c[30:], old[30:]) and same(c[table[1, :2].long()], old[table[1, :2].long()])
    again = dec.step(x, i32(dev, [40] * 5), table=table, counts=counts)  # all of them well again
    assert torch.isfinite(again[:4]).all()
    assert near(again[0], twin.step(x[:1], 40, table=table[:1])[0])
