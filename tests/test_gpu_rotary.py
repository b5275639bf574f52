"""rope on the GPU against 64 bits."""
from __future__ import annotations

import pytest
import torch

from tests import _kv_ref as kvref
from tests import _paged_ref as ref
from tests.test_gpu_kv import DTS, i32, rand, same

pytestmark = pytest.mark.gpu

# cos and sin are off by 2^-23 (the angle's rounding, the sums'), and by 2^-23 more with the
# factor; two products and a sum add 2^-23: 2^-22 of |a| + |b| together, and twice that is allowed
LEAD = 2.0 ** -21


def given(dev, B, T, pos, form, seed=7):
    """(what rope takes, positions [B, T] or [axes, B, T])"""
    first = torch.tensor([pos - b * 3 for b in range(B)], dtype=torch.int32)
    plain = first[:, None] + torch.arange(T, dtype=torch.int32)
    if form == "int":
        return pos, torch.full((B, 1), pos) + torch.arange(T)
    if form == "start":
        return first.to(dev), plain
    g = torch.Generator().manual_seed(seed)
    if form == "tokens":
        p = plain + torch.randint(-40, 40, (B, T), generator=g, dtype=torch.int32)
    else:
        p = plain + torch.randint(-40, 40, (3, B, T), generator=g, dtype=torch.int32)
    return p.to(dev), p


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,T,nh,nkv,hd,dims,pos,form,factor", [
    (1, 1, 32, 4, 128, 128, 0, "int", 1.0),
    (1, 1, 1, 0, 2, 2, 3, "int", 1.0),              # one pair, q alone
    (2, 3, 5, 2, 128, 128, 1000, "start", 1.0),
    (3, 7, 3, 3, 72, 18, 100, "tokens", 1.25),      # an odd number of pairs
    (2, 5, 4, 1, 80, 20, 12345, "axes", 1.0),
    (1, 33, 2, 2, 96, 48, 2**20, "tokens", 0.7),
    (2, 9, 7, 1, 256, 256, 77, "axes", 1.0),
    (1, 4, 3, 1, 64, 62, 2**24 - 50, "start", 1.0),  # positions at the end of the range
    (1, 300, 2, 1, 70, 70, -150, "int", 1.0),       # from negative ones to positive ones
    (4, 1100, 1, 1, 64, 32, 5, "start", 2.0),       # more tokens than one a workgroup
    (1, 2100, 2, 1, 128, 128, 40000, "int", 1.0),
    (1, 4200, 5, 3, 72, 18, 100, "tokens", 1.25),   # pairs through LDS: 9 of them,
    (3, 1100, 10, 2, 80, 20, 7, "axes", 1.0),       # 10, positions on axes,
    (1, 2050, 16, 0, 256, 250, 2**20, "int", 1.0),  # 125 of a wide head,
    (33, 1, 1000, 24, 64, 62, 9, "start", 0.5)])    # 31, and a token's heads shared out
def test_rope_matches_64_bits(pkg, dev, dtype, layout, B, T, nh, nkv, hd, dims, pos, form, factor):
    q, k = rand(dev, B, T, nh, hd, seed=1, dtype=dtype), rand(dev, B, T, nkv, hd, seed=2,
                                                              dtype=dtype)
    n = dims // 2
    axes = [i * 7 % 3 for i in range(n)] if form == "axes" else None
    f = 1.0 / 1e4 ** (torch.arange(n) / n)
    r = pkg.Rotary(f, layout=layout, factor=factor, axes=axes)
    call, p = given(dev, B, T, pos, form)
    got = pkg.rope(q, k if nkv else None, call, r)
    got = got if nkv else (got,)
    for x, y in zip((q, k), got):
        want, size = ref.turned(x, r.inv_freq, p, layout, factor, axes)
        tol = ref.rounded(want, size, dtype, LEAD)
        assert ((y.double().cpu() - want).abs() <= tol).all()
        assert same(y[..., dims:].contiguous(), x[..., dims:].contiguous())
        assert y.shape == x.shape and y.is_contiguous()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,dims,shift", [(128, 128, 0), (128, 64, 0), (80, 20, 0), (64, 64, 1),
                                           (64, 32, 2), (64, 64, 4)])
def test_views_and_in_place(pkg, dev, layout, hd, dims, shift):
    """Views of the fused rows at every alignment, in place and into other views: the bits of
    dense rows; nothing else is written."""
    B, T, nh, nkv = 2, 5, 3, 2
    r = pkg.Rotary.plain(dims, 1e4, layout=layout)
    width = (nh + 2 * nkv) * hd + 16 + shift
    flat = rand(dev, B * T * width + shift + 8, seed=3)
    rows = flat[shift:shift + B * T * width].view(B, T, width)
    q = rows[..., :nh * hd].unflatten(-1, (nh, hd))
    k = rows[..., nh * hd:(nh + nkv) * hd].unflatten(-1, (nkv, hd))
    pos = i32(dev, [10, 300])
    want = pkg.rope(q.contiguous(), k.contiguous(), pos, r)
    got = pkg.rope(q, k, pos, r)
    assert all(same(a, b) for a, b in zip(got, want))
    # heads before tokens, as attention keeps them
    turned = pkg.rope(q.transpose(1, 2).contiguous().transpose(1, 2), None, pos, r)
    assert same(turned, want[0])
    # into views of another buffer
    there = torch.full((B, nh + nkv, T, hd + 8), 3.0, dtype=q.dtype, device=dev)
    views = (there[:, :nh, :, :hd].transpose(1, 2), there[:, nh:, :, :hd].transpose(1, 2))
    got = pkg.rope(q, k, pos, r, out=views)
    assert got[0] is views[0] and all(same(a.contiguous(), b) for a, b in zip(got, want))
    assert (there[..., hd:] == 3.0).all()
    # in place
    before = flat.clone()
    got = pkg.rope(q, k, pos, r, out=(q, k))
    assert got[0] is q and all(same(a.contiguous(), b) for a, b in zip(got, want))
    q.copy_(before[shift:shift + B * T * width].view(B, T, width)[..., :nh * hd]
            .unflatten(-1, (nh, hd)))
    k.copy_(before[shift:shift + B * T * width].view(B, T, width)[..., nh * hd:(nh + nkv) * hd]
            .unflatten(-1, (nkv, hd)))
    assert same(flat, before)


@pytest.mark.parametrize("dtype", DTS)
def test_pairs_through_lds(pkg, dev, dtype):
    """In place in the fused rows, padding, positions outside and values that are not finite,
    where the number of pairs is odd and rows are many: as rows of few tokens."""
    B, T, nh, nkv, hd, dims = 3, 1500, 6, 2, 72, 18
    r = pkg.Rotary.plain(dims, 1e4)
    rows = rand(dev, B, T, (nh + 2 * nkv) * hd, seed=1, dtype=dtype)
    rows[0, 3, 5], rows[1, 7, 30], rows[1, 7, hd - 1] = float("inf"), float("-inf"), float("nan")
    x = rows.unflatten(-1, (-1, hd))
    counts, pos = i32(dev, [T, 0, T - 9]), i32(dev, [2**24 - 700, 5, 0])

    def turned(x, b, lo, hi):
        q, k = x[b:b + 1, lo:hi, :nh], x[b:b + 1, lo:hi, nh:nh + nkv]
        return pkg.rope(q, k, int(pos[b]) + lo, r)

    torch.full_like(x[:, :, :nh], 5.0)  # leaves memory that is not zeros
    got = pkg.rope(x[:, :, :nh], x[:, :, nh:nh + nkv], pos, r, counts=counts)
    for y in got:
        assert torch.isnan(y[0, 700:]).all() and not y[1].any() and not y[2, T - 9:].any()
    for b, n in ((0, 700), (2, T - 9)):
        for lo in range(0, n, 100):
            for a, w in zip(got, turned(x, b, lo, min(lo + 100, n))):
                a, w = a[b, lo:min(lo + 100, n)], w[0]
                assert torch.equal(torch.isfinite(a), torch.isfinite(w))
                a, w = (z.double().nan_to_num(0, 0, 0) for z in (a, w))
                # the same products, summed in either order: one more rounding of each, and
                # then half a step apart at most, or one where that tips
                assert ((a - w).abs() <= 2.01 * kvref.half_step(dtype) * w.abs() + 1e-6).all()
    want = [g.clone() for g in got]
    keep = rows.clone()
    pkg.rope(x[:, :, :nh], x[:, :, nh:nh + nkv], pos, r, counts=counts,
             out=(x[:, :, :nh], x[:, :, nh:nh + nkv]))
    for y, w, lo, n in ((x, want[0], 0, nh), (x, want[1], nh, nkv)):
        for b, c in ((0, T), (2, T - 9)):
            assert same(y[b, :c, lo:lo + n].contiguous(), w[b, :c].contiguous())
    y = keep.unflatten(-1, (-1, hd))
    assert same(x[:, :, nh + nkv:].contiguous(), y[:, :, nh + nkv:].contiguous())
    assert same(x[1], y[1]) and same(x[2, T - 9:], y[2, T - 9:])


def test_one_sequence_without_a_batch(pkg, dev):
    T, n = 6, 32
    q, k = rand(dev, T, 4, 64, seed=1), rand(dev, T, 2, 64, seed=2)
    axes = [i % 3 for i in range(n)]
    r, r3 = pkg.Rotary.plain(64, 1e4), pkg.Rotary.plain(64, 1e4, axes=axes)
    p = i32(dev, [4, 5, 6, 7, 8, 9])
    want = pkg.rope(q[None], k[None], 4, r)
    p3 = torch.stack([p, p + 3, p * 2])
    for got in (pkg.rope(q, k, 4, r), pkg.rope(q, k, i32(dev, [4]), r), pkg.rope(q, k, p, r),
                pkg.rope(q, k, p, r3), pkg.rope(q, k, 4, r3), pkg.rope(q, k, p.expand(3, T), r3)):
        assert all(same(a, b[0]) for a, b in zip(got, want))
    got = pkg.rope(q, k, p3, r3)
    for a, x in zip(got, (q, k)):
        y, size = ref.turned(x[None], r3.inv_freq, p3[:, None], axes=axes)
        assert ((a.double().cpu() - y[0]).abs() <= ref.rounded(y[0], size[0], a.dtype, LEAD)).all()


def test_padding_and_positions_outside(pkg, dev):
    """Padding is left as it is; a position outside gives NaN rows, on any of a token's axes."""
    B, T, n = 5, 4, 16
    q, k = rand(dev, B, T, 3, 40, seed=1), rand(dev, B, T, 1, 40, seed=2)
    r = pkg.Rotary.plain(2 * n, 1e4, axes=[i % 2 for i in range(n)])
    counts = [4, 0, 2, 9, -3]
    outs = tuple(torch.full_like(x, 5.0) for x in (q, k))
    pos = i32(dev, [0, 1, 2, 3, 4])
    pkg.rope(q, k, pos, r, counts=i32(dev, counts), out=outs)
    whole = pkg.rope(q, k, pos, r)
    for x in (q, k):  # leaves memory that is not zeros to the new outputs
        torch.full_like(x, 5.0)
    fresh = pkg.rope(q, k, pos, r, counts=i32(dev, counts))
    for b, c in enumerate(counts):
        c = max(0, min(c, T))
        for a, w, z in zip(outs, whole, fresh):
            assert same(a[b, :c], w[b, :c]) and (a[b, c:] == 5.0).all()
            assert same(z[b, :c], w[b, :c]) and not z[b, c:].any()
    edge = 2**24
    far = pkg.rope(q, k, i32(dev, [edge - 2, edge, -edge, 2**31 - 1, -2**31]), r)
    for y in far:
        assert torch.isfinite(y[0, :2]).all() and torch.isnan(y[0, 2:]).all()
        assert torch.isnan(y[1]).all() and torch.isnan(y[2, 0]).all()
        assert torch.isfinite(y[2, 1:]).all() and torch.isnan(y[3:]).all()
    p = torch.zeros(2, B, T, dtype=torch.int32, device=dev)
    p[0, 1, 2] = edge
    p[1, 3, 0] = -2**31
    for y in pkg.rope(q, k, p, r):
        bad = torch.isnan(y)
        assert bad[1, 2].all() and bad[3, 0].all() and int(bad.sum()) == 2 * y[0, 0].numel()


@pytest.mark.parametrize("dtype", DTS)
def test_values_that_are_not_finite_stay_in_their_pair(pkg, dev, dtype):
    for layout in ("half", "interleaved"):
        for hd, dims in ((128, 64), (24, 18)):
            r = pkg.Rotary.plain(dims, 1e4, layout=layout)
            x = rand(dev, 1, 2, 2, hd, seed=1, dtype=dtype)
            clean = pkg.rope(x, None, 5, r)
            for d, v in ((0, float("inf")), (dims - 1, float("nan")), (dims, float("-inf")),
                         (hd - 1, float("nan"))):
                y = x.clone()
                y[0, 1, 0, d] = v
                got = pkg.rope(y, None, 5, r)
                n, mate = dims // 2, d
                if d < dims:
                    mate = d ^ 1 if layout == "interleaved" else (d + n) % dims
                bad = ~torch.isfinite(got[0, 1, 0])
                assert set(bad.nonzero()[:, 0].tolist()) == {d, mate}
                got[0, 1, 0, [d, mate]] = clean[0, 1, 0, [d, mate]]
                assert same(got, clean)
                if d >= dims:  # passed on as it is
                    assert same(pkg.rope(y, None, 5, r)[0, 1, 0, d:d + 1], y[0, 1, 0, d:d + 1])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_turning_back_is_the_gradient(pkg, dev, layout):
    """The rotation by -p is the transpose of the rotation by p (and its inverse), here against
    the formula's gradient and against differences: the function is linear, so a difference of
    two of its values is exact up to their rounding."""
    B, T, nh, hd, dims = 2, 3, 2, 64, 48
    r = pkg.Rotary.plain(dims, 1e4, layout=layout)
    x, dy = rand(dev, B, T, nh, hd, seed=1), rand(dev, B, T, nh, hd, seed=2)
    p = i32(dev, [3, 1000])[:, None] + torch.arange(T, dtype=torch.int32, device=dev)
    dx = pkg.rope(dy, None, -p, r)
    leaf = x.double().cpu().requires_grad_()
    n, f = dims // 2, r.inv_freq.double()
    a = (p.cpu().double()[..., None] * f)[:, :, None]
    u, v = (leaf[..., :n], leaf[..., n:dims]) if layout == "half" else \
        (leaf[..., 0:dims:2], leaf[..., 1:dims:2])
    s, t = u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()
    y = torch.cat([s, t], -1) if layout == "half" else torch.stack([s, t], -1).flatten(-2)
    torch.cat([y, leaf[..., dims:]], -1).backward(dy.double().cpu())
    _, size = ref.turned(dy, r.inv_freq, -p, layout)
    tol = ref.rounded(leaf.grad, size, x.dtype, LEAD)
    assert ((dx.double().cpu() - leaf.grad).abs() <= tol).all()
    e = rand(dev, B, T, nh, hd, seed=3).double()
    plus, minus = (pkg.rope((x.double() + z * e).to(x.dtype), None, p, r).double() for z in (4, -4))
    step = ((x.double() + 4 * e).to(x.dtype).double() - (x.double() - 4 * e).to(x.dtype).double())
    lhs, rhs = ((plus - minus) * dy.double()).sum(), (step * dx.double()).sum()
    # each value of plus, minus and dx is rounded once: half a step of it
    h = kvref.half_step(x.dtype)
    tol = 1.01 * h * (((plus.abs() + minus.abs()) * dy.double().abs()).sum()
                      + (step.abs() * dx.double().abs()).sum())
    assert (lhs - rhs).abs() <= tol
    back = pkg.rope(pkg.rope(x, None, p, r), None, -p, r).double().cpu()
    _, size = ref.turned(x, r.inv_freq, p, layout)
    # two roundings of values of up to size, the first one turned: its error once more
    assert ((back - x.double().cpu()).abs() <= 4.1 * h * size).all()


def test_streams_devices_and_graphs(pkg, dev):
    B, T = 3, 2
    r = pkg.Rotary.plain(128, 1e6)
    q, k = rand(dev, B, T, 8, 128, seed=1), rand(dev, B, T, 2, 128, seed=2)
    pos = i32(dev, [1, 2, 3])
    want = [pkg.rope(q, k, pos + 100 * i, r) for i in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.rope(q, k, pos, r)
    torch.cuda.current_stream().wait_stream(side)
    assert all(same(a, b) for a, b in zip(got, want[0]))
    graph, at = torch.cuda.CUDAGraph(), pos.clone()
    with torch.cuda.graph(graph):
        got = pkg.rope(q, k, at, r)
    for i in (3, 0, 1, 2, 0):
        at.copy_(pos + 100 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want[i]))
        assert all(same(a, b) for a, b in zip(pkg.rope(q, k, pos + 100 * i, r), want[i]))
