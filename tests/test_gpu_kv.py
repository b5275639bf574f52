"""rope_append, attn_window, kv8_append and attn_kv8 on the GPU against 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from tests import _kv_ref as ref

pytestmark = pytest.mark.gpu
HD = 128
DTS = [torch.bfloat16, torch.float16]
KINDS = [torch.int8, torch.float8_e4m3fn]


def rand(dev, *shape, seed=0, dtype=torch.bfloat16, gain=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * gain).to(dtype)


def starts(pos, B):
    """A first position for each sequence, in [0, pos]."""
    return [pos - b * (pos // 2 + 1) % (pos + 1) for b in range(B)]


def i32(dev, values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def same(a, b):
    """Equal bits, NaN included."""
    if a.dtype.is_floating_point:
        kind = {1: torch.int8, 2: torch.int16, 4: torch.int32}[a.element_size()]
        a, b = a.view(kind), b.view(kind)
    return torch.equal(a, b)


def check(got, want, tol):
    """Every row that the reference has (the others are padding) within the tolerance."""
    rows = ~torch.isnan(want).all(-1)
    got, want, tol = got.double().cpu()[rows], want[rows], tol[rows]
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert (off <= tol).all(), f"off by {(off / tol).max().item():.2f} times the tolerance"


# ------------------------------------------------------------------- rope_append

@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("B,T,nh,nkv,pos", [
    (1, 1, 32, 4, 0), (1, 1, 32, 4, 65535), (1, 7, 7, 1, 1000), (3, 5, 8, 8, 13),
    (2, 70, 6, 2, 100), (1, 300, 4, 4, 1)])
def test_rope_matches_64_bits(pkg, dev, dtype, B, T, nh, nkv, pos):
    rows = pos + T + 3
    width = (nh + 2 * nkv) * HD
    wide = rand(dev, B, T, width + 64, dtype=dtype, seed=1)
    qkv = wide[..., :width]  # rows with a stride of their own
    qw, kw = ((1 + 0.2 * rand(dev, HD, seed=s).float()).to(dtype) for s in (2, 3))
    inv = pkg.rope_inv_freq(HD, 1e6)
    k0, v0 = rand(dev, B, nkv, rows, HD, seed=4, dtype=dtype), rand(dev, B, nkv, rows, HD, seed=5,
                                                                   dtype=dtype)
    k, v = k0.clone(), v0.clone()
    first = starts(pos, B)
    q = pkg.rope_append(qkv, nh, nkv, qw, kw, 1e-6, inv, i32(dev, first), k, v)
    x = qkv.cpu().reshape(B, T, nh + 2 * nkv, HD)
    p = torch.tensor(first)[:, None] + torch.arange(T)
    u = ref.half_step(dtype)
    for lo, n, w, got in ((0, nh, qw, q), (nh, nkv, kw, None)):
        want, size = ref.rope(x[:, :, lo:lo + n], w.cpu(), p[..., None], inv, 1e-6)
        if got is None:
            got = torch.stack([k[b, :, first[b]:first[b] + T].transpose(0, 1) for b in range(B)])
        # fp32: the norm's sum, root and quotient (2^-20 together), sine and cosine (2^-22),
        # the products; then one rounding
        err = 2.0 ** -19 * size
        assert ((got.double().cpu() - want).abs() <= err + u * (want.abs() + err) + 1e-7).all()
    for b in range(B):
        new = slice(first[b], first[b] + T)
        assert same(v[b, :, new].cpu().transpose(0, 1).contiguous(),
                    x[b, :, nh + nkv:].contiguous())
        for a, a0 in ((k, k0), (v, v0)):  # the other rows as they were
            assert same(a[b, :, :first[b]], a0[b, :, :first[b]])
            assert same(a[b, :, first[b] + T:], a0[b, :, first[b] + T:])


def test_rope_rows_padding_and_positions_outside(pkg, dev):
    """first_row, counts, a given output whose padding stays, and device positions outside."""
    B, T, nh, nkv = 4, 6, 4, 2
    qkv = rand(dev, B, T, (nh + 2 * nkv) * HD, seed=1)
    w = torch.ones(HD, dtype=torch.bfloat16, device=dev)
    inv = pkg.rope_inv_freq(HD, 1e4)
    counts = [6, 0, 3, 9]  # more than T: T
    k, v = (torch.full((B, nkv, 10, HD), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    out = torch.full((B, T, nh, HD), 5.0, dtype=torch.bfloat16, device=dev)
    pkg.rope_append(qkv, nh, nkv, w, w, 1e-6, inv, i32(dev, [5, 6, 900, 70000]), k, v,
                    first_row=2, counts=i32(dev, counts), out=out)
    whole = pkg.rope_append(qkv, nh, nkv, w, w, 1e-6, inv, i32(dev, [5, 6, 900, 70000]),
                            k.clone(), v.clone(), first_row=4)
    for b, c in enumerate(counts):
        c = min(c, T)
        assert same(out[b, :c], whole[b, :c]) and (out[b, c:] == 5.0).all()
        assert (v[b, :, :2] == 7.0).all() and (v[b, :, 2 + c:] == 7.0).all()
        assert same(v[b, :, 2:2 + c].transpose(0, 1).contiguous(),
                    qkv[b, :c].view(c, nh + 2 * nkv, HD)[:, nh + nkv:].contiguous())
    # a cache of 10 rows: from 8 on two tokens fit; -1 and 10 are outside
    k0, v0 = k.clone(), v.clone()
    q = pkg.rope_append(qkv, nh, nkv, w, w, 1e-6, inv, i32(dev, [8, -1, 10, 2**31 - 1]), k, v)
    assert torch.isfinite(q[0, :2]).all() and torch.isnan(q[0, 2:]).all()
    assert torch.isnan(q[1:]).all()
    assert same(k[1:], k0[1:]) and same(v[1:], v0[1:])
    assert same(k[0, :, :8], k0[0, :, :8]) and not same(k[0, :, 8:], k0[0, :, 8:])


# ------------------------------------------------------------------- attn_window

def case(dev, B, T, nh, nkv, rows, dtype, seed=0):
    q = rand(dev, B, T, nh, HD, seed=seed, dtype=dtype, gain=1.5)
    k = rand(dev, B, nkv, rows, HD, seed=seed + 1, dtype=dtype)
    v = rand(dev, B, nkv, rows, HD, seed=seed + 2, dtype=dtype) + 0.25
    return q, k, v


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("B,T,nh,nkv,pos,window,sinks", [
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
    (1, 5, 8, 1, 4095, 1000, 70),
    (2, 8, 32, 4, 64, 5000, 4),       # a window longer than the context
    (1, 17, 32, 4, 0, None, 0),
    (1, 33, 6, 2, 31, 16, 5),
    (1, 63, 4, 4, 1, 64, 0),
    (2, 64, 8, 2, 0, 65, 1),
    (1, 65, 32, 4, 63, 1, 0),
    (1, 129, 14, 2, 200, 37, 100),
    (1, 300, 8, 1, 777, 250, 65),
    (2, 257, 4, 2, 0, None, 0),
    (1, 500, 2, 2, 1500, 640, 128),
])
def test_attn_window_matches_64_bits(pkg, dev, dtype, B, T, nh, nkv, pos, window, sinks):
    rows = pos + T + 5
    q, k, v = case(dev, B, T, nh, nkv, rows, dtype, seed=pos + T)
    first = starts(pos, B)
    # nothing behind a sequence's own tokens may be read into its rows
    for b in range(B):
        k[b, :, first[b] + T:] = math.nan
        v[b, :, first[b] + T:] = math.inf
    want, tol = ref.attention(q, k, v, first, [T] * B, window, sinks)
    got = pkg.attn_window(q, k, v, i32(dev, first), window=window, sinks=sinks)
    check(got, want, tol)
    if B == 1:  # a host position, without the batch dimension
        one = pkg.attn_window(q[0], k[0], v[0], pos, window=window, sinks=sinks)
        check(one[None], want, tol)


@pytest.mark.parametrize("B,nh,nkv,T", [
    (70, 4, 1, 1),     # more sequences than a wave has lanes
    (150, 16, 2, 2),   # more kv heads than share 512 workgroups
    (300, 3, 1, 1), (600, 2, 2, 1),  # 1200 kv heads: a workgroup each
    (1, 32, 4, 4), (2, 31, 1, 1), (1, 33, 1, 1)])  # 32, 31 and 33 rows
@pytest.mark.parametrize("eight", [False, True])
def test_many_sequences_of_different_ages(pkg, dev, eight, B, nh, nkv, T):
    g = torch.Generator().manual_seed(B)
    first = (torch.rand(B, generator=g) ** 3 * 900).int().tolist()
    counts = [T - (b % 7 == 3) for b in range(B)]
    rows = 900 + T
    q, k, v = case(dev, B, T, nh, nkv, rows, torch.bfloat16, seed=B)
    keep = [0, 1, B // 3, B // 2, B - 1] + sorted(range(B), key=lambda b: -first[b])[:3]
    keep = sorted({b for b in keep if b < B})
    sub = lambda x: torch.stack([x[b] for b in keep])  # noqa: E731
    pos, cnt = [first[b] for b in keep], [counts[b] for b in keep]
    if eight:
        cache = pkg.KV8Cache.empty(nkv, rows, batch=B, device=dev)
        pkg.kv8_append(k.transpose(1, 2), v.transpose(1, 2), cache, 0,
                       counts=i32(dev, [p + c for p, c in zip(first, counts)]))
        got = pkg.attn_kv8(q, cache, i32(dev, first), counts=i32(dev, counts))
        kk, vv = cache.values()
        end = [p + c for p, c in zip(pos, cnt)]
        kk, vv = sub(kk).cpu(), sub(vv).cpu()
        for i, (b, e) in enumerate(zip(keep, end)):
            kk[i, :, e // 64 * 64:e] = cache.k_tail[b, :, :e % 64].float().cpu()
            vv[i, :, e // 64 * 64:e] = cache.v_tail[b, :, :e % 64].float().cpu()
    else:
        got = pkg.attn_window(q, k, v, i32(dev, first), counts=i32(dev, counts))
        kk, vv = sub(k), sub(v)
    want, tol = ref.attention(sub(q), kk, vv, pos, cnt, None, 0)
    check(sub(got), want, tol)


@pytest.mark.parametrize("T,nh", [(3, 4), (20, 8)])
def test_masked_infinities_in_the_tail(pkg, dev, T, nh):
    """Tokens of the unfinished block with NaN and infinities reach the later rows alone."""
    pos = 64 * 3 + 5
    kv = rand(dev, 2, 1, pos + T, 1, HD, seed=6)
    bad = pos + T - 2
    kv[0, 0, bad, 0, 3] = math.nan
    kv[1, 0, bad, 0, 9] = math.inf
    cache = pkg.KV8Cache.empty(1, pos + T, device=dev)
    want8 = ref.Cache8(1, 1, cache.max_len // 64, torch.int8, torch.bfloat16)
    pkg.kv8_append(kv[0], kv[1], cache, 0)
    want8.append(kv, [0], [pos + T])
    q = rand(dev, 1, T, nh, HD, seed=8)
    got = pkg.attn_kv8(q, cache, pos)
    k, v = want8.rows([pos + T])
    want, tol = ref.attention(q, k, v, [pos], [T - 2], None, 0)
    check(got[:, :T - 2], want[:, :T - 2], tol[:, :T - 2])
    assert torch.isnan(got[:, T - 2:]).all()


@pytest.mark.parametrize("T", [1, 4, 40, 150])
def test_attn_window_strides(pkg, dev, T):
    """[max_len, n_kv_heads, head_dim] caches and q as a view of the fused rows."""
    B, nh, nkv, pos = 2, 8, 2, 200
    rows = pos + T
    fused = rand(dev, B, T, nh + 2 * nkv, HD, seed=5)
    q = fused[:, :, :nh]
    k, v = (rand(dev, B, rows + 9, nkv + 1, HD, seed=s).transpose(1, 2)[:, 1:, :rows]
            for s in (6, 7))
    assert not q.is_contiguous() and not k.is_contiguous()
    want, tol = ref.attention(q, k, v, [pos] * B, [T] * B, 77, 3, scale=0.11)
    got = pkg.attn_window(q, k, v, pos, window=77, sinks=3, scale=0.11)
    check(got, want, tol)
    swapped = q.transpose(1, 2).contiguous().transpose(1, 2)  # [B, nh, T, d] in memory
    assert same(pkg.attn_window(swapped, k, v, pos, window=77, sinks=3, scale=0.11), got)


@pytest.mark.parametrize("T,nh", [(1, 8), (3, 8), (6, 16), (100, 8), (70, 14)])
def test_attn_window_padding_stays(pkg, dev, T, nh):
    B, nkv, pos = 4, 2, [100, 37, 0, 260]
    q, k, v = case(dev, B, T, nh, nkv, 260 + T, torch.bfloat16, seed=3)
    counts = [T, 0, (T + 1) // 2, T + 7]
    out = torch.full((B, T, nh, HD), 5.0, dtype=torch.bfloat16, device=dev)
    got = pkg.attn_window(q, k, v, i32(dev, pos), window=50, sinks=2, counts=i32(dev, counts),
                          out=out)
    assert got.data_ptr() == out.data_ptr()
    c = [min(n, T) for n in counts]
    for b in range(B):
        assert (out[b, c[b]:] == 5.0).all()
    want, tol = ref.attention(q, k, v, pos, c, 50, 2)
    check(out, want, tol)
    new = pkg.attn_window(q, k, v, i32(dev, pos), window=50, sinks=2, counts=i32(dev, counts))
    for b in range(B):
        assert same(new[b, :c[b]], out[b, :c[b]]) and (new[b, c[b]:] == 0).all()


@pytest.mark.parametrize("T", [1, 2, 90])
def test_attn_window_positions_outside(pkg, dev, T):
    B, nh, nkv, rows = 5, 8, 2, 100
    q, k, v = case(dev, B, T, nh, nkv, rows, torch.float16, seed=3)
    pos = [99, -1, 100, 2**31 - 1, 10]
    got = pkg.attn_window(q, k, v, i32(dev, pos))
    assert torch.isnan(got[1:4]).all() and torch.isnan(got[0, 1:]).all()
    want, tol = ref.attention(q, k, v, pos, [1, 0, 0, 0, T], None, 0)
    check(got, want, tol)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("T,nh,window,sinks", [(1, 8, 20, 2), (4, 8, 20, 2), (12, 8, 9, 3),
                                               (140, 8, 33, 5), (140, 2, None, 0)])
def test_masked_infinities_stay_out(pkg, dev, dtype, T, nh, window, sinks):
    """Keys and values with NaN and infinities reach exactly the rows that see them."""
    nkv, pos = 1, 150
    rows = pos + T
    q, k, v = case(dev, 1, T, nh, nkv, rows, dtype, seed=9)
    bad = {30: math.nan, 75: math.inf, 100: -math.inf}
    if T > 1:
        bad |= {pos + T // 2: math.nan, pos + T - 1: math.inf}
    for j, x in bad.items():
        v[0, 0, j, j % HD] = x
        v[0, 0, j, (j + 64) % HD] = x
        if j != pos + T - 1:
            k[0, 0, j, 5] = math.nan
    got = pkg.attn_window(q, k, v, pos, window=window, sinks=sinks)[0].cpu()
    ok = [t for t in range(T) if not any(ref.see(pos + t, rows, window, sinks)[j] for j in bad)]
    if window is not None:
        assert ok
    for t in range(T):
        hit = [j for j in bad if ref.see(pos + t, rows, window, sinks)[j]]
        if any(j != pos + T - 1 for j in hit):  # a NaN key: the row is NaN
            assert torch.isnan(got[t]).all(), t
        elif hit:  # the infinity alone
            assert not torch.isfinite(got[t][:, [(pos + T - 1) % HD, (pos + T + 63) % HD]]).any()
    kz, vz = k.clone(), v.clone()
    for j in bad:
        kz[0, 0, j], vz[0, 0, j] = 0, 0
    want, tol = ref.attention(q, kz, vz, [pos], [T], window, sinks)
    for t in ok:
        check(got[None, t:t + 1], want[:, t:t + 1], tol[:, t:t + 1])


@pytest.mark.parametrize("T", [1, 64])
def test_attn_window_extreme_scores(pkg, dev, T):
    """Scores that grow along the context by far more than fp32's exponent range, both ways."""
    nh = nkv = 1
    rows = 300 + T
    for sign in (1.0, -1.0):
        q, k, v = case(dev, 1, T, nh, nkv, rows, torch.bfloat16, seed=4)
        q[..., 1:] = 0
        q[..., 0] = 50.0
        k[..., 1:] = 0
        k[0, 0, :, 0] = (sign * torch.linspace(-50, 50, rows, device=dev)).to(torch.bfloat16)
        want, tol = ref.attention(q, k, v, [300], [T], None, 0)
        got = pkg.attn_window(q, k, v, 300)
        check(got, want, tol)


def test_long_cache_offsets(pkg, dev):
    """A batch of caches whose elements pass 2^32, read at its far end."""
    B, nkv, rows = 9, 4, 1 << 20
    k = torch.empty(B, nkv, rows, HD, dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 32
    at = rows - 1
    k[-1, :, -300:] = rand(dev, nkv, 300, HD, seed=1, dtype=torch.float16)
    v[-1, :, -300:] = rand(dev, nkv, 300, HD, seed=2, dtype=torch.float16)
    k[:, :, :3] = rand(dev, B, nkv, 3, HD, seed=3, dtype=torch.float16)
    v[:, :, :3] = rand(dev, B, nkv, 3, HD, seed=4, dtype=torch.float16)
    for T in (1, 40):
        q = rand(dev, B, T, 8, HD, seed=5, dtype=torch.float16)
        first = i32(dev, [0] * (B - 1) + [at - T + 1])
        counts = i32(dev, [min(T, 3)] * (B - 1) + [T])
        got = pkg.attn_window(q, k, v, first, window=200, sinks=3, counts=counts)
        kk = torch.cat([k[-1:, :, :3], k[-1:, :, -300:]], 2)
        vv = torch.cat([v[-1:, :, :3], v[-1:, :, -300:]], 2)
        want, tol = ref.attention(q[-1:], kk, vv, [303 - T], [T], 200, 3)
        check(got[-1:], want, tol)
        want, tol = ref.attention(q[:1], k[:1, :, :3], v[:1, :, :3], [0], [min(T, 3)], None, 0)
        check(got[:1], want, tol)


# ------------------------------------------------------------------- the 8-bit cache

def history(dev, B, n, total, dtype, seed=0):
    """[2, B, total, n, 128]: keys with strong channels, values; magnitudes vary by block."""
    x = rand(dev, 2, B, total, n, HD, seed=seed, dtype=torch.float32)
    x[0, ..., 7] *= 12
    x *= torch.exp(torch.randn(total // 16 + 1, generator=torch.Generator().manual_seed(seed)))[
        torch.arange(total) // 16].to(dev)[:, None, None]
    return x.to(dtype)


def compare(cache, want, B):
    k, v = cache.values()
    for s, (x, sc, tail) in enumerate(((k, cache.k_scale, cache.k_tail),
                                       (v, cache.v_scale, cache.v_tail))):
        wsc = want.scale[s].float()
        assert same(torch.nan_to_num(sc.cpu(), -1.0), torch.nan_to_num(wsc, -1.0))
        vals = (want.elem[s].float() * wsc[..., None, None]).reshape(x.shape)
        assert torch.equal(torch.nan_to_num(x.cpu(), 12345.0), torch.nan_to_num(vals, 12345.0))
        assert same(tail.cpu(), want.tail[s])


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,steps", [
    (1, [1] * 70), (2, [63, 1, 1, 64, 65]), (4, [200]), (3, [30, 100, 5, 57, 64]),
    (1, [64, 64]), (2, [129, 1, 61, 1, 1])])
def test_kv8_append_is_exact(pkg, dev, dtype, kind, n, steps):
    """Bit for bit the exact quotients, however the tokens arrive."""
    B, total = 2, sum(steps)
    kv = history(dev, B, n, total, dtype, seed=len(steps))
    blocks = -(-total // 64)
    cache = pkg.KV8Cache.empty(n, total, batch=B, dtype=dtype, kind=kind, device=dev)
    want = ref.Cache8(B, n, blocks, kind, dtype)
    at = 0
    for m in steps:
        new = kv[:, :, at:at + m]
        pkg.kv8_append(new[0], new[1], cache, at)
        want.append(new, [at] * B, [m] * B)
        at += m
    compare(cache, want, B)
    whole = pkg.KV8Cache.empty(n, total, batch=B, dtype=dtype, kind=kind, device=dev)
    pkg.kv8_append(kv[0], kv[1], whole, 0)
    assert same(whole.k, cache.k) and same(whole.v, cache.v)
    assert same(whole.k_scale, cache.k_scale) and same(whole.v_scale, cache.v_scale)
    r = total % 64
    assert same(whole.k_tail[:, :, :r], cache.k_tail[:, :, :r])


@pytest.mark.parametrize("kind", KINDS)
def test_kv8_ties_and_edges(pkg, dev, kind):
    """Quotients on and next to ties, blocks of zeros, of tiny and of non-finite values."""
    n, total = 1, 64 * 6
    x = torch.zeros(2, 1, total, n, HD, dtype=torch.float16, device=dev)
    # a scale of exactly 1 (largest 127 or 448): halves are ties
    full = 127.0 if kind == torch.int8 else 448.0
    line = torch.arange(64 * HD, device=dev).float().view(64, HD)
    x[:, 0, :64, 0] = (((line % 508) / 4 - 63.5) if kind == torch.int8 else
                       torch.ldexp(16 + (line % 16) / 2, ((line // 16) % 12 - 10).int())).half()
    x[:, 0, 0, 0, 0] = full
    x[:, 0, 64:128, 0] = (line * 2.0 ** -24).half()  # subnormal halves
    x[:, 0, 192, 0, 3] = math.nan
    x[:, 0, 256, 0, 4] = -math.inf
    x[:, 0, 320:, 0] = 65504.0
    cache = pkg.KV8Cache.empty(n, total, dtype=torch.float16, kind=kind, device=dev)
    want = ref.Cache8(1, n, 6, kind, torch.float16)
    pkg.kv8_append(x[0], x[1], cache, 0)
    want.append(x, [0], [total])
    compare(cache, want, 1)
    y = rand(dev, 2, 1, 64, n, HD, seed=1).to(torch.bfloat16) * 2.0 ** -120
    cache = pkg.KV8Cache.empty(n, 64, dtype=torch.bfloat16, kind=kind, device=dev)
    want = ref.Cache8(1, n, 1, kind, torch.bfloat16)
    pkg.kv8_append(y[0], y[1], cache, 0)
    want.append(y, [0], [64])
    compare(cache, want, 1)


def test_kv8_append_padding_positions_strides(pkg, dev):
    """Ragged counts, device positions (some outside), strided tokens; the rest untouched."""
    B, n, T, blocks = 6, 2, 150, 4
    kv = history(dev, B, n, T, torch.bfloat16, seed=2)
    pos, counts = [0, 63, 100, -1, 256, 250], [150, 0, 92, 150, 3, 150]
    cache = pkg.KV8Cache.empty(n, blocks * 64, batch=B, device=dev)
    want = ref.Cache8(B, n, blocks, torch.int8, torch.bfloat16)
    old = history(dev, B, n, 250, torch.bfloat16, seed=3)
    held = [0, 63, 100, 0, 0, 250]
    pkg.kv8_append(old[0], old[1], cache, 0, counts=i32(dev, held))
    want.append(old, [0] * B, held)
    compare(cache, want, B)
    turned = kv.transpose(2, 3).contiguous().transpose(2, 3)  # [B, n, T, d] in memory
    pkg.kv8_append(turned[0], turned[1], cache, i32(dev, pos), counts=i32(dev, counts))
    want.append(kv, pos, counts)
    compare(cache, want, B)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T,nh,nkv,pos,window,sinks", [
    (1, 1, 32, 4, 0, None, 0), (1, 1, 32, 4, 63, None, 0), (1, 1, 32, 4, 64, None, 0),
    (2, 1, 7, 1, 1000, 130, 3), (3, 1, 8, 8, 700, 1, 1), (1, 1, 40, 1, 333, 100, 70),
    (1, 2, 32, 4, 127, 64, 4), (2, 5, 8, 1, 190, None, 0), (1, 8, 16, 4, 1000, 500, 65),
    (1, 17, 32, 4, 0, None, 0), (1, 64, 8, 2, 0, None, 0), (1, 65, 4, 4, 63, 20, 1),
    (2, 100, 14, 2, 333, 90, 64), (1, 257, 8, 1, 127, None, 0)])
def test_attn_kv8_matches_64_bits(pkg, dev, dtype, kind, B, T, nh, nkv, pos, window, sinks):
    first = starts(pos, B)
    total = pos + T
    kv = history(dev, B, nkv, total, dtype, seed=pos)
    cache = pkg.KV8Cache.empty(nkv, total + 30, batch=B, dtype=dtype, kind=kind, device=dev)
    want8 = ref.Cache8(B, nkv, cache.max_len // 64, kind, dtype)
    for at, m in ((first, [0] * B), ([0] * B, first), (first, [T] * B)):
        new = kv if at != first else torch.stack(
            [kv[:, b, first[b]:first[b] + T] for b in range(B)], 1)
        pkg.kv8_append(new[0], new[1], cache, i32(dev, at), counts=i32(dev, m))
        want8.append(new, at, m)
    q = rand(dev, B, T, nh, HD, seed=8, dtype=dtype, gain=0.4)
    k, v = want8.rows([p + T for p in first])
    want, tol = ref.attention(q, k, v, first, [T] * B, window, sinks)
    got = pkg.attn_kv8(q, cache, i32(dev, first), window=window, sinks=sinks)
    check(got, want, tol)
    if B == 1:
        check(pkg.attn_kv8(q[0], cache, pos, window=window, sinks=sinks)[None], want, tol)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,nh", [(1, 4), (6, 4), (130, 2)])
def test_attn_kv8_block_scales(pkg, dev, dtype, kind, T, nh):
    """Value blocks of very different magnitudes, zeros among them, up and down."""
    total = 64 * 14 + T
    kv = rand(dev, 2, 1, total, 1, HD, seed=4, dtype=torch.float32)
    steps = [0, 6, -9, -9, 3, 14, None, 0, -4, 10, None, 2, -14, 5, 0, 0, 1]
    for i, p in enumerate(steps):
        kv[1, :, 64 * i:64 * i + 64] *= 0.0 if p is None else 2.0 ** p
    kv = kv.to(dtype)
    cache = pkg.KV8Cache.empty(1, total, dtype=dtype, kind=kind, device=dev)
    want8 = ref.Cache8(1, 1, cache.max_len // 64, kind, dtype)
    pkg.kv8_append(kv[0], kv[1], cache, 0)
    want8.append(kv, [0], [total])
    q = rand(dev, 1, T, nh, HD, seed=8, dtype=dtype)
    k, v = want8.rows([total])
    for window, sinks in ((None, 0), (70, 0), (200, 65)):
        want, tol = ref.attention(q, k, v, [total - T], [T], window, sinks)
        check(pkg.attn_kv8(q, cache, total - T, window=window, sinks=sinks), want, tol)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,nh", [(1, 4), (6, 4), (130, 2)])
def test_attn_kv8_of_one_key(pkg, dev, dtype, kind, T, nh):
    """A token that sees itself alone gets its value: the weight cancels, rounded or not.

    Left are the output's rounding (half a step) and 2^-16, what a sum of two bf16 numbers is
    off by; 2^-20 holds the fp32 operations."""
    total = 64 * 6
    kv = history(dev, 1, 1, total, dtype, seed=6)
    cache = pkg.KV8Cache.empty(1, total, dtype=dtype, kind=kind, device=dev)
    want8 = ref.Cache8(1, 1, cache.max_len // 64, kind, dtype)
    pkg.kv8_append(kv[0], kv[1], cache, 0)
    want8.append(kv, [0], [total])
    q = rand(dev, 1, T, nh, HD, seed=8, dtype=dtype)
    got = pkg.attn_kv8(q, cache, total - T, window=1).double().cpu()
    want = want8.rows([total])[1][0, 0, total - T:total].double().cpu()[None, :, None]
    tol = want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -16 + 2.0 ** -20) + 2.0 ** -25
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,nh", [(1, 8), (2, 8), (5, 24), (120, 8)])
def test_attn_kv8_padding_outside_and_bad_blocks(pkg, dev, kind, T, nh):
    """Ragged counts, positions outside, and blocks that read as NaN outside the window."""
    B, nkv = 5, 2
    total = 450 + T
    first, counts = [400, 63, 0, -1, 449], [T, 0, (T + 1) // 2, T, T]
    kv = history(dev, B, nkv, total, torch.bfloat16, seed=5)
    kv[:, 0, 70, 0, 3] = math.nan   # block 1 of head 0: not seen from 400 on
    cache = pkg.KV8Cache.empty(nkv, total, batch=B, kind=kind, device=dev)
    want8 = ref.Cache8(B, nkv, cache.max_len // 64, kind, torch.bfloat16)
    held = [max(p, 0) for p in first]
    pkg.kv8_append(kv[0], kv[1], cache, 0, counts=i32(dev, held))
    want8.append(kv, [0] * B, held)
    new = kv[:, :, :T]
    pkg.kv8_append(new[0], new[1], cache, i32(dev, first), counts=i32(dev, counts))
    want8.append(new, first, counts)
    out = torch.full((B, T, nh, HD), 5.0, dtype=torch.bfloat16, device=dev)
    q = rand(dev, B, T, nh, HD, seed=8, gain=0.4)
    pkg.attn_kv8(q, cache, i32(dev, first), window=200, sinks=3, counts=i32(dev, counts), out=out)
    assert torch.isnan(out[3]).all()
    k, v = want8.rows([max(p, 0) + c for p, c in zip(first, counts)])
    want, tol = ref.attention(q, k, v, first, [c if b != 3 else 0 for b, c in enumerate(counts)],
                               200, 3)
    check(out, want, tol)
    for b in (0, 1, 2, 4):
        assert (out[b, counts[b]:] == 5.0).all()


# ------------------------------------------------------------------- together

def test_positions_of_a_captured_graph(pkg, dev):
    """A decode token's three calls, captured once and replayed over positions, against the
    same calls made eagerly, both caches; eager work and synchronisations in between."""
    B, nh, nkv, rows = 3, 8, 2, 400
    w = (1 + 0.1 * rand(dev, HD, seed=1).float()).to(torch.bfloat16)
    inv = pkg.rope_inv_freq(HD, 1e6)
    steps = [rand(dev, B, 1, (nh + 2 * nkv) * HD, seed=20 + i) for i in range(6)]
    at = [[0, 62, 300], [1, 63, 301], [2, 64, 302], [3, 65, 303], [4, 66, 304], [5, 67, 399]]

    def state():
        k, v = (rand(dev, B, nkv, rows, HD, seed=s) for s in (3, 4))
        c8 = pkg.KV8Cache.empty(nkv, rows, batch=B, device=dev)
        pkg.kv8_append(k.transpose(1, 2), v.transpose(1, 2), c8, 0,
                       counts=i32(dev, at[0]))
        return k, v, c8, pkg.Workspace()

    def step(qkv, pos, st):
        k, v, c8, ws = st
        q = pkg.rope_append(qkv, nh, nkv, w, w, 1e-6, inv, pos, k, v)
        a = pkg.attn_window(q, k, v, pos, window=100, sinks=4, workspace=ws)
        new = qkv.view(B, 1, nh + 2 * nkv, HD)[:, :, nh:]
        pkg.kv8_append(new[:, :, :nkv], new[:, :, nkv:], c8, pos)
        return a, pkg.attn_kv8(q, c8, pos, workspace=ws)

    eager, taped = state(), state()
    pos, qkv = i32(dev, at[0]), steps[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(qkv, pos, state())  # loads the kernels
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = step(qkv, pos, taped)
    for x, p in zip(steps, at):
        qkv.copy_(x)
        pos.copy_(i32(dev, p))
        graph.replay()
        wa, wb = step(x, i32(dev, p), eager)
        torch.cuda.synchronize()
        assert same(a, wa) and same(b, wb), p
        assert same(taped[0], eager[0]) and same(taped[2].k_tail, eager[2].k_tail)
    assert same(taped[2].k, eager[2].k) and same(taped[2].v_scale, eager[2].v_scale)


@pytest.mark.parametrize("T", [2, 60])
def test_chunks_of_a_captured_graph(pkg, dev, T):
    """A chunk's attention over both caches, split along the context, captured without a
    workspace and replayed over positions and counts."""
    nh, nkv, rows = 16, 2, 4000
    q, k, v = case(dev, 1, T, nh, nkv, rows, torch.bfloat16, seed=T)
    c8 = pkg.KV8Cache.empty(nkv, rows, device=dev)
    pkg.kv8_append(k.transpose(1, 2), v.transpose(1, 2), c8, 0)
    pos, counts = i32(dev, [0]), i32(dev, [T])

    def step():
        return (pkg.attn_window(q, k, v, pos, window=3000, sinks=4, counts=counts),
                pkg.attn_kv8(q, c8, pos, counts=counts))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = step()
    # whole blocks, so that the appended tail is never asked for
    for p, n in ((0, T), (3904 - T, T), (64 - T, T), (1920 - T + 1, T - 1), (3840 - T, T)):
        pos.fill_(p)
        counts.fill_(n)
        graph.replay()
        wa, wb = step()
        torch.cuda.synchronize()
        # the graph's own zeros are of its capture: rows behind the count stay
        assert same(a[:, :n], wa[:, :n]) and same(b[:, :n], wb[:, :n]), (p, n)


@pytest.mark.parametrize("T", [1, 3, 100])
def test_other_stream_and_repeats(pkg, dev, T):
    """The same bits on every call, on another stream than the tensors' own as well."""
    q, k, v = case(dev, 2, T, 32, 4, 5000 + T, torch.bfloat16, seed=2)
    ws = pkg.Workspace()
    first = pkg.attn_window(q, k, v, 5000, window=3000, sinks=4, workspace=ws)
    for _ in range(3):
        assert same(pkg.attn_window(q, k, v, 5000, window=3000, sinks=4, workspace=ws), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = pkg.attn_window(q, k, v, 5000, window=3000, sinks=4)
    side.synchronize()
    assert same(other, first)


def test_a_conversation(pkg, dev):
    """A prompt, a padded second chunk and single tokens through rope_append, both caches and
    both attentions, against 64 bits with the exact 16-bit cache rows."""
    B, nh, nkv, window, sinks = 2, 16, 2, 90, 4
    w = (1 + 0.1 * rand(dev, HD, seed=1).float()).to(torch.bfloat16)
    inv = pkg.rope_inv_freq(HD, 1e6)
    rows = 320
    k, v = (torch.zeros(B, nkv, rows, HD, dtype=torch.bfloat16, device=dev) for _ in range(2))
    c8 = pkg.KV8Cache.empty(nkv, rows, batch=B, device=dev)
    want8 = ref.Cache8(B, nkv, c8.max_len // 64, torch.int8, torch.bfloat16)
    held = [0, 0]
    for i, (T, counts) in enumerate([(150, [150, 150]), (40, [40, 23]), (1, [1, 1]), (1, [1, 1]),
                                     (3, [3, 2])]):
        qkv = rand(dev, B, T, (nh + 2 * nkv) * HD, seed=30 + i)
        pos, cnt = i32(dev, held), i32(dev, counts)
        q = pkg.rope_append(qkv, nh, nkv, w, w, 1e-6, inv, pos, k, v, counts=cnt)
        new = torch.stack([torch.stack([torch.nn.functional.pad(
            x[b, :, held[b]:held[b] + counts[b]], (0, 0, 0, T - counts[b])).transpose(0, 1)
            for b in range(B)]) for x in (k, v)])
        pkg.kv8_append(new[0], new[1], c8, pos, counts=cnt)
        want8.append(new, held, counts)
        bounds = {"window": window, "sinks": sinks, "counts": cnt}
        a = pkg.attn_window(q, k, v, pos, **bounds)
        a8 = pkg.attn_kv8(q, c8, pos, **bounds)
        want, tol = ref.attention(q, k, v, held, counts, window, sinks)
        check(a, want, tol)
        ends = [h + c for h, c in zip(held, counts)]
        k8, v8 = want8.rows(ends)
        want, tol = ref.attention(q, k8, v8, held, counts, window, sinks)
        check(a8, want, tol)
        held = ends
    compare(c8, want8, B)
