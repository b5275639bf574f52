"""The cache operators at the edges of their ranges: far positions, value blocks of extreme and
zero scales, splits beyond one round of the merges, what 8 bits do to a prompt."""
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


def i32(dev, values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def check(got, want, tol):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert (off <= tol).all(), f"off by {(off / tol).max().item():.2f} times the tolerance"


def caches(pkg, dev, kv, kind, room=0):
    """An 8-bit cache of the tokens kv [2, B, T, n, 128] and its reference."""
    _, B, T, n, _ = kv.shape
    cache = pkg.KV8Cache.empty(n, T + room, batch=B, dtype=kv.dtype, kind=kind, device=dev)
    want = ref.Cache8(B, n, cache.max_len // 64, kind, kv.dtype)
    pkg.kv8_append(kv[0], kv[1], cache, 0)
    want.append(kv, [0] * B, [T] * B)
    return cache, want


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("pos", [1 << 17, 1 << 20, (1 << 22) + 12345, (1 << 24) - 5])
def test_rope_far_positions(pkg, dev, dtype, pos):
    """The rotation up to the last position that fp32 holds exactly."""
    T, nh, nkv = 5, 3, 1
    qkv = rand(dev, 1, T, (nh + 2 * nkv) * HD, seed=1, dtype=dtype)
    qw, kw = ((1 + 0.2 * rand(dev, HD, seed=s).float()).to(dtype) for s in (2, 3))
    inv = pkg.rope_inv_freq(HD, 1e6)
    k, v = (torch.zeros(1, nkv, T, HD, dtype=dtype, device=dev) for _ in range(2))
    x = qkv.cpu().view(1, T, nh + 2 * nkv, HD)
    p = torch.arange(pos, pos + T)[None, :, None]
    for at in (pos, i32(dev, [pos])):
        q = pkg.rope_append(qkv, nh, nkv, qw, kw, 1e-6, inv, at, k, v, first_row=0)
        for lo, n, w, got in ((0, nh, qw, q), (nh, nkv, kw, k.transpose(1, 2))):
            want, size = ref.rope(x[:, :, lo:lo + n], w.cpu(), p, inv, 1e-6)
            # the norm's sum, root and quotient 2^-20, the sines and cosines of the product's
            # two parts 2^-21; then one rounding
            err = 2.0 ** -19 * size
            check(got, want, err + ref.half_step(dtype) * (want.abs() + err) + 1e-7)


@pytest.mark.parametrize("kind", KINDS)
def test_append_quotients_that_underflow(pkg, dev, kind):
    """Elements so far below their block's largest that x / scale is below fp32's range."""
    x = torch.zeros(2, 1, 128, 1, HD, dtype=torch.bfloat16, device=dev)
    x[:, 0, 0] = 1e30
    small = [1e-20, -1e-20, 9.2e-41, -9.2e-41, 1e-38, -1e-38, 1e-8, -1e-8, 0.0, -0.0]
    for i, e in enumerate(small):
        x[:, 0, 1 + i] = e
    x[:, 0, 64] = 1e9
    for i, e in enumerate(small):
        x[:, 0, 65 + i, 0, ::2] = e
    cache, want = caches(pkg, dev, x, kind)
    for s, (got, sc) in enumerate(zip(cache.values(), (cache.k_scale, cache.v_scale))):
        assert torch.equal(sc.cpu(), want.scale[s].float())
        vals = (want.elem[s].float() * sc.cpu()[..., None, None]).reshape(got.shape)
        assert torch.equal(got.cpu(), vals)
    q = rand(dev, 1, 2, 4, HD, seed=1)
    assert torch.isfinite(pkg.attn_kv8(1e-30 * q, cache, 126)).all()


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,nh,n,more", [(1, 4, 20, 6), (6, 4, 20, 6), (130, 2, 20, 6),
                                         (50, 4, 6, 0), (50, 4, 5, 0)])  # the last: one split
def test_zero_block_behind_large_blocks(pkg, dev, dtype, kind, T, nh, n, more):
    """n blocks of scales up to 1 with a sum that grows along the context, then a block of
    zeros, then ordinary ones."""
    total = 64 * (n + 1 + more) + T
    kv = rand(dev, 2, 1, total, 1, HD, seed=4, dtype=torch.float32)
    big = 127.0 if kind == torch.int8 else 400.0
    kv[1, :, :64 * n, :, 17] = big
    kv[1, :, 64 * n:64 * n + 64] = 0
    kv = kv.to(dtype)
    cache, want8 = caches(pkg, dev, kv, kind)
    q = rand(dev, 1, T, nh, HD, seed=8, dtype=dtype, gain=0.01)
    k, v = want8.rows([total])
    for window, sinks in ((None, 0), (64 * 10, 64)):
        want, tol = ref.attention(q, k, v, [total - T], [T], window, sinks)
        check(pkg.attn_kv8(q, cache, total - T, window=window, sinks=sinks), want, tol)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("T,nh", [(2, 8), (3, 8), (90, 4)])
def test_blocks_of_scale_zero(pkg, dev, dtype, kind, which, T, nh):
    """A scale of 0 (an empty cache's, or another quantiser's for zeros): the block's values are
    zeros, also where a row sees part of the block alone."""
    total = 64 * 8 + T
    cache, want8 = caches(pkg, dev, rand(dev, 2, 1, total, 1, HD, seed=4, dtype=dtype), kind)
    for i in (0, 2, 5, 6):
        for s, (name, sc) in enumerate((("k", cache.k_scale), ("v", cache.v_scale))):
            if which in (name, "both"):
                sc[..., i] = 0
                want8.scale[s, ..., i] = 0
    q = rand(dev, 1, T, nh, HD, seed=8, dtype=dtype)
    k, v = want8.rows([total])
    for window, sinks in ((None, 0), (90, 0), (150, 20), (1, 0)):
        want, tol = ref.attention(q, k, v, [total - T], [T], window, sinks)
        check(pkg.attn_kv8(q, cache, total - T, window=window, sinks=sinks), want, tol)


@pytest.mark.parametrize("kind", [None] + KINDS)
@pytest.mark.parametrize("T,nh", [(1, 4), (6, 4), (130, 2)])
def test_values_near_the_end_of_bf16(pkg, dev, kind, T, nh):
    """bf16 values up to 2.5e38: the average is finite where the sum of the values under weights
    of at most 1 is; scores that grow along the context make the running maximum late."""
    total, pos = 64 * 6 + T, 64 * 6
    kv = rand(dev, 2, 1, total, 1, HD, seed=4, dtype=torch.float32)
    kv[1] = kv[1].clamp(-3, 3) * 1e37
    kv[1, :, ::7, :, 5] = 2.5e38
    kv[0, ..., 0] = torch.linspace(0, 12, total, device=dev)[None, :, None]
    kv = kv.to(torch.bfloat16)
    q = rand(dev, 1, T, nh, HD, seed=8, gain=0.1)
    q[..., 0] = 3.0
    if kind is None:
        k, v = (x.transpose(1, 2).contiguous() for x in kv)
        go = lambda **b: pkg.attn_window(q, k, v, pos, **b)  # noqa: E731
    else:
        cache, want8 = caches(pkg, dev, kv, kind)
        k, v = want8.rows([total])
        go = lambda **b: pkg.attn_kv8(q, cache, pos, **b)  # noqa: E731
    for window, sinks in ((1, 0), (3, 0), (2, 1)):
        want, tol = ref.attention(q, k, v, [pos], [T], window, sinks)
        check(go(window=window, sinks=sinks), want, tol)
    # rows of small weights on many large values of both signs: each sum stays in fp32
    kv[1] = torch.where(kv[1].abs() > 2e38, kv[1] / 4, kv[1])
    kv[1, :, 1::2] = -kv[1, :, 0:total - 1:2][:, :kv[1, :, 1::2].shape[1]]
    if kind is None:
        k, v = (x.transpose(1, 2).contiguous() for x in kv)
        go = lambda **b: pkg.attn_window(q, k, v, pos, **b)  # noqa: E731
    else:
        cache, want8 = caches(pkg, dev, kv, kind)
        k, v = want8.rows([total])
        go = lambda **b: pkg.attn_kv8(q, cache, pos, **b)  # noqa: E731
    want, tol = ref.attention(q, k, v, [pos], [T], 40, 4)
    check(go(window=40, sinks=4), want, tol)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,nh", [(1, 4), (6, 4), (130, 2)])
def test_bf16_blocks_of_very_different_magnitudes(pkg, dev, kind, T, nh):
    """Value blocks from 2^-90 to 2^100 in one cache, upwards, downwards and mixed."""
    total = 64 * 14 + T
    base = rand(dev, 2, 1, total, 1, HD, seed=4, dtype=torch.float32)
    mixed = [0, -90, 100, None, -90, -40, 60, 0, 100, -60, None, 20, -90, 100, 0, 0, 0]
    for steps in (mixed, sorted((s or 0) for s in mixed), sorted(((s or 0) for s in mixed),
                                                                  reverse=True), [-90] * 17):
        kv = base.clone()
        for i, p in enumerate(steps):
            kv[1, :, 64 * i:64 * i + 64] *= 0.0 if p is None else 2.0 ** p
        cache, want8 = caches(pkg, dev, kv.to(torch.bfloat16), kind)
        q = rand(dev, 1, T, nh, HD, seed=8, gain=0.5)
        k, v = want8.rows([total])
        for window, sinks in ((None, 0), (130, 64)):
            want, tol = ref.attention(q, k, v, [total - T], [T], window, sinks)
            # a workgroup's rows share the unit of their sums: what a row sees is kept to 2^-60
            # of the largest value among the cache's blocks
            tol += 2.0 ** -60 * v.abs().max().item()
            check(pkg.attn_kv8(q, cache, total - T, window=window, sinks=sinks), want, tol)


def splits(pkg, B, T, nh, nkv, keys, rows):
    need = pkg.lib().i4_attn_window_workspace_bytes(B, T, nh, nkv, keys, 0, 0)
    return need / ((HD + 2) * 4 * rows)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("T,nh,pos,least", [(4, 8, 8000, 17), (20, 4, 8000, 17), (33, 2, 6000, 17),
                                            (3, 6, 30000, 33)])
def test_merge_of_many_splits(pkg, dev, dtype, eight, T, nh, pos, least):
    """More splits than one round of the merge's loads, with a workgroup a row."""
    assert splits(pkg, 1, T, nh, 1, pos + T, T * nh) >= least
    kv = rand(dev, 2, 1, pos + T, 1, HD, seed=T, dtype=dtype)
    q = rand(dev, 1, T, nh, HD, seed=8, dtype=dtype)
    if eight:
        cache, want8 = caches(pkg, dev, kv, torch.int8)
        k, v = want8.rows([pos + T])
        got = pkg.attn_kv8(q, cache, pos)
    else:
        k, v = (x.transpose(1, 2).contiguous() for x in kv)
        got = pkg.attn_window(q, k, v, pos)
    want, tol = ref.attention(q, k, v, [pos], [T], None, 0)
    check(got, want, tol)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("counted", [True, False])
@pytest.mark.parametrize("B,nh,nkv,pos", [(1, 8, 1, 9000), (1, 4, 2, 32000), (2, 16, 1, 16500)])
def test_merge_of_many_parts(pkg, dev, dtype, eight, counted, B, nh, nkv, pos):
    """More parts than one round of the few-row merge, by the last workgroup or in a launch."""
    assert splits(pkg, B, 1, nh, nkv, pos + 1, 16 * B * nkv) > 32
    kv = rand(dev, 2, B, pos + 1, nkv, HD, seed=B, dtype=dtype)
    q = rand(dev, B, 1, nh, HD, seed=8, dtype=dtype)
    ws = pkg.Workspace()
    if not counted:
        ws.counters = lambda device: None
    first = [pos - 700 * b for b in range(B)]
    if eight:
        cache, want8 = caches(pkg, dev, kv, torch.int8)
        k, v = want8.rows([p + 1 for p in first])
        for b in range(B):  # each sequence's own unfinished block
            cache.k_tail[b] = kv[0, b, first[b] // 64 * 64:][:64].transpose(0, 1)[
                :, torch.arange(64) % (first[b] % 64 + 1)]
            cache.v_tail[b] = kv[1, b, first[b] // 64 * 64:][:64].transpose(0, 1)[
                :, torch.arange(64) % (first[b] % 64 + 1)]
            for s, x in enumerate((k, v)):
                n = first[b] % 64 + 1
                x[b, :, first[b] // 64 * 64:first[b] + 1] = (
                    (cache.k_tail, cache.v_tail)[s][b, :, :n].double().cpu())
        got = pkg.attn_kv8(q, cache, i32(dev, first), workspace=ws)
    else:
        k, v = (x.transpose(1, 2).contiguous() for x in kv)
        got = pkg.attn_window(q, k, v, i32(dev, first), workspace=ws)
    want, tol = ref.attention(q, k, v, first, [1] * B, None, 0)
    check(got, want, tol)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("kind", [None] + KINDS)
@pytest.mark.parametrize("T,nh,window", [(1, 8, 2), (2, 8, 9), (16, 1, 20)])
def test_few_rows_keep_their_weights(pkg, dev, dtype, kind, T, nh, window):
    """Up to 16 rows of a kv head: a weight is a sum of two 16-bit numbers, off by the square of
    half a step.  Values that cancel under the weights leave the output's rounding out of it; the
    oracle with weights of one number is off by more than the tolerance."""
    total, pos = 64 * 6 + T - 1, 64 * 6 - 1
    kv = rand(dev, 2, 1, total, 1, HD, seed=4, dtype=torch.float32)
    q = rand(dev, 1, T, nh, HD, seed=8, dtype=dtype, gain=0.1)
    kk = kv[0, 0, :, 0].to(dtype).double()
    w = torch.softmax(kk[pos - window + 1:pos + 1] @ q[0, 0, 0].double() / math.sqrt(HD), 0)
    # the last of the first row's values cancels the others
    vv = kv[1, 0, pos - window + 1:pos + 1, 0].to(dtype).double()
    kv[1, 0, pos, 0] = (-(w[:-1, None] * vv[:-1]).sum(0) / w[-1]).float()
    kv = kv.to(dtype)
    if kind is None:
        k, v = (x.transpose(1, 2).contiguous() for x in kv)
        got = pkg.attn_window(q, k, v, pos, window=window)
    else:
        cache, want8 = caches(pkg, dev, kv, kind)
        k, v = want8.rows([total])
        got = pkg.attn_kv8(q, cache, pos, window=window)
    u = 2.0 ** -8 if kind is not None else ref.half_step(dtype)  # 8-bit values: bf16 weights
    two, one = torch.empty(T, nh, HD, dtype=torch.float64), 0.0
    tol = two.clone()
    for t in range(T):
        j = ref.see(pos + t, pos + t + 1, window, 0).nonzero()[:, 0]
        kd, vd = (x.double().cpu()[0, 0][j] for x in (k, v))
        s = q[0, t].double().cpu() @ kd.T / math.sqrt(HD)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        mass = e @ vd.abs() / e.sum(-1, keepdim=True)
        size = (q[0, t].double().cpu().abs() @ kd.abs().T).amax(-1, keepdim=True) / math.sqrt(HD)
        two[t] = e @ vd / e.sum(-1, keepdim=True)
        # as in the reference's tolerance, with u^2 in the place of u for the weights
        off = (u * u + 2.0 ** -16 * size + 2.0 ** -18) * mass
        tol[t] = off + ref.half_step(dtype) * (two[t].abs() + off) + 2.0 ** -25
        r = e.to(torch.bfloat16 if kind is not None else dtype).double()
        one = max(one, (((r @ vd / e.sum(-1, keepdim=True)) - two[t]).abs() / tol[t]).max().item())
    assert one > 1.5
    check(got[0], two, tol)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("B,T,nh,nkv,pos,window,sinks", [
    (3, 300, 32, 4, 5000, 2048, 4), (1, 1500, 16, 4, 0, None, 0), (1, 200, 32, 4, 3000, 2000, 64)])
def test_tiles_repeat(pkg, dev, dtype, B, T, nh, nkv, pos, window, sinks):
    """Prompts and chunks over both caches give the same bits on every call."""
    kv = rand(dev, 2, B, pos + T, nkv, HD, seed=T, dtype=dtype)
    q = rand(dev, B, T, nh, HD, seed=8, dtype=dtype)
    k, v = (x.transpose(1, 2).contiguous() for x in kv)
    cache = pkg.KV8Cache.empty(nkv, pos + T, batch=B, dtype=dtype, device=dev)
    pkg.kv8_append(kv[0], kv[1], cache, 0)
    first = None
    for _ in range(4):
        got = (pkg.attn_window(q, k, v, pos, window=window, sinks=sinks),
               pkg.attn_kv8(q, cache, pos, window=window, sinks=sinks))
        if first is None:
            first = got
        assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, first))


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_over_8_bits_reads_whole_blocks(pkg, dev, kind):
    """A prompt's queries read the blocks that their call finished in 8 bits, their own among
    them, with later tokens in the scale; token by token the unfinished block is in 16 bits."""
    T, nh = 100, 2
    kv = rand(dev, 2, 1, T, 1, HD, seed=4)
    q = rand(dev, 1, T, nh, HD, seed=8)
    cache, whole8 = caches(pkg, dev, kv, kind)
    k, v = whole8.rows([T])
    want, tol = ref.attention(q, k, v, [0], [T], None, 0)
    prompt = pkg.attn_kv8(q, cache, 0)
    check(prompt, want, tol)
    one = pkg.KV8Cache.empty(1, T, kind=kind, device=dev)
    one8 = ref.Cache8(1, 1, 2, kind, torch.bfloat16)
    for t in range(T):
        pkg.kv8_append(kv[0, :, t:t + 1], kv[1, :, t:t + 1], one, t)
        one8.append(kv[:, :, t:t + 1], [t], [1])
        k, v = one8.rows([t + 1])
        wt, tt = ref.attention(q[:, t:t + 1], k, v, [t], [1], None, 0)
        check(pkg.attn_kv8(q[:, t:t + 1], one, t), wt, tt)
    assert torch.equal(one.k, cache.k) and torch.equal(one.v_scale, cache.v_scale)
    # a later token's infinity: all rows of its finished block, none of a tail's earlier rows
    for at in (60, 90):
        x = kv.clone()
        x[1, 0, at, 0, 3] = math.inf
        cache, _ = caches(pkg, dev, x, kind)
        got = pkg.attn_kv8(q, cache, 0)
        if at == 60:
            assert got.isnan().all()
        else:
            assert torch.equal(got[:, :at], prompt[:, :at])
            assert not torch.isfinite(got[:, at:, :, 3]).any()
