"""ThinkerAttention and ThinkerDecoder with prompts, a bounded context and an 8-bit cache."""
from __future__ import annotations

import pytest
import torch

from tests import _kv_ref as ref

pytestmark = pytest.mark.gpu
H, NH, NKV, HD = 1024, 8, 2, 128


def build(pkg, dev, seed=0, layers=1, max_len=320, dtype=torch.bfloat16, **context):
    g = torch.Generator(device=dev).manual_seed(seed)

    def ct(e, N, K):
        p = torch.randint(-2**31, 2**31, (e, N, K // 8), dtype=torch.int32, device=dev,
                          generator=g)
        sc = (torch.rand(e, N, K // 32, device=dev, generator=g) * 0.004 + 0.001).to(dtype)
        return pkg.QWeight(p, sc, None, "ct", 32, N, K)

    def vec(n):
        return (torch.rand(n, device=dev, generator=g) * 0.4 + 0.8).to(dtype)

    def layer():
        qkv = pkg.PackedQKV.from_qweights(ct(1, NH * HD, H), ct(1, NKV * HD, H),
                                          ct(1, NKV * HD, H))
        o = pkg.PackedLinear.from_qweight(ct(1, H, NH * HD))
        attn = pkg.ThinkerAttention(qkv, o, vec(HD), vec(HD), vec(H), NH, NKV, HD,
                                    max_len=max_len, **context)
        wr = (torch.randn(16, H, device=dev, generator=g) * 0.05).to(dtype)
        return pkg.ThinkerDecoderLayer(attn, pkg.FusedPackedMoE.from_stacked(
            ct(16, 2 * 512, H), ct(16, H, 512), wr, 4, norm_weight=vec(H)))

    return pkg.ThinkerDecoder([layer() for _ in range(layers)])


def tokens(dev, n, seed=9, dtype=torch.bfloat16):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(n, H, generator=g, device=dev).to(dtype)


def near(a, b, dtype=torch.bfloat16):
    """Two roundings apart at each of q|k|v, the rotated rows, the attention output and the
    layer's output: at most 8 steps of the largest value."""
    a, b = a.double(), b.double()
    assert torch.isfinite(a).all()
    return (a - b).abs().max() <= 16 * ref.half_step(dtype) * b.abs().max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_equals_token_by_token(pkg, dev, dtype):
    """A prompt, a chunk and single tokens against the decode step's own entries."""
    h = tokens(dev, 140, dtype=dtype)
    a, b = (build(pkg, dev, dtype=dtype).layers[0].attn for _ in range(2))
    one = torch.cat([a(h[i:i + 1], i) for i in range(140)])
    many = torch.cat([b(h[:90], 0), b(h[90:139], 90), b(h[139:], 139)])
    assert near(many, one, dtype)
    assert near(b.k_cache[:, :140], a.k_cache[:, :140], dtype)
    assert near(b.v_cache[:, :140], a.v_cache[:, :140], dtype)


def test_wide_window_is_no_window(pkg, dev):
    h = tokens(dev, 100)
    a, b = build(pkg, dev).layers[0], build(pkg, dev, window=320, sinks=4).layers[0]
    assert not b.fused()
    for x, pos in ((h[:70], 0), (h[70:71], 70), (h[71:], 71)):
        assert near(b.attn(x, pos), a.attn(x, pos))


@pytest.mark.parametrize("context", [
    {"window": 40, "sinks": 3}, {"kv_dtype": torch.int8},
    {"kv_dtype": torch.float8_e4m3fn, "window": 50, "sinks": 64}])
def test_bounded_and_8_bit_attention(pkg, dev, context):
    """The module's attention against 64 bits from its own projections, and the two launches
    around it."""
    attn = build(pkg, dev, **context).layers[0].attn
    h = tokens(dev, 260)
    from qwen3_omni_duplex_amd import kv, ops

    kc, vc = (torch.zeros(1, NKV, 320, HD, dtype=torch.bfloat16, device=dev) for _ in range(2))
    want8 = ref.Cache8(1, NKV, 5, context.get("kv_dtype", torch.int8), torch.bfloat16)
    at = 0
    for T in (150, 1, 1, 70, 5, 1):
        x = h[at:at + T]
        got = attn(x, at if T > 1 else torch.tensor([at], dtype=torch.int32, device=dev))
        qkv = attn.qkv.lin(ops.rmsnorm(x, attn.input_norm_w, attn.eps))
        q = kv.rope_append(qkv, NH, NKV, attn.q_norm_w, attn.k_norm_w, attn.eps, attn.inv_freq, at,
                           kc[0], vc[0])
        k, v = kc, vc
        if attn.kv8 is not None:
            want8.append(torch.stack([c[:, :, at:at + T].transpose(1, 2) for c in (kc, vc)]),
                         [at], [T])
            k, v = want8.rows([at + T])
        want, tol = ref.attention(q[None], k, v, [at], [T], context.get("window"),
                                  context.get("sinks", 0))
        a = (kv.attn_kv8(q, attn.kv8, at, window=attn.window, sinks=attn.sinks)
             if attn.kv8 is not None else
             kv.attn_window(q, kc[0], vc[0], at, window=attn.window, sinks=attn.sinks))
        assert ((a.double().cpu() - want[0]).abs() <= tol[0]).all()
        assert near(got, x + attn.o_proj(a.view(T, -1)))
        at += T
    attn.reset_cache()
    if attn.kv8 is not None:
        assert not attn.kv8.k_scale.any() and not attn.kv8.values()[0].any()


@pytest.mark.parametrize("context", [{}, {"window": 60, "sinks": 4}, {"kv_dtype": torch.int8}])
def test_decoder_prompt_then_steps(pkg, dev, context):
    """A decoder's prompt, then its decode steps eager and replayed from one graph."""
    dec, twin = (build(pkg, dev, layers=2, **context) for _ in range(2))
    h = tokens(dev, 80)
    assert torch.equal(dec.step(h[:70], 0), twin.step(h[:70], 0))
    pos, x = torch.tensor([70], dtype=torch.int32, device=dev), h[70:71].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        build(pkg, dev, layers=2, **context).step(x, pos)  # loads the kernels
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dec.step(x, pos)
    for i in range(70, 76):
        x.copy_(h[i:i + 1])
        pos.fill_(i)
        graph.replay()
        want = twin.step(h[i:i + 1], i)
        torch.cuda.synchronize()
        assert near(y, want) and torch.isfinite(y).all(), i


def test_module_refuses(pkg, dev):
    attn = build(pkg, dev, max_len=128).layers[0].attn
    for T, pos in ((2, 127), (1, 128), (129, 0), (1, -1)):
        with pytest.raises(ValueError, match="outside the cache"):
            attn(tokens(dev, T), pos)
    for bad in ({"window": 0}, {"sinks": 2}, {"window": 4, "sinks": -1}):
        with pytest.raises(ValueError, match="window"):
            build(pkg, dev, **bad)


def test_leading_dimension_of_one(pkg, dev):
    """[1, T, H] is [T, H], for a prompt and for one token."""
    a, b = (build(pkg, dev, layers=2) for _ in range(2))
    h = tokens(dev, 9)
    for x, pos in ((h[:8], 0), (h[8:], 8)):
        got, want = a.step(x[None], pos), b.step(x, pos)
        assert got.shape == (1, *want.shape) and torch.equal(got[0], want)
    with pytest.raises(ValueError, match="several sequences"):
        a.step(h[:2, None], 0)


@pytest.mark.parametrize("context", [{}, {"kv_dtype": torch.int8}])
def test_scratch_of_a_decoder(pkg, dev, context):
    """A long chunk far into a conversation leaves no scratch behind, and steps share one."""
    dec = build(pkg, dev, layers=3, max_len=65536, **context)
    T, pos = 1040, 64 * 936  # a whole block: the chunk can be appended twice
    need = pkg.lib().i4_attn_window_workspace_bytes(1, T, NH, NKV, pos + T, 0, 0)
    assert need > 1 << 25
    h = tokens(dev, T)
    for l in dec.layers:
        if l.attn.kv8 is not None:  # a cache of zeros
            l.attn.kv8.k_scale.fill_(1.0), l.attn.kv8.v_scale.fill_(1.0)
    first = dec.step(h, pos)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    again = dec.step(h, pos)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - held < need // 2  # the result
    assert torch.equal(first, again)
    dec.step(h[:2], pos)  # few rows: kept, once
    assert all(l.attn.context_workspace.buf is None for l in dec.layers)
    assert 0 < dec.context_workspace.buf.numel() <= 1 << 25


def test_8_bit_cache_follows_the_dtype(pkg, dev):
    """half() moves the unfinished block with the norms; the finished ones have no dtype."""
    h = tokens(dev, 100, dtype=torch.float16)
    a, b = (build(pkg, dev, kv_dtype=t).layers[0].attn for t in (torch.int8, None))
    a.half(), b.half()
    assert a.kv8.k_tail.dtype == a.kv8.v_tail.dtype == torch.float16
    for lo, hi in ((0, 60), (60, 61)):  # all of them still in 16 bits
        assert near(a(h[lo:hi], lo), b(h[lo:hi], lo), torch.float16)
    k8 = a.kv8.tensors
    a.bfloat16()
    assert a.kv8.k.data_ptr() == k8[0].data_ptr() and a.kv8.k_tail.dtype == torch.bfloat16
    assert torch.equal(a.kv8.k_tail, k8[4].bfloat16())
    assert torch.isfinite(a(h[61:].bfloat16(), 61)).all()


def test_end_of_an_8_bit_cache(pkg, dev):
    """Host and device positions end at the same one: max_len in whole blocks."""
    h = tokens(dev, 128)
    for step in (lambda p: p, lambda p: torch.tensor([p], dtype=torch.int32, device=dev)):
        attn = build(pkg, dev, max_len=100, kv_dtype=torch.int8).layers[0].attn
        assert attn.max_len == 128
        attn(h[:127], 0)
        assert torch.isfinite(attn(h[127:], step(127))).all()
    assert torch.isnan(attn(h[127:], step(128))).all()
    with pytest.raises(ValueError, match="outside the cache"):
        attn(h[127:], 128)
