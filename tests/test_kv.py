"""What rope_append, attn_window, kv8_append and attn_kv8 refuse, on the host and before any
launch (no compute call is made here), and the references of their GPU tests."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from tests import _kv_ref as ref

P = 0x10000  # an aligned address that nothing reads
NULL, SHAPE, DTYPE, ALIGN, WORKSPACE, STRIDE = -1, -2, -3, -4, -7, -9


def cache(lb, **kw):
    base = dict(k=P, v=P, batch_stride=4 * 256 * 128, head_stride=256 * 128, row_stride=128,
                batch=2, n_kv_heads=4, max_len=256, head_dim=128, dtype=2)
    return lb.KVCacheC(**{**base, **kw})


def cache8(lb, **kw):
    base = dict(k=P, v=P, k_scale=P, v_scale=P, k_tail=P, v_tail=P, batch=2, n_kv_heads=4,
                blocks=4, head_dim=128, dtype=2, format=0)
    return lb.KV8CacheC(**{**base, **kw})


BAD_TOKENS = [
    (dict(T=0), SHAPE), (dict(T=-3), SHAPE), (dict(pos=-1), SHAPE), (dict(pos=256), SHAPE),
    (dict(pos=250, T=7), SHAPE), (dict(pos=2**31 - 1, T=2**20), SHAPE),
    (dict(nh=6), SHAPE), (dict(nh=2), SHAPE), (dict(nh=2048), SHAPE), (dict(xt=0), DTYPE),
    (dict(xt=1), DTYPE), (dict(pos_dev=P + 2), ALIGN), (dict(counts=P + 1), ALIGN),
    (dict(pos_dev=P, T=2**20 + 1), SHAPE),
]
BAD_CACHE = [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(k=P + 8), ALIGN), (dict(v=P + 2), ALIGN),
    (dict(head_dim=64), SHAPE), (dict(batch=0), SHAPE), (dict(n_kv_heads=0), SHAPE),
    (dict(max_len=0), SHAPE), (dict(max_len=2**20 + 1), SHAPE), (dict(row_stride=120), STRIDE),
    (dict(row_stride=132), ALIGN), (dict(head_stride=64), STRIDE), (dict(batch_stride=0), STRIDE),
    (dict(row_stride=2**30), STRIDE), (dict(dtype=0), DTYPE), (dict(dtype=7), DTYPE),
]
BAD_CACHE8 = [(dict([(n, None)]), NULL) for n in ("k", "v", "k_scale", "v_scale", "k_tail",
                                                   "v_tail")] + [
    (dict(k=P + 4), ALIGN), (dict(v_tail=P + 4), ALIGN), (dict(head_dim=64), SHAPE),
    (dict(batch=0), SHAPE), (dict(n_kv_heads=0), SHAPE), (dict(blocks=0), SHAPE),
    (dict(blocks=2**14 + 1), SHAPE), (dict(dtype=0), DTYPE), (dict(format=2), DTYPE),
    (dict(format=-1), DTYPE)]


def call_rope(lb, lib, c=None, **kw):
    a = {**dict(qkv=P, xt=2, T=1, bs=16 * 128, ts=16 * 128, nh=8, qw=P, kw=P, pos_dev=None, pos=0,
                first=-1, counts=None, out=P), **kw}
    tab = (ctypes.c_float * 64)()
    return lib.i4_rope_append(a["qkv"], a["xt"], a["T"], a["bs"], a["ts"], a["nh"], a["qw"],
                              a["kw"], 1e-6, tab if a.get("tab", True) else None, a["pos_dev"],
                              a["pos"], a["first"], a["counts"], a["out"],
                              ctypes.byref(c or cache(lb)), None)


def call_attn(lb, lib, c=None, eight=False, **kw):
    a = {**dict(q=P, xt=2, T=1, bs=8 * 128, ts=8 * 128, hs=128, nh=8, pos_dev=None, pos=0,
                counts=None, window=0, sinks=0, scale=0.1, out=P, ws=P, wsb=1 << 40, counters=None), **kw}
    fn = lib.i4_attn_kv8 if eight else lib.i4_attn_window
    return fn(a["q"], a["xt"], a["T"], a["bs"], a["ts"], a["hs"], a["nh"],
              ctypes.byref(c or (cache8(lb) if eight else cache(lb))), a["pos_dev"], a["pos"],
              a["counts"], a["window"], a["sinks"], a["scale"], a["out"], a["ws"], a["wsb"],
              a["counters"], None)


def call_append(lb, lib, c=None, **kw):
    a = {**dict(k=P, v=P, xt=2, T=1, bs=512, ts=512, hs=128, pos_dev=None, pos=0, counts=None),
         **kw}
    return lib.i4_kv8_append(a["k"], a["v"], a["xt"], a["T"], a["bs"], a["ts"], a["hs"],
                             ctypes.byref(c or cache8(lb)), a["pos_dev"], a["pos"], a["counts"],
                             None)


@pytest.fixture
def lb(pkg):
    from qwen3_omni_duplex_amd import _lib

    return _lib


@pytest.mark.parametrize("bad,code", BAD_TOKENS + [
    (dict(qkv=None), NULL), (dict(qw=None), NULL), (dict(kw=None), NULL), (dict(out=None), NULL),
    (dict(tab=False), NULL), (dict(first=256), SHAPE), (dict(first=250, T=7), SHAPE),
    (dict(first=0, pos=2**24), SHAPE), (dict(T=2, ts=100), STRIDE), (dict(bs=100), STRIDE),
    (dict(qkv=P + 2), ALIGN), (dict(bs=16 * 128 + 1), ALIGN), (dict(out=P + 8), ALIGN)])
def test_rope_refuses(lb, pkg, bad, code):
    assert call_rope(lb, pkg.lib(), **bad) == code


@pytest.mark.parametrize("bad,code", BAD_CACHE)
def test_cache_refused(lb, pkg, bad, code):
    c = cache(lb, **bad)
    assert call_rope(lb, pkg.lib(), c) == code
    assert call_attn(lb, pkg.lib(), c) == code


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("bad,code", BAD_TOKENS + [
    (dict(q=None), NULL), (dict(out=None), NULL), (dict(window=-1), SHAPE),
    (dict(sinks=-1, window=4), SHAPE), (dict(sinks=4), SHAPE), (dict(scale=0.0), SHAPE),
    (dict(scale=-1.0), SHAPE), (dict(scale=math.inf), SHAPE), (dict(scale=math.nan), SHAPE),
    (dict(T=2, ts=64), STRIDE), (dict(hs=64), STRIDE), (dict(bs=64), STRIDE),
    (dict(q=P + 8), ALIGN), (dict(out=P + 8), ALIGN), (dict(hs=132), ALIGN),
    (dict(ts=8 * 128 + 4, T=2), ALIGN), (dict(counters=P + 2), ALIGN)])
def test_attention_refuses(lb, pkg, eight, bad, code):
    assert call_attn(lb, pkg.lib(), eight=eight, **bad) == code


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("bad,code", [(dict(ws=None), WORKSPACE), (dict(wsb=1 << 10), WORKSPACE),
                                      (dict(ws=P + 128), ALIGN)])
def test_workspace_refused(lb, pkg, eight, bad, code):
    c = cache8(lb, blocks=128) if eight else cache(lb, max_len=8192, head_stride=8192 * 128,
                                                   batch_stride=4 * 8192 * 128)
    need = pkg.lib().i4_attn_window_workspace_bytes(2, 1, 8, 4, 8001, 0, 0)
    assert need > 1 << 10 and pkg.lib().i4_attn_window_workspace_bytes(2, 1, 8, 4, 64, 0, 0) == 0
    assert call_attn(lb, pkg.lib(), c, eight=eight, pos=8000, **bad) == code


def test_workspace_sizes(pkg):
    """No size overflows, and a bound never asks for more than none."""
    size = pkg.lib().i4_attn_window_workspace_bytes
    big = 2**31 - 1
    for T, nh, nkv in ((1, 32, 4), (4, 32, 4), (5, 32, 4), (300, 8, 8)):
        most = size(2, T, nh, nkv, 1 << 20, 0, 0)
        assert 0 < most < 1 << 31
        for window, sinks in ((1, 0), (100, big), (big, big), (big, 0), (5000, 64)):
            assert 0 <= size(2, T, nh, nkv, 1 << 20, window, sinks) <= 2 * most
    assert size(0, 1, 8, 4, 64, 0, 0) == size(1, 0, 8, 4, 64, 0, 0) == 0
    assert size(1, 1, 9, 4, 64, 0, 0) == size(1, 1, 8, 0, 64, 0, 0) == 0


@pytest.mark.parametrize("bad,code", BAD_CACHE8)
def test_cache8_refused(lb, pkg, bad, code):
    c = cache8(lb, **bad)
    assert call_append(lb, pkg.lib(), c) == code
    assert call_attn(lb, pkg.lib(), c, eight=True) == code
    assert pkg.lib().i4_kv8_values(ctypes.byref(c), P, P, None) == code


@pytest.mark.parametrize("bad,code", [
    (dict(T=0), SHAPE), (dict(pos=-1), SHAPE), (dict(pos=250, T=7), SHAPE), (dict(k=None), NULL),
    (dict(v=None), NULL), (dict(xt=1), DTYPE), (dict(k=P + 8), ALIGN), (dict(hs=132), ALIGN),
    (dict(T=2, ts=64), STRIDE), (dict(bs=64), STRIDE), (dict(counts=P + 2), ALIGN)])
def test_append_refuses(lb, pkg, bad, code):
    assert call_append(lb, pkg.lib(), **bad) == code


def test_values_refuses(lb, pkg):
    c = cache8(lb)
    assert pkg.lib().i4_kv8_values(ctypes.byref(c), None, P, None) == NULL
    assert pkg.lib().i4_kv8_values(ctypes.byref(c), P, P + 4, None) == ALIGN


def test_cpu_tensors_are_refused(pkg):
    x = torch.zeros(1, 1, 8, 128, dtype=torch.bfloat16)
    k = torch.zeros(1, 4, 64, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.attn_window(x, k, k, 0)
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.KV8Cache.empty(4, 64, device="cpu")
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.rope_append(x.view(1, 1, -1), 4, 2, x, x, 1e-6, pkg.rope_inv_freq(128, 1e6), 0, k, k)


def test_python_refuses(pkg, monkeypatch):
    """Argument checks that come before any address is taken, on CPU tensors."""
    from qwen3_omni_duplex_amd import _lib, kv

    monkeypatch.setattr(_lib, "require_device", lambda *ts: torch.device("cpu"))
    q = torch.zeros(2, 3, 8, 128, dtype=torch.bfloat16)
    k = torch.zeros(2, 4, 64, 128, dtype=torch.bfloat16)
    cpu = torch.device("cpu")
    for bad, match in (
            (dict(window=0), "at least 1"), (dict(sinks=3), "window"),
            (dict(out=torch.zeros(2, 3, 8, 64, dtype=torch.bfloat16)), "contiguous"),
            (dict(out=torch.zeros(3, 2, 8, 128, dtype=torch.bfloat16)), "contiguous"),
            (dict(out=torch.zeros(2, 3, 8, 128)), "contiguous")):
        with pytest.raises(RuntimeError, match=match):
            kv.attn_window(q, k, k, 0, **bad)
    for pos in (-1, 62, 2**31, 2**32, 2**40 + 3):  # 3 tokens, 64 rows
        with pytest.raises(RuntimeError, match="outside"):
            kv.attn_window(q, k, k, pos)
    with pytest.raises(RuntimeError, match="batch"):
        kv.attn_window(q[:1], k, k, 0)
    with pytest.raises(RuntimeError, match="dimensions"):
        kv.attn_window(q[0, 0], k, k, 0)
    with pytest.raises(RuntimeError, match="strides"):
        kv.attn_window(q, k, k.transpose(0, 1).contiguous().transpose(0, 1), 0)
    with pytest.raises(RuntimeError, match="last dimension"):
        kv.attn_window(q, k.mT, k.mT, 0)
    for t in (torch.zeros(2), torch.zeros(1, dtype=torch.int32),
              torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(RuntimeError, match="int32"):
            kv._int32(t, 2, cpu, "pos")
    w, inv = torch.zeros(128, dtype=torch.bfloat16), pkg.rope_inv_freq(128, 1e6)
    x = torch.zeros(2, 3, 16 * 128, dtype=torch.bfloat16)
    for args, kw, match in (
            ((x, 8, 4, w[:64], w, 1e-6, inv, 0, k, k), {}, "head_dim"),
            ((x, 8, 4, w.float(), w, 1e-6, inv, 0, k, k), {}, "dtype"),
            ((x, 9, 4, w, w, 1e-6, inv, 0, k, k), {}, "head counts"),
            ((x, 8, 4, w, w, 1e-6, inv[:32], 0, k, k), {}, "inv_freq"),
            ((x, 8, 4, w, w, 1e-6, inv, 0, k.half(), k.half()), {}, "dtype"),
            ((x, 8, 4, w, w, 1e-6, inv, 0, k, k), {"first_row": -1}, "first_row"),
            ((x, 8, 4, w, w, 1e-6, inv, 0, k, k), {"first_row": 62}, "first_row"),
            ((x, 8, 4, w, w, 1e-6, inv, 0, k, k), {"first_row": 2**32}, "first_row"),
            ((x, 8, 4, w, w, 1e-6, inv, 62, k, k), {}, "outside"),
            ((x, 8, 4, w, w, 1e-6, inv, 2**32, k, k), {"first_row": 0}, "outside")):
        with pytest.raises(RuntimeError, match=match):
            kv.rope_append(*args, **kw)
    c = pkg.KV8Cache.empty(4, 100, batch=2, device="cpu")
    assert c.max_len == 128 and c.v.shape == (2, 4, 2, 128, 64)
    kk = torch.zeros(2, 3, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="does not match"):
        kv.kv8_append(kk[:, :, :2], kk[:, :, :2], c, 0)
    with pytest.raises(RuntimeError, match="agree"):
        kv.kv8_append(kk, kk.half(), c, 0)
    for pos in (-1, 126, 2**32):
        with pytest.raises(RuntimeError, match="outside"):
            kv.kv8_append(kk, kk, c, pos)
        with pytest.raises(RuntimeError, match="outside"):
            kv.attn_kv8(q, c, pos)
    t = list(c._t)
    for i, bad, match in ((0, t[0].view(torch.uint8), "int8 or float8"), (0, t[0][:, :, 0], "k is"),
                          (1, t[1].transpose(3, 4), "v must"), (2, t[2].double(), "float32"),
                          (3, t[3][:1], "v_scale"), (4, t[4].half(), "one dtype"),
                          (5, t[5][:, :, :32], "v_tail")):
        with pytest.raises(RuntimeError, match=match):
            pkg.KV8Cache(*(bad if j == i else y for j, y in enumerate(t)))


def test_reference_quantisation():
    """The reference's e4m3 grid rounding against torch's own, and int8 against hand values."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(64, 128, generator=g)
    e, s = ref.quantise(x, torch.float8_e4m3fn)
    assert s == pytest.approx(x.abs().max().item() / 448, rel=1e-6)
    near = (x.double() / s).float().to(torch.float8_e4m3fn).double()
    assert (e != near).float().mean() < 1e-3  # double rounding through fp32 aside
    y = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 63.49]])
    e, s = ref.quantise(y, torch.int8)
    assert s == 1.0 and e.tolist() == [[127, 0, 2, 2, 0, -2, 63]]
    e, s = ref.quantise(torch.tensor([[448.0, 17.0, 19.0, 0.5 * 2 ** -9, 1.5 * 2 ** -9]]),
                        torch.float8_e4m3fn)
    assert s == 1.0 and e.tolist() == [[448.0, 16.0, 20.0, 0.0, 2 * 2.0 ** -9]]
    assert math.isnan(ref.quantise(torch.tensor([[1.0, math.inf]]), torch.int8)[1])


def test_reference_visibility():
    assert ref.see(5, 8, None, 0).tolist() == [True] * 6 + [False] * 2
    assert ref.see(5, 8, 2, 1).nonzero()[:, 0].tolist() == [0, 4, 5]
    assert ref.see(0, 3, 1, 9).nonzero()[:, 0].tolist() == [0]


def test_module_refuses_several_sequences(pkg):
    """A batch of sequences is not read as the tokens of one (made before any launch)."""
    attn = pkg.ThinkerAttention.__new__(pkg.ThinkerAttention)
    torch.nn.Module.__init__(attn)
    attn.max_len = 64
    layer = pkg.ThinkerDecoderLayer.__new__(pkg.ThinkerDecoderLayer)
    torch.nn.Module.__init__(layer)
    layer.attn = attn
    for shape in ((2, 1, 16), (2, 3, 16), (2, 1, 1, 16)):
        for call in (attn, layer.unfused, pkg.ThinkerDecoder([layer]).unfused):
            with pytest.raises(ValueError, match="several sequences"):
                call(torch.zeros(shape), 0)
    with pytest.raises(ValueError, match="no token"):
        attn(torch.zeros(1, 0, 16), 0)


def test_scratch_of_long_chunks_is_the_calls_own(pkg):
    """What a workspace keeps is bounded, and a decoder's layers share one."""
    from qwen3_omni_duplex_amd import kv

    ws, cpu = pkg.Workspace(), torch.device("cpu")
    big, counters = kv._scratch(ws, kv.KEPT_BYTES + 1, cpu)
    assert big.numel() > kv.KEPT_BYTES and counters is None and ws.buf is None
    small, counters = kv._scratch(ws, 1000, cpu)
    assert ws.buf is small and counters is not None
    size = pkg.lib().i4_attn_window_workspace_bytes
    for B in (1, 3, 70, 256, 600):  # calls that count their parts
        for T, nh, nkv in ((1, 32, 4), (16, 2, 2), (2, 32, 4), (1, 16, 1)):
            assert size(B, T, nh, nkv, 1 << 20, 0, 0) <= kv.KEPT_BYTES

    class Attn(torch.nn.Module):
        def forward(self, h, pos, workspace=None):
            seen.append(workspace)
            return h

    seen = []
    layer = pkg.ThinkerDecoderLayer.__new__(pkg.ThinkerDecoderLayer)
    torch.nn.Module.__init__(layer)
    layer.attn, layer._fused = Attn(), False
    layer.moe = lambda h, residual: h
    dec = pkg.ThinkerDecoder([layer, layer])
    dec.step(torch.zeros(3, 16), 0)
    assert seen == [dec.context_workspace] * 2


def test_capture_on_another_device_than_the_current_one(pkg, monkeypatch):
    """Scratch of a call on cuda:1 goes by cuda:1's stream while cuda:0 is current."""
    import contextlib

    from qwen3_omni_duplex_amd import _lib, kv, ops

    now = [0]

    @contextlib.contextmanager
    def device(d):
        old, now[0] = now[0], d.index
        yield
        now[0] = old

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] in capturing)
    monkeypatch.setattr(_lib, "stream", lambda dev: 7)
    monkeypatch.setattr(kv, "_STREAM_WS", {})
    for capturing, want in (({1}, (False, True)), ({0}, (True, False)), (set(), (False, False))):
        for i in (0, 1):
            dev = torch.device("cuda", i)
            assert ops._capturing(dev) is want[i] and now[0] == 0
            got = []
            monkeypatch.setattr(kv.Workspace, "get", lambda self, n, d: got.append(self))
            monkeypatch.setattr(kv.Workspace, "counters", lambda self, d: None)
            kv._scratch(None, 100, dev)
            kept = kv._STREAM_WS.get((i, 7))
            assert (got[0] is not kept) == want[i]
    assert not ops._capturing(torch.device("cpu"))


def test_launches_past_the_grid_limit_are_refused(lb, pkg):
    """2^24 workgroups of 256 threads are more than a launch holds."""
    lib = pkg.lib()
    c = cache(lb, batch=16, max_len=1 << 20, head_stride=128 << 20, batch_stride=512 << 20)
    assert call_rope(lb, lib, c, T=1 << 20, bs=2048 << 20) == SHAPE
    for batch, T in ((1 << 14, 1), (1 << 14, 17)):  # few rows, and tiles of them
        many = dict(batch=batch, n_kv_heads=1024)
        big = cache(lb, **many, head_stride=256 * 128, batch_stride=1024 * 256 * 128)
        a = dict(T=T, nh=1024, ts=1024 * 128, bs=1024 * 128 * T)
        assert call_attn(lb, lib, big, **a) == SHAPE
        assert call_attn(lb, lib, cache8(lb, **many), eight=True, **a) == SHAPE
    c8 = cache8(lb, batch=1024, n_kv_heads=1024, blocks=16)
    assert lib.i4_kv8_values(ctypes.byref(c8), P, P, None) == SHAPE
