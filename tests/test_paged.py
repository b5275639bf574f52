"""What rope, paged_append and attn_paged refuse, on the host and before any launch (no compute
call is made here); the lookup of a page on the CPU; and the references of their GPU tests."""
from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from tests import _kv_ref as kvref
from tests import _paged_ref as ref
from tests.test_kv import ALIGN, BAD_TOKENS, DTYPE, NULL, P, SHAPE, STRIDE, WORKSPACE

CSRC = Path(__file__).resolve().parents[1] / "qwen3-omni-duplex_amd" / "csrc"


@pytest.fixture
def lb(pkg):
    from qwen3_omni_duplex_amd import _lib

    return _lib


def table(n=64, value=0.5):
    return (ctypes.c_float * n)(*[value] * n)


def rotary(lb, **kw):
    tab = kw.pop("tab", None) or table()
    base = dict(inv_freq=ctypes.addressof(tab), axes=None, factor=1.0, pairs=64, layout=0)
    c = lb.RotaryC(**{**base, **kw})
    c.keep = tab
    return c


def cache(lb, **kw):
    base = dict(k=P, v=P, table=P, page_stride=4 * 64 * 128, head_stride=64 * 128,
                table_stride=4, batch=2, n_kv_heads=4, pages=10, page=64, table_len=4,
                head_dim=128, dtype=2)
    return lb.PagedCacheC(**{**base, **kw})


def heads(lb, **kw):
    base = dict(x=P, y=P, xb=4 * 8 * 128, xt=8 * 128, xh=128, yb=4 * 8 * 128, yt=8 * 128, yh=128,
                heads=8)
    return lb.HeadsC(**{**base, **kw})


def at(c):
    return None if c is None else ctypes.byref(c)


def call_rope(lb, lib, q=None, k=None, r=None, turn=None, **kw):
    a = {**dict(xt=2, B=2, T=4, hd=128, pos_dev=None, pos=0, counts=None), **kw}
    return lib.i4_rope(at(q or heads(lb)), at(k), a["xt"], a["B"], a["T"], a["hd"],
                       at(r or rotary(lb)), a["pos_dev"], a["pos"], at(turn), a["counts"], 0, None)


def call_append(lb, lib, c=None, r=None, turn=None, **kw):
    a = {**dict(qkv=P, xt=2, T=1, bs=16 * 128, ts=16 * 128, nh=8, qw=P, kw=P, pos_dev=None, pos=0,
                counts=None, out=P), **kw}
    return lib.i4_paged_append(a["qkv"], a["xt"], a["T"], a["bs"], a["ts"], a["nh"], a["qw"],
                               a["kw"], 1e-6, at(r or rotary(lb)), a["pos_dev"], a["pos"], at(turn),
                               a["counts"], 0, a["out"], at(c or cache(lb)), None)


def call_attn(lb, lib, c=None, **kw):
    a = {**dict(q=P, xt=2, T=1, bs=8 * 128, ts=8 * 128, hs=128, nh=8, pos_dev=None, pos=0,
                counts=None, window=0, sinks=0, scale=0.1, out=P, ws=P, wsb=1 << 40,
                counters=None), **kw}
    return lib.i4_attn_paged(a["q"], a["xt"], a["T"], a["bs"], a["ts"], a["hs"], a["nh"],
                             at(c or cache(lb)), a["pos_dev"], a["pos"], a["counts"], 0, a["window"],
                             a["sinks"], a["scale"], a["out"], a["ws"], a["wsb"], a["counters"],
                             None)


BAD_CACHE = [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(table=None), NULL), (dict(k=P + 8), ALIGN),
    (dict(v=P + 2), ALIGN), (dict(table=P + 2), ALIGN), (dict(head_dim=64), SHAPE),
    (dict(batch=0), SHAPE), (dict(batch=65536), SHAPE), (dict(n_kv_heads=0), SHAPE),
    (dict(n_kv_heads=1025), SHAPE), (dict(pages=0), SHAPE), (dict(page=8), SHAPE),
    (dict(page=48), SHAPE), (dict(page=2048), SHAPE), (dict(page=0), SHAPE),
    (dict(page=-64), SHAPE), (dict(table_len=0), SHAPE), (dict(table_len=2**14 + 1), SHAPE),
    (dict(table_len=-1), SHAPE), (dict(page_stride=64), STRIDE), (dict(page_stride=2**60), STRIDE),
    (dict(head_stride=64), STRIDE), (dict(head_stride=2**60), STRIDE),
    (dict(table_stride=3), STRIDE), (dict(page_stride=4 * 64 * 128 + 4), ALIGN),
    (dict(head_stride=64 * 128 + 4), ALIGN), (dict(dtype=0), DTYPE), (dict(dtype=7), DTYPE)]


@pytest.mark.parametrize("bad,code", BAD_CACHE)
def test_cache_refused(lb, pkg, bad, code):
    assert call_append(lb, pkg.lib(), cache(lb, **bad)) == code
    assert call_attn(lb, pkg.lib(), cache(lb, **bad)) == code


BAD_ROTARY = [
    (dict(inv_freq=None), NULL), (dict(pairs=0), SHAPE), (dict(pairs=129), SHAPE),
    (dict(pairs=-1), SHAPE), (dict(layout=2), SHAPE), (dict(layout=-1), SHAPE),
    (dict(factor=math.inf), SHAPE), (dict(factor=math.nan), SHAPE),
    (dict(tab=table(64, math.nan)), SHAPE), (dict(tab=table(64, math.inf)), SHAPE),
    (dict(tab=table(64, -17.0)), SHAPE)]


@pytest.mark.parametrize("bad,code", BAD_ROTARY)
def test_rotary_refused(lb, pkg, bad, code):
    assert call_append(lb, pkg.lib(), r=rotary(lb, **bad)) == code
    assert call_rope(lb, pkg.lib(), r=rotary(lb, **bad)) == code


@pytest.mark.parametrize("bad,code", [
    (dict(pos=None), NULL), (dict(axes=0), SHAPE), (dict(axes=5), SHAPE), (dict(axes=2), SHAPE),
    (dict(pos=P + 2), ALIGN), (dict(axis_stride=-1), STRIDE), (dict(batch_stride=-4), STRIDE)])
def test_given_positions_refused(lb, pkg, bad, code):
    t = lb.TurnC(**{**dict(pos=P, axis_stride=8, batch_stride=4, axes=3), **bad})
    axes = (ctypes.c_uint8 * 64)(*[i % 3 for i in range(64)])
    r = rotary(lb, axes=ctypes.addressof(axes))
    assert call_append(lb, pkg.lib(), r=r, turn=t) == code
    assert call_rope(lb, pkg.lib(), r=r, turn=t) == code


def test_several_axes_need_the_pairs_axes(lb, pkg):
    t = lb.TurnC(P, 8, 4, 3)
    assert call_rope(lb, pkg.lib(), turn=t) == NULL
    assert call_append(lb, pkg.lib(), turn=t) == NULL


@pytest.mark.parametrize("bad,code", [b for b in BAD_TOKENS if "nh" not in b[0]] + [
    (dict(qkv=None), NULL), (dict(out=None), NULL), (dict(nh=6), SHAPE), (dict(nh=2048), SHAPE),
    (dict(T=2, ts=100), STRIDE), (dict(bs=100), STRIDE), (dict(qkv=P + 2), ALIGN),
    (dict(bs=16 * 128 + 1), ALIGN), (dict(out=P + 8), ALIGN), (dict(qw=P + 8), ALIGN),
    (dict(kw=P + 2), ALIGN)])
def test_append_refuses(lb, pkg, bad, code):
    assert call_append(lb, pkg.lib(), **bad) == code


def test_append_refuses_parts_of_a_vector(lb, pkg):
    for pairs, layout in ((60, 0), (4, 0), (65, 1), (72, 0)):
        assert call_append(lb, pkg.lib(), r=rotary(lb, pairs=pairs, layout=layout,
                                                   tab=table(72))) == SHAPE


@pytest.mark.parametrize("bad,code", BAD_TOKENS + [
    (dict(q=None), NULL), (dict(out=None), NULL), (dict(window=-1), SHAPE),
    (dict(sinks=-1, window=4), SHAPE), (dict(sinks=4), SHAPE), (dict(scale=0.0), SHAPE),
    (dict(scale=math.nan), SHAPE), (dict(T=2, ts=64), STRIDE), (dict(hs=64), STRIDE),
    (dict(bs=64), STRIDE), (dict(q=P + 8), ALIGN), (dict(out=P + 8), ALIGN),
    (dict(hs=132), ALIGN), (dict(counters=P + 2), ALIGN)])
def test_attention_refuses(lb, pkg, bad, code):
    assert call_attn(lb, pkg.lib(), **bad) == code


@pytest.mark.parametrize("bad,code", [(dict(ws=None), WORKSPACE), (dict(wsb=1 << 10), WORKSPACE),
                                      (dict(ws=P + 128), ALIGN)])
def test_workspace_refused(lb, pkg, bad, code):
    c = cache(lb, table_len=128, table_stride=128)
    assert call_attn(lb, pkg.lib(), c, pos=8000, **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(xt=0), DTYPE), (dict(xt=7), DTYPE), (dict(B=0), SHAPE), (dict(B=65536), SHAPE),
    (dict(T=0), SHAPE), (dict(T=2**20 + 1), SHAPE), (dict(B=65535, T=2**20), SHAPE),
    (dict(hd=0), SHAPE), (dict(hd=127), SHAPE), (dict(hd=258), SHAPE), (dict(hd=126), SHAPE),
    (dict(pos=2**24 - 3), SHAPE), (dict(pos=-2**24), SHAPE), (dict(pos_dev=P + 2), ALIGN),
    (dict(counts=P + 1), ALIGN)])
def test_rope_refuses(lb, pkg, bad, code):
    assert call_rope(lb, pkg.lib(), **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(x=None), NULL), (dict(y=None), NULL), (dict(heads=0), SHAPE), (dict(heads=1025), SHAPE),
    (dict(xh=127), STRIDE), (dict(yh=0), STRIDE), (dict(xt=-1024), STRIDE), (dict(yb=8), STRIDE),
    (dict(x=P + 1), ALIGN), (dict(y=P + 1), ALIGN)])
def test_rope_rows_refused(lb, pkg, bad, code):
    assert call_rope(lb, pkg.lib(), heads(lb, **bad)) == code
    assert call_rope(lb, pkg.lib(), k=heads(lb, **bad)) == code


def test_python_refuses(pkg, monkeypatch):
    """Argument checks that come before any address is taken, on CPU tensors."""
    from qwen3_omni_duplex_amd import _lib

    monkeypatch.setattr(_lib, "require_device", lambda *ts: torch.device("cpu"))
    bf = torch.bfloat16
    R = pkg.Rotary
    for bad, match in ((dict(layout="other"), "layout"), (dict(factor=math.nan), "factor"),
                       (dict(axes=[0, 1]), "axes"), (dict(axes=[4] * 64), "axes")):
        with pytest.raises(RuntimeError, match=match):
            R(torch.ones(64), **bad)
    for f in (torch.ones(0), torch.ones(129), torch.ones(2, 2), torch.full((4,), math.nan),
              torch.full((4,), 17.0)):
        with pytest.raises(RuntimeError, match="inv"):
            R(f)
    with pytest.raises(RuntimeError, match="scale"):
        R.scaled(64, 1e4, 0.5)
    for shape in ((4, 2, 48, 128), (4, 2, 8, 128), (4, 2, 2048, 128)):
        with pytest.raises(RuntimeError, match="power of two"):
            pkg.PagedCache(torch.zeros(shape, dtype=bf), torch.zeros(shape, dtype=bf))
    k = torch.zeros(4, 2, 16, 128, dtype=bf)
    for a, b, match in ((k, k[:3], "agree"), (k, k.half(), "agree"), (k[0], k[0], "agree"),
                        (k.transpose(1, 2), k.transpose(1, 2), "dense"),
                        (k.float(), k.float(), "float16")):
        with pytest.raises(RuntimeError, match=match):
            pkg.PagedCache(a, b)
    with pytest.raises(RuntimeError, match="their own"):
        pkg.PagedCache(k, k)
    c = pkg.PagedCache(k, k.clone())
    q = torch.zeros(2, 3, 4, 128, dtype=bf)
    t = torch.zeros(2, 2, dtype=torch.int32)
    for bad in (t.long(), t[:1], torch.zeros(2, 0, dtype=torch.int32), t[0], t.t().contiguous().t(),
                t[None]):
        with pytest.raises(RuntimeError, match="table"):
            pkg.attn_paged(q, c, bad, 0)
    for pos in (-1, 30, 2**31, 2**32):
        with pytest.raises(RuntimeError, match="outside"):
            pkg.attn_paged(q, c, t, pos)
    with pytest.raises(RuntimeError, match="window"):
        pkg.attn_paged(q, c, t, 0, sinks=3)
    r, x, w = R.plain(128, 1e4), torch.zeros(2, 3, 8 * 128, dtype=bf), torch.ones(128, dtype=bf)
    for bad, match in ((dict(qkv=x[..., :-128]), "width"), (dict(qw=w.half()), "norm"),
                       (dict(qkv=x.half()), "dtype"), (dict(kw=w[:64]), "norm"),
                       (dict(r=R.plain(24, 1e4)), "multiple of 16"),
                       (dict(r=R.plain(192, 1e4)), "at most"), (dict(pos=30), "outside"),
                       (dict(turn=torch.zeros(2, 2, dtype=torch.int32)), "positions"),
                       (dict(turn=torch.zeros(3, 2, 3, dtype=torch.int32)), "axes"),
                       (dict(turn=torch.zeros(2, 3)), "int32"),
                       (dict(out=torch.zeros(2, 3, 4, 64, dtype=bf)), "out")):
        a = {**dict(qkv=x, qw=w, kw=w, r=r, pos=0, turn=None, out=None), **bad}
        with pytest.raises(RuntimeError, match=match):
            pkg.paged_append(a["qkv"], 4, a["qw"], a["kw"], 1e-6, a["r"], a["pos"], c, t,
                             turn=a["turn"], out=a["out"])
    for bad, match in ((dict(k=q.half()), "dtype"), (dict(k=q[:1]), "match"),
                       (dict(k=q[..., :64]), "match"), (dict(r=R.plain(192, 1e4)), "turn"),
                       (dict(pos=2**24 - 2), "outside"), (dict(pos=-2**24), "outside"),
                       (dict(pos=torch.zeros(3, dtype=torch.int32)), "int32"),
                       (dict(pos=torch.zeros(3, 2, dtype=torch.int32)), "positions"),
                       (dict(pos=torch.zeros(2, 2, 3, dtype=torch.int32)), "axes"),
                       (dict(out=(q,)), "each"), (dict(k=None, out=(q[..., :64],)), "out must"),
                       (dict(k=None, out=(q.half(),)), "out must")):
        a = {**dict(k=q, r=r, pos=0, out=None), **bad}
        with pytest.raises(RuntimeError, match=match):
            pkg.rope(q, a["k"], a["pos"], a["r"], out=a["out"])
    room = torch.zeros(2, 4, 4, 128, dtype=bf)
    for x, y in ((room[:, :3], room[:, 1:]), (room[:, 1:], room[:, :3])):
        with pytest.raises(RuntimeError, match="overlap"):
            pkg.rope(x, None, 0, r, out=(y, None))
    f = torch.zeros(2, 3, 8 * 128, dtype=bf).unflatten(2, (8, 128))
    for a, b, out in ((f[:, :, :4], f[:, :, 3:], (f[:, :, :4], f[:, :, 3:])),
                      (f[:, :, :4], f[:, :, :4], (f[:, :, :4], q)),
                      (f[:, :, :4], f[:, :, 4:], (q, q)),
                      (f[:, :, :4], f[:, :, 4:], (f[:, :, 4:], f[:, :, :4])),
                      (f[:, :, :4], f[:, :, 4:], (f[:, :, :4], f[:, :, 3:7]))):
        with pytest.raises(RuntimeError, match="overlap"):
            pkg.rope(a, b, 0, r, out=out)
    with pytest.raises(RuntimeError, match="overlap"):
        pkg.attn_paged(q, c, t, 0, out=q)
    rows = torch.zeros(2 * 3 * 8 * 128, dtype=bf)
    with pytest.raises(RuntimeError, match="overlap"):
        pkg.paged_append(rows.view(2, 3, -1), 4, w, w, 1e-6, r, 0, c, t,
                         out=rows[:2 * 3 * 4 * 128].view(2, 3, 4, 128))
    with pytest.raises(RuntimeError, match="apart"):
        pkg.rope(q, None, 0, r, out=(q[:1].expand(2, 3, 4, 128), None))


def test_structs_are_packed_as_declared(pkg, monkeypatch):
    """The bytes that the wrappers pass are the structs' own."""
    from qwen3_omni_duplex_amd import _lib, paged, rotary

    monkeypatch.setattr(_lib, "require_device", lambda *ts: torch.device("cpu"))
    assert rotary._heads(1, 2, 3, 4, 5, 6, 7, -8, 9) == bytes(_lib.HeadsC(1, 2, 3, 4, 5, 6, 7, -8, 9))
    assert rotary._turn(1, 2, 3, 4) == bytes(_lib.TurnC(1, 2, 3, 4))
    assert paged._paged(*range(1, 14)) == bytes(_lib.PagedCacheC(*range(1, 14)))
    c = pkg.PagedCache(*(torch.zeros(4, 2, 16, 128, dtype=torch.float16) for _ in range(2)))
    t = torch.zeros(3, 9, dtype=torch.int32)[:, :5]
    got, keys = c._with(t, 3)
    s = _lib.PagedCacheC.from_buffer_copy(got)
    assert keys == 80 and (s.k, s.v, s.table) == (c.k.data_ptr(), c.v.data_ptr(), t.data_ptr())
    assert (s.page_stride, s.head_stride, s.table_stride) == (2 * 16 * 128, 16 * 128, 9)
    assert (s.batch, s.n_kv_heads, s.pages, s.page, s.table_len, s.head_dim, s.dtype) == \
        (3, 2, 4, 16, 5, 128, 1)


def test_overlap_of_views(pkg):
    from qwen3_omni_duplex_amd.rotary import overlaps

    f = torch.zeros(3, 5, 10 * 16).unflatten(2, (10, 16))
    q, k, v = f[:, :, :4], f[:, :, 4:6], f[:, :, 6:]
    assert not any(overlaps(a, b) for a, b in ((q, k), (k, q), (k, v), (q, v), (v, k)))
    assert overlaps(q, q) and overlaps(f[:, :, :5], k) and overlaps(k, f[:, :, 5:])
    assert not overlaps(f[:, :2], f[:, 2:4].clone()) and overlaps(f[:, 1:3], f[:, 2:4])
    assert not overlaps(f[:1], f[1:2]) and not overlaps(f[:, :1, :4], f[:, :1, 4:])
    assert not overlaps(f[:, :1, :4], f[:, 1:2, :4])
    h = f.transpose(1, 2)  # heads before tokens
    assert not overlaps(h[:, :, :2], h[:, :, 2:]) and overlaps(h[:, :, :3], h[:, :, 2:])
    assert overlaps(f, f[:, :, :, ::2].expand(3, 5, 10, 8)) and overlaps(f[0:1].expand(3, 5, 10, 16), f)
    w = torch.zeros(4096)
    for i in range(300):  # against the elements themselves
        g = torch.Generator().manual_seed(i)
        n = torch.randint(1, 4, (2, 3), generator=g).tolist()
        s = torch.randint(1, 30, (3,), generator=g).tolist()
        o = torch.randint(0, 60, (2,), generator=g).tolist()
        x, y = (w.as_strided(n[k], s, o[k]) for k in (0, 1))
        ids = [set(torch.arange(4096).as_strided(n[k], s, o[k]).flatten().tolist()) for k in (0, 1)]
        assert overlaps(x, y) or not ids[0] & ids[1]  # it may refuse what is apart, never the reverse
    one = torch.zeros(64).view(1, 1, 4, 16)
    assert not overlaps(one[:, :, :2], one[:, :, 2:]) and overlaps(one[:, :, :3], one[:, :, 2:])


def test_pools_that_overlap(pkg, monkeypatch):
    """k and v share no element: not one tensor, not pages or heads apart of one; beside each
    other in one allocation in any way they may lie."""
    monkeypatch.setattr(pkg.paged._lib, "require_device", lambda *ts: torch.device("cuda", 0))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    x = torch.zeros(7, 4, 16, 128, dtype=torch.bfloat16)
    for k, v in ((x, x), (x[:6], x[1:]), (x[1:], x[:6]), (x[:, :3], x[:, 1:])):
        with pytest.raises(RuntimeError, match="pools of their own"):
            pkg.PagedCache(k, v)
    for k, v in ((x[:3], x[3:6]), (x[:, :2], x[:, 2:]), (x[::2][:3], x[1::2]), (x[:, ::2], x[:, 1::2]),
                 (x.transpose(0, 1)[:2], x.transpose(0, 1)[2:])):
        assert pkg.PagedCache(k, v).page == 16


def test_copies(pkg, monkeypatch):
    """A copied handle holds its own tensors' addresses."""
    import copy
    import pickle

    from qwen3_omni_duplex_amd import _lib

    monkeypatch.setattr(_lib, "require_device", lambda *ts: torch.device("cpu"))
    c = pkg.PagedCache(*(torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16) for _ in range(2)))
    d = copy.deepcopy(c)
    assert d.k.data_ptr() != c.k.data_ptr() and d._c[4] == d.k.data_ptr() and d.pages == 4
    r = pkg.Rotary.plain(32, 1e4, axes=[0, 1] * 8, factor=1.5, layout="interleaved")
    for s in (copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert torch.equal(s.inv_freq, r.inv_freq) and repr(s) == repr(r)
        assert s._c.inv_freq == s.inv_freq.data_ptr() != r.inv_freq.data_ptr()


def test_cpu_tensors_are_refused(pkg):
    x = torch.zeros(1, 1, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.rope(x, None, 0, pkg.Rotary.plain(128, 1e4))
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.PagedCache.empty(4, 8, device="cpu")


def test_page_lookup_stays_inside_the_pool(tmp_path):
    """Whatever a table holds, the row that is read lies inside a page of the pool; entries
    outside it are said to be bad."""
    src = tmp_path / "page.cpp"
    src.write_text('#include "i4_page.h"\n'
                   'extern "C" long long row(int id, int pages, long long ps, long long hs, '
                   'int shift, int g, int j, int* bad) {\n'
                   '  const i4::PageRows r = i4::page_rows_of(id, pages, ps, hs, shift, 256, g, j);\n'
                   '  *bad = r.bad;\n  return r.at;\n}\n')
    so = tmp_path / "page.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-Wall", "-Werror", "-D__host__=",
                    "-D__device__=", "-I", str(CSRC), str(src), "-o", str(so)], check=True)
    row = ctypes.CDLL(str(so)).row
    row.restype = ctypes.c_longlong
    row.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_longlong, ctypes.c_longlong,
                    ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    bad = ctypes.c_int()
    for pages in (1, 7, 2**31 - 1):
        for shift in (4, 6, 10):
            page = 256 << shift
            for ps, hs in ((4 * page, page), (page, pages * page)):
                for id in (0, 1, 6, 7, pages - 1, pages % 2**31, -1, -2**31, 2**31 - 1, 2**30):
                    for g in (0, 3):
                        for j in (0, 15, 16, 1023, 2**20 - 1):
                            at = row(id, pages, ps, hs, shift, g, j, bad)
                            ok = 0 <= id < pages
                            assert bad.value == (not ok)
                            assert at == (id if ok else 0) * ps + g * hs + \
                                j % (1 << shift) * 256


def test_tables(pkg):
    """Rotary's tables against their definitions in 64 bits."""
    d, theta = 64, 1e4
    i = torch.arange(0, d, 2, dtype=torch.double)
    want = theta ** (-i / d)
    near = dict(rtol=2.0 ** -22, atol=0)  # a few roundings of an fp32 power and quotient
    plain = pkg.Rotary.plain(d, theta)
    assert torch.equal(plain.inv_freq, pkg.rope_inv_freq(d, theta)) and plain.dims == d
    torch.testing.assert_close(plain.inv_freq.double(), want, **near)
    s = pkg.Rotary.scaled(d, theta, 4.0, layout="interleaved")
    torch.testing.assert_close(s.inv_freq.double(), want / 4, **near)
    assert s.factor == 1.0 and s.layout == "interleaved"
    y = pkg.Rotary.scaled(d, theta, 16.0, 4096)
    turns = 4096 * want / (2 * math.pi)
    for f, g, n in zip(y.inv_freq.double(), want, turns):
        keep = min(max((n.item() - 1) / 31, 0), 1)
        assert math.isclose(f, g * (keep + (1 - keep) / 16), rel_tol=2.0 ** -22)
    assert (turns > 32).any() and (turns < 1).any() and ((turns > 1) & (turns < 32)).any()
    assert math.isclose(y.factor, 1 + 0.1 * math.log(16))
    assert pkg.Rotary.scaled(d, theta, 1.0, 4096).factor == 1.0


def test_reference_rotation():
    """The reference is a rotation: complex numbers, either pairing; its inverse is by -p."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 2, 12, generator=g, dtype=torch.double)
    f = torch.rand(4, generator=g)
    p = torch.tensor([[0, 5, -7], [100, 3, 2**20]])
    for layout in ("half", "interleaved"):
        y, size = ref.turned(x, f, p, layout, 1.5)
        z = torch.view_as_complex((x[..., :8].unflatten(-1, (4, 2)) if layout == "interleaved" else
                                   x[..., :8].unflatten(-1, (2, 4)).transpose(-1, -2)).contiguous())
        z = z * torch.polar(torch.tensor(1.5, dtype=torch.double),
                            p.double()[..., None, None] * f.double())
        w = torch.view_as_real(z)
        w = w.flatten(-2) if layout == "interleaved" else w.transpose(-1, -2).flatten(-2)
        torch.testing.assert_close(y[..., :8], w)
        assert torch.equal(y[..., 8:], x[..., 8:]) and (y.abs() <= size * (1 + 1e-12)).all()
        back, _ = ref.turned(y, f, -p, layout, 1 / 1.5)
        torch.testing.assert_close(back, x)
    axes = [0, 1, 2, 0]
    p3 = torch.stack([p, p + 1, 2 * p])
    y, _ = ref.turned(x, f, p3, axes=axes)
    for a in range(3):
        one, _ = ref.turned(x, f, p3[a])
        for i in (i for i in range(4) if axes[i] == a):
            assert torch.equal(y[..., i], one[..., i]) and torch.equal(y[..., 4 + i], one[..., 4 + i])


def test_reference_pages():
    """Rows gathered by a table are the pool's, and attention over them is the dense one's."""
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(2, 2, 48, 128, generator=g)
    tab = torch.tensor([[4, 0, 5], [2, 6, 1]])
    pool = torch.full((8, 2, 16, 128), math.nan)
    for b in range(2):
        for i in range(3):
            pool[tab[b, i]] = rows[b, :, 16 * i:16 * i + 16]
    assert torch.equal(ref.gathered(pool, tab), rows)
    tab[1, 0] = -1
    x = ref.gathered(pool, tab)
    assert torch.isnan(x[1, :, :16]).all() and torch.equal(x[1, :, 16:], rows[1, :, 16:])
    q = torch.randn(2, 1, 4, 128, generator=g)
    out, _ = kvref.attention(q, x, x, [47, 47], [1, 1], 20, 0)
    assert torch.isfinite(out).all()  # the missing page is behind the window
