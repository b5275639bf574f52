"""ThinkerAttention and ThinkerDecoder with caches in pages."""
from __future__ import annotations

import pytest
import torch

from tests import _kv_ref as ref
from tests.test_gpu_kv import i32
from tests.test_gpu_kv_module import H, HD, NKV, build, near, tokens

pytestmark = pytest.mark.gpu


def tables(dev, rows):
    return torch.tensor(rows, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("context", [{}, {"window": 50, "sinks": 3}])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_session_is_the_contiguous_cache(pkg, dev, dtype, context):
    """Prompts, chunks and single tokens, with and without a batch dimension and with either kind
    of position, against the module over one run of rows."""
    a = build(pkg, dev, dtype=dtype, window=context.get("window", 320),
              sinks=context.get("sinks", 0)).layers[0].attn
    b = build(pkg, dev, dtype=dtype, pages=30, page=16, **context).layers[0].attn
    table = tables(dev, torch.randperm(30).tolist()[:20])
    h = tokens(dev, 140, dtype=dtype)
    for lo, hi in ((0, 90), (90, 91), (91, 139), (139, 140)):
        want = a(h[lo:hi], lo)
        got = b(h[lo:hi], lo, table=table)
        assert got.shape == want.shape and near(got, want, dtype)
        again = b(h[None, lo:hi], i32(dev, [lo]), table=table[None])
        assert again.shape == (1, *want.shape) and near(again[0], want, dtype)


def test_sessions_as_one_batch(pkg, dev):
    """A decoder's padded batch of sessions of different ages: each row of a session is what it is
    alone, in a pool of its own."""
    dec = build(pkg, dev, layers=2, pages=40, page=16)
    alone = [build(pkg, dev, layers=2, pages=40, page=16) for _ in range(3)]
    ids = torch.randperm(40, generator=torch.Generator().manual_seed(3)).tolist()
    table = tables(dev, [ids[:13], ids[13:26], ids[26:39]])
    h = torch.stack([tokens(dev, 200, seed=s) for s in (1, 2, 3)])
    pos = [0, 0, 0]
    for counts in ([60, 1, 33], [1, 1, 1], [7, 90, 1], [1, 0, 1], [1, 1, 1]):
        T = max(counts)
        x = torch.zeros(3, T, H, dtype=h.dtype, device=dev)
        for b, n in enumerate(counts):
            x[b, :n] = h[b, pos[b]:pos[b] + n]
        got = dec.step(x, i32(dev, pos), table=table, counts=i32(dev, counts))
        assert got.shape == x.shape and torch.isfinite(got).all()
        for b, n in enumerate(counts):
            if n:
                want = alone[b].step(x[b, :n], pos[b], table=table[b])
                assert near(got[b, :n], want)
                pos[b] += n


def test_shared_prefix(pkg, dev):
    """Two sessions on one prompt's pages, each with a page of its own behind them."""
    dec, twin = (build(pkg, dev, layers=2, pages=12, page=16) for _ in range(2))
    h = tokens(dev, 70)
    prompt = tables(dev, [3, 4, 5, 6])
    dec.step(h[:64], 0, table=prompt)
    twin.step(h[:64], 0, table=prompt)
    x = torch.stack([h[64:65], h[65:66]])
    got = dec.step(x, 64, table=tables(dev, [[3, 4, 5, 6, 7], [3, 4, 5, 6, 9]]))
    for b, p in ((0, 7), (1, 9)):
        assert near(got[b], twin.step(x[b], 64, table=tables(dev, [3, 4, 5, 6, p])))


def test_rotary_of_the_module(pkg, dev):
    """Positions on three axes against 64 bits: the module's keys."""
    from qwen3_omni_duplex_amd import ops
    from tests import _paged_ref as pref

    r = pkg.Rotary.plain(HD, 1e6, axes=pkg.interleaved_axes([24, 20, 20]))
    attn = build(pkg, dev, pages=4, page=16, rotary=r).layers[0].attn
    T = 20
    h = tokens(dev, T)
    t = torch.arange(T, dtype=torch.int32)
    turn = torch.stack([t // 8 + 3, t % 8, t * 5]).to(dev)
    y = attn(h, 7, table=tables(dev, [2, 0, 1]), turn=turn)
    assert torch.isfinite(y).all()
    qkv = attn.qkv.lin(ops.rmsnorm(h, attn.input_norm_w, attn.eps)).view(1, T, -1, HD)
    k = pref.normed(qkv[:, :, -2 * NKV:-NKV], attn.k_norm_w)
    want, size = pref.turned(k, r.inv_freq, turn[:, None], axes=r.axes)
    got = pref.gathered(attn.paged.k, tables(dev, [[2, 0, 1]]))[0, :, 7:7 + T].transpose(0, 1)
    tol = pref.rounded(want, size, torch.bfloat16, 2.0 ** -19)
    assert ((got.double() - want[0]).abs() <= tol[0]).all()
    # equal along the axes: the plain rotation
    plain = build(pkg, dev, pages=4, page=16).layers[0].attn
    attn.reset_cache()
    assert torch.equal(attn(h, 7, table=tables(dev, [2, 0, 1])),
                       plain(h, 7, table=tables(dev, [2, 0, 1])))


def test_a_captured_step_serves_every_table(pkg, dev):
    """One graph of a batch's step, replayed at other positions and with other pages, eager steps
    of the same decoder in between."""
    dec, twin = (build(pkg, dev, layers=2, pages=30, page=16) for _ in range(2))
    h = torch.stack([tokens(dev, 60, seed=s) for s in (1, 2)])
    table = tables(dev, [list(range(0, 8)), list(range(8, 16))])
    for d in (dec, twin):
        d.step(h[:, :50], 0, table=table)
    x, pos, tab = h[:, 50:51].clone(), i32(dev, [50, 50]), table.clone()
    build(pkg, dev, layers=2, pages=30, page=16).step(x, pos, table=tab)  # loads the kernels
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = dec.step(x, pos, table=tab)
    for i in range(50, 56):
        x.copy_(h[:, i:i + 1])
        pos.copy_(i32(dev, [i, i]))
        if i == 53:  # the second session moves to other pages
            moved = torch.tensor([list(range(0, 8)), list(range(20, 28))], dtype=torch.int32)
            for d in (dec, twin):
                for l in d.layers:
                    for c in (l.attn.paged.k, l.attn.paged.v):
                        c[20:28] = c[8:16]
                        c[8:16] = float("nan")
            table = moved.to(dev)
        tab.copy_(table)
        graph.replay()
        want = twin.step(h[:, i:i + 1], i32(dev, [i, i]), table=table)
        torch.cuda.synchronize()
        assert near(y, want) and torch.isfinite(y).all(), i
        assert near(dec.step(h[:, i:i + 1], i, table=table), want)  # the same token again


def test_dtype_moves_the_pool(pkg, dev):
    attn = build(pkg, dev, pages=4, page=16, dtype=torch.bfloat16).layers[0].attn
    h = tokens(dev, 20)
    table = tables(dev, [1, 3])
    attn(h, 0, table=table)
    k = attn.paged.k
    attn.half()
    assert attn.paged.k.dtype == torch.float16 and torch.equal(attn.paged.k, k.half())
    attn.reset_cache()
    assert not attn.paged.k.any() and not attn.paged.v.any()


def test_module_refuses(pkg, dev):
    plain, paged = build(pkg, dev), build(pkg, dev, pages=4, page=16)
    h, table = tokens(dev, 3), tables(dev, [0, 1])
    with pytest.raises(ValueError, match="table"):
        plain.step(h, 0, table=table)
    with pytest.raises(ValueError, match="table"):
        plain.step(h[:1], 0, table=table)
    with pytest.raises(ValueError, match="need a cache in pages"):
        plain.step(h, 0, counts=i32(dev, [2]))
    with pytest.raises(ValueError, match="table"):
        paged.step(h, 0)
    with pytest.raises(RuntimeError, match="outside"):
        paged.step(h, 30, table=table)
    with pytest.raises(RuntimeError, match="table"):
        paged.step(torch.stack([h, h]), 0, table=table)
    with pytest.raises(ValueError, match=r"\[B, T, H\]"):
        paged.step(h[None, None], 0, table=table)
    with pytest.raises(ValueError, match="16 bits"):
        build(pkg, dev, pages=4, kv_dtype=torch.int8)
    with pytest.raises(ValueError, match="needs a cache in pages"):
        build(pkg, dev, rotary=pkg.Rotary.plain(HD, 1e6))
