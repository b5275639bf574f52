"""What the documents promise of the paged cache and the rotary embeddings beyond single calls."""
from __future__ import annotations

import pytest
import torch

from tests import _kv_ref as kvref
from tests import _paged_ref as ref
from tests.test_gpu_kv import i32, rand, same

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
