"""The operators of a long conversation's key/value cache, as measurable cases.

A duplex session runs one token per 80 ms frame for hours, takes prompt chunks in between, and
shares the GPU with other sessions.  The cases are the attention side of that, at the Thinker's
32 query and 4 key/value heads of 128 unless a case says otherwise:

  rope     rope_append: q/k RMSNorm and rotary embedding of the fused q|k|v rows, k and v into
           the cache's rows
  window   attn_window: attention of one token or many over a 16-bit cache, bounded by a sliding
           window with the first tokens kept visible, or over everything
  append   kv8_append: tokens into a cache of 8 bits with a scale for each block of 64 tokens and
           head; the unfinished block stays in 16 bits
  kv8      attn_kv8: the attention of `window` over that 8-bit cache

Where `own` is false, run() computes them in elementary torch operations in fp32.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HD, BLOCK, EPS, THETA = 128, 64, 1e-6, 1_000_000.0
NH, NKV = 32, 4            # the Thinker's heads
FULL = {"int8": 127.0, "e4m3": 448.0}  # the largest value of the 8-bit formats
TINY = 2.0 ** -100         # a block whose largest value is below is scaled as if it were this


def _package():
    name = "qwen3_omni_duplex_amd"
    if name not in sys.modules:
        root = ROOT / "qwen3-omni-duplex_amd"
        spec = importlib.util.spec_from_file_location(name, root / "__init__.py",
                                                      submodule_search_locations=[str(root)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _case(op, batch, tokens, pos, dtype, **kw):
    c = {"op": op, "batch": batch, "tokens": tokens, "pos": pos, "dtype": dtype, "heads": NH,
         "kv_heads": NKV}
    return {**c, **kw}


def listed():
    return [
        # one frame's token of one session, 1024 positions in
        {"name": "rope_token", **_case("rope", 1, 1, 1024, "bf16")},
        # a 3001-token prompt from an empty cache
        {"name": "rope_prompt", **_case("rope", 1, 3001, 0, "bf16")},
        # one frame's token, 5000 positions in, a window of 1024 and four first tokens
        {"name": "window_token", **_case("window", 1, 1, 5000, "bf16", window=1024, sinks=4)},
        # the tokens of 24 sessions of different ages, up to 20000 positions in
        {"name": "window_batch", **_case("window", 24, 1, 20000, "fp16", window=8192, sinks=16)},
        # a padded batch of three prompt chunks of up to 500 tokens
        {"name": "window_chunks", **_case("window", 3, 500, 7001, "bf16", window=2048, sinks=4,
                                          ragged=True)},
        # a 6001-token prompt that attends everything before each token
        {"name": "window_prompt", **_case("window", 1, 6001, 0, "bf16", window=0, sinks=0)},
        # the tokens of 16 sessions into their 8-bit caches
        {"name": "append_token", **_case("append", 16, 1, 447, "bf16", fmt="int8")},
        # a 4001-token prompt behind 63 cached tokens
        {"name": "append_prompt", **_case("append", 1, 4001, 63, "bf16", fmt="e4m3")},
        # one frame's token over an 8191-token 8-bit cache
        {"name": "kv8_token", **_case("kv8", 1, 1, 8191, "bf16", window=0, sinks=0, fmt="int8")},
        # the tokens of 32 sessions, up to 32000 positions each
        {"name": "kv8_batch", **_case("kv8", 32, 1, 32000, "bf16", window=0, sinks=0, fmt="int8")},
        # a 300-token chunk, 4000 positions in, under a window
        {"name": "kv8_chunk", **_case("kv8", 1, 300, 4000, "fp16", window=3000, sinks=64,
                                      fmt="e4m3")},
        # a 5000-token prompt over its own 8-bit cache
        {"name": "kv8_prompt", **_case("kv8", 1, 5000, 0, "bf16", window=0, sinks=0, fmt="int8")},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "window", "window", "append", "kv8", "kv8"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 4, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 7, 8, 8])
    more = {"heads": heads, "kv_heads": kv_heads}
    if rng.random() < 0.5:  # sessions' tokens, or a few tokens each
        batch, tokens = _spread(rng, 1, 32), rng.choice([1, 1, 1, 2, 3, 5, 8])
        pos = _spread(rng, 1, 30000 if op in ("window", "kv8") else 800) - 1
    else:                   # prompt chunks and prompts
        batch, tokens = rng.choice([1, 1, 2, 3]), _spread(rng, 9, 2500)
        pos = rng.choice([0, _spread(rng, 1, 3000)])
    if op in ("rope", "append"):
        more["ragged"] = batch > 1 and rng.random() < 0.5
    if op in ("window", "kv8"):
        more["window"] = rng.choice([0, _spread(rng, 1, 9000)])
        more["sinks"] = rng.choice([0, 1, 4, _spread(rng, 5, 300)]) if more["window"] else 0
        more["ragged"] = batch > 1 and rng.random() < 0.5
    if op in ("append", "kv8"):
        more["fmt"] = rng.choice(["int8", "e4m3"])
    return _case(op, batch, tokens, pos, dtype, **more)


# --------------------------------------------------------------------------- inputs

def _positions(c):
    """The first position of each sequence: the oldest session is at `pos`, the others younger."""
    return [c["pos"] - (b * 7919) % (c["pos"] // 2 + 1) for b in range(c["batch"])]


def _counts(c):
    """How many of the padded tokens each sequence has (the first has all)."""
    if not c.get("ragged"):
        return [c["tokens"]] * c["batch"]
    return [c["tokens"] - (b * 613) % (c["tokens"] + 1) for b in range(c["batch"])]


def _rows(n):
    return -(-n // BLOCK) * BLOCK


def _keys(g, shape, dtype):
    """Keys as they are after their norm: unit rows with a gain for each dimension."""
    gain = torch.exp(0.3 * torch.randn(HD, generator=g, device=DEV))
    return (torch.randn(*shape, generator=g, device=DEV) * gain).to(dtype)


def _values(g, shape, dtype):
    """Values: a row of its own for each token around a mean for each dimension."""
    mean = 0.5 * torch.randn(HD, generator=g, device=DEV)
    return (torch.randn(*shape, generator=g, device=DEV) + mean).to(dtype)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt, B, T = DT[c["dtype"]], c["batch"], c["tokens"]
    nh, nkv = c["heads"], c["kv_heads"]
    rows = _rows(c["pos"] + T)
    at, counts = _positions(c), _counts(c)
    # one sequence's position is a number in hand; several sessions keep theirs on the device
    s = {"case": c, "rows": rows,
         "pos": torch.tensor(at, dtype=torch.int32, device=DEV),
         "counts": torch.tensor(counts, dtype=torch.int32, device=DEV) if c.get("ragged") else None}
    s["where"] = c["pos"] if B == 1 else s["pos"]
    if c["op"] == "rope":
        s["qkv"] = torch.randn(B, T, (nh + 2 * nkv) * HD, generator=g, device=DEV).to(dt)
        s["qw"], s["kw"] = ((1 + 0.2 * torch.randn(HD, generator=g, device=DEV)).to(dt)
                            for _ in range(2))
        # a host table, as the rotary embedding's inverse frequencies are kept
        s["inv_freq"] = 1.0 / THETA ** (torch.arange(0, HD, 2, dtype=torch.float) / HD)
        s["k"], s["v"] = (torch.randn(B, nkv, rows, HD, generator=g, device=DEV).to(dt)
                          for _ in range(2))
    elif c["op"] == "window":
        s["q"] = 1.5 * torch.randn(B, T, nh, HD, generator=g, device=DEV).to(dt)
        s["k"], s["v"] = _keys(g, (B, nkv, rows, HD), dt), _values(g, (B, nkv, rows, HD), dt)
    else:
        if c["op"] == "append":
            s["k_new"] = _keys(g, (B, T, nkv, HD), dt)
            s["v_new"] = _values(g, (B, T, nkv, HD), dt)
        else:
            s["q"] = 1.5 * torch.randn(B, T, nh, HD, generator=g, device=DEV).to(dt)
        k = _keys(g, (B, nkv, rows, HD), dt).view(B, nkv, -1, BLOCK, HD)
        v = _values(g, (B, nkv, rows, HD), dt).view(B, nkv, -1, BLOCK, HD)
        # the unfinished block of each sequence, before an append or at the attention
        end = s["pos"].long() + (0 if c["op"] == "append" else
                                 torch.tensor(counts, device=DEV))
        last = (end // BLOCK).clamp(max=rows // BLOCK - 1)
        b = torch.arange(B, device=DEV)
        s["k_tail"], s["v_tail"] = k[b, :, last].contiguous(), v[b, :, last].contiguous()
        s["k8"], s["ks"] = _quantise(k, c["fmt"])
        v8, s["vs"] = _quantise(v, c["fmt"])
        s["v8"] = v8.transpose(-1, -2).contiguous()  # value blocks are kept [dim][token]
        if own:  # the handle that a session keeps for its cache
            s["cache"] = _package().KV8Cache(s["k8"], s["v8"], s["ks"], s["vs"], s["k_tail"],
                                             s["v_tail"])
    return s


# --------------------------------------------------------------------------- plain forms

def _quantise(x, fmt):
    """8-bit blocks of [..., 64, 128] and their fp32 scales: the largest magnitude over the
    format's largest value, and each quotient rounded once (in 64 bits: values next to a
    border), ties to even."""
    big = x.float().abs().amax((-1, -2)).clamp(min=TINY)
    scale = (big.double() / FULL[fmt]).float()
    y = x.double() / scale.double()[..., None, None]
    if fmt == "int8":
        return torch.round(y).to(torch.int8), scale
    step = torch.exp2(torch.frexp(y)[1].clamp(min=-5).double() - 4)
    return (torch.round(y / step) * step).float().to(torch.float8_e4m3fn), scale


def _plain_attention(s, k, v):
    """softmax(q k^T / sqrt(d)) v over the visible positions, k and v [B, kv heads, rows, d] fp32."""
    c = s["case"]
    B, T, nh, nkv = c["batch"], c["tokens"], c["heads"], c["kv_heads"]
    G, L = nh // nkv, k.shape[2]
    q = s["q"].float().view(B, T, nkv, G, HD).permute(0, 2, 3, 1, 4).reshape(B, nkv, G * T, HD)
    scores = (q @ k.transpose(-1, -2) * (1.0 / math.sqrt(HD))).view(B, nkv, G, T, L)
    p = (s["pos"][:, None] + torch.arange(T, device=DEV))[:, :, None]
    j = torch.arange(L, device=DEV)
    see = j <= p
    if c["window"]:
        see = see & ((j > p - c["window"]) | (j < c["sinks"]))
    scores = scores.masked_fill(~see[:, None, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = (e.view(B, nkv, G * T, L) @ v).view(B, nkv, G, T, HD) / e.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, nh, HD).to(s["q"].dtype)
    if s["counts"] is not None:  # the padding's rows are zeros
        o = o * (torch.arange(T, device=DEV) < s["counts"][:, None])[:, :, None, None]
    return o


def _plain_rope(s):
    c = s["case"]
    B, T, nh, nkv = c["batch"], c["tokens"], c["heads"], c["kv_heads"]
    dt = s["qkv"].dtype
    x = s["qkv"].view(B, T, nh + 2 * nkv, HD)
    p = s["pos"][:, None] + torch.arange(T, device=DEV)
    angle = p.double()[..., None] * s["inv_freq"].to(DEV).double()  # far positions
    cos, sin = (torch.cat([f, f], -1).float()[:, :, None] for f in (angle.cos(), angle.sin()))

    def rotated(y, w):
        y = y.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
        return (y * cos + torch.cat([-y[..., HD // 2:], y[..., :HD // 2]], -1) * sin).to(dt)

    q = rotated(x[:, :, :nh], s["qw"])
    k, v = rotated(x[:, :, nh:nh + nkv], s["kw"]), x[:, :, nh + nkv:]
    n = torch.arange(s["rows"], device=DEV) - s["pos"][:, None]
    count = s["counts"] if s["counts"] is not None else torch.full_like(s["pos"], T)
    new = ((n >= 0) & (n < count[:, None]))[:, None, :, None]
    at = n.clamp(0, T - 1)[:, :, None, None].expand(B, s["rows"], nkv, HD)
    for name, y in (("k", k), ("v", v)):
        s[name].copy_(torch.where(new, y.gather(1, at).transpose(1, 2), s[name]))
    if s["counts"] is not None:
        q = q * (torch.arange(T, device=DEV) < count[:, None])[:, :, None, None]
    return q, s["k"], s["v"]


def _plain_append(s):
    c = s["case"]
    B, T, nkv, fmt = c["batch"], c["tokens"], c["kv_heads"], c["fmt"]
    nblk = s["rows"] // BLOCK
    count = s["counts"] if s["counts"] is not None else torch.full_like(s["pos"], T)
    first, r = s["pos"] // BLOCK, s["pos"] % BLOCK
    nb = -(-(T + BLOCK - 1) // BLOCK)
    # the touched blocks' tokens: the tail's, then the new ones
    n = torch.arange(nb * BLOCK, device=DEV) - r[:, None]
    new = ((n >= 0) & (n < count[:, None]))[:, None, :, None]
    at = n.clamp(0, T - 1)[:, :, None, None].expand(B, nb * BLOCK, nkv, HD)
    done = (r + count) // BLOCK  # blocks that are finished now
    i = torch.arange(nblk, device=DEV) - first[:, None]
    write = ((i >= 0) & (i < done[:, None]))[:, None, :]
    blk = i.clamp(0, nb - 1)[:, None, :].expand(B, nkv, nblk)
    # the unfinished block and its tokens' slots in the tail
    slot = torch.arange(BLOCK, device=DEV)
    lo = torch.where(done > 0, torch.zeros_like(r), r)
    put = ((slot >= lo[:, None]) & (slot < (r + count - done * BLOCK)[:, None]))[:, None, :, None]
    part = done.clamp(max=nb - 1).long()
    out = []
    for a, f, sc, tail, y in (("k8", False, "ks", "k_tail", s["k_new"]),
                              ("v8", True, "vs", "v_tail", s["v_new"])):
        seq = torch.cat([s[tail], s[tail].new_zeros(B, nkv, (nb - 1) * BLOCK, HD)], 2)
        seq = torch.where(new, y.gather(1, at).transpose(1, 2), seq).view(B, nkv, nb, BLOCK, HD)
        q8, scale = _quantise(seq, fmt)
        q8 = q8.transpose(-1, -2) if f else q8
        w, bits = write[..., None, None], q8.contiguous().view(torch.int8)
        got = bits.gather(2, blk[..., None, None].expand(-1, -1, -1, *q8.shape[-2:]))
        s[a].view(torch.int8).copy_(torch.where(w, got, s[a].view(torch.int8)))
        s[sc].copy_(torch.where(write, scale.gather(2, blk), s[sc]))
        s[tail].copy_(torch.where(put, seq[torch.arange(B, device=DEV), :, part], s[tail]))
        out += [_stands_for(s[a], s[sc], f), s[sc], s[tail]]
    return out


def _stands_for(x, scale, turned):
    """The values of 8-bit blocks as [B, kv heads, rows, d] fp32."""
    y = x.float() * scale[..., None, None]
    y = y.transpose(-1, -2) if turned else y
    return y.reshape(*y.shape[:2], -1, HD)


def _plain_kv8(s):
    c = s["case"]
    count = s["counts"] if s["counts"] is not None else torch.full_like(s["pos"], c["tokens"])
    last = (s["pos"] + count) // BLOCK  # the unfinished block
    here = (torch.arange(s["rows"], device=DEV) // BLOCK == last[:, None])[:, None, :, None]
    kv = []
    for a, f, sc, tail in (("k8", False, "ks", "k_tail"), ("v8", True, "vs", "v_tail")):
        x = _stands_for(s[a], s[sc], f)
        t = s[tail].float().repeat(1, 1, s["rows"] // BLOCK, 1)
        kv.append(torch.where(here, t, x))
    return _plain_attention(s, *kv)


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "rope":
            return _plain_rope(s)
        if c["op"] == "window":
            return _plain_attention(s, s["k"].float(), s["v"].float())
        return _plain_append(s) if c["op"] == "append" else _plain_kv8(s)
    pkg = _package()
    if c["op"] == "rope":
        q = pkg.rope_append(s["qkv"], c["heads"], c["kv_heads"], s["qw"], s["kw"], EPS,
                            s["inv_freq"], s["where"], s["k"], s["v"], counts=s["counts"])
        return q, s["k"], s["v"]
    if c["op"] == "append":
        cache = s["cache"]
        pkg.kv8_append(s["k_new"], s["v_new"], cache, s["where"], counts=s["counts"])
        k, v = cache.values()
        return [k, cache.k_scale, cache.k_tail, v, cache.v_scale, cache.v_tail]
    bounds = {"window": c["window"] or None, "sinks": c["sinks"], "counts": s["counts"]}
    if c["op"] == "window":
        return pkg.attn_window(s["q"], s["k"], s["v"], s["where"], **bounds)
    return pkg.attn_kv8(s["q"], s["cache"], s["where"], **bounds)


# --------------------------------------------------------------------------- work and 64 bits

def _visible(c):
    """(query, key) pairs of one head, and the distinct keys that they cover, over the batch."""
    pairs = keys = 0
    for p0, n in zip(_positions(c), _counts(c)):
        if n == 0:
            continue
        w = c["window"] or 1 << 30
        lo, hi = max(0, p0 - w + 1), p0 + n  # the first query's first key, the last one's end
        keys += hi - lo + min(c["sinks"], lo)
        pairs += sum(min(p + 1, w) + min(c["sinks"], max(0, p + 1 - w)) for p in range(p0, hi))
    return pairs, keys


def work(case):
    c = case
    nh, nkv, tokens = c["heads"], c["kv_heads"], sum(_counts(c))
    if c["op"] == "rope":  # the fused rows in, q and the cache rows out
        return {"bytes": 2 * 2 * tokens * (nh + 2 * nkv) * HD, "flops": 8 * tokens * nh * HD}
    if c["op"] == "append":
        # tokens in (16 bits) and out (8 bits), and the cache's values, which come back in fp32
        rows = c["batch"] * _rows(c["pos"] + c["tokens"])
        return {"bytes": 2 * nkv * HD * (tokens * (2 + 1) + rows * (1 + 4)),
                "flops": 4 * tokens * nkv * HD}
    pairs, keys = _visible(c)
    size = 2 if c["op"] == "window" else 1
    return {"bytes": 2 * keys * nkv * HD * size + 2 * 2 * tokens * nh * HD,
            "flops": 4 * HD * nh * pairs}


def _exact_attention(s, k_of, v_of):
    """k_of(b, h), v_of(b, h): one head's rows in fp64."""
    c = s["case"]
    T, nh, G = c["tokens"], c["heads"], c["heads"] // c["kv_heads"]
    out = torch.zeros(c["batch"], T, nh, HD, dtype=torch.float64, device=DEV)
    for b, (p0, n) in enumerate(zip(_positions(c), _counts(c))):
        if n == 0:
            continue
        row = torch.arange(p0, p0 + n, device=DEV)[:, None]
        col = torch.arange(p0 + n, device=DEV)[None]
        hidden = col > row
        if c["window"]:
            hidden |= (col <= row - c["window"]) & (col >= c["sinks"])
        for h in range(nh):
            x = s["q"][b, :n, h].double() @ k_of(b, h // G)[:p0 + n].T / math.sqrt(HD)
            x[hidden] = -math.inf
            out[b, :n, h] = torch.softmax(x, -1) @ v_of(b, h // G)[:p0 + n]
    return out


def _exact_block(x, fmt):
    """A block's values after 8 bits, and its scale, in fp64."""
    x = x.double()
    scale = (x.abs().max().clamp(min=TINY) / FULL[fmt]).float().double()
    y = x / scale
    if fmt == "int8":
        return torch.round(y) * scale, scale
    grid = torch.arange(127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()
    mid = (grid[1:] + grid[:-1]) / 2
    m = y.abs()
    i = torch.bucketize(m, mid)                   # the nearest of the format's values,
    tie = torch.bucketize(m, mid, right=True) - i  # and the even one of two as near
    return torch.sign(y) * grid[i + tie * (i & 1)] * scale, scale


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    T, nh, nkv, at, counts = c["tokens"], c["heads"], c["kv_heads"], _positions(c), _counts(c)
    if c["op"] == "window":
        return _exact_attention(s, lambda b, h: s["k"][b, h].double(),
                                lambda b, h: s["v"][b, h].double())
    if c["op"] == "kv8":
        def rows(x, scale, tail, turned):
            def of(b, h):
                y = x[b, h].double() * scale[b, h].double()[:, None, None]
                y = (y.transpose(1, 2) if turned else y).reshape(-1, HD)
                end = at[b] + counts[b]
                if end % BLOCK:
                    y = torch.cat([y[:end // BLOCK * BLOCK], tail[b, h, :end % BLOCK].double()])
                return y
            return of
        return _exact_attention(s, rows(s["k8"], s["ks"], s["k_tail"], False),
                                rows(s["v8"], s["vs"], s["v_tail"], True))
    if c["op"] == "rope":
        q = torch.zeros(c["batch"], T, nh, HD, dtype=torch.float64, device=DEV)
        k, v = s["k"].double(), s["v"].double()
        for b, (p0, n) in enumerate(zip(at, counts)):
            x = s["qkv"][b, :n].double().view(n, nh + 2 * nkv, HD)
            turn = torch.arange(p0, p0 + n, device=DEV).double()[:, None, None] * \
                s["inv_freq"].to(DEV).double()
            turn = torch.polar(torch.ones_like(turn), turn)
            for lo, m, w in ((0, nh, s["qw"]), (nh, nkv, s["kw"])):
                y = x[:, lo:lo + m]
                y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
                z = torch.complex(y[..., :HD // 2], y[..., HD // 2:]) * turn
                y = torch.cat([z.real, z.imag], -1)
                if lo:
                    k[b, :, p0:p0 + n] = y.transpose(0, 1)
                else:
                    q[b, :n] = y
            v[b, :, p0:p0 + n] = x[:, nh + nkv:].transpose(0, 1)
        return q, k, v
    out = []
    for x, scale, tail, new, turned in ((s["k8"], s["ks"], s["k_tail"], s["k_new"], False),
                                        (s["v8"], s["vs"], s["v_tail"], s["v_new"], True)):
        y = x.double() * scale.double()[..., None, None]
        y = y.transpose(-1, -2).contiguous() if turned else y
        scale, tail = scale.double(), tail.double()
        for b, (p0, n) in enumerate(zip(at, counts)):
            first, r = p0 // BLOCK, p0 % BLOCK
            for h in range(nkv):
                seq = torch.cat([tail[b, h, :r], new[b, :n, h].double()])
                for i in range(len(seq) // BLOCK):
                    y[b, h, first + i], scale[b, h, first + i] = _exact_block(
                        seq[i * BLOCK:(i + 1) * BLOCK], c["fmt"])
                rest = len(seq) % BLOCK
                tail[b, h, :rest] = seq[len(seq) - rest:]
        out += [y.reshape(*y.shape[:2], -1, HD), scale, tail]
    return out
