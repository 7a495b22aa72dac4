"""Serving from a key/value cache held in 4 bits, as a program that decodes with
adaptive splash attention runs it: tokens' keys and values are quantised as
they are written, attention reads the 4-bit cache in place, and a sequence's
keys and values are read back where the dense path needs them.

The cache is paged.  A row (one token's key or value of one head) is d
channels in groups of 32; a group has a scale s and an offset m, both
bfloat16, and one code c of 4 bits for each channel, standing for m + c s:

  m = the largest bfloat16 at most min(x)
  s = the smallest bfloat16 >= 2^-126 with 15 s >= max(x) - m (0 if max(x) = m)
  c = the number of borders m + (k + 1/2) s, k = 0..14, below x

  codes   uint8 [pages, heads, page_size, 16 G], G = ceil(d / 32): channel
          32 g + 8 o + 2 j + h is the nibble h (0: low) of byte 16 g + 4 o + j
          in a value row and of byte 4 G o + 4 g + j in a key row
  params  bfloat16 [pages, heads, page_size, G, 2]: s, m

Position t of sequence b is row t % page_size of page table[b, t // page_size].

Attention is alpha-entmax over the visible keys (position at most the
query's): z = (alpha - 1) clamp(scale q.k, -10, 10), p = max(z - tau, 0) ^
(1 / (alpha - 1)) with tau such that the p of a row sum to one, out = sum p v.
A row that sees no key gives zeros.

A case is a dict of plain values:

  call    "attend": attention of NQ query tokens at the end of each sequence
          "write":  n new tokens of each sequence go into the cache, then
                    come back as the values that their codes stand for
          "read":   n positions of each sequence, from the first
  B, H, HK (query and key/value heads; write and read have H = HK), d, page,
  dtype, alpha, n (cached tokens, or tokens written or read), NQ
  start   tokens in the cache before a write
  ragged  sequences of unequal length up to n, every eighth of them an empty slot
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_TINY = 2.0 ** -126


def _case(name, call, B, HK, d, n, dtype="bfloat16", **kw):
    c = dict(name=name, call=call, B=B, H=HK, HK=HK, d=d, page=64, dtype=dtype, alpha=1.5, n=n,
             NQ=1, start=0, ragged=False)
    c.update(kw)
    return c


def listed():
    return [
        # One user, a short chat, the benchmark's heads: latency is all there is.
        _case("attend_one_short", "attend", 1, 16, 64, 512),
        # An ordinary decode step of a small batch with shared key/value heads.
        _case("attend_batch", "attend", 8, 8, 128, 2048, H=32),
        # A continuous batch: unequal lengths, empty slots, small pages, fp16.
        _case("attend_ragged", "attend", 24, 8, 64, 4095, "float16", H=16, page=16, ragged=True),
        # Checking a few drafted tokens at once, fp32, a head dimension between
        # the tile widths, the sparser weights of a smaller window.
        _case("attend_drafts_fp32", "attend", 3, 5, 80, 1537, "float32", H=15, NQ=5, alpha=2.0,
              page=32),
        # One user at the end of a very long document.
        _case("attend_one_long", "attend", 1, 8, 128, 131072, H=32),
        # A loaded server with long contexts: the cache's bytes are all there is.
        _case("attend_batch_long", "attend", 16, 8, 128, 32768, H=32),
        # Long contexts, one query head to a key head, weights spread over
        # many keys.
        _case("attend_spread", "attend", 4, 16, 64, 16384, "bfloat16", alpha=1.25),
        # A decode step's new token of each sequence.
        _case("write_decode", "write", 32, 8, 128, 1, start=1000),
        # A prompt of one user, longer than a page and not a whole number of them.
        _case("write_prompt", "write", 1, 8, 128, 16001, start=37),
        # Prompts of unequal length, fp32, a last group of channels that is not full.
        _case("write_ragged_fp32", "write", 9, 6, 80, 700, "float32", ragged=True, page=32),
        # A cached prefix read back for a chunked prompt.
        _case("read_prefix", "read", 1, 16, 64, 4096),
        # A batch of contexts read back.
        _case("read_batch", "read", 8, 8, 128, 8191, "float16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    call = rng.choice(["attend", "attend", "attend", "write", "read"])
    d = rng.choice([64, 128, 128, 8 * rng.randrange(2, 17)])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    hk = rng.choice([1, 2, 4, 8, 8, 16, rng.randrange(1, 17)])
    B = _log(rng, 1, 48)
    c = dict(call=call, B=B, H=hk, HK=hk, d=d, page=rng.choice([16, 32, 64, 64, 128]), dtype=dtype,
             alpha=1.5, n=1, NQ=1, start=0, ragged=rng.random() < 0.5)
    if call == "attend":
        c["H"] = hk * rng.choice([1, 2, 3, 4, 4, 8])
        c["NQ"] = rng.choice([1, 1, 1, rng.randrange(2, 9)])
        c["alpha"] = rng.choice([1.5, 1.5, 1.25, 4 / 3, 2.0, round(rng.uniform(1.1, 2.0), 3)])
        # at most the key rows and the scores of the largest listed case
        rows = 16 * 8 * 32768 // max(1, c["H"] * c["NQ"] // (4 * hk))
    else:
        rows = 8 * (8192 if dtype == "float32" else 16384)
        if call == "write":
            c["start"] = rng.choice([0, 0, rng.randrange(1, 2000)])
    c["n"] = _log(rng, 1, max(2, min(65536, rows * 128 // (B * hk * max(32, d)))))
    return c


def _counts(c):
    """Tokens of each sequence (a plain rule of the case, so that its work is known)."""
    if not c["ragged"]:
        return [c["n"]] * c["B"]
    return [0 if b % 8 == 7 else c["n"] if b % 8 == 0 else 1 + (b * 7919 + 13) % 97 * (c["n"] - 1) // 96
            for b in range(c["B"])]


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------
def _groups(x):
    """[..., d] -> [..., G, 32]; the missing channels of a last group repeat
    its first one, which leaves its minimum and maximum as they are."""
    d = x.shape[-1]
    G = -(-d // 32)
    if d % 32:
        x = torch.cat([x, x[..., 32 * (G - 1):32 * (G - 1) + 1].expand(*x.shape[:-1], 32 * G - d)], -1)
    return x.unflatten(-1, (G, 32))


def _quantise(x):
    """codes uint8 [..., G, 32] and params bfloat16 [..., G, 2] of rows [..., d].
    In 64 bits: a value next to a border decides a code."""
    d = x.shape[-1]
    x = _groups(x.double())
    lo = x.amin(-1, keepdim=True).float()
    bits = lo.view(torch.int32)
    cut = bits & -65536
    m = torch.where((lo < 0) & (cut != bits), cut + 65536, cut).view(torch.float32).double()
    span = x.amax(-1, keepdim=True) - m
    cut = (span / 15).clamp_min(_TINY).float().view(torch.int32) & -65536
    s = torch.where(15 * cut.view(torch.float32).double() < span, cut + 65536, cut)
    s = torch.where(span > 0, s.view(torch.float32), 0.0).double()
    codes = ((x - m) / s.clamp_min(_TINY) - 0.5).ceil().clamp(0, 15).to(torch.uint8)
    if d % 32:
        codes[..., -1, d % 32:] = 0
    return codes, torch.cat([s, m], -1).to(torch.bfloat16)


def _pack(codes, key):
    """codes [..., G, 32] -> bytes [..., 16 G] in a key row's order or a value row's."""
    c = codes.unflatten(-1, (4, 4, 2))  # [..., G, o, j, h]
    c = c[..., 0] | (c[..., 1] << 4)
    return (c.transpose(-3, -2) if key else c).flatten(-3)


def _unpack(codes, params, d, key):
    """bytes [..., 16 G], params [..., G, 2] -> the values [..., d] in 32 bits."""
    G = params.shape[-2]
    c = codes.unflatten(-1, (4, G, 4)).transpose(-3, -2) if key else codes.unflatten(-1, (G, 4, 4))
    c = torch.stack([c & 15, c >> 4], -1).flatten(-3)  # [..., G, 32]
    p = params.float()
    return (c.float() * p[..., :1] + p[..., 1:]).flatten(-2)[..., :d]


def _gather(pool, table):
    """[pages, HK, page, X] through [B, P] -> [B, HK, P page, X]."""
    t = pool[table]  # [B, P, HK, page, X]
    return t.transpose(1, 2).flatten(2, 3)


def _rows(st, key, n):
    name = "k" if key else "v"
    codes = _gather(st[name + "_codes"], st["table"])[:, :, :n]
    params = _gather(st[name + "_params"].flatten(-2), st["table"])[:, :, :n]
    return _unpack(codes, params.unflatten(-1, (-1, 2)), st["d"], key)


def _plain_attend(st):
    q, c, am1 = st["q"], st["case"], st["case"]["alpha"] - 1.0
    B, H, NQ, d = q.shape
    HK, n = c["HK"], st["n"]
    k, v = _rows(st, True, n), _rows(st, False, n)
    r = q.float().reshape(B, HK, H // HK * NQ, d)
    s = torch.matmul(k, r.transpose(2, 3).contiguous()).transpose(2, 3).contiguous()
    z = am1 * (s * st["scale"]).clamp(-10.0, 10.0)
    at = st["lengths"].long()[:, None] - NQ + torch.arange(NQ, device=q.device)
    at = at[:, None, :].expand(B, H, NQ).reshape(B, HK, -1, 1)
    seen = torch.arange(n, device=q.device) <= at
    z = z.masked_fill(~seen, -1e30)
    # tau lies within one of the largest z; a general alpha has no closed form
    # for it, so the bracket is halved down to the resolution of 32 bits
    top = z.amax(-1, keepdim=True)
    tau, step = top - 1.0, 0.5
    for _ in range(24):
        tau = torch.where((z - (tau + step)).clamp_min(0.0).pow(1.0 / am1).sum(-1, keepdim=True) >= 1.0,
                          tau + step, tau)
        step *= 0.5
    p = (z - tau).clamp_min(0.0).pow(1.0 / am1).masked_fill(~seen, 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return torch.matmul(p, v).reshape(B, H, NQ, d).to(q.dtype)


def _plain_write(st):
    c, page = st["case"], st["case"]["page"]
    B, HK, n, d = st["k"].shape
    i = torch.arange(n, device=st["k"].device)
    at = st["start"].long()[:, None] + i
    # the padding behind a sequence goes to the pool's last page, which no table names
    fine = i < st["counts"][:, None]
    pages = torch.where(fine, st["table"].gather(1, at // page), st["k_codes"].shape[0] - 1)
    for name in ("k", "v"):
        codes, params = _quantise(st[name].transpose(1, 2))  # [B, n, HK, G, 32]
        st[name + "_codes"][pages, :, at % page] = _pack(codes, name == "k")
        st[name + "_params"][pages, :, at % page] = params
    return _plain_read(st)


def _plain_read(st):
    at = st["start"].long()[:, None] + torch.arange(st["n"], device=st["table"].device)
    fine = (at < st["ends"][:, None])[:, None, :, None]
    page = st["case"]["page"]
    pages, rows = st["table"].gather(1, at // page), at % page
    dtype = _DTYPES[st["case"]["dtype"]]
    k = _unpack(st["k_codes"][pages, :, rows], st["k_params"][pages, :, rows], st["d"], True)
    v = _unpack(st["v_codes"][pages, :, rows], st["v_params"][pages, :, rows], st["d"], False)
    return tuple(torch.where(fine, t.transpose(1, 2), 0.0).to(dtype) for t in (k, v))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(g, shape, dev):
    return torch.randn(shape, generator=g, device=dev)


def _keys_values(g, B, HK, n, d, dtype, dev):
    """Keys with channels of unequal size and offset, as projections give
    them, and plain values."""
    gain = (0.5 * _normal(g, (HK, 1, d), dev)).exp()
    k = (_normal(g, (B, HK, n, d), dev) + 0.3 * _normal(g, (HK, 1, d), dev)) * gain
    return k.to(dtype), _normal(g, (B, HK, n, d), dev).to(dtype), gain


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    c = dict(case)
    B, H, HK, d, n, page = (c[x] for x in ("B", "H", "HK", "d", "n", "page"))
    dtype, G = _DTYPES[c["dtype"]], -(-c["d"] // 32)
    P = -(-(c["start"] + n) // page)
    counts = torch.tensor(_counts(c), dtype=torch.int32, device=dev)
    # a pool whose pages were handed out in no order; its last page stays free
    table = torch.randperm(B * P, generator=g, device=dev).reshape(B, P)
    st = {"case": c, "d": d, "n": n, "table": table}
    for name in ("k", "v"):
        st[name + "_codes"] = torch.zeros((B * P + 1, HK, page, 16 * G), dtype=torch.uint8, device=dev)
        st[name + "_params"] = torch.zeros((B * P + 1, HK, page, G, 2), dtype=torch.bfloat16, device=dev)
    k, v, gain = _keys_values(g, B, HK, n, d, dtype, dev)
    if c["call"] == "write":
        st.update(k=k, v=v, counts=counts, start=torch.full((B,), c["start"], dtype=torch.int32, device=dev))
    else:
        st.update(start=torch.zeros((B,), dtype=torch.int32, device=dev))
        for name, x in (("k", k), ("v", v)):
            for b in range(B):  # one sequence at a time: the 64-bit copies are large
                codes, params = _quantise(torch.nn.functional.pad(x[b], (0, 0, 0, P * page - n)))
                pages = _pack(codes, name == "k").unflatten(1, (P, page)).transpose(0, 1)
                st[name + "_codes"][table[b]] = pages
                st[name + "_params"][table[b]] = params.unflatten(1, (P, page)).transpose(0, 1)
    st["ends"] = st["start"] + counts
    if c["call"] == "attend":
        # heads from spread to peaked: scores with deviations from 0.5 to 2.5
        sharp = torch.linspace(0.5, 2.5, H, device=dev)[:, None, None]
        q = _normal(g, (B, H, c["NQ"], d), dev) * sharp
        q = q / gain.repeat_interleave(H // HK, 0) ** 0.5
        st.update(q=q.to(dtype), lengths=counts, scale=d ** -0.5)
    st["pages"] = table.to(torch.int32)
    if own:
        st["cache"] = _package().QuantizedKVCache.from_tensors(
            st["k_codes"], st["k_params"], st["v_codes"], st["v_params"], d)
    return st


def _package():
    root = os.path.join(os.getcwd(), "adaptive-splash-attention_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import splash_attention

    return splash_attention


def run(st):
    c = st["case"]
    if not own:
        return {"attend": _plain_attend, "write": _plain_write, "read": _plain_read}[c["call"]](st)
    if c["call"] == "attend":
        return st["cache"].attention(st["q"], st["pages"], st["lengths"], alpha=c["alpha"],
                                     sm_scale=st["scale"])
    if c["call"] == "write":
        st["cache"].write(st["k"], st["v"], st["pages"], st["start"], st["counts"])
    return st["cache"].read(st["pages"], st["ends"], st["n"], _DTYPES[c["dtype"]], start=st["start"])


# ---------------------------------------------------------------------------
# Work and exact results
# ---------------------------------------------------------------------------
def work(case):
    """Attention: every key's codes and params, one value row to a query row
    (the fewest that weights summing to one can need: alpha-entmax gives most
    keys no weight), queries and results.  Write: the tokens in, their rows
    out, and rows in and values out for the read; read: the latter."""
    c = case
    size, G = (4 if c["dtype"] == "float32" else 2), -(-c["d"] // 32)
    row = 16 * G + 4 * G
    tokens = sum(_counts(c))
    if c["call"] == "attend":
        rows = c["B"] * c["H"] * c["NQ"]
        pairs = tokens * c["H"] * c["NQ"]
        return {"bytes": tokens * c["HK"] * row + rows * (row + 2 * c["d"] * size) + 4 * tokens // c["page"],
                "flops": 2 * pairs * c["d"]}
    back = 2 * tokens * c["HK"] * row + 2 * c["B"] * c["n"] * c["HK"] * c["d"] * size
    values = 2 * tokens * c["HK"] * c["d"]
    if c["call"] == "read":
        return {"bytes": back, "flops": 2 * values}
    return {"bytes": back + values * size + 2 * tokens * c["HK"] * row, "flops": 6 * values}


def _stored(x):
    """The 64-bit values that rows [..., d] are stored as: each group's codes
    counted border by border."""
    out = torch.empty_like(x, dtype=torch.float64)
    for a in range(0, x.shape[-1], 32):
        y = x[..., a:a + 32].double()
        low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        m = low.to(torch.bfloat16)
        m = torch.where(m.double() > low, torch.nextafter(m, torch.full_like(m, -math.inf)), m).double()
        s = ((high - m) / 15).to(torch.bfloat16)
        s = torch.where(15 * s.double() >= high - m, s, torch.nextafter(s, torch.full_like(s, math.inf)))
        s = torch.where(high > m, s.double().clamp_min(_TINY), 0.0)
        code = torch.zeros_like(y)
        for k in range(15):
            code += (y > m + (k + 0.5) * s).double()
        out[..., a:a + 32] = m + code * s
    return out


def exact(case, seed):
    c = case
    dev = torch.device("cuda")
    B, H, HK, d, n, NQ = (c[x] for x in ("B", "H", "HK", "d", "n", "NQ"))
    g = torch.Generator(device=dev).manual_seed(seed)
    torch.randperm(B * -(-(c["start"] + n) // c["page"]), generator=g, device=dev)  # the pages come first
    k, v, gain = _keys_values(g, B, HK, n, d, _DTYPES[c["dtype"]], dev)
    counts = _counts(c)
    if c["call"] != "attend":
        out = []
        for x in (k, v):
            y = torch.zeros(x.shape, dtype=torch.float64, device=dev)
            for b, t in enumerate(counts):
                if t:
                    y[b, :, :t] = _stored(x[b, :, :t])
            out.append(y)
        return tuple(out)
    sharp = torch.linspace(0.5, 2.5, H, device=dev)[:, None, None]
    q = _normal(g, (B, H, NQ, d), dev) * sharp
    q = (q / gain.repeat_interleave(H // HK, 0) ** 0.5).to(_DTYPES[c["dtype"]]).double()
    q = q.reshape(B, HK, H // HK * NQ, d)
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    e = 1.0 / (c["alpha"] - 1.0)
    for b, t in enumerate(counts):
        if not t:
            continue
        s = q[b] @ _stored(k[b, :, :t]).transpose(1, 2).contiguous() * d ** -0.5  # [HK, rows, t]
        last = (t - NQ + torch.arange(NQ, device=dev)).repeat(H // HK)[:, None]
        z = (c["alpha"] - 1.0) * s.clamp(-10.0, 10.0)
        z[:, torch.arange(t, device=dev) > last] = -1e3
        lo = z.amax(-1, keepdim=True) - 1.0
        hi = lo + 1.0
        for _ in range(54):
            mid = 0.5 * (lo + hi)
            big = (z - mid).clamp_min(0.0).pow(e).sum(-1, keepdim=True) >= 1.0
            lo, hi = torch.where(big, mid, lo), torch.where(big, hi, mid)
        p = (z - lo).clamp_min(0.0).pow(e)
        p = torch.where(last >= 0, p / p.sum(-1, keepdim=True), 0.0)
        out[b] = p @ _stored(v[b, :, :t])
    return out.reshape(B, H, NQ, d)
