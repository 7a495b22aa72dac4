"""The 4-bit cache on the GPU: codes against the 64-bit definition (equal, not
near), attention against 64-bit alpha-entmax, and the ways a serving program
calls them."""
from __future__ import annotations

import math

import pytest
import torch

import splash_attention as sa

import _cache as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(dev, pages, heads, d, page, fill=0xA5):
    """A cache whose every byte is `fill` (as params: finite odd values)."""
    c = sa.QuantizedKVCache(pages, heads, d, page, device=dev)
    for t in c.tensors():
        t.view(torch.uint8).fill_(fill)
    return c


def table_of(B, P, pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:B * P].reshape(B, P).to(torch.int32)


def stored(c, table, b, t):
    """codes, s, m of position t's key row and value row (all heads), float64."""
    page, row = int(table[b, t // c.page_size]), t % c.page_size
    kc, kp, vc, vp = (x[page, :, row].cpu() for x in c.tensors())
    return ref.unpack(kc, kp, c.head_dim, True), ref.unpack(vc, vp, c.head_dim, False)


def hard_rows(n, d, dtype, seed):
    """Rows that are hard to quantise: on the borders, constant, offset,
    huge, tiny, not finite, with a minimum far below the step."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g)
    big = 6e4 if dtype == torch.float16 else 3e38
    for i in range(n):
        kind = i % 10
        if kind == 1:  # borders and codes of a power-of-two step: ties
            x[i] = torch.randint(0, 31, (d,), generator=g) * 0.25 - 3.0
        elif kind == 2:
            x[i] = x[i, 0]
        elif kind == 3:
            x[i] = x[i] * 1e-3 + 100.0
        elif kind == 4:
            x[i] = x[i].sign() * big
        elif kind == 5:
            x[i] = x[i] * (2.0 ** -20 if dtype == torch.float16 else 2.0 ** -130)
        elif kind == 6:
            x[i, ::5] = math.nan
            x[i, 1::7] = math.inf
            x[i, 2::9] = -math.inf
        elif kind == 7:  # a minimum far below the step, ties above it
            x[i] = torch.randint(1, 31, (d,), generator=g) * 0.5
            x[i, ::32] = -2.0 ** (-20 - i % 3)
            x[i, 1::32] = 15.0
        elif kind == 8:
            x[i] = 0.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page", [(64, 64), (128, 16), (80, 32), (96, 64), (1, 16), (20, 128), (33, 32), (127, 16), (8, 256)])
def test_written_codes_are_the_definitions(dev, dtype, d, page):
    """Codes, scales and offsets equal the 64-bit definition's; every other
    byte of the pool stays as it was; read gives m + c s rounded once."""
    B, H, n = 3, 2, 40
    start, counts = [0, page - 3, 5], [40, 23, 0]
    P = -(-(page + n) // page)
    pages = B * P + 2
    c = make(dev, pages, H, d, page)
    table = table_of(B, P, pages)
    K = hard_rows(B * H * n, d, dtype, 1).reshape(B, H, n, d)
    V = hard_rows(B * H * n, d, dtype, 2).reshape(B, H, n, d).flip(2).contiguous()
    i32 = dict(dtype=torch.int32, device=dev)
    c.write(K.to(dev), V.to(dev), table.to(dev), torch.tensor(start, **i32), torch.tensor(counts, **i32))
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(B):
        for i in range(counts[b]):
            t = start[b] + i
            touched[table[b, t // page], t % page] = True
            for (got, src) in zip(stored(c, table, b, t), (K, V)):
                for a, w in zip(got, ref.quantise(src[b, :, i])):
                    assert torch.equal(a, w), (b, i)
    for x in c.tensors():
        left = x.cpu().view(torch.uint8).reshape(pages, H, page, -1)
        assert bool((left.permute(0, 2, 1, 3)[~touched] == 0xA5).all())
    ends = torch.tensor([s + m for s, m in zip(start, counts)], **i32)
    for out in TYPES:
        got = c.read(table.to(dev), ends, n, out, torch.tensor(start, **i32))
        for g, src in zip(got, (K, V)):
            assert g.shape == (B, H, n, d) and g.dtype == out
            want = ref.values(*ref.quantise(src)).to(torch.float32).to(out)
            for b in range(B):
                assert torch.equal(g[b, :, :counts[b]].cpu(), want[b, :, :counts[b]])
                assert not bool(g[b, :, counts[b]:].any())


def test_codes_past_the_head_dimension_are_zero(dev):
    c = make(dev, 1, 1, 20, 16)
    K = torch.randn(1, 1, 1, 20, device=dev)
    z = torch.zeros(1, dtype=torch.int32, device=dev)
    c.write(K, K, z[None], z)
    (kc, _, _), (vc, _, _) = (ref.unpack(x[0, :, 0].cpu(), p[0, :, 0].cpu(), 32, key) for x, p, key in
                              ((c.k_codes, c.k_params, True), (c.v_codes, c.v_params, False)))
    assert not bool(kc[..., 20:].any()) and not bool(vc[..., 20:].any())


@pytest.mark.parametrize("layout", ["bnhd", "expanded", "sliced", "odd_offset", "channel_stride"])
def test_write_reads_any_layout(dev, layout):
    B, H, n, d = 2, 3, 21, 64
    x = torch.randn(B, H, n, d, device=dev).bfloat16()
    if layout == "bnhd":
        y = x.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "expanded":
        x = x[:, :1].expand(B, H, n, d)
        y = x
    elif layout == "sliced":
        y = torch.cat([x, x], -1)[..., :d]
    elif layout == "odd_offset":
        y = torch.empty(x.numel() + 1, device=dev, dtype=x.dtype)[1:].view(x.shape).copy_(x)
    else:
        y = torch.stack([x, x], -1)[..., 0]
    i = torch.zeros(B, dtype=torch.int32, device=dev)
    table = torch.arange(2 * B, dtype=torch.int32, device=dev).reshape(B, 2)
    a, b = make(dev, 2 * B, H, d, 16), make(dev, 2 * B, H, d, 16)
    a.write(x.contiguous(), x.contiguous(), table, i)
    b.write(y, y, table.long(), i.long())
    for s, t in zip(a.tensors(), b.tensors()):
        assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))


def test_tokens_without_a_page_are_dropped(dev):
    """Negative positions, positions past the table and entries that are not
    pages: nothing is written for them, and they read as zeros."""
    B, H, d, page = 4, 2, 64, 16
    c = make(dev, 3, H, d, page)
    table = torch.tensor([[0, -1], [3, 1], [-(2 ** 31), 2 ** 31 - 1], [2, 2 ** 20]], dtype=torch.int32, device=dev)
    start = torch.tensor([10, -5, 0, 28], dtype=torch.int32, device=dev)
    K = torch.randn(B, H, 25, d, device=dev)
    before = [t.clone() for t in c.tensors()]
    c.write(K, K, table, start)
    changed = [(t.view(torch.uint8) != s.view(torch.uint8)).reshape(3, H, page, -1).any(-1).any(1).cpu()
               for t, s in zip(c.tensors(), before)]
    want = torch.zeros(3, page, dtype=torch.bool)
    want[0, 10:] = True  # sequence 0: page 0 from row 10, then no page
    want[1, :4] = True   # sequence 1: positions 16 .. 19 (0 .. 15 have no page)
    for got in changed:
        assert not bool((got & ~want).any())
    assert bool((changed[0][want]).all())
    lengths = torch.tensor([32, 20, 32, 40], dtype=torch.int32, device=dev)
    k, v = c.read(table, lengths, 40, torch.float32)
    fine = torch.zeros(B, 40, dtype=torch.bool)
    fine[0, :16] = fine[1, 16:20] = fine[3, :16] = True
    for t in (k, v):
        assert not bool(t.cpu().permute(0, 2, 1, 3)[~fine].any())
    assert torch.equal(k[0, :, 10:16], c.read(table[:1], lengths[:1], 6, torch.float32, start[:1])[0][0])


def test_read_defaults_and_extremes(dev):
    c = make(dev, 4, 1, 32, 16)
    K = torch.randn(1, 1, 64, 32, device=dev)
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device=dev)
    z = torch.zeros(1, dtype=torch.int32, device=dev)
    c.write(K, K, table, z)
    k, _ = c.read(table, z + 64)
    assert k.shape == (1, 1, 64, 32) and k.dtype == torch.bfloat16
    assert not bool(c.read(table, z, 5)[0].any())
    assert not bool(c.read(table, z + 2 ** 31 - 1, 5, start=z + 2 ** 31 - 3)[0].any())
    assert torch.equal(c.read(table, z + 64, 3, start=z - 1)[0][:, :, 1:], k[:, :, :2])


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def filled(dev, lengths, HK, d, page, dtype, seed, kscale=1.0):
    B = len(lengths)
    n = max(max(lengths), 1)
    P = -(-n // page)
    pages = B * P + 3
    c = make(dev, pages, HK, d, page)
    table = table_of(B, P, pages, seed).to(dev)
    g = torch.Generator().manual_seed(seed)
    K = torch.randn(B, HK, n, d, generator=g) * kscale + 0.3
    V = torch.randn(B, HK, n, d, generator=g)
    L = torch.tensor(lengths, dtype=torch.int32, device=dev)
    c.write(K.to(dtype).to(dev), V.to(dtype).to(dev), table, torch.zeros_like(L), L)
    k, v = c.read(table, L, n, torch.float32)
    return c, table, L, k.double().cpu(), v.double().cpu()


def check_attention(out, q, k, v, lengths, q_idx, alpha, scale, what=""):
    """out against 64-bit attention over the cached values.

    Scores: q.k is a sum of codes 16 + c <= 31 times the queries, minus 16
    times their sum, in fp32.  About a hundred roundings of 2^-24 of partial
    sums near 30 s |q|_2 (the 32 terms of a group have random signs) add as
    their root: 10 * 2^-24 * 30 * s |q|_2 per group; z carries (alpha - 1)
    scale of it and its own rounding, 2^-24 |z|.  A weight moves by e
    v^(e-1) dz, tau by at most dz, and the normaliser by as much again: out
    by at most 4 sens dz max|v|, sens = sum e v^(e-1).  The powers' own error
    (hardware exp2 and log2: 2^-22 of the exponent's argument, at most e
    log2(1/v) ~ 40) adds 2^-17 for a general alpha; 16-bit outputs round once
    more, by half a step."""
    B, H, NQ, d = q.shape
    HK = k.shape[1]
    q64 = q.double().cpu()
    half = torch.finfo(q.dtype).eps / 2
    for b in range(B):
        n = lengths[b]
        vis = torch.tensor([max(0, min(n, int(p) + 1)) for p in q_idx[b]])
        for h in range(H):
            kk, vv = k[b, h // (H // HK), :n], v[b, h // (H // HK), :n]
            want, sens = ref.entmax_attention(q64[b, h], kk, vv, vis, alpha, scale)
            if not n:
                assert not bool(out[b, h].any()), what
                continue
            s = (kk.amax() - kk.amin()) / 15
            dz = (alpha - 1) * (abs(scale) * 10 * 2.0 ** -24 * 30 * float(s) * math.sqrt(d / 32)
                                * q64[b, h].norm(dim=1) + 10 * 2.0 ** -24)
            tol = (4 * sens * dz + 2.0 ** -17) * float(vv.abs().amax())
            got = out[b, h].double().cpu()
            err = (got - want).abs() - half * want.abs()
            assert bool((err <= tol[:, None]).all()), \
                f"{what} b {b} h {h}: {float((err - tol[:, None]).max()):.3e} past {tol.max():.3e}"
            assert not bool(got[vis == 0].any())


def default_idx(lengths, NQ):
    return [[n - NQ + i for i in range(NQ)] for n in lengths]


SHAPES = [
    # lengths, HK, rep, NQ, d, page
    ([1], 1, 1, 1, 64, 64),
    ([5, 0, 64, 65], 2, 2, 1, 64, 16),
    ([300], 1, 16, 1, 128, 64),
    ([257, 31], 2, 3, 2, 80, 32),
    ([511, 2, 0], 3, 5, 4, 96, 128),
    ([129], 1, 7, 5, 32, 16),
    ([40, 700], 2, 1, 64, 64, 256),
    ([90], 2, 20, 3, 24, 16),
    ([33, 100], 1, 2, 1, 1, 16),
    ([70], 1, 1, 3, 127, 32),
    ([2048], 1, 4, 1, 128, 64),
    # past the one-block plan
    ([2500, 17, 0], 2, 4, 1, 64, 64),
    ([3001], 1, 9, 3, 128, 16),
    ([5000, 4999], 1, 1, 1, 100, 256),
    ([9000], 1, 2, 1, 33, 128),
    ([70001], 1, 2, 1, 32, 64),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[1:])) + f"_n{s[0][0]}")
def test_attention_matches_64_bits(dev, dtype, shape):
    lengths, HK, rep, NQ, d, page = shape
    c, table, L, k, v = filled(dev, lengths, HK, d, page, dtype, 3)
    g = torch.Generator().manual_seed(4)
    q = (torch.randn(len(lengths), HK * rep, NQ, d, generator=g) * 1.5).to(dtype)
    out = c.attention(q.to(dev), table, L, alpha=1.5, sm_scale=d ** -0.5)
    assert out.dtype == dtype and out.shape == q.shape
    check_attention(out, q, k, v, lengths, default_idx(lengths, NQ), 1.5, d ** -0.5, str(shape))


@pytest.mark.parametrize("alpha", [1.05, 1.2, 1.25, 4 / 3, 1.5, 1.75, 2.0, 2.5, 3.0])
@pytest.mark.parametrize("n", [200, 2300])
def test_attention_over_alphas(dev, alpha, n):
    if alpha > 2:
        # e < 1: a weight's slope grows without bound at the support's edge.
        # Keys that are spread enough keep the edge free of near ties.
        n = n // 8
    c, table, L, k, v = filled(dev, [n], 1, 64, 32, torch.float32, 5)
    q = torch.randn(1, 4, 1, 64, generator=torch.Generator().manual_seed(6)) * 1.5
    out = c.attention(q.to(dev), table, L, alpha=alpha)
    check_attention(out, q, k, v, [n], [[n - 1]], alpha, 0.125, f"alpha {alpha}")


@pytest.mark.parametrize("n,qscale", [(900, 1e-4), (900, 0.0), (900, 0.1), (1500, 1e-4), (1500, 0.0), (12000, 1e-4), (12000, 0.0), (20000, 0.05), (2000, 40.0)])
@pytest.mark.parametrize("alpha", [1.5, 2.0, 1.25, 2.5])
def test_flat_and_peaked_rows(dev, n, qscale, alpha):
    """Near-uniform rows, whose candidates fit no list, rows with every score
    equal, and rows past the score clamp."""
    c, table, L, k, v = filled(dev, [n], 1, 64, 64, torch.float32, 7)
    q = torch.randn(1, 2, 1, 64, generator=torch.Generator().manual_seed(8)) * qscale
    out = c.attention(q.to(dev), table, L, alpha=alpha)
    check_attention(out, q, k, v, [n], [[n - 1]], alpha, 0.125)


@pytest.mark.parametrize("n", [150, 2500])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales_of_any_sign(dev, n, scale):
    c, table, L, k, v = filled(dev, [n], 2, 64, 32, torch.bfloat16, 20)
    for rep in (1, 3, 6, 10):  # each number of key tiles that share a result
        q = torch.randn(1, 2 * rep, 1, 64, generator=torch.Generator().manual_seed(rep)).bfloat16()
        out = c.attention(q.to(dev), table, L, sm_scale=scale)
        check_attention(out, q, k, v, [n], [[n - 1]], 1.5, scale)


@pytest.mark.parametrize("n", [100, 3000])
def test_query_positions(dev, n):
    """Any positions, in any order: before the first key, past the last."""
    c, table, L, k, v = filled(dev, [n, n // 2], 2, 64, 16, torch.bfloat16, 9)
    idx = [[0, -1, n - 1, 5 * n], [n // 3, 7, -2 ** 31, 2 ** 31 - 1]]
    q = torch.randn(2, 4, 4, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    out = c.attention(q.to(dev), table, L, torch.tensor(idx, device=dev))
    check_attention(out, q, k, v, [n, n // 2], idx, 1.5, 0.125)


@pytest.mark.parametrize("n", [100, 3000])
def test_max_length_bounds_the_keys(dev, n):
    c, table, L, k, v = filled(dev, [n], 1, 64, 16, torch.float32, 10)
    q = torch.randn(1, 2, 1, 64, generator=torch.Generator().manual_seed(1))
    same = c.attention(q.to(dev), table, L, max_length=n)
    assert torch.allclose(same, c.attention(q.to(dev), table, L, max_length=10 * n), atol=1e-6)
    m = n - 37
    out = c.attention(q.to(dev), table, L, torch.full((1, 1), n, device=dev), max_length=m)
    check_attention(out, q, k[:, :, :m], v[:, :, :m], [m], [[n]], 1.5, 0.125)
    check_attention(c.attention(q.to(dev), table, L + 10 ** 6, torch.full((1, 1), n - 1, device=dev)),
                    q, k, v, [n], [[n - 1]], 1.5, 0.125)


@pytest.mark.parametrize("n,page", [(200, 16), (2600, 64)])
def test_keys_of_missing_pages_are_not_seen(dev, n, page):
    c, table, L, k, v = filled(dev, [n], 2, 64, page, torch.float32, 11)
    bad = table.clone()
    bad[0, 1], bad[0, 3] = -1, 2 ** 30
    keep = torch.ones(n, dtype=torch.bool)
    keep[page:2 * page] = keep[3 * page:4 * page] = False
    q = torch.randn(1, 4, 1, 64, generator=torch.Generator().manual_seed(2))
    out = c.attention(q.to(dev), bad, L)
    check_attention(out, q, k[:, :, keep], v[:, :, keep], [int(keep.sum())], [[n]], 1.5, 0.125)
    assert not bool(c.attention(q.to(dev), torch.full_like(bad, -1), L).any())


@pytest.mark.parametrize("n", [64, 2200])
def test_rows_that_are_not_finite(dev, n):
    """A query row with a NaN or an infinity scores -10 throughout: the mean
    of its visible values.  Other rows do not notice."""
    c, table, L, k, v = filled(dev, [n], 1, 64, 64, torch.float32, 12)
    for dtype in TYPES:
        q = torch.randn(1, 4, 1, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
        clean = c.attention(q.to(dev), table, L)
        q[0, 1, 0, 5] = math.nan
        q[0, 3, 0, 40] = math.inf
        out = c.attention(q.to(dev), table, L)
        assert torch.equal(out[:, ::2], clean[:, ::2])
        mean = v[0, 0].mean(0)
        for h in (1, 3):
            assert float((out[0, h, 0].double().cpu() - mean).abs().max()) <= 2e-6 + torch.finfo(dtype).eps


@pytest.mark.parametrize("layout", ["bnhd", "expanded", "odd_offset", "channel_stride", "broadcast"])
def test_attention_reads_any_query_layout(dev, layout):
    c, table, L, _, _ = filled(dev, [300, 120], 2, 64, 32, torch.bfloat16, 13)
    x = torch.randn(2, 4, 3, 64, device=dev).bfloat16()
    if layout == "bnhd":
        y = x.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "expanded":
        x = x[:, :1].expand(2, 4, 3, 64)
        y = x
    elif layout == "broadcast":
        x = x[:1, :1, :1].expand(2, 4, 3, 64)
        y = x
    elif layout == "odd_offset":
        y = torch.empty(x.numel() + 1, device=dev, dtype=x.dtype)[1:].view(x.shape).copy_(x)
    else:
        y = torch.stack([x, x], -1)[..., 0]
    assert torch.equal(c.attention(y, table.long(), L.long()), c.attention(x.contiguous(), table, L))


@pytest.mark.parametrize("n", [1000, 6000])
def test_same_bits_every_time_and_on_another_stream(dev, n):
    c, table, L, _, _ = filled(dev, [n, n // 3], 2, 128, 64, torch.bfloat16, 14)
    q = torch.randn(2, 8, 1, 128, device=dev).bfloat16()
    first = c.attention(q, table, L)
    for _ in range(3):
        assert torch.equal(c.attention(q, table, L), first)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        a = c.attention(q, table, L)
    with torch.cuda.stream(t):
        b = c.attention(q, table, L)
    torch.cuda.synchronize()
    assert torch.equal(a, first) and torch.equal(b, first)


@pytest.mark.parametrize("long", [False, True])
def test_decode_loop_against_the_dense_path(dev, long):
    """Prompt through the cache, then tokens one by one: each step's output is
    splash_attention's (exact threshold) on the values read back."""
    B, HK, rep, d, page = 2, 2, 2, 64, 32
    n0, steps = (2301 if long else 61), 5
    P = -(-(n0 + steps) // page)
    c = make(dev, B * P, HK, d, page)
    table = table_of(B, P, B * P).to(dev)
    g = torch.Generator().manual_seed(15)
    x = [torch.randn(B, HK, n0 + steps, d, generator=g).bfloat16().to(dev) for _ in range(2)]
    z = torch.zeros(B, dtype=torch.int32, device=dev)
    c.write(x[0][:, :, :n0], x[1][:, :, :n0], table, z)
    attn = sa.AdaptiveSplashAttention(head_dim=d, alpha=1.5, k_keep=32, tau_mode="exact")
    for t in range(n0, n0 + steps):
        c.write(x[0][:, :, t:t + 1], x[1][:, :, t:t + 1], table, z + t)
        q = (torch.randn(B, HK * rep, 1, d, generator=g) * 1.5).to(dev)
        out = attn.decode(q, c, table, z + t + 1)
        k, v = (y.repeat_interleave(rep, 1) for y in c.read(table, z + t + 1, t + 1, torch.float32))
        with torch.no_grad():
            want = attn(q, k, v, torch.full((B * HK * rep, 1), t, device=dev, dtype=torch.int32))
        # both sides round scores in fp32: check_attention's bound, 1e-4 at these sizes
        assert float((out - want).abs().max()) <= 1e-4


@pytest.mark.parametrize("n", [200, 3000])
def test_captured_steps_replay(dev, n):
    """A decode step (write, attend, read) captured into a graph and replayed
    as its inputs change, with eager work between; two graphs of one cache."""
    B, HK, d, page = 2, 2, 64, 32
    c, table, L, _, _ = filled(dev, [n, n - 9], HK, d, page, torch.bfloat16, 16)
    k = torch.randn(B, HK, 1, d, device=dev).bfloat16()
    q = torch.randn(B, 4, 1, d, device=dev).bfloat16()
    start = L - 1

    def step():
        c.write(k, k, table, start)
        return c.attention(q, table, L), c.read(table, L, n, torch.bfloat16)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphs.append((gr, step()))
    for i in range(6):
        k.normal_()
        q.normal_()
        gr, outs = graphs[i % 2]
        gr.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i
        torch.zeros(1 << 20, device=dev).sum().item()


@pytest.mark.parametrize("HK,rep,n", [(100, 4, 2500), (100, 16, 900), (200, 1, 5000)])
def test_many_tiles_in_one_launch(dev, HK, rep, n):
    """Enough tiles for one launch with long rows: dots past 64 KB of LDS,
    captured and replayed, against the split of the same rows (few heads)."""
    d = 32
    c, table, L, k, v = filled(dev, [n, n - 70], HK, d, 64, torch.bfloat16, 21)
    q = torch.randn(2, HK * rep, 1, d, device=dev).bfloat16()
    out = c.attention(q, table, L)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        again = c.attention(q, table, L)
    for _ in range(3):
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, out)
        torch.zeros(1 << 18, device=dev).sum().item()
    for h in (0, HK - 1):
        check_attention(out[:, h * rep:(h + 1) * rep], q[:, h * rep:(h + 1) * rep], k[:, h:h + 1], v[:, h:h + 1],
                        [n, n - 70], default_idx([n, n - 70], 1), 1.5, d ** -0.5)


@pytest.mark.parametrize("alpha", [1.5, 1.25])
@pytest.mark.parametrize("rep,qscale", [(16, 1e-3), (16, 0.3), (5, 0.0), (1, 1e-3)])
def test_flat_rows_of_many_tiles(dev, rep, qscale, alpha):
    """Rows whose candidates fit no list, several to a block, some blocks with
    more rows than waves."""
    HK, n, d = 100, 900, 32
    c, table, L, k, v = filled(dev, [n, 650], HK, d, 64, torch.float32, 24)
    q = torch.randn(2, HK * rep, 1, d, generator=torch.Generator().manual_seed(9)) * qscale
    out = c.attention(q.to(dev), table, L, alpha=alpha)
    for h in (0, 57):
        check_attention(out[:, h * rep:(h + 1) * rep], q[:, h * rep:(h + 1) * rep], k[:, h:h + 1], v[:, h:h + 1],
                        [n, 650], default_idx([n, 650], 1), alpha, d ** -0.5)


def test_check_write(dev):
    """The debug check: every token of a write has a row, and its own."""
    c = make(dev, 4, 1, 32, 16)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    c.check_write(t([[0, 1], [2, 3]]), t([0, 5]), 20)
    c.check_write(t([[0, 1], [0, 3]]), t([0, 16]), 16)           # a shared page, one writer
    c.check_write(t([[0, 1], [0, -1]]), t([0, 0]), 20, t([20, 0]))
    with pytest.raises(ValueError, match="same row"):
        c.check_write(t([[0, 1], [0, 3]]), t([0, 10]), 16)
    with pytest.raises(ValueError, match="no row"):
        c.check_write(t([[0, 1], [2, 4]]), t([0, 0]), 20)
    with pytest.raises(ValueError, match="no row"):
        c.check_write(t([[0, 1]]), t([30]), 3)
    with pytest.raises(ValueError, match="no row"):
        c.check_write(t([[0, 1]]), t([-1]), 3)


def test_two_threads_call_at_once(dev):
    """Calls of one cache from two threads, each on a stream of its own."""
    import threading

    c, table, L, _, _ = filled(dev, [3000, 100], 2, 64, 32, torch.bfloat16, 22)
    qs = [torch.randn(2, 4, n, 64, device=dev).bfloat16() for n in (1, 3)]
    want = [c.attention(q, table, L) for q in qs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(c.attention(qs[i], table, L))
            torch.cuda.current_stream().synchronize()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    for g, w in zip(got, want):
        assert len(g) == 20 and all(torch.equal(x, w) for x in g)


def test_a_wide_page_table_of_short_sequences(dev):
    """The table is as wide as the longest context that a server allows."""
    c, table, L, k, v = filled(dev, [70, 3], 2, 64, 16, torch.float32, 23)
    wide = torch.full((2, 8192), -1, dtype=torch.int32, device=dev)
    wide[:, :table.size(1)] = table
    q = torch.randn(2, 4, 1, 64, generator=torch.Generator().manual_seed(5))
    check_attention(c.attention(q.to(dev), wide, L), q, k, v, [70, 3], [[69], [2]], 1.5, 0.125)
    check_attention(c.attention(q.to(dev), wide, L, max_length=100), q, k, v, [70, 3], [[69], [2]], 1.5, 0.125)


def test_compiled_steps(dev):
    """Through torch.compile, as custom operators, without a graph break."""
    c, table, L, _, _ = filled(dev, [100, 50], 2, 64, 16, torch.float32, 17)
    k = torch.randn(2, 2, 1, 64, device=dev)
    q = torch.randn(2, 4, 1, 64, device=dev)

    def step(k, q):
        c.write(k, k, table, L - 1)
        return c.attention(q, table, L), c.read(table, L, 7, torch.float32)[1]

    want = [t.clone() for t in step(k, q)]
    got = torch.compile(step, fullgraph=True, backend="eager")(k, q)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_gradients_are_refused(dev):
    c, table, L, _, _ = filled(dev, [20], 1, 64, 16, torch.float32, 18)
    q = torch.randn(1, 1, 1, 64, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradients"):
        c.attention(q, table, L)
    with pytest.raises(RuntimeError, match="no gradients"):
        c.write(q, q, table, L - 1)
    with torch.no_grad():
        c.attention(q, table, L)


def test_from_tensors_uses_the_pool_in_place(dev):
    c, table, L, _, _ = filled(dev, [50], 1, 96, 16, torch.float32, 19)
    twin = sa.QuantizedKVCache.from_tensors(*c.tensors(), 96)
    q = torch.randn(1, 1, 1, 96, device=dev)
    assert torch.equal(twin.attention(q, table, L), c.attention(q, table, L))
    bad = list(c.tensors())
    with pytest.raises(ValueError, match="shape"):
        sa.QuantizedKVCache.from_tensors(*bad, 64)
    with pytest.raises(TypeError, match="k_codes"):
        sa.QuantizedKVCache.from_tensors(bad[0].int(), *bad[1:], 96)
    with pytest.raises(ValueError, match="contiguous"):
        sa.QuantizedKVCache.from_tensors(bad[0], bad[1], torch.cat([bad[2]] * 2, -1)[..., ::2], bad[3], 96)


def test_rows_past_32_bit_offsets(dev):
    """A pool whose codes pass 2^31 bytes: rows of its last page."""
    d, page, heads = 128, 256, 16
    pages = 2 ** 31 // (page * heads * 64) + 9
    c = sa.QuantizedKVCache(pages, heads, d, page, device=dev)
    assert c.k_codes.numel() > 2 ** 31
    n = 300
    table = torch.tensor([[pages - 1, pages - 2], [0, 1]], dtype=torch.int32, device=dev)
    K, V = (torch.randn(2, heads, n, d, device=dev).bfloat16() for _ in range(2))
    K[1], V[1] = K[0], V[0]
    z = torch.zeros(2, dtype=torch.int32, device=dev)
    c.write(K, V, table, z)
    k, v = c.read(table, z + n, n)
    assert torch.equal(k[0], k[1]) and torch.equal(v[0], v[1]) and bool(k[0].any())
    q = torch.randn(1, heads, 1, d, device=dev).bfloat16().expand(2, heads, 1, d)
    out = c.attention(q, table, z + n)
    assert torch.equal(out[0], out[1]) and bool(out[0].any())
