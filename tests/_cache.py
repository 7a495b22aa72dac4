"""64-bit definitions of the 4-bit cache and the attention over it, on the CPU."""
from __future__ import annotations

import math

import torch

TINY = 2.0 ** -126


def floor_bf16(x):
    """The largest bfloat16 at most x (float64 in and out)."""
    m = x.to(torch.bfloat16)
    down = torch.nextafter(m, torch.full_like(m, -math.inf))
    return torch.where(m.double() > x, down, m).double()


def ceil_bf16(x):
    s = x.to(torch.bfloat16)
    up = torch.nextafter(s, torch.full_like(s, math.inf))
    return torch.where(s.double() < x, up, s).double()


def quantise(x):
    """codes, s, m (float64, [..., d] and [..., G]) of rows [..., d]."""
    x = torch.nan_to_num(x.double(), nan=0.0).clamp(-2.0 ** 126, 2.0 ** 126)
    codes, ss, ms = torch.zeros_like(x), [], []
    for a in range(0, x.shape[-1], 32):
        y = x[..., a:a + 32]
        m = floor_bf16(y.amin(-1))
        span = y.amax(-1) - m
        s = torch.where(span > 0, ceil_bf16((span / 15).clamp_min(TINY)), 0.0)
        # bf16(span / 15) may round onto a number whose 15-fold is below span
        s = torch.where(15 * s < span, torch.nextafter(s.to(torch.bfloat16),
                                                       torch.tensor(math.inf).bfloat16()).double(), s)
        for k in range(15):
            codes[..., a:a + 32] += (y > m[..., None] + (k + 0.5) * s[..., None]).double()
        ss.append(s)
        ms.append(m)
    return codes, torch.stack(ss, -1), torch.stack(ms, -1)


def values(codes, s, m):
    d = codes.shape[-1]
    def wide(t):
        return t.repeat_interleave(32, -1)[..., :d]
    return codes * wide(s) + wide(m)


def unpack(codes, params, d, key):
    """codes (float64 [..., d]), s, m of raw cache rows [..., 16 G], [..., G, 2]."""
    G = params.shape[-2]
    c = codes.reshape(*codes.shape[:-1], 4, G, 4).transpose(-3, -2) if key else \
        codes.reshape(*codes.shape[:-1], G, 4, 4)
    c = torch.stack([c & 15, c >> 4], -1).reshape(*codes.shape[:-1], 32 * G)
    p = params.double()
    return c.double()[..., :d], p[..., 0], p[..., 1]


def entmax_attention(q, k, v, vis, alpha, scale):
    """q [R, d], k, v [n, d] in float64; row r sees keys < vis[r].  Returns
    out [R, d] and each row's sensitivity sum e v^(e-1)."""
    R, n = q.shape[0], k.shape[0]
    e = 1.0 / (alpha - 1.0)
    out, sens = torch.zeros_like(q), torch.zeros(R, dtype=torch.float64)
    if not n:
        return out, sens
    z = (alpha - 1.0) * (q @ k.T * scale).clamp(-10, 10)
    z = torch.where(torch.arange(n) < vis[:, None], z, -1e9)
    lo = z.amax(1, keepdim=True) - 1
    hi = lo + 1
    for _ in range(60):
        mid = 0.5 * (lo + hi)
        big = (z - mid).clamp_min(0).pow(e).sum(1, keepdim=True) >= 1
        lo, hi = torch.where(big, mid, lo), torch.where(big, hi, mid)
    u = (z - lo).clamp_min(0)
    p = u.pow(e)
    ok = vis > 0
    out[ok] = (p / p.sum(1, keepdim=True))[ok] @ v
    sens[ok] = (e * torch.where(u > 0, u.pow(e - 1), 0.0).sum(1))[ok]
    return out, sens
