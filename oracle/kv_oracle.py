"""Rotary positions, the paged key-value cache and one-token attention, restated in 64 bits on the CPU.

Caches are (k, v, k_exp, v_exp) with k, v [pages, kv_heads, page_size, dim] in bf16, or as e4m3 bytes with int8
exponents [pages, kv_heads, page_size]; a row of a quantised cache stands for code * 2^exp."""

from __future__ import annotations

import math

import torch

E_MIN, E_MAX = -110, 119


def e4m3_values() -> torch.Tensor:
    """The 256 values of e4m3 codes from the format: sign, 4 exponent bits (bias 7), 3 of fraction; code
    0x7f / 0xff is NaN."""
    out = []
    for b in range(256):
        e, f = (b >> 3) & 15, b & 7
        v = math.nan if (b & 127) == 127 else (f / 8 * 2.0**-6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
        out.append(-v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


def rope(x, positions, inv_freq, interleaved=False, factor=1.0):
    """x [T, heads, dim] in float64 with its pairs turned."""
    x = x.double().clone()
    r = inv_freq.numel()
    t = positions.double()[:, None] * inv_freq.double()
    c, s = (t.cos() * factor)[:, None], (t.sin() * factor)[:, None]
    ia = torch.arange(0, 2 * r, 2) if interleaved else torch.arange(r)
    ib = ia + 1 if interleaved else ia + r
    a, b = x[..., ia], x[..., ib]
    x[..., ia], x[..., ib] = a * c - b * s, b * c + a * s
    return x


def exponent(x):
    """The exponent of each row (last axis) of bf16 values: the smallest e with amax <= 448 * 2^e, clamped."""
    out = []
    for r in x.double().reshape(-1, x.shape[-1]):
        r = r[r.isfinite()]
        top = float(r.abs().max()) if r.numel() else 0.0
        e = 0
        if top > 0:
            e = math.floor(math.log2(top / 448)) - 1
            while 448 * 2.0**e < top:
                e += 1
            e = min(max(e, E_MIN), E_MAX)
        out.append(e)
    return torch.tensor(out, dtype=torch.int8).reshape(x.shape[:-1])


def quantise(x):
    """(values that the codes stand for in float64, exponents) of bf16 rows: nearest e4m3, ties to the even
    code; what is not finite becomes NaN."""
    e = exponent(x)
    grid = e4m3_values()[:127]  # the positive ones, ascending: code = index
    y = x.double() * torch.exp2(-e.double())[..., None]
    a = y.abs().clamp_max(448).nan_to_num(0.0).contiguous()
    hi = torch.searchsorted(grid, a).clamp_max(126)
    lo = (hi - 1).clamp_min(0)
    dh, dl = grid[hi] - a, a - grid[lo]
    code = torch.where(dl < dh, lo, torch.where(dh < dl, hi, torch.where(lo % 2 == 0, lo, hi)))
    v = grid[code] * torch.where(y < 0, -1.0, 1.0)
    return torch.where(x.double().isfinite(), v, math.nan) * torch.exp2(e.double())[..., None], e


def values(cache, exps):
    """What a cache buffer holds, in float64."""
    if exps is None:
        return cache.double()
    return e4m3_values()[cache.view(torch.uint8).long()] * torch.exp2(exps.double())[..., None]


def tokens(cache, exps, table, row, n):
    """The first n tokens of a row: [kv_heads, n, dim]; tokens of a page outside the cache are None places
    (second result: which tokens have a page)."""
    size, pages = cache.shape[2], cache.shape[0]
    at = torch.arange(n)
    page = table[row].long()[at // size] if n else at
    ok = (page >= 0) & (page < pages)
    page = torch.where(ok, page, 0)
    e = None if exps is None else exps[page, :, at % size]
    return values(cache[page, :, at % size], e).transpose(0, 1), ok


def attention(q, k_cache, v_cache, k_exp, v_exp, table, lengths, scale=None, window=0):
    """(out [rows, q_heads, dim], lse, spread = sum p |v|, reach = max scale * sum |q k|), all float64."""
    rows, q_heads, dim = q.shape
    kv_heads, size = k_cache.shape[1], k_cache.shape[2]
    g = q_heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(rows, q_heads, dim, dtype=torch.float64)
    spread = torch.zeros_like(out)
    lse = torch.full((rows, q_heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros(rows, q_heads, dtype=torch.float64)
    for r in range(rows):
        n = min(int(lengths[r]), table.shape[1] * size)
        if n <= 0:
            continue
        k, ok = tokens(k_cache, k_exp, table, r, n)
        v, _ = tokens(v_cache, v_exp, table, r, n)
        if window:
            ok = ok & (torch.arange(n) >= n - window)
        if not ok.any():
            continue
        k, v = k[:, ok], v[:, ok]
        for h in range(kv_heads):
            of = slice(h * g, (h + 1) * g)
            s = q[r, of].double() @ k[h].T * scale
            p = s.softmax(-1)
            out[r, of], lse[r, of] = p @ v[h], s.logsumexp(-1)
            spread[r, of] = p @ v[h].abs()
            reach[r, of] = (q[r, of].double().abs() @ k[h].abs().T).amax(-1) * abs(scale)
    return out, lse, spread, reach
