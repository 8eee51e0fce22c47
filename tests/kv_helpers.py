"""Seeded paged caches for the tests: pages dealt out of order, every place that no token holds poisoned with NaN
(bf16) or NaN codes and huge exponents (e4m3), unused table entries outside the cache."""

import torch

from oracle import kv_oracle

BF = torch.bfloat16


def paged(lengths, kv_heads, dim, size, quant, seed, capacity=None, like=None):
    """dict of k, v, k_exp, v_exp, table, lengths, status on the CPU."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // size) for n in lengths]
    per_row = max(need + [1] + ([-(-capacity // size)] if capacity else []))
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), per_row), -7, dtype=torch.int32)
    used = torch.zeros(pages, size, dtype=torch.bool)
    for r, n in enumerate(lengths):
        mine, order = order[:need[r]], order[need[r]:]
        table[r, :need[r]] = torch.tensor(mine, dtype=torch.int32)
        for i, p in enumerate(mine):
            used[p, :min(size, n - i * size)] = True
    d = {"table": table, "lengths": torch.tensor(lengths, dtype=torch.int64), "status": torch.zeros(1, dtype=torch.int32)}
    shape = (pages, kv_heads, size, dim)
    for name in ("k", "v"):
        x = torch.randn(shape, generator=g)
        x *= torch.exp2(torch.randint(-3, 3, shape[:3], generator=g).float())[..., None]  # rows of different sizes
        x = x.to(BF)
        hole = ~used[:, None, :].expand(shape[:3])
        if quant:
            v, e = kv_oracle.quantise(x)
            code = (v * torch.exp2(-e.double())[..., None]).float().to(torch.float8_e4m3fn)
            code.view(torch.uint8)[hole] = 0x7F
            e[hole] = torch.where(torch.rand(e[hole].shape, generator=g) < 0.5, 127, -128).to(torch.int8)
            d[name], d[name + "_exp"] = code, e
        else:
            x[hole] = torch.nan
            d[name], d[name + "_exp"] = x, None
    return d


def to_cuda(d):
    return {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in d.items()}


def held(d):
    return d["k"], d["v"], d["k_exp"], d["v_exp"]


def check_attention(out, lse, d, q, scale=None, window=0):
    """Against the oracle. The bounds count, in the order below: rounding the output to bf16 (half a step, 2^-8
    of the value); one rounding of each weight to 11 bits (2^-11, the sum's weights are not rounded), the
    logits' error as the weights' (twice it, once from the sum), and the fp32 accumulations, n / 16 tensor
    steps that each lose at most 2^-22 of the terms so far, all against sum p |v|. A logit adds dim / 16 such
    steps and a few fp32 roundings against scale * sum |q k|."""
    ref, rlse, spread, reach = kv_oracle.attention(q, *held(d), d["table"], d["lengths"], scale, window)
    out, lse = out.double().cpu(), lse.double().cpu()
    n = int(d["lengths"].max()) if d["lengths"].numel() else 0
    logit = reach * (q.shape[-1] / 16 + 4) * 2.0**-22
    tol = ref.abs() * 2.0**-8 + spread * (2.0**-11 + 2 * logit + (n / 16 + 8) * 2.0**-22)[..., None] + 1e-30
    assert out.isfinite().all()
    assert ((out - ref).abs() <= tol).all(), float(((out - ref).abs() / tol).max())
    empty = rlse == -torch.inf
    assert torch.equal(lse == -torch.inf, empty)
    ltol = logit + rlse.abs() * 2.0**-22 + (n / 16 + 8) * 2.0**-22
    assert ((lse - rlse).abs()[~empty] <= ltol[~empty]).all(), float(((lse - rlse).abs() / ltol)[~empty].max())
    assert (out[empty] == 0).all()
