"""dm3::paged_attention against the 64-bit oracle, alone and in a decode loop with the cache."""

import math
import subprocess
import sys

import pytest
import torch

from oracle import kv_oracle
from tests.conftest import ROOT
from tests.kv_helpers import check_attention, held, paged, to_cuda

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _q(rows, heads, dim, seed, size=1.0):
    return (torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(seed)) * size).to(BF)


def _run(dm3, d, q, scale=None, window=0):
    dev = to_cuda(d)
    out, lse = dm3.ops.paged_attention(q.cuda(), *held(dev), dev["table"], dev["lengths"], dev["status"], scale, window)
    assert int(dev["status"]) == 0
    return out, lse


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 8), (3, 4), (1, 16), (2, 5), (1, 24), (4, 1)])
@pytest.mark.parametrize("quant", [False, True])
def test_heads(dm3, dim, kv_heads, group, quant):
    d = paged([130, 0, 1, 15, 16, 17, 77], kv_heads, dim, 48, quant, dim + group)
    q = _q(7, kv_heads * group, dim, group, 2.0)
    check_attention(*_run(dm3, d, q), d, q)


@pytest.mark.parametrize("size", [16, 32, 80, 256])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("window", [0, 1, 16, 100, 5000])
def test_lengths_pages_and_windows(dm3, size, quant, window):
    lengths = [0, 1, 2, size - 1, size, size + 1, 333, 1024, 1500, 2049]
    d = paged(lengths, 2, 128, size, quant, size + window, capacity=2500)
    q = _q(len(lengths), 6, 128, window)
    check_attention(*_run(dm3, d, q, 0.07, window), d, q, 0.07, window)


@pytest.mark.parametrize("quant", [False, True])
def test_long_row(dm3, quant):
    d = paged([40003, 7], 1, 64, 64, quant, 3)
    q = _q(2, 8, 64, 3)
    check_attention(*_run(dm3, d, q), d, q)


def _spread(rows, longest, empty, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(1, longest + 1, (rows,), generator=g)
    n[torch.rand(rows, generator=g) < empty] = 0
    return n.tolist()


@pytest.mark.parametrize("rows,longest,empty,capacity", [(300, 90, 0.3, 9000), (129, 400, 0.0, 9000), (128, 33, 0.9, 9000), (1, 3000, 0.0, 200000),
                                                         (3, 2500, 0.4, 200000), (700, 5, 0.5, 9000), (40, 700, 0.0, 700)])
@pytest.mark.parametrize("kv_heads,group,dim,quant,window", [(2, 4, 128, False, 0), (1, 12, 64, True, 0), (3, 20, 64, False, 50), (1, 9, 256, True, 0)])
def test_many_and_ragged_rows(dm3, rows, longest, empty, capacity, kv_heads, group, dim, quant, window):
    """Rows of all lengths in one sequence cut into equal shares: cuts inside rows, at their ends, and over many of them."""
    d = paged(_spread(rows, longest, empty, rows + dim), kv_heads, dim, 16, quant, rows, capacity=capacity)
    q = _q(rows, kv_heads * group, dim, rows)
    check_attention(*_run(dm3, d, q, None, window), d, q, None, window)


@pytest.mark.parametrize("rows,longest", [(128, 900), (100, 900), (101, 200)])
@pytest.mark.parametrize("quant", [False, True])
def test_longest_rows_first(dm3, rows, longest, quant):
    """More units than run at once, in a table of 1,000 tokens a row: rows of equal lengths, of none, and in any order."""
    n = _spread(rows, longest, 0.1, rows)
    n[3:40] = [n[3]] * 37
    d = paged(n, 3, 64, 16, quant, rows, capacity=1000)
    q = _q(rows, 6, 64, rows)
    check_attention(*_run(dm3, d, q), d, q)


def test_nothing_to_see(dm3):
    d = paged([0, 0, 0], 2, 64, 16, False, 1)
    q = _q(3, 4, 64, 1)
    out, lse = _run(dm3, d, q)
    assert (out == 0).all() and (lse == -math.inf).all()
    e = torch.zeros(0, 4, 64, dtype=BF, device="cuda")
    dev = to_cuda(d)
    out, lse = dm3.ops.paged_attention(e, *held(dev), dev["table"][:0], dev["lengths"][:0], dev["status"])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    wide = paged([0, 0, 0], 2, 64, 16, False, 1, capacity=100000)
    out, lse = _run(dm3, wide, q)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = dm3.ops.paged_attention(q.cuda(), *held(dev), dev["table"][:, :0], dev["lengths"], dev["status"])
    assert (out == 0).all() and (lse == -math.inf).all() and int(dev["status"]) == 0


@pytest.mark.parametrize("quant", [False, True])
def test_sharp_and_shifted_logits(dm3, quant):
    """One token far above the others, early or late; all logits equal; a large common offset; logits of both signs
    whose exp leaves fp32's range; a negative and a zero scale; value rows of very different sizes."""
    dim, n = 128, 300
    base = paged([n] * 6, 1, dim, 32, False, 2)
    k = base["k"].float()
    row = lambda r, t: (int(base["table"][r, t // 32]), 0, t % 32)  # noqa: E731
    q = _q(6, 8, dim, 5).float()
    for r, t in ((0, 3), (1, n - 1)):
        k[row(r, t)] = q[r, 0] * 3
    for t in range(n):
        k[row(2, t)] = k[row(2, 0)]
        k[row(3, t)] = k[row(3, t)] + q[3, 1] * 5
        k[row(4, t)] = k[row(4, t)] * 60
    v = base["v"].float() * torch.exp2(torch.randint(-60, 40, base["v"].shape[:3], generator=torch.Generator().manual_seed(1)).float())[..., None]
    base["k"], base["v"] = k.to(BF), v.to(BF)
    if quant:
        hole = base["k"].isnan().all(-1)
        for name in ("k", "v"):
            x, e = kv_oracle.quantise(base[name].nan_to_num(0.0))
            base[name] = (x * torch.exp2(-e.double())[..., None]).float().to(torch.float8_e4m3fn)
            base[name].view(torch.uint8)[hole] = 0x7F
            base[name + "_exp"] = e
    q = q.to(BF)
    for scale in (None, 1.0, -0.3, 0.0):
        check_attention(*_run(dm3, base, q, scale), base, q, scale)


def test_queries_of_extreme_size(dm3):
    """Queries near the ends of bf16's range: only the products with the scale have to be in range."""
    for quant in (False, True):
        d = paged([50, 33], 1, 64, 16, quant, 6)
        for size in (2.0**100, 2.0**-100):
            q = _q(2, 4, 64, 7, size)
            check_attention(*_run(dm3, d, q, 1.0 / size), d, q, 1.0 / size)


def test_value_rows_of_extreme_size(dm3):
    """Quantised value rows whose exponents lie at either end, alone and mixed, short and long: weights and sums stay in range."""
    for lengths in ([700, 20000], [33, 64, 1]):
        d = paged(lengths, 1, 64, 16, True, 8)
        q = _q(len(lengths), 4, 64, 2, 2.0)
        e = d["v_exp"].clone()
        for low, high in ((-110, -110), (119, 119), (-110, 119)):
            d["v_exp"] = torch.where(torch.rand(e.shape, generator=torch.Generator().manual_seed(1)) < 0.9, low, high).to(torch.int8)
            out, lse = _run(dm3, d, q)
            scale = 2.0 ** -max(low, high)  # the check's absolute floor is far from these values
            d["v_exp"] = (d["v_exp"].int() - max(low, high)).clamp(min=-128).to(torch.int8)
            # 448 * 2^119 is the largest value a cache holds; a sum of weights of one cannot exceed it
            check_attention(out.double() * scale, lse, d, q)


def test_bad_pages_and_lengths(dm3):
    """Tokens of a page outside the cache are left out and reported, a length behind the table is cut and reported."""
    for quant in (False, True):
        d = paged([100, 64], 2, 64, 16, quant, 4)
        q = _q(2, 4, 64, 4)
        for page in (-1, d["k"].shape[0], 2**31 - 1):
            d["table"][0, 2] = page
            dev = to_cuda(d)
            out, lse = dm3.ops.paged_attention(q.cuda(), *held(dev), dev["table"], dev["lengths"], dev["status"])
            assert int(dev["status"]) == 4
            check_attention(out, lse, d, q)
        for capacity in (112, 100000):
            d = paged([0, 100, 40], 2, 64, 16, quant, 4, capacity=capacity)
            dev = to_cuda(d)
            dev["table"] = dev["table"].clone()
            full = dev["table"].shape[1] * 16
            dev["table"][0] = dev["table"][1, 0]  # a row with pages to the end, and a length behind them
            dev["lengths"][0] = full + 1
            out, lse = dm3.ops.paged_attention(q[:1].expand(3, -1, -1).cuda(), *held(dev), dev["table"], dev["lengths"], dev["status"])
            assert int(dev["status"]) == 4
            d["table"], d["lengths"] = dev["table"].cpu(), torch.tensor([full, 100, 40])
            check_attention(out, lse, d, q[:1].expand(3, -1, -1))
        d = paged([100, 112], 2, 64, 16, quant, 4)
        d["lengths"][1] = 1 << 41
        dev = to_cuda(d)
        out, lse = dm3.ops.paged_attention(q.cuda(), *held(dev), dev["table"], dev["lengths"], dev["status"])
        assert int(dev["status"]) == 4
        d["lengths"][1] = 112
        check_attention(out, lse, d, q)
        d["lengths"][1] = -5
        out, lse = _run(dm3, d, q)
        d["lengths"][1] = 0
        check_attention(out, lse, d, q)


def test_strided_queries_and_narrow_tables(dm3):
    d = paged([70, 40, 12], 2, 64, 16, False, 9, capacity=400)
    whole = _q(3, 12, 64, 2)
    dev = to_cuda(d)
    wd = whole.cuda()
    for q, qd in ((whole[:, 2:6], wd[:, 2:6]), (whole[:, ::3], wd[:, ::3]), (whole[:, :1].expand(3, 4, 64), wd[:, :1].expand(3, 4, 64)),
                  (whole.view(3, 24, 32)[:, 1:9].reshape(3, 4, 64), wd.view(3, 24, 32)[:, 1:9].reshape(3, 4, 64))):
        for cols in (5, 9, 25):
            out, lse = dm3.ops.paged_attention(qd, *held(dev), dev["table"][:, :cols], dev["lengths"], dev["status"])
            check_attention(out, lse, d, q)
    odd = torch.empty(3 * 4 * 64 + 1, dtype=BF, device="cuda")[1:].view(3, 4, 64).copy_(wd[:, :4])
    out, lse = dm3.ops.paged_attention(odd, *held(dev), dev["table"], dev["lengths"], dev["status"])
    check_attention(out, lse, d, whole[:, :4])
    assert int(dev["status"]) == 0


def test_same_answer_every_time(dm3):
    d = paged([5000, 37, 2048, 900], 2, 128, 32, False, 12)
    q = _q(4, 8, 128, 1)
    first = _run(dm3, d, q)
    for _ in range(5):
        again = _run(dm3, d, q)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_shared_pages(dm3):
    """Two rows whose tables share a prefix's pages."""
    d = paged([64, 64], 1, 64, 16, True, 12)
    d["table"][1, :2] = d["table"][0, :2]
    q = _q(2, 2, 64, 1)
    check_attention(*_run(dm3, d, q), d, q)


@pytest.mark.parametrize("quant", [False, True])
def test_frames_together(dm3, quant):
    """Prompt reading (rotate, cache, read back), then decode frames (rotate, cache, attend) from one captured graph,
    with pages reserved between replays, against the oracle on the same tokens."""
    g = torch.Generator().manual_seed(20)
    rows, kv, qh, dim, rot, size, layers = 2, 2, 8, 128, 32, 16, 2
    prompt, frames = [37, 21], 30
    rope = dm3.Rope(rot, 1e5)
    cache = dm3.KVCache(layers, rows, 128, kv, dim, page_size=size, quantised=quant)
    total = sum(prompt)
    row = torch.cat([torch.full((n,), r) for r, n in enumerate(prompt)])
    pos = torch.cat([torch.arange(n) for n in prompt])
    hist = {(layer, r): ([], []) for layer in range(layers) for r in range(rows)}

    def remember(layer, k, v, rows_, pos_):
        kr = kv_oracle.rope(k, pos_, rope.inv_freq.cpu(), False, 1.0).to(BF)
        for i, r in enumerate(rows_.tolist()):
            for x, to in zip((kr[i], v[i]), hist[layer, r]):
                to.append(kv_oracle.quantise(x)[0] if quant else x.double())

    for r, n in enumerate(prompt):
        cache.reserve(r, n)
    for layer in range(layers):
        qkv = torch.randn(total, qh + 2 * kv, dim, generator=g).to(BF)
        q, k, v = qkv.cuda().split([qh, kv, kv], 1)
        cache.write(layer, k, v, pos.cuda(), row.cuda(), q, rope)
        remember(layer, *qkv.split([qh, kv, kv], 1)[1:], row, pos)
        rk, rv = cache.read(layer, torch.tensor(prompt).cuda(), max(prompt))
        for r, n in enumerate(prompt):
            want = torch.stack(hist[layer, r][0], 1)
            # a bf16 key may be the neighbour of the oracle's rounding; a quantised one is exact
            assert (rk[r, :, :n].double().cpu() - want).abs().max() <= (0 if quant else want.abs().max() * 2.0**-7)
            assert torch.equal(rv[r, :, :n].double().cpu(), torch.stack(hist[layer, r][1], 1))

    position = torch.tensor(prompt, device="cuda")
    inputs = [torch.zeros(rows, qh + 2 * kv, dim, dtype=BF, device="cuda") for _ in range(layers)]

    def frame():
        outs = []
        lengths = position + 1
        for layer in range(layers):
            q, k, v = inputs[layer].split([qh, kv, kv], 1)
            q = cache.write(layer, k, v, position, None, q, rope)
            outs.append((q, *cache.attend(layer, q, lengths)))
        return outs

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for r, n in enumerate(prompt):
        cache.reserve(r, n + 1)
    with torch.cuda.stream(side):
        frame()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = frame()
    for f in range(frames):
        for r, n in enumerate(prompt):
            cache.reserve(r, n + f + 1)
        now = torch.tensor([n + f for n in prompt])
        position.copy_(now)
        fresh = [torch.randn(rows, qh + 2 * kv, dim, generator=g).to(BF) for _ in range(layers)]
        for to, x in zip(inputs, fresh):
            to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for layer in range(layers):
            remember(layer, *fresh[layer].split([qh, kv, kv], 1)[1:], torch.arange(rows), now)
            if f % 7 and f != frames - 1:
                continue
            q, out, lse = (x.double().cpu() for x in outs[layer])
            for r in range(rows):
                k, v = (torch.stack(x, 1) for x in hist[layer, r])
                for h in range(qh):
                    s = k[h // 4] @ q[r, h] * dim ** -0.5
                    want = s.softmax(-1) @ v[h // 4]
                    # a bf16 key off by one step moves a logit by 2^-7 of scale * sum |q k| at most (part of rot only);
                    # that is the tolerance's larger part for the bf16 cache, the operators' own rounding for e4m3
                    off = 0.0 if quant else float((q[r, h, :rot].abs() @ k[h // 4][:, :rot].abs().T).max()) * dim ** -0.5 * 2.0**-7
                    spread = s.softmax(-1) @ v[h // 4].abs()
                    assert ((out[r, h] - want).abs() <= want.abs() * 2.0**-8 + spread * (2 * off + 2.0**-10)).all()
                    assert abs(float(lse[r, h] - s.logsumexp(-1))) <= off + 1e-4
    assert cache.check() == 0
    assert torch.equal(cache.table[0, :5].cpu() >= 0, torch.ones(5, dtype=torch.bool))


def test_one_table_for_all_rows(dm3):
    """A table of one row expanded over all of them (stride 0): rows that read the same tokens."""
    d = paged([90], 2, 64, 16, False, 3)
    dev = to_cuda(d)
    q = _q(3, 4, 64, 1)
    n = torch.tensor([90, 40, 0])
    out, lse = dm3.ops.paged_attention(q.cuda(), *held(dev), dev["table"].expand(3, -1), n.cuda(), dev["status"])
    d["table"], d["lengths"] = d["table"].expand(3, -1).contiguous(), n
    check_attention(out, lse, d, q)
    k, _ = dm3.ops.kv_read(*held(dev), dev["table"].expand(3, -1), n.cuda(), 90, dev["status"])
    assert torch.equal(k[1, :, :40], k[0, :, :40]) and int(dev["status"]) == 0


@pytest.mark.parametrize("quant", [False, True])
def test_nan_and_infinity_that_are_seen(dm3, quant):
    """A NaN key makes its row NaN, a NaN value its column; an infinite value (bf16) its column infinite. Rows beside them
    are as they were."""
    d = paged([100, 100, 100, 100], 1, 64, 16, quant, 3)
    q = _q(4, 4, 64, 1, 0.1)
    at = lambda r, t: (int(d["table"][r, t // 16]), 0, t % 16)  # noqa: E731
    if quant:
        d["k"].view(torch.uint8)[at(1, 50)][5] = 0x7F
        d["v"].view(torch.uint8)[at(2, 50)][5] = 0x7F
    else:
        d["k"][at(1, 50)][5] = math.nan
        d["v"][at(2, 50)][5] = math.nan
        d["v"][at(3, 50)][5] = math.inf
    dev = to_cuda(d)
    out, lse = dm3.ops.paged_attention(q.cuda(), *held(dev), dev["table"], dev["lengths"], dev["status"])
    ref, rlse, _, _ = kv_oracle.attention(q, *held(d), d["table"], d["lengths"])
    out, lse = out.double().cpu(), lse.double().cpu()
    assert out[1].isnan().all() and lse[1].isnan().all()
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out == math.inf, ref == math.inf)
    ok = ref.isfinite()
    assert (out - ref)[ok].abs().max() <= ref[ok].abs().max() * 2.0**-7
    assert (lse - rlse)[rlse.isfinite()].abs().max() < 1e-4


@pytest.mark.parametrize("lengths", [[1, 3], [900, 1, 700], [20000, 5, 40], [33] * 40])
@pytest.mark.parametrize("quant", [False, True])
def test_rows_of_nan(dm3, lengths, quant):
    """Rows all of whose logits are NaN, by the query of one head or by every key: NaN in out and lse, not "nothing seen"."""
    d = paged(lengths, 1, 64, 16, quant, 3)
    q = _q(len(lengths), 4, 64, 1, 0.1)
    q[0, 2, 7] = math.nan
    n = lengths[1]
    for t in range(n):
        at = (int(d["table"][1, t // 16]), 0, t % 16)
        if quant:
            d["k"].view(torch.uint8)[at][t % 64] = 0x7F
        else:
            d["k"][at][t % 64] = math.nan
    dev = to_cuda(d)
    out, lse = dm3.ops.paged_attention(q.cuda(), *held(dev), dev["table"], dev["lengths"], dev["status"])
    ref, rlse, _, _ = kv_oracle.attention(q, *held(d), d["table"], d["lengths"])
    out, lse = out.double().cpu(), lse.double().cpu()
    assert ref[1].isnan().all() and rlse[1].isnan().all() and ref[0, 2].isnan().all() and int(ref.isnan().sum()) == 5 * 64
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(lse.isnan(), rlse.isnan())
    ok = rlse.isfinite()
    assert (out - ref)[ok].abs().max() <= ref[ok].abs().max() * 2.0**-7 and (lse - rlse)[ok].abs().max() < 1e-4


def test_captured_without_a_first_call(dm3):
    """The first call of a process's kernels may be a captured one."""
    code = """
import torch, sys
sys.path.insert(0, ".")
import drama3_b200 as dm3
c = dm3.KVCache(1, 2, 64, 1, 192, page_size=16, quantised=True)
[c.reserve(r, 64) for r in range(2)]
x = torch.randn(2, 1, 192, device="cuda").bfloat16()
pos, rope = torch.tensor([0, 0], device="cuda"), dm3.Rope(64)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    q = c.write(0, x, x, pos, None, x, rope)
    out, lse = c.attend(0, q, pos + 1)
    k, v = c.read(0, pos + 1, 4)
g.replay()
torch.cuda.synchronize()
assert torch.equal(out, v[:, :, 0]) and c.check() == 0
print("fine")
"""
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert got.stdout.strip() == "fine", got.stderr[-2000:]


def test_two_graphs_and_two_streams(dm3):
    """Two captured graphs and eager calls on several streams, all in flight at once, keep apart."""
    ds = [paged([900 + 50 * i, 333], 2, 64, 32, bool(i % 2), 30 + i) for i in range(3)]
    qs = [_q(2, 8, 64, i) for i in range(3)]
    dev = [(to_cuda(d), q.cuda()) for d, q in zip(ds, qs)]
    call = lambda i: dm3.ops.paged_attention(dev[i][1], *held(dev[i][0]), dev[i][0]["table"], dev[i][0]["lengths"], dev[i][0]["status"])  # noqa: E731
    want = [call(i) for i in range(3)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(i))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i < 2:
                    graphs[i].replay()
                else:
                    out2 = call(2)
    torch.cuda.synchronize()
    for got, w in zip([*outs, out2], want):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


@pytest.mark.parametrize("dim,group,quant", [(64, 4, True), (64, 16, True), (128, 4, False), (128, 16, True), (192, 4, False), (192, 12, True), (256, 8, True)])
@pytest.mark.parametrize("rows,row_bytes", [(2, 40 << 20), (16, 5 << 18), (400, 1 << 17)])
def test_waits_that_run_out(dm3, dim, group, quant, rows, row_bytes):
    """With the shortest limit waits run out, in every layout (equal shares, clusters, a CTA a unit) and with rings of an even and an odd
    number of units: the call ends all the same and its status says so; the calls after it have the right answer again.
    Where all copies stay ahead of the products no wait runs out and the answer is right; not over long bf16 rows, which
    wait for memory."""
    tokens = row_bytes // (dim if quant else 2 * dim)
    cache = dm3.KVCache(1, rows, tokens, 1, dim, page_size=16, quantised=quant)
    g = torch.Generator("cuda").manual_seed(dim)
    for x in (cache.k, cache.v):
        x.view(torch.uint8).random_(0, 64, generator=g)  # e4m3 below 2, bf16 below 2^-1
    for r in range(rows):
        cache.reserve(r, tokens)
    q = torch.randn(rows, group, dim, generator=g, device="cuda").to(BF)
    lengths = torch.full((rows,), tokens, device="cuda")
    want = cache.attend(0, q, lengths)
    assert cache.check() == 0 and want[0].isfinite().all() and want[1].isfinite().all()
    flush = torch.zeros(1 << 26, device="cuda")
    try:
        torch.cuda.synchronize()
        dm3.ops.set_wait_limit(1)
        ran_out = []
        for _ in range(4):
            flush += 1  # the cache's rows are not in L2
            out, lse = cache.attend(0, q, lengths)
            ran_out.append(cache.check())
            assert ran_out[-1] == 1 or ran_out[-1] == 0 and torch.equal(out, want[0]) and torch.equal(lse, want[1])
        print("status", ran_out)
        assert any(ran_out) or quant or rows > 2
    finally:
        torch.cuda.synchronize()
        dm3.ops.set_wait_limit(1_000_000_000)
    for _ in range(3):
        out, lse = cache.attend(0, q, lengths)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert cache.check() == 0


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("group", [4, 16])
@pytest.mark.parametrize("lengths,capacity,window", [([1, 17, 40, 100, 130], None, 0), ([90] * 150, 700, 0), ([90] * 150, 700, 21), ([3000, 77], 100000, 0),
                                                     ([100, 60], None, 0)])
def test_what_is_not_seen_decides_nothing(dm3, dim, group, lengths, capacity, window):
    """Equal bits whatever the places behind a row's length, before its window, and of pages that it does not have hold, and whatever
    earlier calls left in shared memory."""
    d = paged(lengths, 1, dim, 16, True, dim + group, capacity=capacity)
    if len(lengths) == 2 and lengths[0] == 100:
        d["table"][:, 0] = -1  # the first tile has no page
    hole = (d["k"].view(torch.uint8) == 0x7F).all(-1)
    dev, q = to_cuda(d), _q(len(lengths), group, dim, 3).cuda()
    if window:  # what the window leaves out
        for r, n in enumerate(lengths):
            for t in range(n - window):
                hole[int(d["table"][r, t // 16]), 0, t % 16] = True
    hole = hole.cuda()
    other = dm3.KVCache(1, 200, 500, 1, dim, page_size=16, quantised=True)
    other.table.random_(0, other.k.shape[1])
    for x in (other.k_exp, other.v_exp):
        x.random_(-110, 120)
    lens = torch.full((200,), 500, device="cuda")
    first = None
    for e in (0, 3, 127, -128, -60, 0):
        for name in ("k", "v"):
            dev[name].view(torch.uint8)[hole] = 0x7F if e else 0x11
            dev[name + "_exp"][hole] = e
        if e:
            other.attend(0, q[:1].expand(200, -1, -1), lens)
        got = dm3.ops.paged_attention(q, *held(dev), dev["table"], dev["lengths"], dev["status"], None, window)
        first = first or got
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1]), e


@pytest.mark.parametrize("tokens,rows,capacity", [(2500, 1, 0), (8000, 300, 0), (5000, 3, 200000), (600000, 1, 0)])
@pytest.mark.parametrize("low,high", [(-110, -110), (-110, 119), (119, 119), (-110, -60)])
@pytest.mark.parametrize("group", [2, 16])
def test_sums_at_the_ends_of_the_exponents(dm3, tokens, rows, capacity, low, high, group):
    """Many tokens whose logits lie just under what raises the maximum (2^8 in units of log2) above the first one's, over value rows with
    exponents at either end: a term of the sum is 2^(14 - exponent), 2^124 at -110, and thousands of them are added."""
    dim, size = 64, 16
    g = torch.Generator().manual_seed(tokens + high)
    pages = 40
    k, ke = torch.zeros(pages, 1, size, dim), torch.zeros(pages, 1, size, dtype=torch.int8)
    k[1:, :, :, 0], ke[1:] = 352.0, -6  # 352 * 2^-6 = 5.5 = 7.93 ln 2; page 0's logits are 0
    d = {"k": k.to(torch.float8_e4m3fn), "k_exp": ke, "status": torch.zeros(1, dtype=torch.int32)}
    d["v"] = (torch.randn(pages, 1, size, dim, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    pick = torch.rand(pages, 1, size, generator=g) < 0.9
    pick[0] = True
    e = torch.where(pick, low, high)
    per_row = -(-max(tokens, capacity) // size)
    table = torch.randint(1, pages, (rows, per_row), generator=g, dtype=torch.int32)
    table[:, :40] = 0  # the first steps of the warps
    d["table"], d["lengths"] = table, torch.full((rows,), tokens, dtype=torch.int64)
    q = torch.zeros(rows, group, dim)
    q[:, :, 0] = 1.0
    q = q.to(BF)
    d["v_exp"] = e.to(torch.int8)
    out, lse = _run(dm3, d, q, 1.0)
    assert out.isfinite().all() and lse.isfinite().all()
    # rows are alike: a few of them against the oracle, the values brought near 1
    d["v_exp"] = (e - max(low, high)).clamp(min=-128).to(torch.int8)
    few = {**d, "table": table[:2], "lengths": d["lengths"][:2]}
    check_attention(out[:2].double() * 2.0 ** -max(low, high), lse[:2], few, q[:2], 1.0)


@pytest.mark.parametrize("lengths", [[70, 90, 30], [3000, 40, 2000], [90] * 300])
def test_infinite_logits(dm3, lengths):
    """A logit of -inf is a token that is not seen, a row of them a row that sees nothing; one of +inf makes its head's out and lse NaN."""
    d = paged(lengths, 1, 64, 16, False, 5)
    q = _q(len(lengths), 4, 64, 6, 0.1)
    q[:, :, 3] = torch.tensor([1.0, -1.0, 0.5, -2.0]).to(BF)
    at = lambda r, t: (int(d["table"][r, t // 16]), 0, t % 16)  # noqa: E731
    for t in range(lengths[0]):
        d["k"][at(0, t)][3] = -math.inf  # heads 0 and 2 of row 0 see nothing, 1 and 3 are infinite
    d["k"][at(1, 25)][3] = -math.inf  # of row 1, heads 0 and 2 see one token less
    dev = to_cuda(d)
    out, lse = dm3.ops.paged_attention(q.cuda(), *held(dev), dev["table"], dev["lengths"], dev["status"])
    assert out[:2, 1::2].isnan().all() and lse[:2, 1::2].isnan().all()
    assert (out[0, ::2] == 0).all() and (lse[0, ::2] == -math.inf).all()
    # the rest against the oracle, the token left out by its page: a copy of row 1 without it
    n = lengths[1]
    k, _ = kv_oracle.tokens(d["k"], None, d["table"], 1, n)
    v, _ = kv_oracle.tokens(d["v"], None, d["table"], 1, n)
    keep = torch.arange(n) != 25
    for h in (0, 2):
        s = q[1, h].double() @ k[0, keep].T * 64 ** -0.5
        want = s.softmax(-1) @ v[0, keep]
        spread = s.softmax(-1) @ v[0, keep].abs()
        assert ((out[1, h].double().cpu() - want).abs() <= want.abs() * 2.0**-8 + spread * 2.0**-10).all()
        assert abs(float(lse[1, h]) - float(s.logsumexp(-1))) < 1e-4
    rest = {**d, "table": d["table"][2:], "lengths": d["lengths"][2:]}
    check_attention(out[2:], lse[2:], rest, q[2:])


@pytest.mark.parametrize("above", [0, 12, 24, 33, 60])
@pytest.mark.parametrize("lengths", [[200, 50], [20000, 300], [400] * 300])
def test_value_rows_beside_a_larger_one(dm3, above, lengths):
    """One value row 2^above times the others' size with a single value that is not 0: the other values of out come from the
    other rows alone. A weight is held to 2^-11 of it, or to 2^-31 of the row's largest (the last places of fp16 below a
    weight that is 2^6 at least): that bounds each of out's values."""
    dim = 64
    d = paged(lengths, 1, dim, 16, True, 9)
    q = _q(len(lengths), 4, dim, 2, 0.3)
    few = min(len(lengths), 3)
    for r in range(len(lengths)):
        at = (int(d["table"][r, 1]), 0, 4)
        d["v"].view(torch.uint8)[at] = 0
        d["v"][at][5] = 256.0
        d["v_exp"][at] = above
    out, lse = _run(dm3, d, q)
    out, lse = out[:few], lse[:few]
    small = {**d, "table": d["table"][:few], "lengths": d["lengths"][:few]}
    ref, rlse, spread, reach = kv_oracle.attention(q[:few], *held(small), small["table"], small["lengths"])
    floor = torch.zeros_like(ref)
    for r in range(few):
        n = lengths[r]
        k, _ = kv_oracle.tokens(d["k"], d["k_exp"], d["table"], r, n)
        page, at = d["table"][r].long()[torch.arange(n) // 16], torch.arange(n) % 16
        code, e = d["v"].double()[page, 0, at], d["v_exp"].double()[page, 0, at]
        p = (q[r].double() @ k[0].T * dim ** -0.5).softmax(-1)
        floor[r] = (p * torch.exp2(e)).amax(-1, keepdim=True) * 2.0**-31 * code.abs().sum(0)
    n, logit = max(lengths), reach * (dim / 16 + 4) * 2.0**-22
    tol = ref.abs() * 2.0**-8 + spread * (2.0**-11 + 2 * logit + (n / 16 + 8) * 2.0**-22)[..., None] + floor
    assert ((out.double().cpu() - ref).abs() <= tol).all()
    assert ((lse.double().cpu() - rlse).abs() <= logit + rlse.abs() * 2.0**-22 + (n / 16 + 8) * 2.0**-22).all()
