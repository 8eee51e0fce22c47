"""dm3::rope, dm3::kv_write and dm3::kv_read against the 64-bit oracle."""

import pytest
import torch

from oracle import kv_oracle
from tests.kv_helpers import held, paged, to_cuda

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _inv(rot, base=1e4):
    return base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)


def _near(y, x, ref, rot, factor=1.0):
    """bf16 rounding (half a step), and fp32 sines, cosines and products (a few 2^-24 of |a| + |b|, which one
    row's largest value bounds)."""
    y = y.double().cpu()
    tol = ref.abs() * 2.0**-8 + x.double().abs().amax(-1, keepdim=True) * factor * 2.0**-20 + 2.0**-133
    assert ((y - ref).abs() <= tol).all(), float(((y - ref).abs() / tol).max())
    assert torch.equal(y[..., rot:], x.double()[..., rot:])


@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 64, 64), (2, 18, 256, 64), (37, 5, 128, 128), (3, 4, 192, 96), (300, 3, 72, 36),
                                                  (5, 2, 10, 6), (2, 1, 2, 2), (700, 1, 1024, 1024), (1, 70, 40, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(dm3, tokens, heads, dim, rot, interleaved):
    g = torch.Generator().manual_seed(tokens * 7 + dim)
    x = torch.randn(tokens, heads, dim, generator=g).to(BF)
    pos = torch.randint(-50, 1 << 20, (tokens,), generator=g)
    pos[0] = 0 if tokens > 1 else 99991
    y = dm3.ops.rope(x.cuda(), pos.cuda(), _inv(rot).cuda(), interleaved, 1.25)
    assert y.shape == x.shape and y.is_contiguous()
    _near(y, x, kv_oracle.rope(x, pos, _inv(rot), interleaved, 1.25), rot, 1.25)


def test_rope_strides_and_alignment(dm3):
    g = torch.Generator().manual_seed(9)
    whole = torch.randn(21, 9, 130, generator=g).to(BF)
    pos = torch.arange(1000, 1021)
    for x in (whole[:, 2:5, :128], whole[::2, :, 1:129], whole.transpose(0, 1)[:, :, :64], whole[:, :, :128].expand(21, 9, 128),
              whole[:, :1, 2:66].expand(21, 6, 64), whole[:, :, ::2], whole[:0]):
        p = pos[:x.shape[0]] if x.shape[0] <= 21 else torch.arange(x.shape[0])
        dev = whole.cuda()
        xd = torch.as_strided(dev, x.shape, x.stride(), x.storage_offset())
        rot = 32 if x.shape[2] % 2 == 0 else 16
        y = dm3.ops.rope(xd, p.cuda(), _inv(rot).cuda())
        if x.shape[0]:
            _near(y, x, kv_oracle.rope(x, p, _inv(rot)), rot)


def test_rope_class(dm3):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(6, 3, 128, generator=g).to(BF)
    pos = torch.arange(6) + 70000
    r = dm3.Rope(64, 1e6, True, "yarn", 4.0, 32768)
    f, factor = dm3.rope_frequencies(64, 1e6, "yarn", 4.0, 32768)
    _near(r(x.cuda(), pos.cuda()), x, kv_oracle.rope(x, pos, f, True, factor), 64, factor)


def _write_case(dim, kv_heads, q_heads, size, quant, seed, spans):
    """A cache with some tokens, and new ones for the rows: (cache dict, k, v, q, rows, positions)."""
    g = torch.Generator().manual_seed(seed)
    d = paged([a + b for a, b in spans], kv_heads, dim, size, quant, seed)
    rows = torch.cat([torch.full((b,), r) for r, (a, b) in enumerate(spans)] + [torch.zeros(0)]).long()
    pos = torch.cat([torch.arange(a, a + b) for a, b in spans] + [torch.zeros(0)]).long()
    mix = torch.randperm(len(rows), generator=g)
    qkv = torch.randn(len(rows), q_heads + 2 * kv_heads, dim, generator=g)
    qkv = (qkv * torch.exp2(torch.randint(-8, 8, qkv.shape[:2], generator=g).float())[..., None]).to(BF)
    return d, qkv, rows[mix], pos[mix]


def _expect_cache(d, k, v, rows, pos, quant):
    """The caches' values after the write: float64 [pages, heads, size, dim] and exponents."""
    size = d["k"].shape[2]
    at, of = d["table"][rows, pos // size].long(), pos % size
    out = []
    for name, x in (("k", k), ("v", v)):
        val = kv_oracle.values(d[name], d[name + "_exp"])
        exp = None
        if quant:
            vals, e = kv_oracle.quantise(x)
            exp = d[name + "_exp"].clone()
            val[at, :, of], exp[at, :, of] = vals, e
        else:
            val[at, :, of] = x.double()
        out.append((val, exp))
    return out


@pytest.mark.parametrize("dim,kv_heads,q_heads,size,rot", [(64, 1, 1, 16, 64), (128, 8, 32, 32, 128), (192, 3, 6, 48, 48), (256, 2, 16, 64, 64),
                                                           (128, 5, 0, 16, 0), (64, 12, 12, 128, 32), (256, 1, 40, 16, 16)])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_kv_write(dm3, dim, kv_heads, q_heads, size, rot, quant, interleaved):
    spans = [(0, 5), (3, 0), (15, 1), (17, 30), (2 * size - 1, 2)]
    d, qkv, rows, pos = _write_case(dim, kv_heads, q_heads, size, quant, dim + kv_heads, spans)
    dev, qd = to_cuda(d), qkv.cuda()
    q, k, v = qkv.split([q_heads, kv_heads, kv_heads], 1)
    qc, kc, vc = qd.split([q_heads, kv_heads, kv_heads], 1)
    inv = _inv(rot, 1e5) if rot else None
    out = dm3.ops.kv_write(kc, vc, pos.cuda(), dev["table"], *held(dev), dev["status"], rows.cuda(), qc if q_heads else None,
                           None if inv is None else inv.cuda(), interleaved, 1.5 if rot else 1.0)
    turn = (lambda x: kv_oracle.rope(x, pos, inv, interleaved, 1.5)) if rot else (lambda x: x.double())
    if q_heads:
        _near(out, q, turn(q), rot, 1.5)
    else:
        assert out.numel() == 0
    # what lies in the cache: a bf16 key is a rounding of the rotated one, a quantised key is the exact one's code
    kr = turn(k)
    if not quant:
        size_ = d["k"].shape[2]
        got = dev["k"].cpu()[d["table"][rows, pos // size_].long(), :, pos % size_]
        _near(got, k, kr, rot, 1.5)
        kr = got
    for name, (val, exp) in zip(("k", "v"), _expect_cache(d, kr.to(BF), v, rows, pos, quant)):
        now = kv_oracle.values(dev[name].cpu(), None if exp is None else dev[name + "_exp"].cpu())
        assert torch.equal(now.nan_to_num(1e30), val.nan_to_num(1e30)), name  # every other place as it was, poison included
        if quant:
            assert torch.equal(dev[name + "_exp"].cpu(), exp)
    assert int(dev["status"]) == 0


@pytest.mark.parametrize("tokens", [700, 4800, 9001])
@pytest.mark.parametrize("quant", [False, True])
def test_many_tokens(dm3, tokens, quant):
    """Enough tokens for blocks of several a CTA, the last one cut short: every one where it belongs."""
    dim, size = 64, 16
    g = torch.Generator().manual_seed(tokens)
    c = dm3.KVCache(1, 3, tokens, 1, dim, page_size=size, quantised=quant)
    c.reserve(1, tokens)
    x = torch.randn(tokens, 5, dim, generator=g).to(BF)
    q, k, v = x.split([3, 1, 1], 1)
    xd = x.cuda()
    pos = torch.randperm(tokens, generator=g)
    rope = dm3.Rope(32, 1e5, True)
    out = c.write(0, xd[:, 3:4], xd[:, 4:], pos.cuda(), torch.ones(tokens, dtype=torch.int64).cuda(), xd[:, :3], rope)
    inv = rope.inv_freq.cpu()
    _near(out, q, kv_oracle.rope(q, pos, inv, True), 32)
    _near(rope(xd, pos.cuda()), x, kv_oracle.rope(x, pos, inv, True), 32)
    rk, rv = c.read(0, torch.tensor([0, tokens, 0]).cuda(), tokens)
    kr = kv_oracle.rope(k, pos, inv, True)[:, 0]
    if quant:
        assert torch.equal(rk[1, 0].double().cpu()[pos], kv_oracle.quantise(kr.to(BF))[0])
        assert torch.equal(rv[1, 0].double().cpu()[pos], kv_oracle.quantise(v[:, 0])[0])
    else:
        _near(rk[1].transpose(0, 1)[pos.cuda()], k, kr[:, None], 32)
        assert torch.equal(rv[1, 0].cpu()[pos], v[:, 0])
    assert (rk[0] == 0).all() and (rk[2] == 0).all() and c.check() == 0


@pytest.mark.parametrize("dim,kv_heads,q_heads,rot", [(64, 1, 3, 64), (128, 2, 5, 96), (192, 1, 2, 48), (256, 1, 0, 256)])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_one_call_and_many(dm3, dim, kv_heads, q_heads, rot, quant, interleaved):
    """Tokens of one long call, padding among them, get the bits that they get in short calls."""
    tokens, step = 6113, 1201
    g = torch.Generator().manual_seed(dim)
    rows, pos = torch.randint(0, 2, (tokens,), generator=g), torch.randperm(tokens, generator=g)
    rows[torch.randperm(tokens, generator=g)[:57]] = -1
    x = torch.randn(tokens, q_heads + 2 * kv_heads, dim, generator=g).to(BF).cuda()
    q, k, v = x.split([q_heads, kv_heads, kv_heads], 1)
    rope, rows, pos = dm3.Rope(rot, 1e4, interleaved), rows.cuda(), pos.cuda()
    one, many = (dm3.KVCache(1, 2, tokens, kv_heads, dim, quantised=quant) for _ in range(2))
    for c in (one, many):
        c.reserve(0, tokens), c.reserve(1, tokens)
    full = torch.full((2,), tokens).cuda()
    out = one.write(0, k, v, pos, rows, q if q_heads else None, rope)
    parts = [many.write(0, k[a:a + step], v[a:a + step], pos[a:a + step], rows[a:a + step], q[a:a + step] if q_heads else None, rope)
             for a in range(0, tokens, step)]
    assert torch.equal(out, torch.cat(parts)) and one.check() == 0 and many.check() == 0
    seen = torch.zeros(2, tokens, dtype=torch.bool, device="cuda")
    seen[rows[rows >= 0], pos[rows >= 0]] = True
    for a, b in zip(one.read(0, full, tokens), many.read(0, full, tokens)):
        a, b = a.transpose(1, 2)[seen], b.transpose(1, 2)[seen]
        assert a.isfinite().all() and torch.equal(a, b)
    if q_heads:
        assert (out[rows < 0] == 0).all()


def test_traced_calls_are_the_same(dm3):
    """Under torch.compile the ops are traced as operators, with the same results and the same writes."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 8, 64, generator=g).to(BF).cuda()
    rope = dm3.Rope(64, device="cuda")
    pos = torch.tensor([17, 4]).cuda()

    def frame(cache, x, pos):
        q = cache.write(0, x[:, :2], x[:, 2:4], pos, None, x[:, 4:], rope)
        out, lse = cache.attend(0, q, pos + 1)
        k, v = cache.read(0, pos + 1, 20)
        return rope(q, pos), out, lse, k, v

    got = []
    for traced in (False, True):
        cache = dm3.KVCache(1, 2, 32, 2, 64, page_size=16, quantised=True)
        for r in range(2):
            cache.reserve(r, 32)
        fn = torch.compile(frame, backend="aot_eager", dynamic=False, fullgraph=True) if traced else frame
        got.append([*fn(cache, x, pos), cache.k.view(torch.uint8).clone(), cache.v_exp.clone()])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_gradients_are_refused(dm3):
    """No operator here has a gradient: one that is asked for is an error, not a silent zero."""
    x = torch.randn(2, 1, 64, dtype=BF, device="cuda", requires_grad=True)
    y = dm3.Rope(64)(x, torch.arange(2).cuda())
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_kv_write_extremes(dm3):
    """Rows of zeros, one huge value, the largest and smallest bf16, subnormals, infinities and NaN; ties."""
    dim = 64
    rows = torch.zeros(12, 1, dim)
    rows[1, 0, 3] = 1.0
    rows[2, 0, :] = torch.finfo(BF).max
    rows[3, 0, :2] = torch.tensor([1.0, 2.0**-126])
    rows[4, 0, :] = 2.0**-130
    rows[5, 0, :4] = torch.tensor([float("inf"), 1.0, -float("inf"), 3.0])
    rows[6, 0, :3] = torch.tensor([float("nan"), -5.0, 0.1])
    rows[7, 0, :] = float("nan")
    rows[8, 0, :] = torch.linspace(-448, 448, dim)
    rows[9, 0, :6] = torch.tensor([1.0625, 1.1875, 1.3125, 448.0, -1.0625, 2.0**-10 * 3])  # half way between two codes
    rows[10, 0, :2] = torch.tensor([449.0, 0.0])
    rows[11, 0, 0] = -0.0
    x = rows.to(BF)
    c = dm3.KVCache(1, 1, 12, 1, dim, page_size=16, quantised=True)
    c.reserve(0, 12)
    c.write(0, x.cuda(), x.flip(-1).contiguous().cuda(), torch.arange(12).cuda(), torch.zeros(12, dtype=torch.int64).cuda())
    k, v = c.read(0, torch.tensor([12]).cuda(), 12)
    val, e = kv_oracle.quantise(x[:, 0])
    page = int(c.table[0, 0])
    assert torch.equal(c.k_exp[0, page, 0, :12].cpu(), e) and torch.equal(c.v_exp[0, page, 0, :12].cpu(), e)
    assert torch.equal(k[0, 0].double().cpu().nan_to_num(1e30), val.nan_to_num(1e30))
    assert torch.equal(v[0, 0].double().cpu().nan_to_num(1e30), val.flip(-1).nan_to_num(1e30))
    assert k[0, 0, :5].isfinite().all() and c.check() == 0


def test_kv_write_padding_and_bad_places(dm3):
    """Padding tokens (negative row or position) and tokens whose row, position or page does not exist are not cached;
    the latter are reported."""
    d = paged([20, 20], 2, 64, 16, False, 5)  # the table has 2 pages a row
    g = torch.Generator().manual_seed(1)
    k, v, q = (torch.randn(8, h, 64, generator=g).to(BF).cuda() for h in (2, 2, 4))
    for rows, pos, bad in (([0, -1, 1], [3, 4, -9], 0), ([0, 2], [0, 0], 4), ([0, 1 << 40], [0, 0], 4), ([1, 0], [0, 32], 4),
                           ([1, 0], [0, 1 << 62], 4)):
        dev, n = to_cuda(d), len(rows)
        out = dm3.ops.kv_write(k[:n], v[:n], torch.tensor(pos).cuda(), dev["table"], *held(dev), dev["status"],
                               torch.tensor(rows).cuda(), q[:n])
        want = d["k"].clone()
        page = int(d["table"][rows[0], pos[0] // 16])
        want[page, :, pos[0] % 16] = k[0].cpu()
        assert torch.equal(dev["k"].cpu().nan_to_num(9.0), want.nan_to_num(9.0))
        assert int(dev["status"]) == bad
        for i in range(n):
            padding = rows[i] < 0 or pos[i] < 0
            assert torch.equal(out[i], torch.zeros_like(q[i]) if padding else q[i])
    for page in (-1, d["k"].shape[0], 2**31 - 1, -(2**31)):
        dev = to_cuda(d)
        dev["table"][0, 1] = page
        dm3.ops.kv_write(k[:1], v[:1], torch.tensor([17]).cuda(), dev["table"], *held(dev), dev["status"])
        assert int(dev["status"]) == 4 and torch.equal(dev["k"].cpu().nan_to_num(9.0), d["k"].nan_to_num(9.0))


@pytest.mark.parametrize("dim,kv_heads,size", [(64, 1, 16), (128, 8, 32), (192, 3, 48), (256, 2, 64)])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("longest", [1, 67, 700])
def test_kv_read(dm3, dim, kv_heads, size, quant, longest):
    lengths = [longest, 0, 1, min(size, longest), longest - 1]
    d = paged(lengths, kv_heads, dim, size, quant, longest)
    dev = to_cuda(d)
    for L in (longest, longest + 5, max(1, longest // 2), 0):
        k, v = dm3.ops.kv_read(*held(dev), dev["table"], dev["lengths"], L, dev["status"])
        assert k.shape == v.shape == (5, kv_heads, L, dim)
        for name, x in (("k", k), ("v", v)):
            want = torch.zeros(5, kv_heads, L, dim, dtype=torch.float64)
            for r, n in enumerate(lengths):
                n = min(n, L)
                if n:
                    want[r, :, :n] = kv_oracle.tokens(d[name], d[name + "_exp"], d["table"], r, n)[0]
            assert torch.equal(x.double().cpu(), want)
    assert int(dev["status"]) == 0


def test_kv_read_bad_pages(dm3):
    d = paged([40, 33], 1, 64, 16, False, 2)
    dev = to_cuda(d)
    dev["table"][0, 1] = d["k"].shape[0]
    k, _ = dm3.ops.kv_read(*held(dev), dev["table"], dev["lengths"], 48, dev["status"])
    assert int(dev["status"]) == 4 and (k[0, 0, 16:32] == 0).all() and k.isfinite().all()
    dev = to_cuda(d)
    dev["lengths"] = torch.tensor([1 << 40, -3]).cuda()
    dev["table"].clamp_(min=0)
    k, _ = dm3.ops.kv_read(*held(dev), dev["table"], dev["lengths"], 16, dev["status"])
    assert int(dev["status"]) == 4 and torch.equal(k[0].cpu(), kv_oracle.tokens(d["k"], None, d["table"], 0, 16)[0].to(BF))
    assert (k[1] == 0).all()


def test_layers_of_one_buffer(dm3):
    """A cache whose pages hold all layers ([pages, layers, ...]): pages are strided, layers do not touch each other."""
    for quant in (False, True):
        d = paged([30], 2, 64, 16, quant, 8)
        wide = {n: None if d[n] is None else torch.stack([d[n], d[n]], 1).cuda() for n in ("k", "v", "k_exp", "v_exp")}
        one = [None if wide[n] is None else wide[n][:, 1] for n in ("k", "v", "k_exp", "v_exp")]
        t, s, n = d["table"].cuda(), d["status"].cuda(), d["lengths"].cuda()
        x = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(0)).to(BF)
        dm3.ops.kv_write(x.cuda(), x.cuda(), torch.tensor([29]).cuda(), t, *one, s)
        k, _ = dm3.ops.kv_read(*one, t, n, 30, s)
        want = kv_oracle.quantise(x[0])[0] if quant else x[0].double()
        assert torch.equal(k[0, :, 29].double().cpu(), want)
        assert torch.equal(wide["k"][:, 0].cpu().view(torch.uint8), d["k"].view(torch.uint8))  # layer 0 as it was


def test_op_refusals(dm3):
    d = to_cuda(paged([20, 20], 2, 64, 16, False, 5))
    e = to_cuda(paged([20, 20], 2, 64, 16, True, 5))
    k = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
    pos, inv = torch.zeros(2, dtype=torch.int64, device="cuda"), _inv(32).cuda()
    ops, t, s, n = dm3.ops, d["table"], d["status"], d["lengths"]

    def refused(fn, *a, **kw):
        with pytest.raises(RuntimeError):
            fn(*a, **kw)

    refused(ops.rope, k.float(), pos, inv)
    refused(ops.rope, k[0], pos, inv)
    refused(ops.rope, k, pos.int(), inv)
    refused(ops.rope, k, pos[:1], inv)
    refused(ops.rope, k, pos, inv.float())
    refused(ops.rope, k, pos, torch.ones(33, dtype=torch.float64, device="cuda"))
    refused(ops.rope, k, pos.cpu(), inv)
    for c in ((d["k"], d["v"].float(), None, None), (d["k"].float(), d["v"].float(), None, None), (d["k"], d["v"], e["k_exp"], e["v_exp"]),
              (e["k"], e["v"], None, None), (e["k"], e["v"], e["k_exp"], None), (e["k"], e["v"], e["k_exp"], e["v_exp"].int()),
              (d["k"][:, :1], d["v"], None, None), (d["k"].transpose(1, 2), d["v"].transpose(1, 2), None, None),
              (d["k"][..., :32], d["v"][..., :32], None, None)):
        refused(ops.kv_write, k, k, pos, t, *c, s)
        refused(ops.kv_read, *c, t, n, 4, s)
        refused(ops.paged_attention, k, *c, t, n, s)
    c = held(d)
    refused(ops.kv_write, k[:, :1], k[:, :1], pos, t, *c, s)
    refused(ops.kv_write, k, k[:, :, :32], pos, t, *c, s)
    refused(ops.kv_write, k, k, pos[:1], t, *c, s)
    refused(ops.kv_write, k, k, pos, t.long(), *c, s)
    refused(ops.kv_write, k, k, pos, t[0], *c, s)
    refused(ops.kv_write, k, k, pos, t, *c, s.long())
    refused(ops.kv_write, k, k, pos, t, *c, s, pos.int())
    refused(ops.kv_write, k, k, pos, t, *c, s, None, k[:1])
    refused(ops.kv_write, k, k, pos, t, *c, s, None, k, _inv(24).cuda())
    refused(ops.kv_read, *c, t, n, -1, s)
    refused(ops.kv_read, *c, t, n[:1], 4, s)
    refused(ops.paged_attention, k[:, :1], *c, t, n, s)
    refused(ops.paged_attention, k[:1], *c, t, n, s)
    refused(ops.paged_attention, k.float(), *c, t, n, s)
    refused(ops.paged_attention, k, *c, t, n.int(), s)
    refused(ops.paged_attention, k, *c, t, n, s, None, -1)
    refused(ops.paged_attention, k, *c, t, n, s, float("nan"))
    refused(ops.paged_attention, k, *c, t.cpu(), n, s)
