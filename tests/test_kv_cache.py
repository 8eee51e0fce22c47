"""The paged cache and rotary positions without a GPU: the frequencies, the page bookkeeping, the oracle's
quantiser against torch's own e4m3 conversion, shapes under tracing, and every refusal of the C entries and
the ops (arguments are checked before any device work)."""

import copy
import ctypes
import math

import pytest
import torch

from oracle import kv_oracle

BF = torch.bfloat16
P = ctypes.c_void_p(256)  # a non-null, aligned pointer that no refused call reads


def test_oracle_quantiser_is_e4m3_of_a_power_of_two():
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(40, 64, generator=g) * torch.exp2(torch.randint(-30, 30, (40, 1), generator=g).float())).to(BF)
    x[3] = 0
    x[4, 5] = math.inf
    x[5, 6] = math.nan
    v, e = kv_oracle.quantise(x)
    scale = torch.exp2(e.double())[:, None]
    ref = (x.double() / scale).float().to(torch.float8_e4m3fn).double() * scale
    ref[~x.isfinite()] = math.nan
    assert torch.equal(v.nan_to_num(7.0), ref.nan_to_num(7.0)) and int(e[3]) == 0
    top = torch.where(x.isfinite(), x.double().abs(), 0.0).amax(-1)
    busy = top > 0
    assert (top[busy] <= 448 * scale[busy, 0]).all() and (top[busy] > 224 * scale[busy, 0]).all()
    # a half step of e4m3 at most (2^-4 of the value, or half of the smallest code's step)
    ok = x.isfinite()
    assert ((v - x.double()).abs()[ok] <= torch.maximum(x.double().abs() / 16, 2.0**-10 * scale.expand_as(v))[ok]).all()


def test_frequencies(dm3):
    f, factor = dm3.rope_frequencies(64, 1e6)
    assert f.dtype == torch.float64 and factor == 1.0 and f[0] == 1.0
    assert torch.allclose(f, torch.tensor([1e6 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    lin, _ = dm3.rope_frequencies(64, 1e6, "linear", 4.0)
    assert torch.equal(lin, f / 4)
    ntk, _ = dm3.rope_frequencies(64, 1e6, "ntk", 4.0)
    assert ntk[0] == 1.0 and abs(float(ntk[-1] / f[-1]) - 0.25) < 1e-12  # the slowest pair is slowed by stretch
    yarn, factor = dm3.rope_frequencies(64, 1e6, "yarn", 4.0, 32768)
    turns = 32768 * f / (2 * math.pi)
    assert torch.equal(yarn[turns > 32], f[turns > 32]) and torch.equal(yarn[turns < 1], f[turns < 1] / 4)
    assert ((yarn <= f) & (yarn >= f / 4)).all() and abs(factor - (0.1 * math.log(4) + 1)) < 1e-15
    assert dm3.rope_frequencies(2, 100.0, "ntk", 2.0)[0].tolist() == [1.0]
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="cubic"), dict(rotary_dim=8, base=0.0),
                dict(rotary_dim=8, scaling="yarn", stretch=2.0), dict(rotary_dim=8, stretch=0.5)):
        with pytest.raises(ValueError):
            dm3.rope_frequencies(**bad)


def test_pages_are_reserved_and_released(dm3):
    c = dm3.KVCache(layers=2, rows=3, tokens_per_row=100, kv_heads=2, head_dim=64, page_size=16, pages=9, device="cpu")
    assert c.pages_per_row == 7 and c.k.shape == (2, 9, 2, 16, 64) and c.k_exp is None
    assert (c.table == -1).all()
    c.reserve(0, 33)
    first = c.table[0, :3].tolist()
    c.reserve(0, 48)  # the third page has room
    assert c.table[0, :4].tolist() == first + [-1]
    c.reserve(1, 96)
    assert len(set(first) | set(c.table[1, :6].tolist())) == 9
    before = c.table.clone()
    with pytest.raises(RuntimeError, match="free"):
        c.reserve(2, 1)
    with pytest.raises(RuntimeError, match="more than its 7 pages"):
        c.reserve(0, 113)
    assert torch.equal(c.table, before)
    c.release(0)
    assert (c.table[0] == -1).all()
    c.reserve(2, 40)
    assert sorted(c.table[2, :3].tolist()) == sorted(first)
    c.reserve(2, 0)
    for bad in (dict(page_size=24), dict(page_size=8), dict(head_dim=96), dict(kv_heads=0), dict(pages=0)):
        with pytest.raises(ValueError):
            dm3.KVCache(**{**dict(layers=1, rows=1, tokens_per_row=10, kv_heads=1, head_dim=64, device="cpu"), **bad})


def _meta_cache(quant, pages=5, heads=2, size=16, dim=64, device="meta"):
    k = torch.empty(pages, heads, size, dim, dtype=torch.float8_e4m3fn if quant else BF, device=device)
    e = torch.empty(pages, heads, size, dtype=torch.int8, device=device) if quant else None
    return k, torch.empty_like(k), e, None if e is None else torch.empty_like(e)


@pytest.mark.parametrize("quantised", [False, True])
def test_layers_are_views_of_the_buffers(dm3, quantised):
    c = dm3.KVCache(3, 2, 40, 2, 64, page_size=16, quantised=quantised, device="cpu")
    for cache in (c, copy.deepcopy(c)):
        for i in range(-3, 3):
            for view, buffer in zip(cache.layer(i), (cache.k, cache.v, cache.k_exp, cache.v_exp)):
                if buffer is None:
                    assert view is None and not quantised
                else:
                    assert view.data_ptr() == buffer[i].data_ptr() and view.shape == buffer.shape[1:] and view.stride() == buffer[i].stride()
    with pytest.raises(IndexError):
        c.layer(3)
    with pytest.raises(AttributeError):
        c.k = c.k.clone()


def test_fake_impls_trace_on_meta(dm3):
    m = dict(device="meta")
    pos, inv = torch.empty(3, dtype=torch.int64, **m), torch.empty(16, dtype=torch.float64, **m)
    table, status = torch.empty(3, 4, dtype=torch.int32, **m), torch.empty(1, dtype=torch.int32, **m)
    x = torch.empty(3, 8, 64, dtype=BF, **m)
    assert torch.ops.dm3.rope(x, pos, inv).shape == x.shape
    for quant in (False, True):
        c = _meta_cache(quant)
        k = torch.empty(3, 2, 64, dtype=BF, **m)
        assert torch.ops.dm3.kv_write(k, k, pos, table, *c, status).shape == (0,)
        assert torch.ops.dm3.kv_write(k, k, pos, table, *c, status, None, x, inv).shape == x.shape
        rk, rv = torch.ops.dm3.kv_read(*c, table, pos, 33, status)
        assert rk.shape == rv.shape == (3, 2, 33, 64) and rk.dtype == BF
        out, lse = torch.ops.dm3.paged_attention(x, *c, table, pos, status)
        assert out.shape == x.shape and out.dtype == BF and lse.shape == (3, 8) and lse.dtype == torch.float32


def test_ops_refuse_cpu_tensors(dm3):
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        dm3.ops.rope(torch.zeros(1, 1, 64, dtype=BF), torch.zeros(1, dtype=torch.int64), torch.ones(32, dtype=torch.float64))
    c = dm3.KVCache(1, 1, 16, 1, 64, device="cpu")
    n = torch.ones(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        c.attend(0, torch.zeros(1, 1, 64, dtype=BF), n)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        c.read(0, n, 4)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        c.write(0, torch.zeros(1, 1, 64, dtype=BF), torch.zeros(1, 1, 64, dtype=BF), n)


def test_ops_refuse_counts_beyond_32_bits(dm3, monkeypatch):
    """Counts that a C int would cut short; the tensors are expanded views of one element or row."""
    ops, many = dm3.ops, 2**32 + 1
    monkeypatch.setattr(ops, "_same_device", lambda *a: 0)
    monkeypatch.setattr(ops, "_launch", lambda *a: pytest.fail("launched"))
    inv, zero = torch.ones(32, dtype=torch.float64), torch.zeros(1, dtype=torch.int64)
    k, c = torch.zeros(1, 1, 64, dtype=BF), torch.zeros(1, 1, 16, 64, dtype=BF)
    t, s = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for bad in (
        lambda: ops.rope(k.expand(many, 1, 64), zero.expand(many), inv),
        lambda: ops.rope(k.expand(1, many, 64), zero, inv),
        lambda: ops.kv_write(k.expand(many, 1, 64), k.expand(many, 1, 64), zero.expand(many), t, c, c, None, None, s),
        lambda: ops.kv_read(c, c, None, None, t.expand(many, 1), zero.expand(many), 0, s),
        lambda: ops.paged_attention(k, c.expand(many, 1, 16, 64), c.expand(many, 1, 16, 64), None, None, t, zero, s),
    ):
        with pytest.raises(RuntimeError, match="at most|bad head"):
            bad()


# What each C entry is called with, by name; a refusal test changes one of them.
_CACHE = dict(k_cache=P, v_cache=P, page_stride=2 * 16 * 64, k_exp=None, v_exp=None, exp_stride=0, pages=5, page_size=16)
_TABLE = dict(table=P, table_stride=4, table_rows=3, per_row=4)
CALLS = {
    "dm3_rope": dict(x=P, T=3, heads=2, dim=64, ts=128, hs=64, positions=P, inv_freq=P, rot=32, interleaved=0, factor=1.0, y=P, stream=None),
    "dm3_kv_write": dict(q=P, q_heads=4, q_ts=256, q_hs=64, k=P, k_ts=128, k_hs=64, v=P, v_ts=128, v_hs=64, T=3, kv_heads=2, dim=64, rows=None,
                         positions=P, **_TABLE, **_CACHE, inv_freq=P, rot=32, interleaved=0, factor=1.0, q_out=P, status=P, stream=None),
    "dm3_kv_read": dict(**_CACHE, kv_heads=2, dim=64, **_TABLE, lengths=P, max_length=40, k_out=P, v_out=P, status=P, stream=None),
    "dm3_paged_attention": dict(q=P, q_rs=256, q_hs=64, q_heads=4, **_CACHE, kv_heads=2, dim=64, **_TABLE, lengths=P, scale=0.125, window=0, out=P,
                                lse=P, status=P, workspace=P, workspace_bytes=1 << 30, stream=None),
}
ODD = ctypes.c_void_p(264)  # not on 16 bytes
BAD_CACHE = [dict(dim=96), dict(dim=0), dict(kv_heads=0), dict(page_size=8), dict(page_size=40), dict(pages=0), dict(k_cache=None), dict(v_cache=None),
             dict(k_cache=ODD), dict(v_cache=ODD), dict(status=None), dict(k_exp=P), dict(v_exp=P), dict(page_stride=2 * 16 * 64 - 8),
             dict(page_stride=2 * 16 * 64 + 4), dict(k_exp=P, v_exp=P, exp_stride=31, page_stride=2 * 16 * 64), dict(table=None),
             dict(table_stride=3), dict(table_rows=-1), dict(per_row=-1),
             dict(page_size=1 << 28, page_stride=1 << 36, exp_stride=1 << 36, per_row=8, table_stride=8),
             dict(page_size=1 << 28, page_stride=1 << 40, kv_heads=8), dict(k_exp=P, v_exp=P, exp_stride=40),
             dict(k_exp=ctypes.c_void_p(264), v_exp=P, exp_stride=32)]
BAD = {
    "dm3_rope": [dict(T=-1), dict(heads=0), dict(dim=0), dict(rot=0), dict(rot=7), dict(rot=66), dict(rot=2048, dim=4096), dict(x=None),
                 dict(positions=None), dict(inv_freq=None), dict(y=None), dict(heads=1 << 20)],
    "dm3_kv_write": BAD_CACHE + [dict(T=-1), dict(q_heads=-1), dict(rot=24), dict(rot=80), dict(inv_freq=None), dict(k=None), dict(v=None),
                                 dict(positions=None), dict(q=None), dict(q_out=None), dict(k=ODD), dict(q=ODD), dict(v_ts=129), dict(q_out=ODD)],
    "dm3_kv_read": BAD_CACHE + [dict(max_length=-1), dict(lengths=None), dict(k_out=None), dict(v_out=ODD), dict(table_rows=70000)],
    "dm3_paged_attention": BAD_CACHE + [dict(q_heads=3), dict(q_heads=1), dict(q_heads=0), dict(window=-1), dict(scale=math.nan),
                                        dict(scale=math.inf), dict(q=None), dict(lengths=None), dict(out=None), dict(lse=None), dict(q=ODD),
                                        dict(q_rs=250), dict(out=ODD), dict(table_rows=70000)],
}


@pytest.mark.parametrize("name", CALLS)
def test_c_entries_refuse(dm3, name):
    lib = dm3._lib.load()
    for change in BAD[name]:
        args = {**CALLS[name], **change}
        rc = getattr(lib, name)(*args.values())
        assert rc == dm3._lib.DM3_EINVAL, (name, change, rc)
        assert lib.dm3_last_error(), (name, change)


@pytest.mark.parametrize("name", CALLS)
def test_c_entries_with_nothing_to_do(dm3, name):
    """No tokens or no rows: done without a launch."""
    lib = dm3._lib.load()
    change = dict(T=0) if "T" in CALLS[name] else dict(table_rows=0, table=None)
    assert getattr(lib, name)(*{**CALLS[name], **change}.values()) == 0
    assert lib.dm3_last_launch_count() == 0


def _packed(dm3, name, args):
    pack, entry = dm3._lib.packed(name)
    return entry(pack(*(a.value if isinstance(a, ctypes.c_void_p) else a or 0 for a in list(args.values())[:-1])), None)


@pytest.mark.parametrize("name", CALLS)
def test_packed_entries(dm3, name):
    """The packed form of an entry passes on every argument: the same refusals with the same words, the same answer to
    a call with nothing to do; and a count that a C int would cut short is refused."""
    lib = dm3._lib.load()
    for change in BAD[name]:
        args = {**CALLS[name], **change}
        rc, why = getattr(lib, name)(*args.values()), lib.dm3_last_error()
        assert (_packed(dm3, name, args), lib.dm3_last_error()) == (rc, why), (name, change)
    change = dict(T=0) if "T" in CALLS[name] else dict(table_rows=0, table=None)
    assert _packed(dm3, name, {**CALLS[name], **change}) == 0 and lib.dm3_last_launch_count() == 0
    for key, kind in zip(CALLS[name], dm3._lib.SIGNATURES[name][1]):
        if kind is ctypes.c_int:
            for n in (2**31, 2**32, -2**31 - 1):
                assert _packed(dm3, name, {**CALLS[name], key: n}) == dm3._lib.DM3_EINVAL
                assert b"range" in lib.dm3_last_error()
    assert getattr(lib, name + "_packed")(None, None) == dm3._lib.DM3_EINVAL


@pytest.fixture
def stub(dm3, monkeypatch):
    """The ops on CPU tensors with the launch replaced: (ops, names of the entries that were launched directly)."""
    names = []
    monkeypatch.setattr(dm3.ops, "_same_device", lambda *a: 0)
    monkeypatch.setattr(dm3.ops, "_attention_workspace", lambda *a: 0)
    monkeypatch.setattr(dm3.ops, "_launch", lambda device, name, *a: names.append(name))
    return dm3.ops, names


def _op_calls(ops):
    """{name: (call on its tensors, tensors, places of those that could have a gradient)}."""
    x, q = torch.randn(3, 2, 64).to(BF), torch.randn(3, 4, 64).to(BF)
    pos, inv = torch.arange(3), torch.ones(16, dtype=torch.float64)
    k, v = torch.zeros(5, 2, 16, 64, dtype=BF), torch.zeros(5, 2, 16, 64, dtype=BF)
    t, s = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    return {
        "rope": (lambda x, pos, inv: ops.rope(x, pos, inv), (x, pos, inv), (0, 2)),
        "kv_write": (lambda a, b, pos, t, k, v, s, q, inv: ops.kv_write(a, b, pos, t, k, v, None, None, s, None, q, inv),
                     (x, x.clone(), pos, t, k, v, s, q, inv), (0, 1, 4, 5, 7, 8)),
        "kv_read": (lambda k, v, t, n, s: ops.kv_read(k, v, None, None, t, n, 7, s), (k, v, t, pos, s), (0, 1)),
        "paged_attention": (lambda q, k, v, t, n, s: ops.paged_attention(q, k, v, None, None, t, n, s), (q, k, v, t, pos, s), (0, 1, 2)),
    }


OPS = ["rope", "kv_write", "kv_read", "paged_attention"]


@pytest.mark.parametrize("name", OPS)
def test_every_tracer_sees_the_operator(stub, name):
    """Whatever records or watches calls finds the operator, not the allocation of its result; a plain call is a direct one."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    ops, names = stub
    fn, args, _ = _op_calls(ops)[name]
    op = "dm3::" + name
    for mode in ("real", "fake"):
        graph = make_fx(fn, tracing_mode=mode)(*args).graph
        assert ["dm3." + name + ".default"] == [str(n.target) for n in graph.nodes if n.op == "call_function" and "getitem" not in str(n.target)]
    kinds = [n.kind() for n in torch.jit.trace(fn, args, check_trace=False).graph.nodes()]
    assert op in kinds and not any("empty" in k for k in kinds)

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, a=(), kw=None):
            seen.append(func.name())
            return func(*a, **(kw or {}))

    class See(TorchFunctionMode):
        def __torch_function__(self, func, types, a=(), kw=None):
            seen.append(str(func))
            return func(*a, **(kw or {}))

    seen = []
    with Watch():
        fn(*args)
    assert op in seen
    seen = []
    with See():
        fn(*args)
    assert any("dm3" in x and name in x for x in seen)
    before = len(names)
    for plain in (torch.no_grad(), torch.inference_mode(), torch.device("cpu")):  # a default device is no tracer
        with plain, torch.profiler.profile() as prof:
            fn(*args)
        assert not any(e.name.startswith("dm3::") for e in prof.events())
    assert names[before:] == ["dm3_" + name] * 3


@pytest.mark.parametrize("name", OPS)
def test_every_gradient_is_refused(stub, name):
    """A gradient asked for by any input is an error, backwards and forwards, not a silent zero."""
    import torch.autograd.forward_ad as forward

    ops, _ = stub
    fn, args, places = _op_calls(ops)[name]
    for at in places:
        leaf = args[at].clone().requires_grad_()
        # (an in-place write to a leaf is refused by the call itself)
        with pytest.raises(RuntimeError, match="gradient|autograd|in-place"):
            out = fn(*args[:at], leaf, *args[at + 1:])
            (out[0] if isinstance(out, tuple) else out).double().sum().backward()
        with forward.dual_level(), pytest.raises(RuntimeError, match="gradient"):
            fn(*args[:at], forward.make_dual(args[at], torch.ones_like(args[at])), *args[at + 1:])
        with pytest.raises(RuntimeError, match="gradient"):
            torch.func.jvp(lambda x: fn(*args[:at], x, *args[at + 1:]), (args[at],), (torch.ones_like(args[at]),))


def test_a_negative_bound_is_refused(dm3, stub):
    """attend's max_tokens narrows the table; a negative one would count its columns from the end."""
    c = dm3.KVCache(1, 2, 200, 1, 64, page_size=16, device="cpu")
    q, n = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, dtype=torch.int64)
    for bad in (-1, -15, -16, -100):
        with pytest.raises(ValueError, match="max_tokens"):
            c.attend(0, q, n, max_tokens=bad)
    assert stub[1] == []
    for fine in (None, 0, 1, 200, 5000):
        c.attend(0, q, n, max_tokens=fine)
    assert len(stub[1]) == 5


@pytest.mark.parametrize("quant", [False, True])
def test_strides_of_sides_of_one(dm3, stub, monkeypatch, quant):
    """A contiguous page is taken whatever the strides of its sides of one are, and so are the strides of a single page."""
    ops, _ = stub
    got = []
    monkeypatch.setattr(ops, "_launch", lambda device, name, *a: got.append((name, a)))
    dtype = torch.float8_e4m3fn if quant else BF
    t, s, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    q = torch.zeros(2, 4, 64, dtype=BF)
    for pages in (1, 5):
        # one head: [pages, tokens, heads, dim] seen as [pages, heads, tokens, dim]
        flat = [torch.zeros(pages, 16, 1, 64).to(dtype).transpose(1, 2) for _ in range(2)]
        exps = [torch.zeros(pages, 16, 1, dtype=torch.int8).transpose(1, 2) if quant else None for _ in range(2)]
        odd = [torch.as_strided(x, x.shape, (x.stride(0), 7, *x.stride()[2:])) for x in flat]
        alone = [torch.as_strided(x, x.shape, (3 if pages == 1 else x.stride(0), *x.stride()[1:])) for x in flat]
        mixed = [flat[0], odd[1]]
        for c in (flat, odd, alone, mixed):
            ops.kv_write(q[:, :1], q[:, :1], n, t, *c, *exps, s)
            ops.kv_read(*c, *exps, t, n, 4, s)
            ops.paged_attention(q, *c, *exps, t, n, s)
    assert len(got) == 24
    # what the entries are told: pages of 16 tokens of one head
    for name, a in got:
        assert 16 * 64 in a and (not quant or 16 in a), (name, a)
    two = [torch.zeros(5, 2, 16, 64).to(dtype) for _ in range(2)]
    ex = [torch.zeros(5, 2, 16, dtype=torch.int8) if quant else None for _ in range(2)]
    wrong = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in two]
    for c, e in ((wrong, ex), (two, [None if x is None else x.transpose(1, 2).contiguous().transpose(1, 2) for x in ex])):
        if c is two and not quant:
            continue
        with pytest.raises(RuntimeError, match="contiguous"):
            ops.kv_read(*c, *e, t, n, 4, s)


def test_frequencies_of_the_callers(dm3, stub, monkeypatch):
    """A Rope's frequencies and factor can be set: calls and the cache's writes take them."""
    got = []
    monkeypatch.setattr(dm3.ops, "_launch", lambda device, name, *a: got.append(a))
    rope = dm3.Rope(64, scaling="yarn", stretch=4.0, trained_length=100, device="cpu")
    mine = torch.linspace(1.0, 0.1, 16, dtype=torch.float64)
    rope.inv_freq, rope.factor = mine, 1.25
    c = dm3.KVCache(1, 1, 16, 1, 64, device="cpu")
    x, n = torch.zeros(1, 1, 64, dtype=BF), torch.zeros(1, dtype=torch.int64)
    rope(x, n)
    c.write(0, x, x, n, None, x, rope)
    for a in got:
        at = a.index(mine.data_ptr())
        assert a[at + 1] == 32 and a[at + 3] == 1.25
