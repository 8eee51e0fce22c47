"""The attention side of a decode frame and of prompt reading, as cases to measure: rotary positions, the paged
key-value cache (written in bf16 or quantised to e4m3, and read back), and one new token's attention over it.

`run` computes a case in elementary torch operations where `own` is false, and by the calls that a user makes
where it is true. `exact` gives the same outputs from the definitions in 64 bits.

A quantised cache row (one token of one head, D values) holds e4m3 codes c and one exponent e, and stands for
c * 2^e: e is the smallest integer with amax <= 448 * 2^e, kept in [-110, 119]; a row of zeros has e = 0. Keys
are rotated, rounded to bf16, and then quantised."""

import math
import random

import torch

own = False

E_MIN, E_MAX = -110, 119


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode frame: the two guidance rows' query and key heads, a quarter of the head rotated
        dict(name="rope_frame", kind="rope", tokens=2, heads=18, dim=256, rot=64, interleaved=False, scaling="none", far=3000),
        # a long prompt in the interleaved layout, the context stretched four times: positions far out
        dict(name="rope_prompt", kind="rope", tokens=16384, heads=20, dim=128, rot=128, interleaved=True, scaling="yarn", far=120000),
        # the frame's new token of both guidance rows into a quantised cache, and the short rows read back
        dict(name="write_frame_e4m3", kind="write", quant=True, rows=2, longest=1, start=45, q_heads=16, kv_heads=2, dim=256, page=64, rot=64,
             interleaved=False, scaling="none"),
        # one chunk of prompt reading: 128 tokens of both guidance rows, into a bf16 cache
        dict(name="write_chunk_bf16", kind="write", quant=False, rows=2, longest=128, start=896, q_heads=16, kv_heads=2, dim=256, page=64, rot=64,
             interleaved=False, scaling="none"),
        # whole prompts of many requests, of every length, into a quantised cache, and read back for the prompt's attention
        dict(name="write_prompts_e4m3", kind="write", quant=True, rows=13, longest=4001, start=0, q_heads=32, kv_heads=8, dim=128, page=32, rot=128,
             interleaved=False, scaling="linear"),
        # a cached prefix read back to go on with: a few rows of odd lengths, bf16
        dict(name="read_prefix_bf16", kind="read", quant=False, rows=5, longest=1237, kv_heads=2, dim=256, page=64),
        # long quantised rows read back
        dict(name="read_long_e4m3", kind="read", quant=True, rows=4, longest=32768, kv_heads=8, dim=128, page=128),
        # attention of a decode frame: two guidance rows, a few hundred frames so far
        dict(name="attend_frame_bf16", kind="attend", quant=False, rows=2, longest=1021, capacity=2048, q_heads=16, kv_heads=2, dim=256, page=64, window=0,
             empty=False),
        # the same frame late in a long session, quantised
        dict(name="attend_session_e4m3", kind="attend", quant=True, rows=2, longest=131072, capacity=131072, q_heads=16, kv_heads=2, dim=256, page=64,
             window=0, empty=False),
        # serving: many ragged requests with grouped heads, bf16
        dict(name="attend_batch_bf16", kind="attend", quant=False, rows=64, longest=8192, capacity=8192, q_heads=32, kv_heads=8, dim=128, page=16, window=0,
             empty=False),
        # the same over a quantised cache, with larger groups and idle rows
        dict(name="attend_batch_e4m3", kind="attend", quant=True, rows=96, longest=6007, capacity=8192, q_heads=64, kv_heads=4, dim=128, page=48, window=0,
             empty=True),
        # every query head with a head of its own, a sliding window, and idle rows
        dict(name="attend_window_bf16", kind="attend", quant=False, rows=24, longest=5000, capacity=5120, q_heads=12, kv_heads=12, dim=64, page=32,
             window=1000, empty=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "write", "write", "read", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
    page = 16 * _log(rng, 1, 16)
    rot = rng.choice([dim, dim // 2, dim // 4])
    place = dict(rot=rot, interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn"]))
    if kind == "rope":
        tokens, heads = _log(rng, 1, 16384), rng.randint(1, 40)
        while tokens * heads * dim > 16384 * 20 * 128:
            tokens = tokens // 2 + 1
        return dict(kind=kind, tokens=tokens, heads=heads, dim=dim, far=_log(rng, 16, 1 << 20), **place)
    quant = rng.random() < 0.5
    rows, longest = _log(rng, 1, 96), _log(rng, 1, 65536)
    most = (13 * 4001 * 8 * 128) if kind == "write" else (4 * 32768 * 8 * 128) if kind == "read" else (64 * 8192 * 8 * 128)
    while rows * longest * kv_heads * dim > most:
        rows, longest = (rows // 2 + 1, longest) if rows > 8 else (rows, longest * 2 // 3)
    if kind == "read":
        return dict(kind=kind, quant=quant, rows=rows, longest=longest, kv_heads=kv_heads, dim=dim, page=page)
    group = rng.choice([1, 2, 3, 4, 8, 16])
    if kind == "write":
        group = min(group, 8)
        start = _log(rng, 1, 2000) - 1
        longest = max(1, min(longest, most // (rows * kv_heads * dim) - start))
        return dict(kind=kind, quant=quant, rows=rows, longest=longest, start=start, q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, **place)
    capacity = longest + _log(rng, 1, 4096) - 1
    return dict(kind=kind, quant=quant, rows=rows, longest=longest, capacity=capacity, q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page,
                window=rng.choice([0, 0, _log(rng, 1, longest)]), empty=rng.random() < 0.3)


def _lengths(case):
    """Tokens of each row: the first row is the longest, the others are spread below it; idle rows have none."""
    r = random.Random(case["rows"] * 1000003 + case["longest"])
    got = [case["longest"]] + [max(1, round(case["longest"] * r.uniform(0.02, 1.0))) for _ in range(case["rows"] - 1)]
    if case.get("empty"):
        got[1::5] = [0] * len(got[1::5])
    return got


def _span(case):
    """The table's tokens a row: whole pages."""
    n = case.get("capacity") or case["longest"] + case.get("start", 0)
    return -(-n // case["page"]) * case["page"]


def _frequencies(case):
    """(angle a position, in 64 bits, for each rotated pair; factor on the rotated part)."""
    rot, base, kind = case["rot"], 1e6, case["scaling"]
    stretch, trained = 4.0, 32768
    if kind == "ntk":
        base *= stretch ** (rot / (rot - 2)) if rot > 2 else stretch
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if kind == "linear":
        f = f / stretch
    if kind == "yarn":
        # pairs that turn more than 32 times over the trained length stay, those that turn less than once are slowed, a ramp between
        turns = trained * f / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        f = f * keep + f / stretch * (1 - keep)
    return f, (0.1 * math.log(stretch) + 1 if kind == "yarn" else 1.0)


# ------------------------------------------------------------------------------------------------ inputs
def _quantise(x):
    """Codes (as bytes) and exponents of rows of bf16 values, along the last axis; what is not finite becomes NaN."""
    x = x.float()
    fine = x.isfinite()
    part, power = torch.frexp(torch.where(fine, x.abs(), 0.0).amax(-1))
    e = torch.where(part > 0, power - torch.where(part <= 0.875, 9, 8), 0).clamp(E_MIN, E_MAX)
    y = torch.ldexp(x, -e[..., None]).clamp(-448, 448)
    return torch.where(fine, y, math.nan).to(torch.float8_e4m3fn).view(torch.uint8), e.to(torch.int8)


def _cache(case, table, pages, g, dev):
    """A cache whose pages all hold values (rows, or what earlier requests left)."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    s = {}
    for name in ("k", "v"):
        x = torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16)
        if name == "k":  # some channels of keys are much larger than the rest
            x *= (1 + 4 * (torch.arange(case["dim"], device=dev) % 31 == 5)).to(torch.bfloat16)
        if case["quant"]:
            code, e = torch.empty(shape, device=dev, dtype=torch.uint8), torch.empty(shape[:-1], device=dev, dtype=torch.int8)
            step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
            for a in range(0, pages, step):
                code[a:a + step], e[a:a + step] = _quantise(x[a:a + step])
            s[name], s[name + "_exp"] = code.view(torch.float8_e4m3fn), e
        else:
            s[name], s[name + "_exp"] = x, None
    return s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    s = {"case": case}
    if "rot" in case:
        f, s["factor"] = _frequencies(case)
        s["inv_freq"] = f.to(dev)
    if case["kind"] == "rope":
        s["x"] = torch.randn(case["tokens"], case["heads"], case["dim"], generator=g, device=dev, dtype=torch.bfloat16)
        first = random.Random(seed).randint(0, max(0, case["far"] - case["tokens"]))
        s["positions"] = torch.arange(first, first + case["tokens"], device=dev)
        return s
    rows, per_row = case["rows"], _span(case) // case["page"]
    lengths = _lengths(case)
    total = [n + case.get("start", 0) for n in lengths]
    # pages are dealt out in the order that a program's requests came and went; rows have pages for their own tokens only
    pages = sum(-(-n // case["page"]) for n in total) + 3
    order = torch.randperm(pages, generator=g, device=dev).tolist()
    table = torch.zeros(rows, per_row, dtype=torch.int32)
    for i, n in enumerate(total):
        have = -(-n // case["page"])
        table[i, :have] = torch.tensor(order[:have], dtype=torch.int32)
        order = order[have:]
    s["table"] = table.to(dev)
    s.update(_cache(case, table, pages, g, dev))
    s["status"] = torch.zeros(1, dtype=torch.int32, device=dev)
    s["lengths"] = torch.tensor(total, device=dev)
    if case["kind"] == "write":
        t = sum(lengths)
        heads = case["q_heads"] + 2 * case["kv_heads"]
        qkv = torch.randn(t, heads, case["dim"], generator=g, device=dev, dtype=torch.bfloat16)  # as one projection gives them
        s["q"], s["new_k"], s["new_v"] = qkv.split([case["q_heads"], case["kv_heads"], case["kv_heads"]], 1)
        n = torch.tensor(lengths, device=dev)
        s["rows"] = torch.repeat_interleave(torch.arange(rows, device=dev), n)
        s["positions"] = torch.cat([torch.arange(case["start"], case["start"] + x) for x in lengths]).to(dev)
    if case["kind"] == "attend":
        s["q"] = torch.randn(rows, case["q_heads"], case["dim"], generator=g, device=dev, dtype=torch.bfloat16)
        s["scale"] = case["dim"] ** -0.5
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _rotate(s, x, bits):
    """x [tokens, heads, dim] with its first rot dims turned by position * inv_freq, computed in `bits`."""
    c = s["case"]
    rot = c["rot"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]  # 32 bits lose the angles of far positions
    cos, sin = (angle.cos() * s["factor"]).to(bits)[:, None], (angle.sin() * s["factor"]).to(bits)[:, None]
    y = x.to(bits)
    if c["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., rot:]], -1)


def _gather(s, name):
    """A cache's values by the table, in 32 bits: [rows, kv_heads, span, dim]."""
    t = s["table"].long()
    x = s[name][t] if s[name + "_exp"] is None else s[name].view(torch.uint8)[t].view(torch.float8_e4m3fn)
    x = x.float()
    if s[name + "_exp"] is not None:
        x = torch.ldexp(x, s[name + "_exp"][t][..., None].int())
    return x.transpose(1, 2).flatten(2, 3)


def _read(s):
    have = torch.arange(_span(s["case"]), device=s["table"].device) < s["lengths"][:, None]
    return [torch.where(have[:, None, :, None], _gather(s, n), 0.0).bfloat16() for n in ("k", "v")]


def _plain_write(s):
    quant, page = s["case"]["quant"], s["case"]["page"]
    q = _rotate(s, s["q"], torch.float32).bfloat16()
    # a rotated key next to a border between two codes decides which it becomes: 64 bits for those
    k = _rotate(s, s["new_k"], torch.float64 if quant else torch.float32).bfloat16()
    at, of = s["table"][s["rows"], s["positions"] // page].long(), s["positions"] % page
    for name, x in (("k", k), ("v", s["new_v"])):
        if quant:
            code, e = _quantise(x)
            s[name].view(torch.uint8)[at, :, of] = code
            s[name + "_exp"][at, :, of] = e
        else:
            s[name][at, :, of] = x
    return [q] + (_read(s) if quant else [s["k"], s["v"]])


def _plain_attend(s):
    c = s["case"]
    n = s["lengths"][:, None]
    at = torch.arange(_span(c), device=n.device)
    seen = (at < n) & (at >= n - c["window"] if c["window"] else at >= 0)
    seen = seen[:, None, None, :]
    group = c["q_heads"] // c["kv_heads"]
    q = s["q"].float().view(c["rows"], c["kv_heads"], group, c["dim"])
    logit = (q @ _gather(s, "k").transpose(-1, -2) * s["scale"]).masked_fill(~seen, -math.inf)
    most = logit.amax(-1, keepdim=True)
    p = torch.where(seen, (logit - most).exp(), 0.0)
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen.transpose(-1, -2), _gather(s, "v"), 0.0)
    out = torch.where(total > 0, p @ v / total, 0.0)
    lse = torch.where(total > 0, most + total.log(), -math.inf)
    return [out.flatten(1, 2).bfloat16(), lse.flatten(1)]


def run(state):
    s, c = state, state["case"]
    if own:
        from drama3_b200 import ops

        if c["kind"] == "rope":
            return ops.rope(s["x"], s["positions"], s["inv_freq"], c["interleaved"], s["factor"])
        held = (s["k"], s["v"], s["k_exp"], s["v_exp"])
        if c["kind"] == "write":
            q = ops.kv_write(s["new_k"], s["new_v"], s["positions"], s["table"], *held, s["status"], s["rows"], s["q"], s["inv_freq"], c["interleaved"],
                             s["factor"])
            return [q, *(ops.kv_read(*held, s["table"], s["lengths"], _span(c), s["status"]) if c["quant"] else (s["k"], s["v"]))]
        if c["kind"] == "read":
            return list(ops.kv_read(*held, s["table"], s["lengths"], _span(c), s["status"]))
        return list(ops.paged_attention(s["q"], *held, s["table"], s["lengths"], s["status"], s["scale"], c["window"]))
    if c["kind"] == "rope":
        return _rotate(s, s["x"], torch.float32).bfloat16()
    return {"write": _plain_write, "read": _read, "attend": _plain_attend}[c["kind"]](s)


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    dim = case["dim"]
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 4 * n * dim + 8 * case["tokens"], "flops": 3 * n * case["rot"]}
    held = (dim + 1 if case["quant"] else 2 * dim) * 2 * case["kv_heads"]  # bytes of one token's keys and values in the cache
    lengths = _lengths(case)
    if case["kind"] == "read":
        return {"bytes": sum(lengths) * held + case["rows"] * _span(case) * 4 * case["kv_heads"] * dim, "flops": 0}
    if case["kind"] == "write":
        t, qh, kh = sum(lengths), case["q_heads"], case["kv_heads"]
        moved = t * (4 * qh * dim + 4 * kh * dim + held + 16)
        if case["quant"]:  # and read back: the rows' earlier tokens from the cache, all of them as bf16
            moved += case["rows"] * case["start"] * held + case["rows"] * _span(case) * 4 * kh * dim
        return {"bytes": moved, "flops": t * (qh + kh) * case["rot"] * 3}
    seen = sum(min(n, case["window"] or n) for n in lengths)
    return {"bytes": seen * held + case["rows"] * case["q_heads"] * (4 * dim + 4), "flops": 4 * seen * case["q_heads"] * dim}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_turn(s, x):
    """Each rotated pair as a complex number times e^(i angle)."""
    rot, half = s["case"]["rot"], s["case"]["rot"] // 2
    first = range(0, rot, 2) if s["case"]["interleaved"] else range(half)
    first = torch.tensor(list(first), device=x.device)
    second = first + 1 if s["case"]["interleaved"] else first + half
    y = x.double()
    turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device=x.device), torch.outer(s["positions"].double(), s["inv_freq"]))
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_codes(x):
    """The values that a quantised cache holds for rows of bf16 values: each of them to the nearest multiple of its step, ties to even."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448))
    e = e + (448 * torch.exp2(e) < top).double() - (448 * torch.exp2(e - 1) >= top).double()
    e = torch.where(top > 0, e, 0.0).clamp(E_MIN, E_MAX)
    y = x * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0**-6))) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448) * torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_turn(s, s["x"])
    page, table = case["page"], s["table"].long()

    def row(name, i, n):
        """Row i's first n tokens of a cache: [kv_heads, n, dim]."""
        at = torch.arange(n, device=table.device)
        where = (table[i, at // page], slice(None), at % page)
        x = s[name].view(torch.uint8)[where].view(torch.float8_e4m3fn).double() if case["quant"] else s[name][where].double()
        return (x * torch.exp2(s[name + "_exp"][where].double())[..., None] if case["quant"] else x).transpose(0, 1)

    lengths = s["lengths"].tolist()
    if case["kind"] == "attend":
        group = case["q_heads"] // case["kv_heads"]
        out = torch.zeros(case["rows"], case["q_heads"], case["dim"], dtype=torch.float64, device=table.device)
        lse = torch.full((case["rows"], case["q_heads"]), -math.inf, dtype=torch.float64, device=table.device)
        for i, n in enumerate(lengths):
            if n:
                from_ = max(0, n - case["window"]) if case["window"] else 0
                for h in range(case["kv_heads"]):
                    of = slice(h * group, (h + 1) * group)
                    logit = s["q"][i, of].double() @ row("k", i, n)[h, from_:].T * s["scale"]
                    out[i, of], lse[i, of] = logit.softmax(-1) @ row("v", i, n)[h, from_:], logit.logsumexp(-1)
        return [out, lse]
    if case["kind"] == "read":
        got = [torch.zeros(case["rows"], case["kv_heads"], _span(case), case["dim"], dtype=torch.float64, device=table.device) for _ in range(2)]
        for i, n in enumerate(lengths):
            for x, name in zip(got, ("k", "v")):
                x[i, :, :n] = row(name, i, n)
        return got
    q, k, v = _exact_turn(s, s["q"]), _exact_turn(s, s["new_k"]), s["new_v"].double()
    at, of = table[s["rows"], s["positions"] // page], s["positions"] % page
    if not case["quant"]:
        held = [s["k"].double(), s["v"].double()]
        held[0][at, :, of], held[1][at, :, of] = k, v
        return [q, *held]
    got = [torch.zeros(case["rows"], case["kv_heads"], _span(case), case["dim"], dtype=torch.float64, device=table.device) for _ in range(2)]
    for x, name, new in zip(got, ("k", "v"), (_exact_codes(k.bfloat16()), _exact_codes(v))):
        for i in range(case["rows"]):
            x[i, :, :case["start"]] = row(name, i, case["start"])
        x[s["rows"], :, s["positions"]] = new
    return [q, *got]
