"""Measured cases of the serving operators: the norm and rotation of query and key heads in one pass, the
paged key/value cache as it is written and read back, attention of one new token over that cache, and low-rank
adapters of many requests beside a shared projection.

A case is a dict of plain values; `prepare` makes its inputs on the GPU, `run` is one call of the operator: the
plain torch form, or with `own` the framework's kernels (scala-torch_b200/scalatorch/ffm.py) on the same buffers.
`exact` is the operator's definition in 64 bits, written apart from the plain form.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PAGE_TYPES = {"F32": torch.float32, "BF16": torch.bfloat16, "F16": torch.float16, "E4M3": torch.float8_e4m3fn}
_THETA = 500000.0
_EPS = 1e-5
_session = None


def listed():
    return [
        # one token of a small model: nine query heads on three key heads of 64, launch latency alone
        dict(name="norm+rope 1x9/3x64", op="norm_rope", rows=1, heads=9, kv_heads=3, width=64),
        # a decode step of 64 requests at 64 query and 8 key heads of 128
        dict(name="norm+rope 64x64/8x128", op="norm_rope", rows=64, heads=64, kv_heads=8, width=128),
        # prompt tokens of several requests together, read out of the fused projection's rows
        dict(name="norm+rope 8191x32/8x128", op="norm_rope", rows=8191, heads=32, kv_heads=8, width=128),
        # the new tokens of 64 requests go into an 8-bit cache
        dict(name="cache write 64 e4m3", op="cache_write", sequences=64, tokens=1, kv_heads=8, width=128, page=16, dtype="E4M3"),
        # prompts of 7 requests go into an 8-bit cache
        dict(name="cache write 7x2039 e4m3", op="cache_write", sequences=7, tokens=2039, kv_heads=8, width=128, page=16, dtype="E4M3"),
        # cached prompts come back in Float32 for a later chunk's attention
        dict(name="cache read 5x4001 e4m3", op="cache_read", sequences=5, tokens=4001, kv_heads=8, width=128, page=32, dtype="E4M3"),
        # one request of a small model with a short cache: launch latency alone
        dict(name="attend 1x9/3x64 33 bf16", op="attend", batch=1, heads=9, kv_heads=3, width=64, longest=33, page=16, dtype="BF16"),
        # a batch of eight requests with caches of up to 544 tokens, 8 bits
        dict(name="attend 8x64/8x128 544 e4m3", op="attend", batch=8, heads=64, kv_heads=8, width=128, longest=544, page=16, dtype="E4M3"),
        # 24 requests of very different lengths
        dict(name="attend 24x64/8x128 16384 bf16", op="attend", batch=24, heads=64, kv_heads=8, width=128, longest=16384, page=16, dtype="BF16"),
        # one long request alone: the cache's length is all there is to split
        dict(name="attend 1x32/8x128 60001 e4m3", op="attend", batch=1, heads=32, kv_heads=8, width=128, longest=60001, page=64, dtype="E4M3"),
        # one request with its adapter beside a small model's projection
        dict(name="adapted 1x1536x576 r8", op="adapted", rows=1, out=1536, inner=576, used=1, rank=8, dtype="BF16"),
        # 32 requests of 12 adapters, some without one, beside a large projection
        dict(name="adapted 32x4096x14336 r64", op="adapted", rows=32, out=4096, inner=14336, used=12, rank=64, dtype="BF16"),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


_HEADS = ((9, 3, 64), (32, 8, 128), (64, 8, 128), (8, 8, 64), (16, 1, 128), (12, 4, 96), (5, 1, 80), (16, 2, 256), (14, 2, 64))


def draw(rng):
    op = rng.choice(("norm_rope", "cache_write", "cache_read", "attend", "adapted"))
    heads, kv_heads, width = rng.choice(_HEADS)
    page, dtype = rng.choice((8, 16, 32, 64)), rng.choice(("F32", "BF16", "F16", "E4M3"))
    if op == "norm_rope":
        most = max(1, 8191 * 40 * 128 // ((heads + kv_heads) * width))
        return dict(op=op, rows=_between(rng, 1, min(8191, most)), heads=heads, kv_heads=kv_heads, width=width)
    if op in ("cache_write", "cache_read"):
        sequences = _between(rng, 1, 64)
        most = max(1, 7 * 2039 * 8 * 128 // (sequences * kv_heads * width))
        return dict(op=op, sequences=sequences, tokens=_between(rng, 1, min(4001, most)), kv_heads=kv_heads, width=width, page=page, dtype=dtype)
    if op == "attend":
        batch = _between(rng, 1, 64)
        most = 24 * 16384 * 8 * 128 // (batch * kv_heads * width * (2 if dtype == "F32" else 1))
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, width=width, longest=_between(rng, 1, min(60001, most)), page=page, dtype=dtype)
    out, inner = rng.choice(((576, 576), (1536, 576), (576, 1536), (1024, 4096), (4096, 4096), (14336, 4096), (4096, 14336), (1000, 1016)))
    rows = _between(rng, 1, 64)
    return dict(op=op, rows=rows, out=out, inner=inner, used=_between(rng, 1, min(rows, 24)), rank=_between(rng, 2, 64), dtype=rng.choice(("F32", "BF16", "F16")))


# ------------------------------------------------------------------ what a case fixes apart from the seed


def _fixed(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """Cache lengths: the longest, one row that has none yet (batches of four and more), the rest spread over
    the range."""
    r, n = _fixed(case), case["batch"]
    got = [case["longest"]] + [r.randint(1, case["longest"]) for _ in range(n - 1)]
    if n >= 4:
        got[1] = 0
    return got


def _ranks(case):
    """Every second adapter of the pool has half the rank (at least one)."""
    return [case["rank"] if i % 2 == 0 else max(1, case["rank"] // 2) for i in range(case["used"] + 3)]


def _used_rows(case):
    """The adapter of each row before the seed's shuffle: the used ones in turn, and rows without one where there
    are more rows than adapters."""
    turn = case["used"] + (1 if case["rows"] > case["used"] else 0)
    return [i % turn if i % turn < case["used"] else -1 for i in range(case["rows"])]


def _bytes_of(dtype):
    return _PAGE_TYPES[dtype].itemsize


def work(case):
    op = case["op"]
    if op == "norm_rope":
        n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["width"]
        return {"bytes": 8 * n + 4 * case["rows"] + 8 * case["width"], "flops": 7 * n}
    if op in ("cache_write", "cache_read"):
        rows = case["sequences"] * case["tokens"]
        n = 2 * rows * case["kv_heads"] * case["width"]
        scales = 2 * rows * case["kv_heads"] if case["dtype"] == "E4M3" else 0
        return {"bytes": n * (4 + _bytes_of(case["dtype"])) + scales + 8 * rows, "flops": 2 * n}
    if op == "attend":
        keys = sum(_lengths(case))
        heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
        per_key = 2 * kv_heads * (width * _bytes_of(case["dtype"]) + (1 if case["dtype"] == "E4M3" else 0))
        return {"bytes": keys * per_key + 8 * case["batch"] * heads * width, "flops": 4 * keys * heads * width}
    rows, out, inner, size = case["rows"], case["out"], case["inner"], _bytes_of(case["dtype"])
    ranks = _ranks(case)
    factors = sum(ranks[i] for i in range(case["used"])) * (out + inner) * size
    thin = sum(ranks[i] for i in _used_rows(case) if i >= 0) * (out + inner)
    return {"bytes": 2 * out * inner + factors + 4 * rows * (out + inner) + 4 * out + 4 * rows, "flops": 2 * rows * out * inner + 2 * thin}


# ------------------------------------------------------------------ inputs


def _quantise(x):
    """E4M3 rows with a power-of-two scale each: the smallest that brings the row's largest magnitude to 448 or
    below.  Returns the values and the scales' exponents + 127."""
    top = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)
    shift = exponent - 9 + (mantissa > 0.875)
    shift = torch.where(top > 0, shift, torch.zeros_like(shift)).clamp(min=-126)
    return torch.ldexp(x, -shift.unsqueeze(-1)).to(torch.float8_e4m3fn), (shift + 127).to(torch.uint8)


def _cache(case, pages, gen):
    """Pages (pages, heads, page, width) of earlier tokens: unit normal with a few wide channels, as keys have."""
    shape = (pages, case["kv_heads"], case["page"], case["width"])
    made = {}
    for name in ("keys", "values"):
        data = torch.empty(shape, dtype=_PAGE_TYPES[case["dtype"]], device="cuda")
        scales = torch.empty(shape[:3], dtype=torch.uint8, device="cuda") if case["dtype"] == "E4M3" else None
        step = max(1, (1 << 25) // (shape[1] * shape[2] * shape[3]))
        for i in range(0, pages, step):
            x = torch.randn((min(step, pages - i),) + shape[1:], generator=gen, device="cuda")
            if name == "keys":
                x[..., :: max(1, case["width"] // 4)] *= 4.0
            if scales is None:
                data[i:i + step] = x.to(data.dtype)
            else:
                q, e = _quantise(x)
                data[i:i + step], scales[i:i + step] = q, e
        made[name] = data
        if scales is not None:
            made[name[:-1] + "_scales"] = scales
    return made


def _tables(lengths, page, gen, spare=3):
    """Pages handed out in a random order; the unused entries of a table are -1."""
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    width = max(1, max(blocks))
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    table_of = torch.zeros((len(lengths), width), dtype=torch.int64)
    used, at = torch.zeros((len(lengths), width), dtype=torch.bool), 0
    for i, n in enumerate(blocks):
        table_of[i, :n] = torch.arange(at, at + n)
        used[i, :n] = True
        at += n
    return torch.where(used.cuda(), order[table_of.cuda()], table.cuda()), pages


def _open():
    """The program's session, made once."""
    global _session
    if _session is None:
        sys.path.insert(0, os.path.join(_ROOT, "scala-torch_b200"))
        from scalatorch.ffm import B200Session
        _session = B200Session(0, 8 << 30)
    return _session


def _held(t):
    """A torch tensor's memory as a tensor of the session."""
    from scalatorch import ffm
    kinds = {torch.float32: ffm.STB_F32, torch.bfloat16: ffm.STB_BF16, torch.float16: ffm.STB_F16,
             torch.float8_e4m3fn: ffm.STB_E4M3, torch.uint8: ffm.STB_U8, torch.int32: ffm.STB_I32}
    return _session.wrap(t.data_ptr(), tuple(t.shape), kinds[t.dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": dict(case), "seed": seed}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if op == "norm_rope":
        rows, heads, kv_heads, width = case["rows"], case["heads"], case["kv_heads"], case["width"]
        s["fused"] = normal(rows, (heads + 2 * kv_heads) * width) * 1.5  # q | k | v of the fused projection
        s["q_weight"], s["k_weight"] = 1 + 0.2 * normal(width), 1 + 0.2 * normal(width)
        s["positions"] = torch.randint(0, 131072, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        s["q_out"], s["k_out"] = torch.empty((rows, heads, width), device="cuda"), torch.empty((rows, kv_heads, width), device="cuda")
    elif op in ("cache_write", "cache_read"):
        n, tokens = case["sequences"], case["tokens"]
        r = _fixed(case)
        starts = [r.randint(0, 40) for _ in range(n)]
        s["tables"], pages = _tables([a + tokens for a in starts], case["page"], gen)
        s.update(_cache(case, pages, gen))
        s["sequences"] = torch.arange(n, device="cuda", dtype=torch.int32).repeat_interleave(tokens)
        s["positions"] = (torch.tensor(starts, device="cuda").unsqueeze(1) + torch.arange(tokens, device="cuda")).reshape(-1).to(torch.int32)
        shape = (n * tokens, case["kv_heads"], case["width"])
        if op == "cache_write":
            s["key"], s["value"] = normal(*shape), normal(*shape)
            s["key"][..., :: max(1, case["width"] // 4)] *= 4.0
        else:
            s["key"], s["value"] = torch.empty(shape, device="cuda"), torch.empty(shape, device="cuda")
    elif op == "attend":
        lengths = _lengths(case)
        random.Random(seed).shuffle(lengths)
        s["tables"], pages = _tables(lengths, case["page"], gen)
        s.update(_cache(case, pages, gen))
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["query"] = normal(case["batch"], case["heads"], case["width"])
        s["out"] = torch.empty_like(s["query"])
    else:
        rows, out, inner, rank = case["rows"], case["out"], case["inner"], case["rank"]
        ranks = torch.tensor(_ranks(case), dtype=torch.int32, device="cuda")
        slots, kind = len(ranks), _PAGE_TYPES[case["dtype"]]
        s["x"] = normal(rows, inner)
        s["weight"] = (normal(out, inner) / math.sqrt(inner)).to(torch.bfloat16)
        s["bias"] = 0.1 * normal(out)
        s["a"] = (normal(slots, rank, inner) / math.sqrt(inner)).to(kind)
        s["b"] = (normal(slots, out, rank) * 0.1).to(kind)
        s["ranks"], s["scales"] = ranks, 16.0 / ranks.float()
        row_of = _used_rows(case)
        random.Random(seed).shuffle(row_of)
        s["adapters"] = torch.tensor(row_of, dtype=torch.int32, device="cuda")
        s["out"] = torch.empty((rows, out), device="cuda")
    if own:
        _plan(s)
    return s


def _plan(s):
    """What a program of the framework keeps beside its buffers: their tensors, the cache, the adapter pool."""
    session, case = _open(), s["case"]
    h = {k: _held(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "norm_rope":
        heads, kv_heads, width = case["heads"], case["kv_heads"], case["width"]
        h["query"] = session.columns(h["fused"], 0, (heads, width))
        h["key"] = session.columns(h["fused"], heads * width, (kv_heads, width))
    elif case["op"] == "adapted":
        h["weight"] = session.as_weight(h["weight"])
        h["pool"] = session.adapter_pool(h["a"], h["b"], h["ranks"], h["scales"])
    else:
        h["cache"] = session.paged_cache(h["keys"], h["values"], h.get("key_scales"), h.get("value_scales"))
    s["held"] = h


def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s, s["held"])
    return _PLAIN[op](s)


# ------------------------------------------------------------------ the framework's calls


def _own_norm_rope(s, h):
    _session.qk_norm_rope(h["query"], h["key"], h["q_weight"], h["k_weight"], h["positions"], _EPS, _THETA, out=(h["q_out"], h["k_out"]))
    return {"q": s["q_out"], "k": s["k_out"]}


def _written(s):
    return {k: s[k] for k in ("keys", "values", "key_scales", "value_scales") if k in s}


def _own_cache_write(s, h):
    h["cache"].append(h["key"], h["value"], h["tables"], h["sequences"], h["positions"])
    return _written(s)


def _own_cache_read(s, h):
    h["cache"].read(h["tables"], h["sequences"], h["positions"], out=(h["key"], h["value"]))
    return {"key": s["key"], "value": s["value"]}


def _own_attend(s, h):
    h["cache"].attend(h["query"], h["tables"], h["lengths"], out=h["out"])
    return s["out"]


def _own_adapted(s, h):
    _session.linear_adapted(h["x"], h["weight"], h["pool"], h["adapters"], h["bias"], out=h["out"])
    return s["out"]


_OWN = {"norm_rope": _own_norm_rope, "cache_write": _own_cache_write, "cache_read": _own_cache_read, "attend": _own_attend, "adapted": _own_adapted}


# ------------------------------------------------------------------ plain forms


def _plain_norm_rope(s):
    c = s["case"]
    rows, heads, kv_heads, width = c["rows"], c["heads"], c["kv_heads"], c["width"]
    half = width // 2
    frequency = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 * math.log(_THETA) / width))
    angle = s["positions"].double().unsqueeze(1) * frequency
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)

    def turned(x, weight):
        x = x.reshape(rows, -1, width)
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    return {"q": turned(s["fused"][:, :heads * width], s["q_weight"]),
            "k": turned(s["fused"][:, heads * width:(heads + kv_heads) * width], s["k_weight"])}


def _places(s):
    page = s["case"]["page"]
    at = s["positions"].long()
    return s["tables"][s["sequences"].long(), at // page].long(), at % page


def _plain_cache_write(s):
    pages, slots = _places(s)
    if s["case"]["dtype"] == "E4M3":
        (k, ke), (v, ve) = _quantise(s["key"]), _quantise(s["value"])
        s["keys"].view(torch.uint8)[pages, :, slots] = k.view(torch.uint8)
        s["values"].view(torch.uint8)[pages, :, slots] = v.view(torch.uint8)
        s["key_scales"][pages, :, slots], s["value_scales"][pages, :, slots] = ke, ve
    else:
        s["keys"][pages, :, slots] = s["key"].to(s["keys"].dtype)
        s["values"][pages, :, slots] = s["value"].to(s["values"].dtype)
    return _written(s)


def _widened(data, scales):
    """Float32 values of gathered cache rows."""
    if scales is None:
        return data.float()
    return torch.ldexp(data.view(torch.float8_e4m3fn).float(), scales.int().unsqueeze(-1) - 127)


def _gathered(s, name, *where):
    """Cache rows at `where`, in Float32."""
    data, scales = s[name + "s"], s.get(name + "_scales")
    if scales is not None:
        data, scales = data.view(torch.uint8), scales[where]
    return _widened(data[where], scales)


def _plain_cache_read(s):
    pages, slots = _places(s)
    every = torch.arange(s["case"]["kv_heads"], device="cuda")
    where = (pages.unsqueeze(1), every, slots.unsqueeze(1))
    return {"key": _gathered(s, "key", *where), "value": _gathered(s, "value", *where)}


def _plain_attend(s):
    c = s["case"]
    batch, heads, kv_heads, width = c["batch"], c["heads"], c["kv_heads"], c["width"]
    pages = s["tables"].long().clamp(min=0)
    keys, values = (_gathered(s, n, pages).transpose(1, 2).reshape(batch, kv_heads, -1, width) for n in ("key", "value"))
    q = s["query"].reshape(batch, kv_heads, heads // kv_heads, width)
    scores = torch.matmul(q, keys.transpose(2, 3)) / math.sqrt(width)
    seen = torch.arange(keys.shape[2], device="cuda") < s["lengths"].unsqueeze(1)
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p, values) / torch.where(total > 0, total, torch.ones_like(total))
    return y.reshape(batch, heads, width)


def _plain_adapted(s):
    rank = s["case"]["rank"]
    slot = s["adapters"].long().clamp(min=0)
    base = torch.matmul(s["x"], s["weight"].float().t())
    thin = torch.matmul(s["a"][slot].float(), s["x"].unsqueeze(2)).squeeze(2)
    thin = thin * (torch.arange(rank, device="cuda") < s["ranks"][slot].unsqueeze(1))
    delta = torch.matmul(s["b"][slot].float(), thin.unsqueeze(2)).squeeze(2)
    factor = torch.where(s["adapters"] >= 0, s["scales"][slot], torch.zeros_like(s["scales"][slot]))
    return base + delta * factor.unsqueeze(1) + s["bias"]


_PLAIN = {"norm_rope": _plain_norm_rope, "cache_write": _plain_cache_write, "cache_read": _plain_cache_read, "attend": _plain_attend, "adapted": _plain_adapted}


# ------------------------------------------------------------------ definitions in 64 bits


def _e4m3_grid(y):
    """The nearest E4M3 value of each float64 (ties to even): spacing 2^(e - 3) in the binade 2^e, e >= -6."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    e = torch.where(y.abs() >= torch.exp2(e + 1), e + 1, torch.where(y.abs() < torch.exp2(e), e - 1, e)).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm_rope":
        heads, width = case["heads"], case["width"]
        x = s["fused"].double().reshape(case["rows"], -1, width)
        d = torch.arange(width // 2, device="cuda", dtype=torch.float64)
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * _THETA ** (-2 * d / width))
        got = {}
        for name, part, weight in (("q", x[:, :heads], s["q_weight"]), ("k", x[:, heads:heads + case["kv_heads"]], s["k_weight"])):
            y = part * torch.rsqrt(part.square().sum(-1, keepdim=True) / width + _EPS) * weight.double()
            z = torch.complex(y[..., :width // 2].contiguous(), y[..., width // 2:].contiguous()) * turn[:, None, :]
            got[name] = torch.cat((z.real, z.imag), -1)
        return got
    if op in ("cache_write", "cache_read"):
        page = case["page"]
        row_page = s["tables"][s["sequences"].long(), (s["positions"] // page).long()].long()
        row_slot = (s["positions"] % page).long()
        got = {}
        for name in ("key", "value"):
            data, scales = s[name + "s"].double(), s.get(name + "_scales")
            if op == "cache_read":
                if scales is not None:
                    data = data * torch.exp2(scales.double() - 127).unsqueeze(-1)
                got[name] = data[row_page, :, row_slot]
                continue
            x = s[name].double()
            if scales is not None:
                top = x.abs().amax(-1, keepdim=True).clamp(min=1e-300)
                e = torch.ceil(torch.log2(top / 448))
                e = torch.where(torch.exp2(e) * 448 < top, e + 1, torch.where(torch.exp2(e - 1) * 448 >= top, e - 1, e))
                x = _e4m3_grid(x * torch.exp2(-e))
                got[name + "_scales"] = None
            data[row_page, :, row_slot] = x
            got[name + "s"] = data
        return got
    if op == "attend":
        y = torch.zeros(case["batch"], case["heads"], case["width"], dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for i, n in enumerate(s["lengths"].tolist()):
            if n == 0:
                continue
            pages = s["tables"][i, : -(-n // case["page"])].long()
            got = []
            for name in ("key", "value"):
                x = s[name + "s"][pages].double()
                if s.get(name + "_scales") is not None:
                    x = x * torch.exp2(s[name + "_scales"][pages].double() - 127).unsqueeze(-1)
                got.append(x.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["width"])[:, :n])
            k, v = got
            score = torch.einsum("hgd,hnd->hgn", s["query"][i].double().reshape(-1, group, case["width"]), k) * case["width"] ** -0.5
            y[i] = torch.einsum("hgn,hnd->hgd", torch.softmax(score, -1), v).reshape(case["heads"], -1)
        return y
    y = s["x"].double() @ s["weight"].double().t()
    for i, slot in enumerate(s["adapters"].tolist()):
        if slot >= 0:
            r = int(s["ranks"][slot])
            y[i] += s["scales"][slot].double() * (s["b"][slot, :, :r].double() @ (s["a"][slot, :r].double() @ s["x"][i].double()))
    return y + s["bias"].double()
