"""Cases for the serving operators: the paged MX key / value cache, attention over a shared prefix, 4-bit weights.

`listed()` are the cases, `draw()` gives more of the same ranges, `prepare()` makes what a serving program has in hand
before the call, `run()` makes one pass: in elementary torch operations, or, with `own` set, through pto_isa_b200."""
import math

import torch

own = False

FORMATS = {"f16": 0, "bf16": 1, "mxfp8": 2, "mxfp4": 3}  # ops.KV_F16, KV_BF16, KV_MXFP8, KV_MXFP4
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # a decode step of a small batch: one new row a sequence, short contexts handed on in 16 bits
        {"name": "cache_small", "op": "cache", "dtype": "bf16", "fmt": "mxfp8", "batch": 4, "kv_heads": 2, "d": 64,
         "page": 16, "new": 1, "length": 100},
        # chunked prefill: a chunk of every prompt is appended, then the context is read back for the prefill attention
        {"name": "cache_chunk_fp8", "op": "cache", "dtype": "f16", "fmt": "mxfp8", "batch": 8, "kv_heads": 8, "d": 128,
         "page": 64, "new": 512, "length": 4096},
        # the same at four bits, odd chunk and context lengths, pages that end inside every tile
        {"name": "cache_chunk_fp4", "op": "cache", "dtype": "bf16", "fmt": "mxfp4", "batch": 13, "kv_heads": 4, "d": 128,
         "page": 16, "new": 77, "length": 2041},
        # the smallest decode: one request behind a short system prompt, unquantised cache
        {"name": "attn_one_f16", "op": "attn", "dtype": "f16", "fmt": "f16", "batch": 1, "tokens": 1, "heads": 8,
         "kv_heads": 8, "d": 64, "page": 16, "prefix": 512, "own_len": 64, "empty": False},
        # ordinary serving: a batch of chats behind one system prompt, 8-bit cache
        {"name": "attn_chat_fp8", "op": "attn", "dtype": "bf16", "fmt": "mxfp8", "batch": 32, "tokens": 1, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "prefix": 4096, "own_len": 512, "empty": False},
        # verifying four drafted tokens a sequence, odd lengths, sequences that have no key of their own yet
        {"name": "attn_draft_fp8", "op": "attn", "dtype": "f16", "fmt": "mxfp8", "batch": 24, "tokens": 4, "heads": 16,
         "kv_heads": 2, "d": 128, "page": 16, "prefix": 1999, "own_len": 301, "empty": True},
        # a large batch of samples of one long prompt, unquantised cache: many rows a key
        {"name": "attn_samples_f16", "op": "attn", "dtype": "f16", "fmt": "f16", "batch": 128, "tokens": 1, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 128, "prefix": 8192, "own_len": 512, "empty": False},
        # questions about one long document, 4-bit cache
        {"name": "attn_document_fp4", "op": "attn", "dtype": "bf16", "fmt": "mxfp4", "batch": 16, "tokens": 1, "heads": 64,
         "kv_heads": 8, "d": 128, "page": 64, "prefix": 32768, "own_len": 1024, "empty": False},
        # one token through a small projection
        {"name": "w4_small_int4", "op": "w4", "dtype": "f16", "fmt": "int4", "m": 1, "n": 1536, "k": 1536, "group": 128,
         "zero": False, "out32": False},
        # one token through a large projection, the weights of the MX fp4 product
        {"name": "w4_one_mxfp4", "op": "w4", "dtype": "bf16", "fmt": "mxfp4", "m": 1, "n": 8192, "k": 8192, "group": 32,
         "zero": False, "out32": False},
        # a small batch through an up projection, zero points
        {"name": "w4_batch_int4", "op": "w4", "dtype": "bf16", "fmt": "int4", "m": 7, "n": 16384, "k": 4096, "group": 64,
         "zero": True, "out32": False},
        # sixteen rows into the logits of a vocabulary of odd size, in 32 bits
        {"name": "w4_logits_mxfp4", "op": "w4", "dtype": "f16", "fmt": "mxfp4", "m": 16, "n": 32003, "k": 4096, "group": 32,
         "zero": False, "out32": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cache", "attn", "attn", "w4"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "cache":
        while True:
            c = {"op": op, "dtype": dtype, "fmt": rng.choice([dtype, "mxfp8", "mxfp4"]), "batch": _log(rng, 1, 32),
                 "kv_heads": rng.choice([1, 2, 3, 4, 8]), "d": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128]),
                 "new": _log(rng, 1, 512), "length": _log(rng, 16, 4096)}
            c["new"] = min(c["new"], c["length"] // 2 + 1)
            if c["batch"] * c["kv_heads"] * c["d"] * c["length"] <= 8 * 8 * 128 * 4096:
                return c
    if op == "attn":
        while True:
            kv_heads = rng.choice([1, 2, 4, 8])
            c = {"op": op, "dtype": dtype, "fmt": rng.choice([dtype, "mxfp8", "mxfp4"]), "batch": _log(rng, 1, 160),
                 "tokens": rng.choice([1, 1, 1, 2, 5]), "heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 16]),
                 "kv_heads": kv_heads, "d": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128]),
                 "prefix": rng.choice([0, _log(rng, 1, 32768), _log(rng, 64, 32768)]), "own_len": _log(rng, 1, 2048),
                 "empty": rng.random() < 0.3}
            rows = c["batch"] * c["tokens"] * c["heads"]
            keys = c["batch"] * c["kv_heads"] * c["own_len"]
            if rows * c["d"] * (c["prefix"] + c["own_len"]) <= 4096 * 128 * 8704 and keys <= 128 * 8 * 512:
                return c
    fmt = rng.choice(["int4", "mxfp4"])
    group = 32 if fmt == "mxfp4" else rng.choice([32, 64, 128])
    while True:
        c = {"op": op, "dtype": dtype, "fmt": fmt, "m": _log(rng, 1, 16), "n": _log(rng, 64, 32000),
             "k": group * _log(rng, max(2, 256 // group), 12288 // group), "group": group,
             "zero": fmt == "int4" and rng.random() < 0.5, "out32": rng.random() < 0.3}
        if c["n"] * c["k"] <= 32003 * 4096:
            return c


def _own_mean(c):
    mean = 0.75 * c["own_len"]
    return mean * (c["batch"] - 1) / c["batch"] if c["empty"] and c["batch"] > 1 else mean


def work(c):
    per = {"f16": 2.0, "bf16": 2.0, "mxfp8": 1.0 + 1 / 32, "mxfp4": 0.5 + 1 / 32}
    if c["op"] == "cache":
        new = c["batch"] * c["new"] * c["kv_heads"] * c["d"] * 2
        live = 0.75 * c["batch"] * c["length"] * c["kv_heads"] * c["d"] * 2
        out = c["batch"] * c["length"] * c["kv_heads"] * c["d"] * 2 * 2
        return {"bytes": new * (2 + per[c["fmt"]]) + live * per[c["fmt"]] + out, "flops": 0}
    if c["op"] == "attn":
        rows = c["batch"] * c["tokens"] * c["heads"]
        keys = c["kv_heads"] * (c["prefix"] + c["batch"] * _own_mean(c))
        return {"bytes": keys * c["d"] * 2 * per[c["fmt"]] + rows * (c["d"] * 4 + 4),
                "flops": 4.0 * c["d"] * rows * (c["prefix"] + _own_mean(c))}
    scale = 1 if c["fmt"] == "mxfp4" else 4 if c["zero"] else 2
    return {"bytes": c["n"] * (c["k"] / 2 + scale * c["k"] / c["group"]) + c["m"] * (c["k"] * 2 + c["n"] * (4 if c["out32"] else 2)),
            "flops": 2.0 * c["m"] * c["n"] * c["k"]}


# ------------------------------------------------------------------------------------- the MX block format


def _encode(x, fmt):
    """Codes (one a byte, unpacked) and scale bytes of the last dimension's blocks of 32."""
    limit, half, shift, most = (448.0, 0.875, 9, 119) if fmt == "mxfp8" else (6.0, 0.75, 3, 125)
    x = x.to(torch.float64).unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], 0.0, x)
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    e = torch.where(mantissa <= half, exponent - shift, exponent - shift + 1)
    e = torch.where(mantissa == 0, -127, e).clamp(-127, most)
    y = (x * torch.exp2(-e.to(torch.float64))[..., None]).clamp(-limit, limit)
    if fmt == "mxfp8":
        codes = y.float().to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = y.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        a = torch.round(a / step) * step
        codes = torch.where(a <= 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    return codes.flatten(-2), torch.where(bad, 255, e + 127).to(torch.uint8)


def _pack(codes, fmt):
    return codes if fmt == "mxfp8" else codes[..., 0::2] | (codes[..., 1::2] << 4)


def _decode(codes, scale, fmt):
    """What packed codes and scale bytes stand for, in 32 bits."""
    if fmt == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
        v = torch.tensor(E2M1, device=codes.device)[(codes & 7).long()]
        v = torch.where(codes >= 8, -v, v)
    s = torch.where(scale == 255, torch.nan, torch.exp2(scale.double() - 127)).to(torch.float32)
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _rows(data, scale, fmt, pages, within):
    """Cached rows (..., kv_heads, d) at (page, position within it), in 32 bits."""
    at = data[pages, :, within]
    return at.float() if fmt in DTYPES else _decode(at, scale[pages, :, within], fmt)


# ------------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _heads_like(g, shape, dtype):
    """Keys / values as projections give them: some channels larger than the rest."""
    gain = torch.exp(0.5 * torch.randn(shape[-2:], generator=g, device="cuda"))
    return (torch.randn(shape, generator=g, device="cuda") * gain).to(dtype)


def _empty_cache(c, pages):
    """A cache as allocated: what no row was written to holds arbitrary bytes, NaN among them."""
    shape, fmt = (pages, c["kv_heads"], c["page"]), c["fmt"]
    if fmt in DTYPES:
        return [torch.full((*shape, c["d"]), torch.nan, dtype=DTYPES[fmt], device="cuda") for _ in range(2)] + [None, None]
    width = c["d"] if fmt == "mxfp8" else c["d"] // 2
    return [torch.full((*shape, width), 255, dtype=torch.uint8, device="cuda") for _ in range(2)] + \
        [torch.full((*shape, c["d"] // 32), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]


def _put(data, scale, fmt, x, pages, within):
    if fmt in DTYPES:
        data[pages, :, within] = x.to(data.dtype)
        return
    codes, s = _encode(x, fmt)
    data[pages, :, within] = _pack(codes, fmt)
    scale[pages, :, within] = s


def _lengths(g, most, batch):
    n = torch.randint(most - most // 2, most + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = most
    return n


def _table(g, batch, per, first=0):
    """A page table over shuffled pages first .. first + batch * per - 1."""
    return (first + torch.randperm(batch * per, generator=g, device="cuda")).to(torch.int32).view(batch, per)


def _fill(c, cache, g, table, total):
    """Writes `total` rows through `table` (n, pages)."""
    t = torch.arange(total, device="cuda")
    for row in table:
        pages, within = row[t // c["page"]].long(), t % c["page"]
        for data, scale in zip(cache[:2], cache[2:]):
            _put(data, scale, c["fmt"], _heads_like(g, (total, c["kv_heads"], c["d"]), DTYPES[c["dtype"]]), pages, within)


def prepare(c, seed):
    g = _generator(seed)
    if c["op"] == "cache":
        per = -(-c["length"] // c["page"])
        table, n = _table(g, c["batch"], per), _lengths(g, c["length"], c["batch"])
        cache = _empty_cache(c, c["batch"] * per)
        _fill(c, cache, g, table, c["length"])
        # the new rows are the last `new` positions of every sequence, as slices of one fused projection's output
        t = n[:, None] - c["new"] + torch.arange(c["new"], device="cuda", dtype=torch.int32)
        slots = table.gather(1, (t.clamp(min=0) // c["page"]).long()) * c["page"] + t.clamp(min=0) % c["page"]
        slots = torch.where(t < 0, -1, slots).flatten().to(torch.int32)
        fused = _heads_like(g, (slots.numel(), 3 * c["kv_heads"], c["d"]), DTYPES[c["dtype"]])
        return {"case": c, "cache": (*cache, FORMATS[c["fmt"]]), "table": table, "lengths": n, "slots": slots,
                "k": fused[:, c["kv_heads"]:2 * c["kv_heads"]], "v": fused[:, 2 * c["kv_heads"]:]}
    if c["op"] == "attn":
        shared, per = -(-c["prefix"] // c["page"]), -(-c["own_len"] // c["page"])
        cache = _empty_cache(c, shared + c["batch"] * per)
        prefix_pages, table = _table(g, 1, shared)[0], _table(g, c["batch"], per, shared)
        if c["prefix"]:
            _fill(c, cache, g, prefix_pages[None], c["prefix"])
        _fill(c, cache, g, table, c["own_len"])
        n = _lengths(g, c["own_len"], c["batch"])
        if c["empty"] and c["batch"] > 1:
            n[1] = 0
        q = torch.randn(c["batch"], c["tokens"], c["heads"], c["d"], generator=g, device="cuda").to(DTYPES[c["dtype"]])
        return {"case": c, "cache": (*cache, FORMATS[c["fmt"]]), "prefix_pages": prefix_pages, "table": table, "lengths": n, "q": q}
    x = torch.randn(c["m"], c["k"], generator=g, device="cuda").to(DTYPES[c["dtype"]])
    w = torch.randint(0, 256, (c["n"], c["k"] // 2), generator=g, device="cuda", dtype=torch.uint8)
    groups = (c["n"], c["k"] // c["group"])
    if c["fmt"] == "mxfp4":
        scale, zero = torch.randint(115, 124, groups, generator=g, device="cuda", dtype=torch.uint8), None
    else:
        scale = (torch.rand(groups, generator=g, device="cuda") * 0.01 + 0.002).to(DTYPES[c["dtype"]])
        zero = torch.randint(5, 12, groups, generator=g, device="cuda").to(DTYPES[c["dtype"]]) if c["zero"] else None
    return {"case": c, "x": x, "w": w, "scale": scale, "zero": zero}


# ------------------------------------------------------------------------------------- one pass


def run(s):
    c = s["case"]
    return {"cache": _run_cache, "attn": _run_attn, "w4": _run_w4}[c["op"]](s, c)


def _run_cache(s, c):
    dtype = DTYPES[c["dtype"]]
    if own:
        import pto_isa_b200 as pto
        pto.kv_cache_write(s["cache"], s["k"], s["v"], s["slots"])
        return pto.kv_cache_read(s["cache"], s["table"], s["lengths"], c["length"], dtype=dtype)
    k, v, k_scale, v_scale, _ = s["cache"]
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    _put(k, k_scale, c["fmt"], s["k"][live], slots // c["page"], slots % c["page"])
    _put(v, v_scale, c["fmt"], s["v"][live], slots // c["page"], slots % c["page"])
    t = torch.arange(c["length"], device="cuda")
    pages = s["table"][:, t // c["page"]].long()
    seen = (t < s["lengths"][:, None])[..., None, None]
    out = [torch.where(seen, _rows(data, scale, c["fmt"], pages, (t % c["page"]).expand_as(pages)), 0.0) for data, scale in ((k, k_scale), (v, v_scale))]
    return tuple(x.transpose(1, 2).to(dtype).contiguous() for x in out)


def _run_attn(s, c):
    if own:
        import pto_isa_b200 as pto
        return pto.prefix_attn(s["q"], s["cache"], s["prefix_pages"], c["prefix"], s["table"], s["lengths"], return_lse=True)
    k, v, k_scale, v_scale, _ = s["cache"]
    batch, tokens, kv, d = c["batch"], c["tokens"], c["kv_heads"], c["d"]
    g = c["heads"] // kv
    # (kv head, batch, token x group, d)
    q = (s["q"].float() * d ** -0.5).view(batch, tokens, kv, g, d).permute(2, 0, 1, 3, 4).reshape(kv, batch, tokens * g, d)
    t = torch.arange(c["prefix"], device="cuda")
    pages = s["prefix_pages"].long()[t // c["page"]]
    pk, pv = (_rows(data, scale, c["fmt"], pages, t % c["page"]).transpose(0, 1) for data, scale in ((k, k_scale), (v, v_scale)))
    t = torch.arange(c["own_len"], device="cuda")
    pages = s["table"].long()[:, t // c["page"]]
    ok, ov = (_rows(data, scale, c["fmt"], pages, (t % c["page"]).expand_as(pages)).permute(2, 0, 1, 3) for data, scale in ((k, k_scale), (v, v_scale)))
    behind = torch.arange(tokens, device="cuda") - (tokens - 1)
    limit = (s["lengths"][:, None] + behind).repeat_interleave(g, 1)  # (batch, token x group)
    seen = t < limit[..., None]
    live = (t < s["lengths"][:, None])[None, ..., None]
    ok, ov = torch.where(live, ok, 0.0), torch.where(live, ov, 0.0)
    x = torch.cat([torch.matmul(q.flatten(1, 2), pk.transpose(1, 2)).view(kv, batch, tokens * g, -1),
                   torch.where(seen, torch.matmul(q, ok.transpose(2, 3)), -torch.inf)], -1)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., :c["prefix"]].flatten(1, 2), pv).view_as(q) + torch.matmul(p[..., c["prefix"]:], ov)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (torch.log(total) + top)[..., 0]
    o = o.view(kv, batch, tokens, g, d).permute(1, 2, 0, 3, 4).reshape(batch, tokens, c["heads"], d)
    return o.to(DTYPES[c["dtype"]]), lse.view(kv, batch, tokens, g).permute(1, 2, 0, 3).reshape(batch, tokens, c["heads"])


def _run_w4(s, c):
    out = torch.float32 if c["out32"] else DTYPES[c["dtype"]]
    if own:
        import pto_isa_b200 as pto
        return pto.w4_matvec(s["x"], s["w"], s["scale"], zero=s["zero"], out_dtype=out)
    if c["fmt"] == "mxfp4":
        w = _decode(s["w"], s["scale"], "mxfp4")
    else:
        w = torch.stack([s["w"] & 15, s["w"] >> 4], -1).flatten(-2).float().unflatten(-1, (-1, c["group"]))
        w = ((w - (s["zero"].float()[..., None] if c["zero"] else 8.0)) * s["scale"].float()[..., None]).flatten(-2)
    return torch.matmul(s["x"].float(), w.t()).to(out)


# ------------------------------------------------------------------------------------- the definition in 64 bits


def _values64(data, scale, fmt):
    """All that a cache holds, (pages, kv_heads, page, d), from tables of the formats' values."""
    if fmt in DTYPES:
        return data.double()
    i = torch.arange(256)
    if fmt == "mxfp8":
        e, m = (i >> 3) & 15, i & 7
        table = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.pow(torch.tensor(2.0, dtype=torch.float64), e - 10.0))
        table[(i & 127) == 127] = torch.nan
        table = torch.where(i >= 128, -table, table).double().cuda()
        v = table[data.long()]
    else:
        table = torch.tensor(E2M1 + [-x for x in E2M1], dtype=torch.float64, device="cuda")
        v = torch.empty(*data.shape[:-1], data.shape[-1] * 2, dtype=torch.float64, device="cuda")
        v[..., 0::2], v[..., 1::2] = table[(data % 16).long()], table[(data // 16).long()]
    powers = torch.pow(torch.tensor(2.0, dtype=torch.float64), torch.arange(256) - 127.0)
    powers[255] = torch.nan
    return v * powers.cuda()[scale.long()].repeat_interleave(32, -1)


def _nearest64(x, fmt):
    """Rows (..., d) as the format holds them: the scale by comparing with every power, the code by distance."""
    grid = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119]
                        if fmt == "mxfp8" else E2M1, dtype=torch.float64, device="cuda")
    powers = torch.pow(torch.tensor(2.0, dtype=torch.float64, device="cuda"), torch.arange(-127, 120 if fmt == "mxfp8" else 126, device="cuda"))
    x = x.double().unflatten(-1, (-1, 32))
    s = powers[torch.searchsorted(powers * grid[-1], x.abs().amax(-1)).clamp(max=powers.numel() - 1)][..., None]
    a = (x.abs() / s).clamp(max=float(grid[-1]))
    above = torch.searchsorted(grid, a).clamp(max=grid.numel() - 1)
    below = (above - 1).clamp(min=0)
    up, down = grid[above] - a, a - grid[below]
    pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return (torch.sign(x) * grid[pick] * s).flatten(-2)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "w4":
        low, high = (s["w"] % 16).double(), (s["w"] // 16).double()
        codes = torch.stack((low, high), 2).reshape(c["n"], c["k"])
        per = c["group"]
        if c["fmt"] == "mxfp4":
            w = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device="cuda")[codes.long()]
            w *= torch.pow(2.0, s["scale"].double() - 127).repeat_interleave(per, 1)
        else:
            w = codes - (s["zero"].double().repeat_interleave(per, 1) if c["zero"] else 8)
            w *= s["scale"].double().repeat_interleave(per, 1)
        return s["x"].double() @ w.t()
    k, v, k_scale, v_scale, _ = s["cache"]
    kd, vd = _values64(k, k_scale, c["fmt"]), _values64(v, v_scale, c["fmt"])
    ps = c["page"]

    def rows(data, pages, n):  # (kv_heads, n, d)
        return data[pages.long()].transpose(0, 1).reshape(c["kv_heads"], -1, c["d"])[:, :n]

    if c["op"] == "cache":
        out = []
        for data, new in ((kd, s["k"]), (vd, s["v"])):
            new = new.double() if c["fmt"] in DTYPES else _nearest64(new, c["fmt"])
            flat = data.transpose(1, 2).reshape(-1, c["kv_heads"], c["d"]).clone()
            flat[s["slots"][s["slots"] >= 0].long()] = new[s["slots"] >= 0]
            data = flat.view(-1, ps, c["kv_heads"], c["d"]).transpose(1, 2)
            o = torch.zeros(c["batch"], c["kv_heads"], c["length"], c["d"], dtype=torch.float64, device="cuda")
            for b, n in enumerate(s["lengths"].tolist()):
                o[b, :, :n] = rows(data, s["table"][b], n)
            out.append(o)
        return tuple(out)
    g = c["heads"] // c["kv_heads"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:-1], -torch.inf, dtype=torch.float64, device="cuda")
    pk, pv = rows(kd, s["prefix_pages"], c["prefix"]), rows(vd, s["prefix_pages"], c["prefix"])
    for b, n in enumerate(s["lengths"].tolist()):
        for j in range(c["tokens"]):
            left = max(0, n - (c["tokens"] - 1 - j))
            if c["prefix"] + left == 0:
                continue
            kk = torch.cat([pk, rows(kd, s["table"][b], left)], 1)
            vv = torch.cat([pv, rows(vd, s["table"][b], left)], 1)
            x = torch.einsum("hgd,hkd->hgk", s["q"][b, j].double().view(-1, g, c["d"]), kk) / math.sqrt(c["d"])
            lse[b, j] = torch.logsumexp(x, -1).flatten()
            o[b, j] = torch.einsum("hgk,hkd->hgd", torch.softmax(x, -1), vv).reshape(-1, c["d"])
    return o, lse
