"""The serving operators against 64-bit statements of them (tests/serving_ref.py): the paged cache in its four formats,
attention over a shared prefix, products with 4-bit weights, and a decode step that runs them together."""
import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
FORMATS = ["16", "mxfp8", "mxfp4"]


def fmt_of(name, dtype):
    import pto_isa_b200 as p
    return {"16": p.KV_F16 if dtype == F16 else p.KV_BF16, "mxfp8": p.KV_MXFP8, "mxfp4": p.KV_MXFP4}[name]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def status():
    import pto_isa_b200 as p
    torch.cuda.synchronize()
    return p.device_status_record()


def garbage_cache(pages, heads, page, d, fmt):
    """A cache whose every byte is 0xff: NaN in 16 bits, NaN codes, NaN scales."""
    import pto_isa_b200 as p
    c = p.kv_cache_empty(pages, heads, page, d, fmt)
    for t in c[:4]:
        if t is not None:
            t.view(torch.uint8).fill_(255)
    return c


def values(c):
    """All cached values (pages, kv_heads, page, d) as (K, V) in 64 bits, on the host."""
    import pto_isa_b200 as p
    if c.fmt in (p.KV_F16, p.KV_BF16):
        return c.k.double().cpu(), c.v.double().cpu()
    fp4 = c.fmt == p.KV_MXFP4
    return ref.decode(c.k, c.k_scale, fp4), ref.decode(c.v, c.v_scale, fp4)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=123.0), torch.nan_to_num(b, nan=123.0)) and torch.equal(a.isnan(), b.isnan())


# --------------------------------------------------------------------------------------------------- the cache


def odd_rows(n, heads, d, dtype, seed):
    """Rows with what quantisation can go wrong on: zeros, ties, largest and smallest values, outliers, NaN, infinities."""
    x = torch.randn(n, heads, d, generator=gen(seed), device="cuda") * torch.exp2(torch.randint(-12, 8, (n, heads, 1), generator=gen(seed + 1), device="cuda").float())
    x = x.to(dtype)
    flat = x.view(-1, 32)
    top = torch.finfo(dtype).max
    small = 2.0 ** -24 if dtype == F16 else 2.0 ** -133
    specials = [torch.zeros(32), torch.full((32,), -0.0), torch.arange(32) * 0.25 - 4, torch.arange(32) * 1.0, torch.full((32,), top),
                torch.cat([torch.tensor([448.0, -448.0, 6.0, 5.0, 3.5, 2.5]), torch.ones(26)]), torch.arange(32) * small,
                torch.cat([torch.tensor([top, small]), torch.zeros(30)]), torch.cat([torch.tensor([float("nan")]), torch.ones(31)]),
                torch.cat([torch.ones(31), torch.tensor([float("-inf")])]), torch.cat([torch.tensor([449.0]), torch.linspace(-1, 1, 31)]),
                torch.cat([torch.tensor([6.25, 0.25, 0.75, 1.25, 1.75]), torch.zeros(27)])]
    for i, s in enumerate(specials):
        flat[(i * 7) % flat.shape[0]] = s.to(dtype).cuda()
    return x


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", FORMATS)
def test_cache_write_is_the_format_bit_for_bit(name, d, dtype):
    import pto_isa_b200 as p
    heads, page, pages, n = 3, 16, 5, 37
    fmt = fmt_of(name, dtype)
    c = garbage_cache(pages, heads, page, d, fmt)
    fused = torch.cat([torch.zeros(n, 1, d, dtype=dtype, device="cuda"), odd_rows(n, heads, d, dtype, 1), odd_rows(n, heads, d, dtype, 9)], 1)
    k, v = fused[:, 1:1 + heads], fused[:, 1 + heads:]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(2))[:n].to(torch.int32)
    slots[5] = -1
    slots[20] = -2 ** 31
    assert p.kv_cache_write(c, k, v, slots.cuda()) is c
    got = [x.transpose(1, 2).reshape(-1, heads, d) for x in values(c)]
    for have, rows in zip(got, (k, v)):
        want = rows.double().cpu()
        if name != "16":
            want = torch.tensor([ref.quantise_block(b, name == "mxfp4")[0] for b in rows.float().cpu().reshape(-1, 32).tolist()], dtype=torch.float64).view(n, heads, d)
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                assert same(have[s], want[i]), (i, s)
    untouched = sorted(set(range(pages * page)) - set(slots.tolist()))  # every other row still holds 0xff bytes
    for t in c[:4]:
        if t is not None:
            assert (t.transpose(1, 2).reshape(pages * page, heads, -1).contiguous().view(torch.uint8)[untouched] == 255).all()
    assert status()[0] == 0


@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (F16, BF16), (BF16, F16)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", FORMATS)
def test_cache_read(name, d, dtype, out):
    import pto_isa_b200 as p
    heads, page, per, max_len = 2, 32, 3, 71
    lens = torch.tensor([71, 0, 1, 32, 33, -4, 500], dtype=torch.int32)
    batch = len(lens)
    c = garbage_cache(batch * per, heads, page, d, fmt_of(name, dtype))
    n = batch * per * page
    x = [torch.randn(n, heads, d, generator=gen(s), device="cuda").to(dtype) * 3 for s in (3, 4)]
    p.kv_cache_write(c, *x, torch.arange(n, dtype=torch.int32, device="cuda"))
    table = torch.randperm(batch * per, generator=torch.Generator().manual_seed(5)).view(batch, per).to(torch.int32)
    wide = torch.full((batch, per + 2), -7, dtype=torch.int32)
    wide[:, :per] = table
    k, v = p.kv_cache_read(c, wide.cuda()[:, :per], lens.cuda(), max_len, dtype=out)  # rows of a wider table
    for got, all_ in zip((k, v), values(c)):
        want = torch.zeros(batch, heads, max_len, d, dtype=out)
        for b in range(batch):
            live = max(0, min(int(lens[b]), max_len))
            want[b, :, :live] = all_[table[b].long()].transpose(0, 1).reshape(heads, -1, d)[:, :live].to(out)
        assert torch.equal(got.cpu(), want)
    assert status()[0] == 0
    pair = (torch.empty_like(k), torch.empty_like(v))
    again = p.kv_cache_read(c, wide.cuda()[:, :per], lens.cuda(), max_len, dtype=out, out=pair)
    assert again[0] is pair[0] and torch.equal(pair[0], k) and torch.equal(pair[1], v)


def test_cache_bad_indices_touch_nothing_and_are_reported():
    import pto_isa_b200 as p
    c = garbage_cache(2, 1, 16, 64, p.KV_MXFP8)
    x = torch.ones(3, 1, 64, dtype=F16, device="cuda")
    p.kv_cache_write(c, x, x, torch.tensor([0, 32, 31], dtype=torch.int32, device="cuda"))
    assert status() == (1, 0, 10, 32) and status()[0] == 0
    table = torch.tensor([[0, 2], [-1, 1]], dtype=torch.int32, device="cuda")
    k, _ = p.kv_cache_read(c, table, torch.tensor([17, 32], dtype=torch.int32, device="cuda"), 32)
    code, _, where, detail = status()
    assert code == 1 and where == 11 and detail in (2, -1)
    assert (k[0, 0, 0] == 1).all() and (k[0, 0, 16:] == 0).all() and (k[1, 0, :16] == 0).all() and (k[1, 0, 31] == 1).all()
    q = torch.ones(2, 1, 64, dtype=F16, device="cuda")
    one = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    good = torch.tensor([[0], [0]], dtype=torch.int32, device="cuda")
    o = p.prefix_attn(q, c, good[0], 0, torch.tensor([[9], [0]], dtype=torch.int32, device="cuda"), one)
    assert status()[2:] == (11, 9) and (o[0] == 0).all() and (o[1] == 1).all()
    o = p.prefix_attn(q, c, good[0], 0, good, torch.tensor([-3, 1], dtype=torch.int32, device="cuda"))
    assert status()[2:] == (12, -3) and (o[0] == 0).all() and (o[1] == 1).all()
    o = p.prefix_attn(q, c, good[0], 0, good, torch.tensor([1, 17], dtype=torch.int32, device="cuda"), max_seq_len=1)
    assert status()[2:] == (12, 17) and (o == 1).all()
    assert status()[0] == 0


# --------------------------------------------------------------------------------------------------- attention


def make_attention(name, dtype, d, kv_heads, page, prefix, lens, seed, spare=0, scale_k=1.0, extra=0):
    """A cache full of 0xff bytes with the prefix's and the sequences' rows written through a shuffled table."""
    import pto_isa_b200 as p
    batch, most = len(lens), max([0, *lens])
    shared, per = -(-prefix // page), -(-most // page) + spare
    total = shared + batch * per + extra
    c = garbage_cache(max(total, 1), kv_heads, page, d, fmt_of(name, dtype))
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    prefix_pages, table = perm[:shared], perm[shared:shared + batch * per].view(batch, per)

    def put(pages, n, s):
        t = torch.arange(n)
        slots = pages.long()[t // page] * page + t % page
        k, v = (torch.randn(n, kv_heads, d, generator=gen(s + i), device="cuda") for i in (0, 1))
        p.kv_cache_write(c, (k * scale_k).to(dtype), (v + 0.1).to(dtype), slots.to(torch.int32).cuda())
    if prefix:
        put(prefix_pages, prefix, 1000 + seed)
    for b, n in enumerate(lens):
        if n:
            put(table[b], n, 2000 + 17 * b + seed)
    kd, vd = values(c)
    rows = lambda data, pages, n: data[pages.long()].transpose(0, 1).reshape(kv_heads, -1, d)[:, :n].cuda()
    parts = [rows(x, prefix_pages, prefix) if prefix else torch.zeros(kv_heads, 0, d, dtype=torch.float64, device="cuda") for x in (kd, vd)]
    own = [[rows(x, table[b], n) if n else torch.zeros(kv_heads, 0, d, dtype=torch.float64, device="cuda") for b, n in enumerate(lens)] for x in (kd, vd)]
    return c, prefix_pages.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), parts, own


def check_attention(q, c, pages, prefix, table, lens, parts, own, scale=None, **kw):
    import pto_isa_b200 as p
    o, lse = p.prefix_attn(q, c, pages, prefix, table, lens, scale=scale, return_lse=True, **kw)
    q4 = q if q.dim() == 4 else q.unsqueeze(1)
    want, wlse, wv, vsum, qk = ref.attention(q4.double(), *parts, *own, q.shape[-1] ** -0.5 if scale is None else scale)
    keys = prefix + max([0] + [x.shape[1] for x in own[0]])
    ob, lb = ref.attention_bounds(q.dtype, want, wv, vsum, qk, keys, mx=c.fmt >= p.KV_MXFP8)
    o, lse = o.view(q4.shape), lse.view(q4.shape[:-1])
    empty = torch.isinf(wlse)
    assert (o[empty] == 0).all() and (lse[empty] == -torch.inf).all()
    err, lerr = (o.double() - want).abs(), (lse.double() - wlse)[~empty].abs()
    assert (err <= ob).all(), float((err / ob).max())
    assert (lerr <= lb[~empty]).all(), float((lerr / lb[~empty]).max())
    assert status()[0] == 0
    return o, lse


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("prefix,lens,tokens,heads,kv_heads,page", [
    (0, [1], 1, 1, 1, 16), (1, [0], 1, 2, 1, 16), (16, [15, 16, 17], 1, 4, 2, 16), (63, [0, 64, 65, 1], 1, 8, 1, 32),
    (65, [1, 2, 0, 5, 4], 4, 6, 2, 16), (1000, [130, 7, 300], 1, 16, 8, 64), (333, [40, 0, 33], 3, 21, 3, 128),
    (129, [2, 250], 5, 16, 1, 256), (0, [700, 0, 3], 2, 4, 4, 16), (2100, [5] * 40, 1, 8, 2, 64)])
def test_attention(prefix, lens, tokens, heads, kv_heads, page, name, d, dtype):
    made = make_attention(name, dtype, d, kv_heads, page, prefix, lens, 7)
    q = torch.randn(len(lens), tokens, heads, d, generator=gen(11), device="cuda").to(dtype)
    check_attention(q, made[0], made[1], prefix, *made[2:])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", FORMATS)
def test_attention_many_rows(name, dtype):
    """Rows of many sequences over the prefix: whole and ragged row tiles, pieces of uneven length."""
    for batch, tokens, heads, kv_heads, prefix, d in ((70, 1, 8, 2, 1111, 128), (33, 4, 4, 1, 640, 64), (150, 1, 4, 2, 129, 128)):
        lens = [(37 * i) % 90 for i in range(batch)]
        made = make_attention(name, dtype, d, kv_heads, 32, prefix, lens, 13)
        q = torch.randn(batch, tokens, heads, d, generator=gen(12), device="cuda").to(dtype)
        check_attention(q, made[0], made[1], prefix, *made[2:])


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_large_logits_and_scales(name, dtype):
    """Logits of hundreds, a running maximum that keeps growing, a negative and a zero scale; single-token form, strided q."""
    d, prefix, lens = 128, 300, [90, 0, 17]
    made = make_attention(name, dtype, d, 2, 16, prefix, lens, 3, scale_k=6.0)
    fused = torch.randn(3, 14, d, generator=gen(5), device="cuda").to(dtype) * 8
    q = fused[:, 3:11]
    for scale in (None, 1.0, -0.25, 0.0):
        check_attention(q, made[0], made[1], prefix, *made[2:], scale=scale)


def test_attention_small_and_large_cached_values():
    """Blocks far from 1: the scale's power of two outside float16's range for bfloat16 queries, near its ends for float16."""
    import pto_isa_b200 as p
    for dtype, exps in ((BF16, (-60, -20, 0, 20, 60)), (F16, (-12, -6, 0, 4, 8))):
        for name in FORMATS:
            for e in exps:
                d, n = 64, 50
                c = garbage_cache(4, 1, 16, d, fmt_of(name, dtype))
                k, v = (torch.randn(n, 1, d, generator=gen(s), device="cuda") for s in (1, 2))
                v = v * 2.0 ** e
                p.kv_cache_write(c, (k * 2.0 ** -e if dtype == BF16 else k).to(dtype), v.to(dtype), torch.arange(n, dtype=torch.int32, device="cuda"))
                q = torch.randn(2, 3, d, generator=gen(3), device="cuda")
                q = (q * 2.0 ** e if dtype == BF16 else q).to(dtype)
                kd, vd = (x.transpose(0, 1).reshape(1, -1, d)[:, :n].cuda() for x in values(c))
                pages = torch.arange(4, dtype=torch.int32, device="cuda")
                lens = torch.tensor([n, 0], dtype=torch.int32, device="cuda")
                none = torch.zeros(1, 0, d, dtype=torch.float64, device="cuda")
                check_attention(q, c, pages, 0, pages.expand(2, 4).contiguous(), lens, [none, none], [[kd, none], [vd, none]])
                check_attention(q, c, pages, n, pages.expand(2, 4).contiguous(), lens * 0, [kd, vd], [[none] * 2] * 2)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("batch,name", [(20, "16"), (20, "mxfp8"), (20, "mxfp4"), (37, "mxfp8"), (75, "16"), (75, "mxfp4")])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_many_rows_of_any_size(dtype, batch, name, d):
    """Many rows over the prefix (one, two and three tiles of 128): a negative, a zero and a large scale, a maximum that keeps
    growing along the keys, cached values far from 1 in some tiles of the prefix only, rows of q of very different sizes."""
    heads, kv, prefix = 8, 2, 700
    for at, (ek, ev) in enumerate(((0, 0), (-30, 0), (30, 0), (0, 30), (0, -30), (0, -10), (0, 6))):
        if dtype == F16 and (abs(ek) > 8 or abs(ev) > 10):
            continue
        made = make_attention(name, dtype, d, kv, 32, prefix, [3] * batch, 40 + at)
        c, pages, table, lens, parts, own = made
        t = torch.arange(150, 420)  # two whole tiles and parts of two
        slots = (pages[(t // 32).cuda()].long() * 32 + t.cuda() % 32).to(torch.int32)
        k, v = (torch.randn(len(t), kv, d, generator=gen(s), device="cuda") * torch.linspace(0.2, 6, len(t), device="cuda")[:, None, None] for s in (1, 2))
        import pto_isa_b200 as p
        p.kv_cache_write(c, (k * 2.0 ** ek).to(dtype), (v * 2.0 ** ev).to(dtype), slots)
        kd, vd = values(c)
        rows = lambda x: x[pages.long().cpu()].transpose(0, 1).reshape(kv, -1, d)[:, :prefix].cuda()
        size = torch.exp2(torch.randint(-3, 3, (batch, 1, heads, 1), generator=gen(8), device="cuda").float() - max(ek, 0))
        q = (torch.randn(batch, 1, heads, d, generator=gen(6), device="cuda") * size).to(dtype)
        for scale in (None, -0.3, 0.0) if at == 0 else (None,):
            check_attention(q, c, pages, prefix, table, lens, [rows(kd), rows(vd)], own, scale=scale)


def test_attention_many_rows_nan_bad_pages_and_repeats():
    import pto_isa_b200 as p
    for name in FORMATS:
        made = make_attention(name, F16, 128, 1, 16, 400, [0] * 40, 22)
        c, pages, table, lens = made[:4]
        table = torch.zeros(40, 1, dtype=torch.int32, device="cuda")
        q = torch.randn(40, 8, 128, generator=gen(2), device="cuda").to(F16)
        first = p.prefix_attn(q, c, pages, 400, table, lens, return_lse=True)
        for _ in range(3):
            again = p.prefix_attn(q, c, pages, 400, table, lens, return_lse=True)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        # a page that does not exist is left out, and reported
        kd, vd = values(c)
        broken = pages.clone()
        broken[7] = c.k.shape[0]
        o = p.prefix_attn(q, c, broken, 400, table, lens)
        assert status()[2:] == (11, c.k.shape[0])
        keep = torch.cat([pages[:7], pages[8:]]).long().cpu()
        rows = lambda x: x[keep].transpose(0, 1).reshape(1, -1, 128)[:, :384].cuda()
        none = torch.zeros(1, 0, 128, dtype=torch.float64, device="cuda")
        want, _, wv, vsum, qk = ref.attention(q[:, None].double(), rows(kd), rows(vd), [none] * 40, [none] * 40, 128 ** -0.5)
        bound, _ = ref.attention_bounds(F16, want, wv, vsum, qk, 400)
        assert ((o[:, None].double() - want).abs() <= bound).all()
        # a NaN in the prefix reaches everybody, one past its end nobody
        bad = torch.full((1, 1, 128), float("nan"), dtype=F16, device="cuda")
        p.kv_cache_write(c, bad, bad, (pages[12] * 16 + 8).view(1))
        assert torch.isfinite(p.prefix_attn(q, c, pages, 200, table, lens)).all()
        assert p.prefix_attn(q, c, pages, 201, table, lens).isnan().all()


def test_attention_nan_reaches_its_own_rows_only():
    """A cached NaN or infinity reaches the sequence that sees it and nobody else."""
    import pto_isa_b200 as p
    for name in FORMATS:
        made = make_attention(name, F16, 64, 1, 16, 40, [20, 20, 20], 21)
        c, pages, table, lens = made[:4]
        row = torch.ones(1, 1, 64, dtype=F16, device="cuda")
        for value in (float("nan"), float("inf")):
            bad = row * value
            p.kv_cache_write(c, row, bad, (table[1, 0] * 16 + 3).view(1))
            q = torch.randn(3, 2, 64, generator=gen(2), device="cuda").to(F16)
            o = p.prefix_attn(q, c, pages, 40, table, lens)
            assert not torch.isfinite(o[1]).any() and torch.isfinite(o[0]).all() and torch.isfinite(o[2]).all()
            lens2 = torch.tensor([20, 3, 20], dtype=torch.int32, device="cuda")  # the row is past the end now
            assert torch.isfinite(p.prefix_attn(q, c, pages, 40, table, lens2)).all()


def test_attention_is_the_same_every_time_and_writes_its_rows_only():
    import pto_isa_b200 as p
    made = make_attention("mxfp8", F16, 128, 2, 64, 700, [100, 3, 64], 8)
    c, pages, table, lens = made[:4]
    q = torch.randn(3, 2, 8, 128, generator=gen(1), device="cuda").to(F16)
    room = torch.full((5, 2, 8, 128), 7.0, dtype=F16, device="cuda")
    need = p.prefix_attn_workspace_bytes(3, 2, 8, 2, 128, 700, table.shape[1] * 64)
    space = torch.full((need + 4096,), 170, dtype=torch.uint8, device="cuda")
    first, lse = p.prefix_attn(q, c, pages, 700, table, lens, out=room[1:4], return_lse=True, workspace=space[2048:2048 + need])
    first, lse = first.clone(), lse.clone()
    assert (room[0] == 7).all() and (room[4] == 7).all() and (space[:2048] == 170).all() and (space[2048 + need:] == 170).all()
    space.fill_(255)  # what the workspace held before does not matter
    for _ in range(3):
        o, l2 = p.prefix_attn(q, c, pages, 700, table, lens, return_lse=True, workspace=space[2048:2048 + need])
        assert torch.equal(o, first) and torch.equal(l2, lse)


def test_attention_in_a_graph_follows_the_tables_contents():
    """A captured call reads tables and lengths when it is replayed; eager calls and a second graph beside it change nothing."""
    import pto_isa_b200 as p
    made = make_attention("mxfp4", BF16, 64, 2, 16, 100, [60, 60, 60], 5)
    c, pages, table, lens = made[:4]
    q = torch.randn(3, 1, 4, 64, generator=gen(4), device="cuda").to(BF16)
    cases = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([60, 1, 0], [0, 0, 0], [17, 60, 33])]
    want = [p.prefix_attn(q, c, pages, 100, table, n, return_lse=True) for n in cases]
    n1, n2 = lens.clone(), lens.clone()
    graphs, outs = [], []
    for n in (n1, n2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(p.prefix_attn(q, c, pages, 100, table, n, return_lse=True))
        graphs.append(graph)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for a, b in ((0, 1), (1, 2), (2, 0)):
        n1.copy_(cases[a])
        n2.copy_(cases[b])
        torch.cuda.synchronize()
        for _ in range(5):  # both at once: they share no workspace
            with torch.cuda.stream(s1):
                graphs[0].replay()
            with torch.cuda.stream(s2):
                graphs[1].replay()
        torch.cuda.synchronize()
        for out, i in zip(outs, (a, b)):
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


def test_attention_on_another_stream_waits_for_its_inputs():
    import pto_isa_b200 as p
    made = make_attention("16", F16, 128, 2, 64, 500, [10, 20], 6)
    c, pages, table, lens = made[:4]
    q = torch.randn(2, 4, 128, generator=gen(9), device="cuda").to(F16)
    want = p.prefix_attn(q, c, pages, 500, table, lens)
    s = torch.cuda.Stream()
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        late.copy_(q)
        got = p.prefix_attn(late, c, pages, 500, table, lens)
    s.synchronize()
    assert torch.equal(got, want)


def test_cache_offsets_beyond_32_bits():
    """Pages whose byte offsets pass 2^32: written, read back and attended."""
    import pto_isa_b200 as p
    heads, page, d = 8, 128, 128
    pages = (5 << 30) // (heads * page * d)
    c = p.kv_cache_empty(pages, heads, page, d, p.KV_MXFP8)
    last = torch.tensor([pages - 1, pages - 2], dtype=torch.int32, device="cuda")
    n = 200
    t = torch.arange(n, device="cuda")
    slots = (last[t // page] * page + t % page).to(torch.int32)
    k, v = (torch.randn(n, heads, d, generator=gen(s), device="cuda").to(F16) for s in (1, 2))
    p.kv_cache_write(c, k, v, slots)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    back = p.kv_cache_read(c, last[None], lens, n)
    data = [ref.decode(x[[pages - 1, pages - 2]], s[[pages - 1, pages - 2]], False).transpose(0, 1).reshape(heads, -1, d)[:, :n].cuda()
            for x, s in ((c.k, c.k_scale), (c.v, c.v_scale))]
    for got, want in zip(back, data):
        assert torch.equal(got[0].double(), want.to(F16).double())
    q = torch.randn(1, 16, d, generator=gen(3), device="cuda").to(F16)
    none = torch.zeros(heads, 0, d, dtype=torch.float64, device="cuda")
    check_attention(q, c, last, 0, last[None], lens, [none, none], [[data[0]], [data[1]]])
    check_attention(q, c, last, n, last[None], lens * 0, data, [[none], [none]])


# --------------------------------------------------------------------------------------------------- 4-bit weights


def make_w4(kind, dtype, n, k, group, seed):
    w = torch.randint(0, 256, (n, k // 2), generator=gen(seed), device="cuda", dtype=torch.uint8)
    if kind == "mxfp4":
        return w, torch.randint(110, 130, (n, k // 32), generator=gen(seed + 1), device="cuda", dtype=torch.uint8), None
    scale = (torch.rand(n, k // group, generator=gen(seed + 1), device="cuda") * 0.05 - 0.02).to(dtype)
    zero = (torch.rand(n, k // group, generator=gen(seed + 2), device="cuda") * 15).to(dtype) if kind == "zero" else None
    return w, scale, zero


def check_w4(x, w, scale, zero, group, **kw):
    import pto_isa_b200 as p
    y = p.w4_matvec(x, w, scale, zero=zero, **kw)
    weights, mag = ref.w4_weights(w, scale, zero, group)
    want = x.double().cpu() @ weights.t()
    bound = ref.w4_bound(x.dtype, y.dtype, x, mag, want, x.shape[-1])
    err = (y.double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    return y


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kind,group", [("mxfp4", 32), ("int4", 32), ("int4", 64), ("int4", 128), ("zero", 32), ("zero", 64), ("zero", 128)])
def test_w4(kind, group, dtype):
    for m, n, k in ((1, 1, group), (1, 16, 256), (2, 17, 3 * group), (7, 100, 1152), (8, 33, 2048 + group), (9, 64, 640), (16, 129, 4096), (17, 48, 896), (33, 40, 512), (64, 31, 1024)):
        x = torch.randn(m, k, generator=gen(m + k), device="cuda").to(dtype)
        made = make_w4(kind, dtype, n, k, group, 5)
        check_w4(x, *made, group)
        check_w4(x, *made, group, out_dtype=torch.float32)


def test_w4_rows_strides_vectors_and_what_is_written():
    import pto_isa_b200 as p
    n, k = 70, 512
    w, scale, _ = make_w4("mxfp4", F16, n, k, 32, 2)
    wide = torch.randn(5, k + 64, generator=gen(1), device="cuda").to(F16)
    x = wide[:, 32:32 + k]  # rows of a wider matrix
    room = torch.full((7, n), 7.0, dtype=F16, device="cuda")
    y = check_w4(x, w, scale, None, 32, out=room[1:6])
    assert (room[0] == 7).all() and (room[6] == 7).all()
    check_w4(x[2], w, scale, None, 32)  # a vector is one row; other row counts may sum in another order, within the same bound
    assert p.w4_matvec(x[2], w, scale).shape == (n,)
    assert torch.equal(p.w4_matvec(x.contiguous(), w, scale), y)
    assert p.w4_matvec(x[:0], w, scale).shape == (0, n)


def test_w4_every_code_and_scale():
    """All sixteen codes with every scale byte whose products stay finite; a NaN scale byte gives NaN in its row alone."""
    import pto_isa_b200 as p
    for dtype in (F16, BF16):
        k = 32
        codes = torch.arange(16, dtype=torch.uint8, device="cuda").repeat(2)
        w = (codes[0::2] | (codes[1::2] << 4)).expand(254, 16).contiguous()
        scale = torch.arange(254, dtype=torch.uint8, device="cuda").view(254, 1)
        x = torch.zeros(1, k, device="cuda", dtype=dtype)
        for i in range(0, 32, 5):
            x.zero_()
            x[0, i] = 0.25  # one code at a time: exact
            y = p.w4_matvec(x, w, scale, out_dtype=torch.float32)
            want = 0.25 * ref.e2m1_table()[codes[i].long().cpu()] * ref.scale_table()[:254]
            live = (want.abs() >= 2.0 ** -120) & (want.abs() < 2.0 ** 127)
            assert torch.equal(y[0].double().cpu()[live], want[live])
            assert (y[0].double().cpu()[~live & (want.abs() < 1)].abs() <= 2.0 ** -119).all()
        scale[9] = 255
        y = p.w4_matvec(torch.ones(1, k, device="cuda", dtype=dtype), w, scale, out_dtype=torch.float32)
        assert y[0, 9].isnan() and torch.isfinite(y[0, :9]).all() and torch.isfinite(y[0, 10:200]).all()


def test_w4_takes_the_weights_of_the_mx_product():
    """w4_matvec and mx_gemm_fp4 read the same weight bytes: on activations that fp4 holds exactly they agree."""
    import pto_isa_b200 as p
    n, k, m = 256, 512, 8
    w, scale, _ = make_w4("mxfp4", F16, n, k, 32, 3)
    codes = torch.randint(0, 256, (m, k // 2), generator=gen(4), device="cuda", dtype=torch.uint8)
    one = torch.full((m, k // 32), 127, dtype=torch.uint8, device="cuda")
    x = ref.decode(codes, one, True).to(F16).cuda()
    a = check_w4(x, w, scale, None, 32, out_dtype=torch.float32)
    b = p.mx_gemm_fp4(codes, w, one, scale, out_dtype=torch.float32)
    weights, mag = ref.w4_weights(w, scale, None, 32)
    bound = ref.w4_bound(F16, torch.float32, x, mag, x.double().cpu() @ weights.t(), k)
    assert ((a - b).abs().double().cpu() <= 2 * bound).all()


# --------------------------------------------------------------------------------------------------- together


@pytest.mark.parametrize("name", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_steps_of_a_batch_behind_one_prompt(name, dtype):
    """Two decode steps as a server runs them, captured in one graph: projection, cache write, attention, projection; each
    operator's output against its own statement on the inputs it got."""
    import pto_isa_b200 as p
    batch, heads, kv, d, page, prefix, hidden = 5, 8, 2, 64, 16, 150, 256
    made = make_attention(name, dtype, d, kv, page, prefix, [15, 31, 0, 1, 7], 30, spare=1)
    c, pages, table, lens = made[:4]
    wqkv, wo = make_w4("mxfp4", dtype, (heads + 2 * kv) * d, hidden, 32, 40), make_w4("int4", dtype, hidden, heads * d, 64, 50)
    wqkv[1].fill_(122)
    hid = torch.randn(batch, hidden, generator=gen(60), device="cuda").to(dtype)
    slots = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def step():
        slots.copy_(table.gather(1, (lens // page).long()[:, None])[:, 0] * page + lens % page)
        lens.add_(1)
        qkv = p.w4_matvec(hid, wqkv[0], wqkv[1]).view(batch, heads + 2 * kv, d)
        p.kv_cache_write(c, qkv[:, heads:heads + kv], qkv[:, heads + kv:], slots)
        o, lse = p.prefix_attn(qkv[:, :heads], c, pages, prefix, table, lens, return_lse=True)
        return qkv, o, lse, p.w4_matvec(o.view(batch, heads * d), wo[0], wo[1])
    graph = torch.cuda.CUDAGraph()
    before = lens.clone()
    step()
    lens.copy_(before)
    with torch.cuda.graph(graph):
        qkv, o, lse, y = step()
    lens.copy_(before)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for x, w, group, got in ((hid, wqkv, 32, qkv.view(batch, -1)), (o.view(batch, -1), wo, 64, y)):
            weights, mag = ref.w4_weights(w[0], w[1], w[2], group)
            want = x.double().cpu() @ weights.t()
            assert ((got.double().cpu() - want).abs() <= ref.w4_bound(dtype, dtype, x, mag, want, x.shape[-1])).all()
        kd, vd = values(c)
        rows = lambda x, pg, n: x[pg.long().cpu()].transpose(0, 1).reshape(kv, -1, d)[:, :n].cuda()
        for i, s in enumerate(slots.tolist()):  # the new rows are in the cache, quantised
            for data, new in ((kd, qkv[i, heads:heads + kv]), (vd, qkv[i, heads + kv:])):
                want = torch.tensor([ref.quantise_block(blk, name == "mxfp4")[0] for blk in new.float().cpu().reshape(-1, 32).tolist()], dtype=torch.float64).view(kv, d)
                assert same(data[s // page, :, s % page], want)
        n = lens.tolist()
        own = [[rows(x, table[b], n[b]) for b in range(batch)] for x in (kd, vd)]
        want, wlse, wv, vsum, qk = ref.attention(qkv[:, None, :heads].double(), rows(kd, pages, prefix), rows(vd, pages, prefix), *own, d ** -0.5)
        ob, lb = ref.attention_bounds(dtype, want, wv, vsum, qk, prefix + max(n), mx=True)
        assert ((o[:, None].double() - want).abs() <= ob).all() and ((lse[:, None].double() - wlse).abs() <= lb).all()
    assert lens.tolist() == [x + 2 for x in before.tolist()] and status()[0] == 0


def test_cached_context_feeds_the_prefill_attention():
    """kv_cache_read's layout goes into flash_attn_fwd; one query tile over the context equals prefix_attn of its rows."""
    import pto_isa_b200 as p
    made = make_attention("mxfp8", F16, 128, 2, 64, 0, [256, 256], 31)
    c, pages, table, lens, parts, own = made
    k, v = p.kv_cache_read(c, table, lens, 256)
    q = torch.randn(2, 2, 128, 128, generator=gen(3), device="cuda").to(F16)  # (batch, heads, 128 query rows, d)
    o = p.flash_attn_fwd(q, k, v)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    for row in (0, 77, 127):
        single = p.prefix_attn(q[:, :, row].contiguous(), c, none, 0, table, lens)
        want, _, wv, vsum, qk = ref.attention(q[:, None, :, row].double(), *parts, *own, 128 ** -0.5)
        bound, _ = ref.attention_bounds(F16, want, wv, vsum, qk, 256)
        assert ((single[:, None].double() - want).abs() <= bound).all()
        # flash_attn_fwd keeps P relative to a reference up to 2^8 above the maximum: its rounding is of the same size
        assert ((o[:, :, row].double() - single.double()).abs() <= 2 * bound[:, 0]).all()


# --------------------------------------------------------------------------------------------------- blocks, paths, streams


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kind,group", [("mxfp4", 32), ("zero", 64)])
def test_w4_of_any_size(kind, group, dtype):
    """Rows of W of every share a block can get (one to eight tiles of 16, several rounds of 128, one block an SM or two), rows of
    x on both sides of every column tile, k that ends inside a step."""
    for n, k in ((1600, 192), (148 * 16 + 5, 1344), (148 * 40, 576), (9473, 256), (148 * 2 * 60 + 1, 320), (148 * 2 * 130 + 7, 192)):
        made = make_w4(kind, dtype, n, k, group, n % 97)
        for m in (2, 3, 8, 9, 16, 24, 40, 64) if n < 9000 else (1, 5, 16, 33):
            x = torch.randn(m, k, generator=gen(m), device="cuda").to(dtype)
            check_w4(x, *made, group)
    assert status()[0] == 0


@pytest.mark.parametrize("m", [1, 2, 5, 20])
@pytest.mark.parametrize("k", [512, 288])
def test_w4_scales_that_begin_anywhere(m, k):
    for kind, group in (("mxfp4", 32), ("zero", 32)):
        dtype = F16
        w, scale, zero = make_w4(kind, dtype, 50, k, group, 9)
        shifted = []
        for t in (scale, zero):
            if t is not None:
                room = torch.full((t.numel() + 1,), 77, dtype=t.dtype, device="cuda")
                room[1:] = t.flatten()
                shifted.append(room[1:].view(t.shape))
        x = torch.randn(m, k, generator=gen(m), device="cuda").to(dtype)
        y = check_w4(x, w, *shifted, *([None] if zero is None else []), group)
        assert torch.equal(y, check_w4(x, w, scale, zero, group))


@pytest.mark.parametrize("kind,group", [("mxfp4", 32), ("int4", 64)])
@pytest.mark.parametrize("m", [2, 5])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_w4_nan_and_infinities_stay_in_their_rows(kind, group, m, dtype):
    import pto_isa_b200 as p
    n, k = 40, 512
    w, scale, zero = make_w4(kind, dtype, n, k, group, 12)
    x = torch.randn(m, k, generator=gen(2), device="cuda").to(dtype)
    clean = check_w4(x, w, scale, zero, group)
    bad = x.clone()
    bad[1, 300] = float("nan")
    y = p.w4_matvec(bad, w, scale, zero=zero)
    assert y[1].isnan().all() and torch.equal(y[0], clean[0]) and torch.equal(y[2:], clean[2:])
    scale = scale.clone()
    scale[7, 1] = 255 if kind == "mxfp4" else float("nan")
    y = p.w4_matvec(x, w, scale, zero=zero)
    keep = torch.arange(n, device="cuda") != 7
    assert y[:, 7].isnan().all() and torch.equal(y[:, keep], clean[:, keep])


def test_both_ways_into_the_library_agree(monkeypatch):
    """Calls in order go through the extension module, others through the checks in Python: the same results bit for bit."""
    import pto_isa_b200 as p
    from pto_isa_b200 import ops
    assert ops._fast is not None

    def run():
        made = make_attention("mxfp8", BF16, 64, 2, 16, 70, [20, 0, 33], 5)
        q = torch.randn(3, 2, 4, 64, generator=gen(1), device="cuda").to(BF16)
        o, lse = p.prefix_attn(q, made[0], made[1], 70, made[2], made[3], return_lse=True)
        k, v = p.kv_cache_read(made[0], made[2], made[3], 40)
        w, scale, zero = make_w4("zero", BF16, 70, 512, 64, 3)
        x = torch.randn(5, 512, generator=gen(3), device="cuda").to(BF16)
        return [made[0].k[made[2].long()], o, lse, k, v, p.w4_matvec(x, w, scale, zero=zero), p.w4_matvec(x[0], w, scale, out_dtype=torch.float32)]
    direct = run()
    monkeypatch.setattr(ops, "_fast", None)
    for a, b in zip(direct, run()):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_calls_at_the_same_time_do_not_share_anything():
    import pto_isa_b200 as p
    made = make_attention("mxfp8", F16, 128, 2, 64, 900, [70] * 20, 8)
    q = [torch.randn(20, 1, 8, 128, generator=gen(s), device="cuda").to(F16) for s in (1, 2)]
    w = make_w4("int4", F16, 700, 1024, 128, 4)
    x = [torch.randn(6, 1024, generator=gen(s), device="cuda").to(F16) for s in (3, 4)]
    call = lambda i: (p.prefix_attn(q[i], made[0], made[1], 900, made[2], made[3]), p.w4_matvec(x[i], w[0], w[1]))
    alone = [call(0), call(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for o, y in got[i]:
            assert torch.equal(o, alone[i][0]) and torch.equal(y, alone[i][1])
    # two captured calls replayed side by side
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for i in (0, 1):
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in (0, 1):
        assert torch.equal(outs[i][0], alone[i][0]) and torch.equal(outs[i][1], alone[i][1])
    assert status()[0] == 0


@pytest.mark.parametrize("batch", [1, 6])
def test_attention_without_keys_of_their_own(batch):
    """A table without columns: every sequence attends to the prefix alone, few rows and many."""
    c, pages, _, lens, parts, own = make_attention("mxfp8", F16, 128, 1, 16, 300, [0] * batch, 6)
    table = torch.zeros(batch, 0, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, 1, 8, 128, generator=gen(1), device="cuda").to(F16)
    check_attention(q, c, pages, 300, table, lens, parts, own)


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_joins_many_and_few_pieces(name, d):
    """One row over a long cache of its own (the most pieces), and more than a thousand rows of few pieces (a warp each)."""
    long = make_attention(name, F16, d, 1, 16, 0, [9000, 3], 3)
    check_attention(torch.randn(2, 1, 1, d, generator=gen(1), device="cuda").to(F16), long[0], long[1], 0, *long[2:])
    rows = make_attention(name, F16, d, 8, 16, 130, [5, 0, 40] * 14 + [1], 4)
    check_attention(torch.randn(43, 1, 32, d, generator=gen(2), device="cuda").to(F16), rows[0], rows[1], 130, *rows[2:])


# --------------------------------------------------------------------------------------------------- a prefix of many rows and keys
# (sizes past which the prefix goes to the tensor memory kernel: one row tile, and several)

WIDE = [(20, 32, 8, 7700), (300, 8, 2, 2111)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("batch,heads,kv,prefix", WIDE)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_long_prefix_of_many_rows(dtype, batch, heads, kv, prefix, name, d):
    """A negative, a zero and a large scale, a maximum that grows along the keys, cached values far from 1 in some tiles only,
    rows of q of very different sizes."""
    import pto_isa_b200 as p
    for at, (ek, ev) in enumerate(((0, 0), (-30, 0), (30, 0), (0, 30), (0, -30), (0, 6))):
        if dtype == F16 and (abs(ek) > 8 or abs(ev) > 10):
            continue
        c, pages, table, lens, parts, own = make_attention(name, dtype, d, kv, 32, prefix, [3] * batch, 40 + at)
        t = torch.arange(150, 420)
        slots = (pages[(t // 32).cuda()].long() * 32 + t.cuda() % 32).to(torch.int32)
        k, v = (torch.randn(len(t), kv, d, generator=gen(s), device="cuda") * torch.linspace(0.2, 6, len(t), device="cuda")[:, None, None] for s in (1, 2))
        p.kv_cache_write(c, (k * 2.0 ** ek).to(dtype), (v * 2.0 ** ev).to(dtype), slots)
        kd, vd = values(c)
        rows = lambda x: x[pages.long().cpu()].transpose(0, 1).reshape(kv, -1, d)[:, :prefix].cuda()
        size = torch.exp2(torch.randint(-3, 3, (batch, 1, heads, 1), generator=gen(8), device="cuda").float() - max(ek, 0))
        q = (torch.randn(batch, 1, heads, d, generator=gen(6), device="cuda") * size).to(dtype)
        for scale in (None, -0.3, 0.0) if at == 0 else (None,):
            check_attention(q, c, pages, prefix, table, lens, [rows(kd), rows(vd)], own, scale=scale)


@pytest.mark.parametrize("name", FORMATS)
def test_attention_long_prefix_nan_bad_pages_and_repeats(name):
    import pto_isa_b200 as p
    batch, heads, d, prefix = 128, 8, 128, 4897
    c, pages, table, lens = make_attention(name, F16, d, 1, 16, prefix, [0] * batch, 22)[:4]
    table = torch.zeros(batch, 1, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, heads, d, generator=gen(2), device="cuda").to(F16)
    first = p.prefix_attn(q, c, pages, prefix, table, lens, return_lse=True)
    for _ in range(3):
        again = p.prefix_attn(q, c, pages, prefix, table, lens, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    kd, vd = values(c)
    broken = pages.clone()
    broken[7] = c.k.shape[0]
    o = p.prefix_attn(q, c, broken, 4896, table, lens)
    assert status()[2:] == (11, c.k.shape[0])
    keep = torch.cat([pages[:7], pages[8:]]).long().cpu()
    rows = lambda x: x[keep].transpose(0, 1).reshape(1, -1, d)[:, :4880].cuda()
    none = torch.zeros(1, 0, d, dtype=torch.float64, device="cuda")
    want, _, wv, vsum, qk = ref.attention(q[:, None].double(), rows(kd), rows(vd), [none] * batch, [none] * batch, d ** -0.5)
    bound, _ = ref.attention_bounds(F16, want, wv, vsum, qk, 4896, mx=name != "16")
    assert ((o[:, None].double() - want).abs() <= bound).all()
    bad = torch.full((1, 1, d), float("nan"), dtype=F16, device="cuda")
    p.kv_cache_write(c, bad, bad, (pages[306] * 16).view(1))  # position 4896
    assert torch.isfinite(p.prefix_attn(q, c, pages, 4896, table, lens)).all()
    assert p.prefix_attn(q, c, pages, 4897, table, lens).isnan().all()


def test_attention_long_prefix_at_the_same_time_and_replayed():
    import pto_isa_b200 as p
    made = make_attention("mxfp8", BF16, 128, 8, 64, 700, [33] * 128, 8)
    q = [torch.randn(128, 1, 64, 128, generator=gen(s), device="cuda").to(BF16) for s in (1, 2)]
    call = lambda i: p.prefix_attn(q[i], made[0], made[1], 700, made[2], made[3])
    alone = [call(0), call(1)]
    check_attention(q[0], made[0], made[1], 700, *made[2:])
    streams, graphs, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for i in (0, 1):
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
        streams[i].wait_stream(torch.cuda.current_stream())
    eager = []
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
                eager.append((i, call(i)))
    torch.cuda.synchronize()
    assert all(torch.equal(outs[i], alone[i]) for i in (0, 1)) and all(torch.equal(o, alone[i]) for i, o in eager)
    assert status()[0] == 0
