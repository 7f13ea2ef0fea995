"""Edges of the serving operators that test_serving_gpu.py does not reach, against the same 64-bit statements: the tensor memory
kernel with many key tiles a block, every scale byte and code in a cache, what the status record gets."""
import pytest
import torch

import serving_ref as ref
from test_serving_gpu import BF16, F16, FORMATS, check_attention, check_w4, fmt_of, gen, make_attention, make_w4, status, values

pytestmark = pytest.mark.gpu


def pieces_of_prefix(batch, tokens, heads, kv_heads, d, prefix):
    """Pieces that the planner cuts the prefix into, from the workspace of a call whose sequences have no keys of their own."""
    import pto_isa_b200 as p
    tiles = -(-batch * tokens * (heads // kv_heads) // 16)
    return p.prefix_attn_workspace_bytes(batch, tokens, heads, kv_heads, d, prefix, 0) / (tiles * kv_heads * 16 * (4 * d + 8))


def wide_shape(batch, tokens, heads, kv_heads, d, prefix):
    """Key tiles of 128 that a block of the tensor memory kernel takes; asserts that the planner chose that kernel, whose number
    of pieces (a block an SM) is not that of the other (three blocks of 16 rows an SM)."""
    rows = batch * tokens * (heads // kv_heads)
    units, tiles = -(-rows // (256 if rows > 128 else 128)) * kv_heads, -(-prefix // 128)
    per = -(-tiles // min(tiles, max(1, 148 // units)))
    wide = -(-tiles // per) * (1 if rows > 128 else 2)
    small = -(-rows // 16) * kv_heads
    chunk = (-(-prefix // min(-(-444 // small), -(-prefix // 64))) + 63) // 64 * 64
    assert wide != -(-prefix // chunk), "these sizes do not tell the two kernels apart"
    assert pieces_of_prefix(batch, tokens, heads, kv_heads, d, prefix) == wide
    return per


# --------------------------------------------------------------------------------------------------- the tensor memory kernel


def missing_pages(made, page, prefix, kv, d, gone):
    """The prefix's page numbers with those of `gone` (a mask over pages) out of range, and the rows of K and V that are left."""
    c, pages = made[0], made[1]
    broken = torch.where(gone, torch.where(torch.arange(len(gone)) % 2 == 0, c.k.shape[0], -5), pages.cpu()).to(torch.int32)
    keep = (~gone[torch.arange(prefix) // page]).nonzero()[:, 0].cuda()
    return broken.cuda(), [x[:, keep] for x in made[4]]


@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("batch,heads,kv,prefix,d", [(265, 64, 8, 3000, 128), (40, 96, 32, 6000, 128), (265, 64, 8, 3000, 64), (40, 96, 32, 6000, 64)])
def test_attention_prefix_with_many_missing_pages(batch, heads, kv, prefix, d, name):
    """Pages that do not exist all along a prefix of many key tiles a block: left out of every row, reported once, and no wait in the
    kernel runs out over them."""
    page = 16
    assert wide_shape(batch, 1, heads, kv, d, prefix) > 8
    made = make_attention(name, F16, d, kv, page, prefix, [0] * batch, 61)
    gone = torch.rand(-(-prefix // page), generator=torch.Generator().manual_seed(5)) < 0.7
    gone[:24] = True  # whole tiles without a key, the first among them
    broken, parts = missing_pages(made, page, prefix, kv, d, gone)
    import pto_isa_b200 as p
    q = torch.randn(batch, 1, heads, d, generator=gen(6), device="cuda").to(F16)
    table = torch.zeros(batch, 1, dtype=torch.int32, device="cuda")
    o, lse = p.prefix_attn(q, made[0], broken, prefix, table, made[3], return_lse=True)
    code, _, where, detail = status()
    assert (code, where) == (1, 11) and detail in (-5, made[0].k.shape[0])
    want, wlse, wv, vsum, qk = ref.attention(q.double(), *parts, *made[5], d ** -0.5)
    ob, lb = ref.attention_bounds(F16, want, wv, vsum, qk, prefix, mx=name != "16")
    assert ((o.double() - want).abs() <= ob).all() and ((lse.double() - wlse).abs() <= lb).all()
    assert status()[0] == 0


# (batch, tokens, heads, kv_heads, prefix, page, key tiles a block): several query tokens a sequence, pages of 16 to 1024, one
# tile of rows (the last one ragged), an even and an odd number of tiles (the last block's second tile absent), rounds of both
# rings and of the eight descriptions
MANY_TILES = [(40, 1, 96, 32, 6000, 256, 12), (7, 5, 96, 32, 6131, 128, 12), (265, 1, 64, 8, 3000, 1024, 12), (38, 7, 64, 8, 2777, 64, 11),
              (64, 4, 64, 8, 2777, 16, 11)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("batch,tokens,heads,kv,prefix,page,tiles", MANY_TILES)
def test_attention_many_key_tiles_a_block(batch, tokens, heads, kv, prefix, page, tiles, name, dtype, d):
    """The tensor memory kernel over many key tiles, q a slice of a fused projection, own keys of uneven lengths (some shorter than
    the query tokens), keys that grow along the prefix, so that maxima move in late tiles too."""
    import pto_isa_b200 as p
    assert wide_shape(batch, tokens, heads, kv, d, prefix) == tiles
    lens = [(5 * i) % 23 for i in range(batch)]
    c, pages, table, n, parts, own = make_attention(name, dtype, d, kv, page, prefix, lens, 50)
    t = torch.arange(prefix, device="cuda")
    k = torch.randn(prefix, kv, d, generator=gen(1), device="cuda") * torch.linspace(0.05, 4, prefix, device="cuda")[:, None, None]
    v = torch.randn(prefix, kv, d, generator=gen(2), device="cuda") + torch.linspace(-2, 2, prefix, device="cuda")[:, None, None]
    p.kv_cache_write(c, k.to(dtype), v.to(dtype), (pages[t // page] * page + t % page).to(torch.int32))
    kd, vd = values(c)
    rows = lambda x: x[pages.long().cpu()].transpose(0, 1).reshape(kv, -1, d)[:, :prefix].cuda()
    fused = torch.randn(batch, tokens, heads + 2 * kv, d, generator=gen(3), device="cuda").to(dtype)
    check_attention(fused[:, :, :heads], c, pages, prefix, table, n, [rows(kd), rows(vd)], own)


@pytest.mark.parametrize("name", FORMATS)
def test_attention_many_key_tiles_nan_and_repeats(name):
    """The same bits every time, and a NaN in the last key of the prefix reaches every row of its head, past the end none."""
    import pto_isa_b200 as p
    batch, heads, kv, d, prefix = 265, 64, 8, 128, 3001
    assert wide_shape(batch, 1, heads, kv, d, prefix) == 12
    c, pages, table, n = make_attention(name, F16, d, kv, 64, prefix, [0] * batch, 51)[:4]
    table = torch.zeros(batch, 1, dtype=torch.int32, device="cuda")
    q = torch.randn(batch, heads, d, generator=gen(3), device="cuda").to(F16)
    first = p.prefix_attn(q, c, pages, prefix, table, n, return_lse=True)
    for _ in range(5):
        again = p.prefix_attn(q, c, pages, prefix, table, n, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    bad = torch.full((1, kv, d), float("nan"), dtype=F16, device="cuda")
    p.kv_cache_write(c, bad, bad, (pages[3000 // 64] * 64 + 3000 % 64).view(1))
    assert torch.isfinite(p.prefix_attn(q, c, pages, prefix - 1, table, n)).all()
    assert p.prefix_attn(q, c, pages, prefix, table, n).isnan().all()
    assert status()[0] == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("tokens,prefix,lens", [(100, 0, [100, 257, 60]), (77, 301, [300, 0, 78, 1]), (513, 0, [700])])
def test_attention_prompt_chunk(tokens, prefix, lens, name, dtype, d):
    """A chunk of a prompt over its cached context: many query tokens a sequence, more than some sequences have keys."""
    made = make_attention(name, dtype, d, 2, 32, prefix, lens, 52)
    q = torch.randn(len(lens), tokens, 6, d, generator=gen(5), device="cuda").to(dtype)
    check_attention(q, made[0], made[1], prefix, *made[2:])


# --------------------------------------------------------------------------------------------------- scale bytes and codes of any cache
# Caches filled by something else than kv_cache_write: any codes under any scale byte.

SHAPES = [("own", 3, 8, 2, 90), ("prefix", 3, 8, 2, 90), ("long", 20, 32, 8, 7700)]  # batch, heads, kv_heads, keys


def raw_cache(name, kv, page, keys, d, low, high, seed):
    """An MX cache of `keys` positions in page order: every code but e4m3's NaN, scale bytes low .. high."""
    import pto_isa_b200 as p
    c = p.kv_cache_empty(-(-keys // page), kv, page, d, fmt_of(name, F16))
    for i, t in enumerate(c[:4]):
        t.copy_(torch.randint(0, 256, t.shape, generator=gen(seed + i), device="cuda") if i < 2 else
                torch.randint(low[i - 2], high[i - 2] + 1, t.shape, generator=gen(seed + i), device="cuda"))
        if i < 2 and name == "mxfp8":
            t[(t & 127) == 127] = 0x38
    return c


def at(keys, page):
    """(page, row) of positions `keys` of a cache in page order."""
    keys = torch.as_tensor(keys, device="cuda")
    return keys // page, keys % page


def put_block(c, which, keys, page, head, block, codes, byte):
    """Block `block` of `head` at positions `keys` of K (which 0) or V (1): all bytes of codes, and the scale."""
    pg, row = at(keys, page)
    width = c[which].shape[-1] // c[which + 2].shape[-1]
    c[which][pg, head, row, block * width:(block + 1) * width] = codes
    c[which + 2][pg, head, row, block] = byte


def check_raw(c, q, where, keys, scale=None, tiny=False):
    """All `keys` positions as every sequence's own keys, or as the prefix: the values that the cache stands for, and NaN exactly
    where it holds one.  tiny: of values near bfloat16's smallest.  In place of the bound's floor of 1e-30 come three halves of a step
    of 2^-133 below the normal numbers, one for V (the weights' sum is 1), one for the output, one for 32-bit sums there (places
    of 2^-149, at most 2^-150 a key: 2^-137 for 8192)."""
    import pto_isa_b200 as p
    batch, heads, d = q.shape
    kv = c.k.shape[1]
    pages = torch.arange(c.k.shape[0], dtype=torch.int32, device="cuda")
    kd, vd = (x.transpose(0, 1).reshape(kv, -1, d)[:, :keys].cuda() for x in values(c))
    none = torch.zeros(kv, 0, d, dtype=torch.float64, device="cuda")
    own = where == "own"
    table = pages.expand(batch, -1).contiguous()
    lens = torch.full((batch,), keys if own else 0, dtype=torch.int32, device="cuda")
    if where == "long":
        wide_shape(batch, 1, heads, kv, d, keys)
        table = table[:, :0]
    elif not own:
        table = table[:, :1]
    parts, owns = ([none, none], [[kd] * batch, [vd] * batch]) if own else ([kd, vd], [[none] * batch] * 2)
    o, lse = p.prefix_attn(q, c, pages, 0 if own else keys, table, lens, scale=scale, return_lse=True)
    o, lse = o[:, None], lse[:, None]
    want, wlse, wv, vsum, qk = ref.attention(q[:, None].double(), *parts, *owns, d ** -0.5 if scale is None else scale)
    ob, lb = ref.attention_bounds(q.dtype, want, wv, vsum, qk, keys, mx=True)
    if tiny:
        ob = ob - 1e-30 + 3 * 2.0 ** -134
    if q.dtype == F16:  # values past float16's range are infinities of the output
        past = want.abs() >= 65520
        assert (o[past] == torch.where(want[past] > 0, torch.inf, -torch.inf)).all()
        ob = torch.where(past, torch.inf, ob)
        want = torch.where(past, 0.0, want)
        o = torch.where(past, 0.0, o.double())
    assert torch.equal(o.isnan(), want.isnan()) and torch.equal(lse.isnan(), wlse.isnan())
    live, seen = ~want.isnan(), ~wlse.isnan()
    err, lerr = (o.double() - want).abs()[live], (lse.double() - wlse).abs()[seen]
    assert (err <= ob[live]).all(), float((err / ob[live]).max())
    assert (lerr <= lb[seen]).all(), float((lerr / lb[seen]).max())
    assert status()[0] == 0
    return o, lse


MX = ["mxfp8", "mxfp4"]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", MX)
@pytest.mark.parametrize("where,batch,heads,kv,keys", SHAPES)
def test_attention_k_scale_of_nan(where, batch, heads, kv, keys, name, dtype, d):
    """Scale byte 255 is NaN over any codes: the rows of that kv head are NaN, those of the others are not."""
    page = 32
    q = torch.randn(batch, heads, d, generator=gen(4), device="cuda").to(dtype)
    for i, (codes, block) in enumerate(((0xff if name == "mxfp4" else 0xb8, 0), (0x22 if name == "mxfp4" else 0x38, d // 32 - 1), (0, 1))):
        c = raw_cache(name, kv, page, keys, d, (116, 116), (122, 124), 70 + i)
        put_block(c, 0, [keys - 3 - i], page, kv - 1, block, codes, 255)
        o, _ = check_raw(c, q.abs() if i == 0 else q, where, keys)  # one sign throughout: a block of infinities would drop the key
        assert o.isnan().any() and not o.isnan().all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", MX)
@pytest.mark.parametrize("where,batch,heads,kv,keys", SHAPES)
def test_attention_k_of_the_smallest_scales(where, batch, heads, kv, keys, name, d):
    """K blocks of scale byte 0 are multiples of 2^-127, which bfloat16 queries of 2^124 turn into ordinary logits."""
    page = 32
    q = (torch.randn(batch, heads, d, generator=gen(4), device="cuda") * 2.0 ** 124).to(BF16)
    for high in (0, 3):
        c = raw_cache(name, kv, page, keys, d, (0, 116), (high, 124), 80)
        if name == "mxfp8":  # codes below 8, so that no key outweighs all others
            c.k.copy_(torch.where((c.k & 127) > 0x50, c.k & 0xcf, c.k))
        check_raw(c, q, where, keys)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", MX)
@pytest.mark.parametrize("where,batch,heads,kv,keys", SHAPES)
def test_attention_v_of_bfloat16_queries_nan(where, batch, heads, kv, keys, name, d):
    """A NaN scale over any codes and (e4m3) a NaN code make their columns NaN and no others, beside scales that float16 holds and
    beside one that it does not."""
    page = 32
    q = torch.randn(batch, heads, d, generator=gen(4), device="cuda").to(BF16)
    for far in (False, True):
        c = raw_cache(name, kv, page, keys, d, (116, 116), (122, 122), 90)
        if far:
            put_block(c, 1, [keys - 6], page, kv - 1, 1, 0x11, 160)
        put_block(c, 1, [keys - 3], page, kv - 1, 0, 0x22 if name == "mxfp4" else 0x38, 255)
        if name == "mxfp8":
            pg, row = at([keys - 4], page)
            c.v[pg, 0, row, 33] = 0x7f
            c.v[pg, 0, row, 40] = 0xff
            c.v[pg, 0, row, 3] = 0x7e  # 448, the largest code that is a number
        o, _ = check_raw(c, q, where, keys)
        nan = o.isnan().view(batch, kv, -1, d)
        assert nan[:, kv - 1, :, :32].all() and not nan[:, kv - 1, :, 32:].any()
        want = [33, 40] if name == "mxfp8" else []
        assert nan[:, 0, :, want].all() and nan[:, 0].sum() == batch * heads // kv * len(want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", MX)
@pytest.mark.parametrize("where,batch,heads,kv,keys", SHAPES)
def test_attention_v_of_the_smallest_scales(where, batch, heads, kv, keys, name, d):
    """V of scale bytes 0 to 3 in bfloat16, in all blocks and in one beside others of ordinary size; zeros of byte 0 stay zeros."""
    page = 32
    q = torch.randn(batch, heads, d, generator=gen(4), device="cuda").to(BF16)
    for low, high in ((0, 0), (0, 3)):
        c = raw_cache(name, kv, page, keys, d, (116, low), (122, high), 100)
        o, _ = check_raw(c, q, where, keys, tiny=True)
        assert (o != 0).any(-1).all()
    c = raw_cache(name, kv, page, keys, d, (116, 120), (122, 124), 110)
    c.v_scale[..., 0] = 0
    o, _ = check_raw(c, q, where, keys, tiny=True)
    assert (o[..., :32] != 0).any(-1).all()
    c.v[..., :c.v.shape[-1] * 32 // d] &= 0x80 if name == "mxfp8" else 0x88
    o, _ = check_raw(c, q, where, keys, tiny=True)
    assert (o[..., :32] == 0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", MX)
@pytest.mark.parametrize("where,batch,heads,kv,keys", SHAPES)
def test_attention_v_of_float16_queries_nan(where, batch, heads, kv, keys, name, d):
    """As with bfloat16 queries: a NaN scale over any codes and a NaN code make their columns NaN and no others."""
    page = 32
    q = torch.randn(batch, heads, d, generator=gen(4), device="cuda").to(F16)
    for far in (None, 90, 145):
        c = raw_cache(name, kv, page, keys, d, (116, 116), (122, 122), 90)
        if far:  # codes that float16 holds under that scale: zeros, and (e4m3) subnormal ones
            put_block(c, 1, [keys - 6], page, kv - 1, 1, 0x01 if name == "mxfp8" else 0x08, far)
        put_block(c, 1, [keys - 3], page, kv - 1, 0, 0x22 if name == "mxfp4" else 0x38, 255)
        if name == "mxfp8":
            pg, row = at([keys - 4], page)
            c.v[pg, 0, row, 33] = 0x7f
            c.v[pg, 0, row, 40] = 0xff
        o, _ = check_raw(c, q, where, keys)
        nan = o.isnan().view(batch, kv, -1, d)
        assert nan[:, kv - 1, :, :32].all() and not nan[:, kv - 1, :, 32:].any()
        want = [33, 40] if name == "mxfp8" else []
        assert nan[:, 0, :, want].all() and nan[:, 0].sum() == batch * heads // kv * len(want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", MX)
@pytest.mark.parametrize("where,batch,heads,kv,keys", SHAPES)
def test_attention_v_scales_that_float16_does_not_have(where, batch, heads, kv, keys, name, d):
    """With float16 queries V is rounded to float16 once, whatever its scale: 2^-40 .. 2^-16, and 2^16 and up over codes whose
    values float16 holds."""
    page = 32
    q = torch.randn(batch, heads, d, generator=gen(4), device="cuda").to(F16)
    low = 87 if name == "mxfp8" else 95  # a block's largest value from half of float16's smallest on
    for first, last in ((low, low + 6), (low + 7, 103), (low, 112)):
        c = raw_cache(name, kv, page, keys, d, (116, first), (122, last), 120)
        check_raw(c, q, where, keys)
    c = raw_cache(name, kv, page, keys, d, (116, 116), (122, 122), 130)
    if name == "mxfp8":  # subnormal codes, 2^-9 .. 7 * 2^-9, at 2^16 .. 2^20
        c.v.bitwise_and_(0x87)
        c.v_scale.copy_(torch.randint(140, 148, c.v_scale.shape, generator=gen(3), device="cuda"))
    else:  # zeros at 2^16 .. 2^40 beside 0.5 .. 6 at 2^12 and 2^13
        big = torch.rand(c.v_scale.shape, generator=gen(3), device="cuda") < 0.5
        c.v_scale.copy_(torch.where(big, torch.randint(143, 168, big.shape, generator=gen(4), device="cuda"), torch.randint(139, 141, big.shape, generator=gen(5), device="cuda")))
        c.v.copy_(torch.where(big.repeat_interleave(16, -1), c.v & 0x88, c.v))
    o, _ = check_raw(c, q, where, keys)
    assert torch.isfinite(o).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("name", MX)
@pytest.mark.parametrize("where,batch,heads,kv,keys", SHAPES)
def test_attention_blocks_of_zeros(where, batch, heads, kv, keys, name, dtype, d):
    """Scale byte 0 over zeros, as kv_cache_write leaves them: in one block of some keys and values, and in all of some."""
    page = 32
    c = raw_cache(name, kv, page, keys, d, (112, 112), (126, 126), 140)
    for which in (0, 1):
        put_block(c, which, torch.arange(3, keys, 7), page, kv - 1, 1, 0x00, 0)
        for block in range(d // 32):
            put_block(c, which, torch.arange(5, keys, 11), page, 0, block, 0x80 if name == "mxfp8" else 0x88, 0)
    check_raw(c, torch.randn(batch, heads, d, generator=gen(4), device="cuda").to(dtype), where, keys)


# --------------------------------------------------------------------------------------------------- the status record


@pytest.mark.parametrize("batch,prefix", [(3, 0), (3, 40), (20, 7700)])
def test_attention_reports_a_length_whatever_its_bound(batch, prefix):
    """A length that is not 0 where the bound is: cut and reported, like any other, with and without columns of the table."""
    import pto_isa_b200 as p
    c, pages, table, lens, parts, own = make_attention("mxfp8", F16, 128, 8, 16, prefix, [0] * batch, 62, spare=1)
    q = torch.randn(batch, 1, 32, 128, generator=gen(1), device="cuda").to(F16)
    want = check_attention(q, c, pages, prefix, table, lens, parts, own, max_seq_len=0)
    for value in (1, -2):
        bad = lens.clone()
        bad[-1] = value
        for columns, bound in ((1, 0), (0, None)):
            o, lse = p.prefix_attn(q, c, pages, prefix, table[:, :columns], bad, max_seq_len=bound, return_lse=True)
            code, _, where, detail = status()
            assert (code, where, detail) == (1, 12, value) and torch.equal(o, want[0]) and torch.equal(lse, want[1])


# --------------------------------------------------------------------------------------------------- one key that outweighs all others


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", FORMATS)
@pytest.mark.parametrize("where,batch,heads,kv,keys", [("own", 3, 8, 2, 9000), ("prefix", 3, 8, 2, 9000), ("long", 20, 32, 8, 7700)])
def test_attention_keys_behind_one_that_outweighs_them(where, batch, heads, kv, keys, name, d):
    """The first key weighs 2^20 to 2^27 times what another does and has no value: the output is what the others hold.  Float16
    probabilities keep multiples of 2^-24 of what they are taken times, 2^15 by pieces and 2^7 at least in the tensor memory kernel:
    errors of 2^-40 and 2^-32 |v| a key in place of the bound's 2^-25."""
    import pto_isa_b200 as p
    page = 64
    c = p.kv_cache_empty(-(-keys // page), kv, page, d, fmt_of(name, F16))
    v = torch.randn(keys, kv, d, generator=gen(1), device="cuda") + 1
    v[0] = 0
    q = torch.ones(batch, heads, d, dtype=F16, device="cuda")
    pages = torch.arange(c.k.shape[0], dtype=torch.int32, device="cuda")
    none = torch.zeros(kv, 0, d, dtype=torch.float64, device="cuda")
    for power in (20, 25, 27):
        k = torch.zeros(keys, kv, d, device="cuda")
        k[0] = round(power * 0.6931 * d ** -0.5 * 16) / 16
        p.kv_cache_write(c, k.to(F16), v.to(F16), torch.arange(keys, dtype=torch.int32, device="cuda"))
        kd, vd = (x.transpose(0, 1).reshape(kv, -1, d)[:, :keys].cuda() for x in values(c))
        own = where == "own"
        if where == "long":
            wide_shape(batch, 1, heads, kv, d, keys)
        lens = torch.full((batch,), keys if own else 0, dtype=torch.int32, device="cuda")
        parts, owns = ([none, none], [[kd] * batch, [vd] * batch]) if own else ([kd, vd], [[none] * batch] * 2)
        o, lse = p.prefix_attn(q, c, pages, 0 if own else keys, pages.expand(batch, -1).contiguous() if own else pages.new_zeros(batch, 0), lens, return_lse=True)
        want, wlse, wv, vsum, qk = ref.attention(q[:, None].double(), *parts, *owns, d ** -0.5)
        ob, lb = ref.attention_bounds(F16, want, wv, vsum, qk, keys, mx=name != "16")
        ob = ob - (2.0 ** -25 - (2.0 ** -32 if where == "long" else 2.0 ** -40)) * vsum
        err = (o[:, None].double() - want).abs()
        assert (err <= ob).all(), (power, float((err / ob).max()))
        assert ((lse[:, None].double() - wlse).abs() <= lb).all()
    assert status()[0] == 0


# --------------------------------------------------------------------------------------------------- 4-bit weights


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kind,group", [("mxfp4", 32), ("int4", 128), ("zero", 64)])
@pytest.mark.parametrize("m", [1, 2])
def test_w4_few_rows_too_long_for_shared_memory(m, kind, group, dtype):
    """One and two rows whose prepared form does not fit a block's shared memory go with those of more rows, and need a workspace."""
    import pto_isa_b200 as p
    k = 28672 // m + 128
    assert p.lib().pto_b200_w4_matvec_workspace_bytes(m, k, 0 if kind == "mxfp4" else 1) > 0
    for n in (5, 600):
        x = torch.randn(m, k, generator=gen(m), device="cuda").to(dtype)
        check_w4(x, *make_w4(kind, dtype, n, k, group, 8), group)
        check_w4(x, *make_w4(kind, dtype, n, k, group, 9), group, out_dtype=torch.float32)


@pytest.mark.parametrize("m", [1, 4])
@pytest.mark.parametrize("dtype", [BF16])
def test_w4_rows_of_small_elements(m, dtype):
    """bfloat16 rows around the largest element 2^-98 below which they are not brought up to float16's full range: errors of 2^-137
    an element, and those of the sums."""
    import pto_isa_b200 as p
    n, k = 40, 512
    w = torch.randint(0, 256, (n, k // 2), generator=gen(1), device="cuda", dtype=torch.uint8)
    scale = torch.randint(120, 130, (n, k // 32), generator=gen(2), device="cuda", dtype=torch.uint8)
    weights, mag = ref.w4_weights(w, scale, None, 32)
    for e in (-90, -100, -110):
        x = (torch.randn(m, k, generator=gen(3), device="cuda") * 2.0 ** e).to(dtype)
        y = p.w4_matvec(x, w, scale, out_dtype=torch.float32).double().cpu()
        want = x.double().cpu() @ weights.t()
        bound = (k / 32 + 32) * 2.0 ** -22 * (x.double().cpu().abs() @ mag.t()) + 2.0 ** -137 * mag.sum(1) + 2.0 ** -24 * want.abs()
        assert ((y - want).abs() <= bound).all(), e
