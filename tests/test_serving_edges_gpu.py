"""Edges of the serving operators that test_serving_gpu.py does not reach, against the same 64-bit statements: the tensor memory
kernel with many key tiles a block, every scale byte and code in a cache, what the status record gets."""
import pytest
import torch

import serving_ref as ref
from test_serving_gpu import BF16, F16, FORMATS, check_attention, fmt_of, garbage_cache, gen, make_attention, status, values  # noqa: F401

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
