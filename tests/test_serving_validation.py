"""Argument checks of the serving operators (paged cache, attention over a shared prefix, 4-bit weights), without a GPU:
the Python layer with the library replaced by a recorder, and the C entry points' own checks."""
import ctypes

import pytest
import torch

from pto_isa_b200 import _lib, build, ops
from pto_isa_b200._lib import PtoB200Error
from test_ops_validation import rec  # noqa: F401  (the recorder fixture)


def cache(fmt=ops.KV_MXFP8, pages=4, heads=2, page=16, d=64):
    return ops.kv_cache_empty(pages, heads, page, d, fmt, device="cpu")


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def rows(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def table(batch=3, pages=2):
    return torch.zeros(batch, pages, dtype=torch.int32)


def test_cache_shapes():
    c = cache(ops.KV_MXFP4, d=128)
    assert c.k.shape == (4, 2, 16, 64) and c.k_scale.shape == (4, 2, 16, 4) and c.k.dtype == torch.uint8
    c = cache(ops.KV_BF16)
    assert c.v.shape == (4, 2, 16, 64) and c.v.dtype == torch.bfloat16 and c.k_scale is None
    for bad in (dict(page=24), dict(page=8), dict(d=96), dict(fmt=7), dict(heads=0)):
        with pytest.raises(PtoB200Error):
            cache(**bad)


def test_cache_write_checks(rec):  # noqa: F811
    c = cache()
    assert ops.kv_cache_write(c, rows(3, 2, 64), rows(3, 2, 64), i32(0, 1, -1)) is c
    fused = rows(3, 6, 64)
    ops.kv_cache_write(c, fused[:, 2:4], fused[:, 4:], i32(0, 1, 2))  # slices of a fused projection
    assert rec.calls == ["pto_b200_kv_cache_write"] * 2
    ok, s = rows(3, 2, 64), i32(0, 1, 2)
    for k, v, slots, what in [
            (rows(3, 1, 64), rows(3, 1, 64), s, "tokens, 2, 64"), (rows(3, 2, 128), rows(3, 2, 128), s, "tokens, 2, 64"),
            (ok, rows(4, 2, 64), s, "of one type"), (ok, ok.bfloat16(), s, "of one type"), (ok.float(), ok.float(), s, "float16 or bfloat16"),
            (ok, ok, s.long(), "int32"), (ok, ok, i32(0, 1), "of 3"), (ok, ok, s[None], "int32"),
            (rows(3, 2, 128)[..., ::2], ok, s, "contiguous"), (rows(3, 2, 68)[..., 4:], ok, s, "aligned"),
            (rows(3, 2, 65)[..., :64], ok, s, "aligned"), (ok[0], ok[0], s, "3 dimensions")]:
        with pytest.raises(PtoB200Error, match=what):
            ops.kv_cache_write(c, k, v, slots)
    with pytest.raises(PtoB200Error, match="own type"):
        ops.kv_cache_write(cache(ops.KV_F16), ok.bfloat16(), ok.bfloat16(), s)
    assert len(rec.calls) == 2


def test_cache_description_checks(rec):  # noqa: F811
    c = cache()
    k, s = rows(1, 2, 64), i32(0)
    for bad, what in [
            (c._replace(fmt=9), "unknown cache format"), (c._replace(k_scale=None), "needs its scales"),
            (c._replace(v=c.v[:2]), "one type"), (c._replace(k_scale=c.k_scale[..., :1]), "scales are"),
            (c._replace(k=c.k.float(), v=c.v.float()), "type of its format"), (c._replace(fmt=ops.KV_MXFP4, k=c.k[..., :24].contiguous(), v=c.v[..., :24].contiguous()), "head_dim is 64 or 128"),
            (cache(ops.KV_F16)._replace(k_scale=c.k_scale, v_scale=c.v_scale), "no scales"),
            (cache(ops.KV_F16)._replace(fmt=ops.KV_BF16), "type of its format"),
            (c._replace(k=c.k[0], v=c.v[0]), "num_pages")]:
        with pytest.raises(PtoB200Error, match=what):
            ops.kv_cache_write(bad, k, k, s)
    ops.kv_cache_write(tuple(c), k, k, s)  # any 5-tuple of that order
    assert rec.calls == ["pto_b200_kv_cache_write"]


def test_cache_read_checks(rec):  # noqa: F811
    c = cache()
    k, v = ops.kv_cache_read(c, table(), i32(1, 0, 32), 32, dtype=torch.bfloat16)
    assert k.shape == v.shape == (3, 2, 32, 64) and k.dtype == torch.bfloat16
    with pytest.raises(PtoB200Error, match="float16 or bfloat16"):
        ops.kv_cache_read(c, table(), i32(1, 0, 32), 32, dtype=torch.float32)
    with pytest.raises(PtoB200Error, match="page table"):
        ops.kv_cache_read(c, table(2), i32(1, 0, 32), 32)
    with pytest.raises(PtoB200Error, match="page table"):
        ops.kv_cache_read(c, table().long(), i32(1, 0, 32), 32)
    with pytest.raises(PtoB200Error, match="page table"):
        ops.kv_cache_read(c, torch.zeros(2, 3, dtype=torch.int32).t(), i32(1, 0, 32), 32)
    with pytest.raises(PtoB200Error, match="int32"):
        ops.kv_cache_read(c, table(), torch.zeros(3), 32)
    with pytest.raises(PtoB200Error, match="must have shape"):
        ops.kv_cache_read(c, table(), i32(1, 0, 32), 32, out=(torch.zeros(3, 2, 16, 64, dtype=torch.float16), None))
    with pytest.raises(PtoB200Error, match="negative"):
        ops.kv_cache_read(c, table(), i32(1, 0, 32), -1)
    assert rec.calls == ["pto_b200_kv_cache_read"]


@pytest.fixture()
def attn_rec(rec):  # noqa: F811
    rec.pto_b200_prefix_attn_workspace_bytes = lambda *a: 64
    return rec


def test_prefix_attn_checks(attn_rec):
    c = cache(pages=8)
    q, pages, lens = rows(3, 2, 4, 64), i32(0, 1), i32(1, 0, 32)
    assert ops.prefix_attn(q, c, pages, 20, table(), lens).shape == q.shape
    o, lse = ops.prefix_attn(q[:, 0], c, pages, 0, table(), lens, return_lse=True)
    assert o.shape == (3, 4, 64) and lse.shape == (3, 4) and lse.dtype == torch.float32
    fused = rows(3, 2, 8, 64)
    ops.prefix_attn(fused[:, :, :4], c, pages, 32, table(), lens, max_seq_len=5)
    n = len(attn_rec.calls)
    assert n == 3
    call = lambda **kw: ops.prefix_attn(**{**dict(q=q, cache=c, prefix_pages=pages, prefix_len=20, page_table=table(), seq_lens=lens), **kw})
    for kw, what in [
            (dict(q=rows(3, 2, 3, 64)), "multiple of 2"), (dict(q=rows(3, 2, 4, 128)), "multiple of 2"), (dict(q=q.float()), "float16 or bfloat16"),
            (dict(q=rows(3, 0, 4, 64)), "multiple of 2"), (dict(q=rows(4, 64)), "4 dimensions"), (dict(q=rows(3, 2, 4, 128)[..., ::2]), "contiguous"),
            (dict(prefix_len=33), "within prefix_pages"), (dict(prefix_len=-1), "within prefix_pages"), (dict(prefix_pages=pages.long()), "int32"),
            (dict(seq_lens=i32(1, 2)), "of 3"), (dict(page_table=table(2)), "page table"), (dict(max_seq_len=33), "within the page table"),
            (dict(max_seq_len=-1), "within the page table"), (dict(out=q.bfloat16()), "must have shape"),
            (dict(cache=cache(ops.KV_BF16, pages=8)), "own type"), (dict(workspace=torch.zeros(8, dtype=torch.uint8)), "workspace needs 64")]:
        with pytest.raises(PtoB200Error, match=what):
            call(**kw)
    assert len(attn_rec.calls) == n
    assert ops.prefix_attn(rows(0, 2, 4, 64), c, pages, 20, table(0), torch.zeros(0, dtype=torch.int32)).shape == (0, 2, 4, 64)
    assert len(attn_rec.calls) == n  # an empty batch launches nothing


def test_w4_matvec_checks(rec):  # noqa: F811
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    x, w = rows(3, 256), u8(40, 128)
    assert ops.w4_matvec(x, w, u8(40, 8)).shape == (3, 40)
    assert ops.w4_matvec(x[0], w, rows(40, 2), zero=rows(40, 2), out_dtype=torch.float32).shape == (40,)
    n = len(rec.calls)
    assert rec.calls.count("pto_b200_w4_matvec") == 2
    for kw, what in [
            (dict(x=rows(3, 192)), r"\(n, 96\)"), (dict(x=rows(65, 256)), "at most 64"), (dict(x=x.float()), "float16 or bfloat16"),
            (dict(scale=u8(40, 4)), "one scale byte per 32"), (dict(scale=u8(39, 8)), "scale is"), (dict(scale=rows(40, 1)), "32, 64 or 128"),
            (dict(scale=rows(40, 2, dtype=torch.bfloat16)), "x's type"), (dict(zero=rows(40, 8)), "no zeros"),
            (dict(scale=rows(40, 2), zero=rows(40, 4)), "zero is like scale"), (dict(out_dtype=torch.bfloat16), "x's type or float32"),
            (dict(out=rows(3, 41)), "must have shape"), (dict(x=rows(3, 260)[:, 4:]), "aligned"), (dict(x=rows(256, 3).t()), "contiguous"),
            (dict(scale=u8(40, 0)), "scale is"), (dict(w=w.to(torch.int16)), r"\(n, 128\) bytes")]:
        with pytest.raises(PtoB200Error, match=what):
            ops.w4_matvec(**{**dict(x=x, w=w, scale=u8(40, 8)), **kw})
    assert rec.calls.count("pto_b200_w4_matvec") == 2


def test_cpu_tensors_are_refused():
    c = cache()
    for call in (lambda: ops.kv_cache_write(c, rows(1, 2, 64), rows(1, 2, 64), i32(0)),
                 lambda: ops.kv_cache_read(c, table(), i32(0, 0, 0), 16),
                 lambda: ops.prefix_attn(rows(3, 1, 2, 64), c, i32(0), 1, table(), i32(0, 0, 0)),
                 lambda: ops.w4_matvec(rows(1, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8))):
        with pytest.raises(PtoB200Error, match="CUDA"):
            call()


@pytest.fixture(scope="module")
def clib():
    build.build()
    return _lib.lib()


def test_c_entry_points_refuse_before_they_touch_a_device(clib):
    some = ctypes.c_void_p(1 << 20)  # never dereferenced
    desc = lambda **kw: ctypes.byref(ops._CacheStruct(**{**dict(k=1 << 20, v=1 << 20, k_scale=1 << 20, v_scale=1 << 20, num_pages=4, format=2, kv_heads=2, page_size=16, head_dim=64), **kw}))
    s4, s3 = (ctypes.c_int64 * 4)(128, 64, 128, 64), (ctypes.c_int64 * 3)(512, 256, 64)
    write = lambda c, dtype=2, tokens=1, k=some, s=s4: clib.pto_b200_kv_cache_write(c, k, some, dtype, some, tokens, s, None)
    assert write(None) == 1 and write(desc(format=4)) == 1 and write(desc(format=-1)) == 1 and write(desc(), dtype=0) == 1
    assert write(desc(k_scale=None)) == 1 and write(desc(kv_heads=0)) == 1 and write(desc(num_pages=-1)) == 1
    assert write(desc(page_size=48)) == 2 and write(desc(page_size=2048)) == 2 and write(desc(head_dim=96)) == 2
    assert write(desc(k=(1 << 20) + 8)) == 2 and write(desc(v_scale=(1 << 20) + 4)) == 2
    assert write(desc(num_pages=1 << 28)) == 5 and write(desc(format=0), dtype=4) == 1 and write(desc(), tokens=-1) == 1
    assert write(desc(), k=ctypes.c_void_p((1 << 20) + 2)) == 2 and write(desc(), s=(ctypes.c_int64 * 4)(128, 60, 128, 64)) == 2
    assert write(desc(), tokens=0) == 0
    read = lambda c, batch=1, n=16, lens=some, out=some: clib.pto_b200_kv_cache_read(c, some, 4, 4, lens, batch, n, out, some, 2, None)
    assert read(desc(), batch=-1) == 1 and read(desc(), n=-1) == 1 and read(desc(), lens=None) == 1
    assert read(desc(), out=ctypes.c_void_p((1 << 20) + 2)) == 2 and read(desc(), batch=0) == 0 and read(desc(), n=0) == 0

    def attn(c=None, heads=4, tokens=1, batch=1, prefix=16, most=16, q=some, ws=some, ws_bytes=0, s=s3):
        return clib.pto_b200_prefix_attn(c or desc(), q, 2, s, some, prefix, some, 4, 4, some, most, batch, tokens, heads, 1.0, some, None, ws, ws_bytes, None)
    assert attn(heads=3) == 1 and attn(tokens=0) == 1 and attn(prefix=-1) == 1 and attn(q=None) == 1 and attn(most=65) == 1
    assert attn(batch=1 << 26, tokens=2) == 5 and attn(q=ctypes.c_void_p((1 << 20) + 2)) == 2
    assert attn(s=(ctypes.c_int64 * 3)(512, 256, 63)) == 2 and attn(ws=ctypes.c_void_p((1 << 20) + 8)) == 2 and attn(batch=0) == 0
    assert attn(ws_bytes=100) == 1 and b"workspace" in clib.pto_b200_last_error()
    need = clib.pto_b200_prefix_attn_workspace_bytes
    assert need(0, 1, 4, 2, 64, 16, 16) == 0 and need(1, 1, 3, 2, 64, 16, 16) == 0 and need(1, 1, 4, 2, 64, 0, 0) == 0
    assert need(1, 1, 4, 2, 64, 16, 16) > 0

    def w4(m=1, n=8, k=64, group=32, fmt=0, dtype=2, x=some, zero=None, stride=64):
        return clib.pto_b200_w4_matvec(x, stride, some, some, zero, some, m, n, k, group, fmt, dtype, 0, None, 0, None)
    assert w4(m=-1) == 1 and w4(fmt=2) == 1 and w4(dtype=0) == 1 and w4(x=None) == 1 and w4(m=65) == 2 and w4(zero=some) == 1
    assert w4(group=64) == 1 and w4(fmt=1, group=48) == 1 and w4(k=48) == 2 and w4(k=0) == 2 and w4(fmt=1, group=128) == 2
    assert clib.pto_b200_w4_matvec_workspace_bytes(1, 4096, 0) == 0 and clib.pto_b200_w4_matvec_workspace_bytes(3, 4096, 0) > 0
    assert w4(m=3) == 1 and b"workspace" in clib.pto_b200_last_error()
    assert w4(x=ctypes.c_void_p((1 << 20) + 2)) == 2 and w4(stride=60) == 2 and w4(m=0) == 0 and w4(n=0) == 0
    odd = ctypes.c_void_p((1 << 20) + 1)
    assert clib.pto_b200_w4_matvec(some, 64, some, odd, None, some, 1, 8, 64, 32, 1, 2, 0, None, 0, None) == 2
    assert w4(fmt=1, zero=odd) == 2 and clib.pto_b200_w4_matvec(some, 64, some, some, None, odd, 1, 8, 64, 32, 0, 2, 0, None, 0, None) == 2
