"""Host-side tests of the paged cache's operators (``cache_write``, ``cache_read``, ``attention_paged``): bad
arguments are rejected before anything is launched, by the C entry points with hipErrorInvalidValue and by the
PyTorch operators with a message. No GPU is used; arguments that are right in all else end at "must be a GPU
tensor"."""
import ctypes

import pytest
import torch

from megakernel import build as mkbuild

INVALID = 1  # hipErrorInvalidValue
vp, i32, i64, size = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
P, Q, R, S = 4096, 8192, 12288, 16384  # aligned addresses that nothing reads


class Pool(ctypes.Structure):  # mk_paged_cache
    _fields_ = ([(n, vp) for n in ("k_pages", "v_pages", "k_scales", "v_scales")] +
                [(n, i64) for n in ("page_stride", "head_stride", "row_stride", "scale_page_stride",
                                    "scale_head_stride")] +
                [("block_tables", vp), ("table_stride", i64)] +
                [(n, ctypes.c_int32) for n in ("table_entries", "num_pages", "kv_heads", "page_size", "num_seqs")])


def pool(e4m3=False, **kw):
    c = dict(k_pages=P, v_pages=Q, k_scales=R if e4m3 else None, v_scales=S if e4m3 else None, page_stride=8 * 16 * 128,
             head_stride=16 * 128, row_stride=128, scale_page_stride=8 * 16, scale_head_stride=16, block_tables=P,
             table_stride=32, table_entries=32, num_pages=100, kv_heads=8, page_size=16, num_seqs=2)
    c.update(kw)
    return Pool(**c)


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(mkbuild.LIB)
    pp = ctypes.POINTER(Pool)
    lib.mk_cache_write.argtypes = [pp, vp, i64, i64, vp, i64, i64, i32, vp, vp, vp]
    lib.mk_cache_read.argtypes = [pp, vp, vp, vp, vp, vp]
    lib.mk_attention_paged_workspace_bytes.restype = size
    lib.mk_attention_paged_workspace_bytes.argtypes = [i32, i32]
    lib.mk_attention_paged.argtypes = [pp, i32, vp, i64, i64, i32, vp, vp, vp, size, vp]
    return lib


BAD_POOLS = [dict(k_pages=None), dict(v_pages=None), dict(v_pages=P), dict(block_tables=None), dict(k_pages=P + 8),
             dict(v_pages=Q + 8), dict(block_tables=P + 2), dict(page_stride=-8), dict(head_stride=-8), dict(row_stride=-8),
             dict(page_stride=8 * 16 * 128 + 4), dict(head_stride=16 * 128 + 4), dict(row_stride=132), dict(row_stride=(1 << 24) + 8), dict(num_pages=0),
             dict(kv_heads=0), dict(kv_heads=65536), dict(page_size=0), dict(page_size=24), dict(page_size=8192),
             dict(num_seqs=0), dict(table_entries=0), dict(table_stride=-1), dict(table_entries=(1 << 26) + 1),
             dict(k_scales=R), dict(v_scales=S), dict(k_scales=R, v_scales=R)]
BAD_E4M3 = [dict(scale_page_stride=-1), dict(scale_head_stride=-16), dict(row_stride=136)]
OVERLAP = [dict(row_stride=64), dict(head_stride=0), dict(page_stride=0), dict(page_stride=7 * 16 * 128),
           dict(head_stride=15 * 128)]


def _lengths(values):
    return (ctypes.c_int32 * max(1, len(values)))(*values)


@pytest.mark.parametrize("fp32", [0, 1])
def test_cache_write_c(lib, fp32):
    def call(c=None, k=P, ks=(1024, 128), v=P, vs=(1024, 128), begin=P, lengths=(0, 0)):
        arr = _lengths(lengths) if lengths is not None else None
        c = pool() if c is None else c
        return lib.mk_cache_write(ctypes.byref(c) if c else None, k, *ks, v, *vs, fp32, begin, arr, None)

    assert call() == call(k=None) == call(pool(True)) == 0  # no rows: nothing to do
    assert call(False) == call(begin=None) == call(lengths=None) == call(lengths=(3, -1)) == INVALID
    assert call(lengths=(2 ** 31 - 1, 1)) == call(lengths=(2 ** 25, 1)) == INVALID
    one = (1, 1)
    assert call(k=None, lengths=one) == call(v=None, lengths=one) == call(k=P + 8, lengths=one) == INVALID
    assert call(v=P + 8, lengths=one) == call(ks=(1022, 128), lengths=one) == call(vs=(1024, 126), lengths=one) == INVALID
    assert call(ks=(-1024, 128), lengths=one) == call(vs=(1024, -128), lengths=one) == INVALID
    for bad in BAD_POOLS + OVERLAP:
        assert call(pool(**bad)) == INVALID, bad
    for bad in BAD_E4M3 + [dict(scale_head_stride=8), dict(scale_page_stride=0)]:
        assert call(pool(True, **bad)) == INVALID, bad
    # other orders of the dimensions, and a lone head or page of any stride
    assert call(pool(head_stride=128, row_stride=1024)) == call(pool(num_pages=1, page_stride=0)) == 0
    assert call(pool(page_stride=2 * 8 * 16 * 128)) == call(pool(kv_heads=1, head_stride=0)) == 0


def test_cache_read_c(lib):
    def call(c=None, begin=P, lengths=(0, 0), k=P, v=Q):
        arr = _lengths(lengths) if lengths is not None else None
        c = pool() if c is None else c
        return lib.mk_cache_read(ctypes.byref(c) if c else None, begin, arr, k, v, None)

    assert call() == call(pool(True)) == 0
    assert call(False) == call(begin=None) == call(lengths=None) == call(lengths=(-1, 5)) == INVALID
    one = (1, 0)
    assert call(k=None, lengths=one) == call(v=None, lengths=one) == call(k=Q, lengths=one) == INVALID
    assert call(k=P + 8, lengths=one) == call(v=Q + 8, lengths=one) == INVALID
    for bad in BAD_POOLS:
        assert call(pool(**bad)) == INVALID, bad
    for bad in BAD_E4M3:
        assert call(pool(True, **bad)) == INVALID, bad
    for overlap in OVERLAP:  # may be read
        assert call(pool(**overlap)) == 0, overlap


def test_attention_paged_c(lib):
    need = lib.mk_attention_paged_workspace_bytes
    assert need(0, 8) == need(16, 0) == need(12, 8) == need(-16, -8) == 0
    assert 0 < need(8, 8) < need(16, 8) < need(128, 8) == need(200, 8) and need(16, 8) % 256 == 0

    def call(c=None, hq=16, q=P, qs=(2048, 128), fp32=0, lengths=P, out=Q, ws=P, nbytes=1 << 30):
        c = pool() if c is None else c
        return lib.mk_attention_paged(ctypes.byref(c) if c else None, hq, q, *qs, fp32, lengths, out, ws, nbytes, None)

    assert call(False) == call(hq=0) == call(hq=12) == call(hq=-8) == INVALID
    assert call(q=None) == call(lengths=None) == call(out=None) == call(ws=None) == INVALID
    assert call(q=P + 8) == call(out=Q + 8) == call(ws=P + 128) == call(nbytes=need(16, 8) - 1) == INVALID
    assert call(qs=(2044, 128)) == call(qs=(2048, 124)) == call(qs=(-2048, 128)) == call(qs=(2046, 128), fp32=1) == INVALID
    assert call(pool(num_seqs=4097)) == INVALID
    assert call(pool(num_seqs=4096, kv_heads=8192), hq=8192) == INVALID  # 2^32 elements of output
    for bad in BAD_POOLS:
        assert call(pool(**bad)) == INVALID, bad
    for bad in BAD_E4M3:
        assert call(pool(True, **bad)) == INVALID, bad


# ---------------------------------------------------------------------------------------------
# the PyTorch operators
# ---------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def ext():
    import megakernel
    return megakernel.load()


BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def _pages(e4m3, n=10, h=8, p=16):
    make = lambda: torch.zeros(n, h, p, 128).to(E4 if e4m3 else BF)  # noqa: E731
    scales = lambda: torch.full((n, h, p), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu)  # noqa: E731
    return (make(), make()) + ((scales(), scales()) if e4m3 else (None, None))


def _refuses(match, fn, *args):
    with pytest.raises(RuntimeError, match=match):
        fn(*args)


def _calls(ext):
    """The three operators as functions of (k_pages, v_pages, tables, k_scales, v_scales), all else right."""
    i = torch.zeros(2, dtype=torch.int32)
    k, v, q = torch.zeros(5, 8, 128), torch.zeros(5, 8, 128), torch.zeros(2, 16, 128)
    return [lambda kp, vp, t, ks, vs: ext.cache_write(k, v, kp, vp, t, i, [2, 3], ks, vs),
            lambda kp, vp, t, ks, vs: ext.cache_read(kp, vp, t, i, [2, 3], ks, vs),
            lambda kp, vp, t, ks, vs: ext.attention_paged(q, kp, vp, t, i, ks, vs)]


def test_pools_of_the_ops(ext):
    t = torch.zeros(2, 4, dtype=torch.int32)
    bk, bv, _, _ = _pages(False)
    ek, ev, es, fs = _pages(True)
    for f in _calls(ext):
        _refuses("must be a GPU tensor", f, bk, bv, t, None, None)
        _refuses("must be a GPU tensor", f, ek, ev, t, es, fs)
        both = torch.zeros(10, 2, 8, 16, 128, dtype=BF)
        _refuses("must be a GPU tensor", f, both[:, 0], both[:, 1], t, None, None)  # one pool of both
        _refuses("must be a GPU tensor", f, bk.view(10, 16, 8, 128).transpose(1, 2), bv.view(10, 16, 8, 128).transpose(1, 2),
                 t, None, None)
        _refuses("must be a GPU tensor", f, bk, bv, torch.zeros(2, 9, dtype=torch.int32)[:, 2:6], None, None)
        _refuses("k_pages must be", f, bk.float(), bv, t, None, None)
        _refuses("k_pages must be", f, bk[0], bv, t, None, None)
        _refuses("k_pages must be", f, bk[..., :64], bv, t, None, None)
        _refuses("has no pages", f, bk[:0], bv[:0], t, None, None)
        _refuses("power of two", f, bk[:, :, :12], bv[:, :, :12], t, None, None)
        _refuses("power of two", f, bk[:, :, :0], bv[:, :, :0], t, None, None)
        _refuses("v_pages must be like", f, bk, bv.float(), t, None, None)
        _refuses("v_pages must be like", f, bk, bv[:, :4], t, None, None)
        _refuses("v_pages must be like", f, bk, bv.to("meta"), t, None, None)
        _refuses("same strides", f, bk, both[:, 1], t, None, None)
        _refuses("must be distinct", f, bk, bk, t, None, None)
        _refuses("contiguous in its last", f, torch.zeros(10, 8, 16, 256, dtype=BF)[..., ::2], bv, t, None, None)
        far = torch.empty((1 << 24) + 256, dtype=BF).as_strided((1, 1, 2, 128), (0, 0, (1 << 24) + 8, 1))
        _refuses("at most 2\\^24", f, far, far, t, None, None)
        _refuses("16-byte boundaries", f, torch.zeros(10, 8, 16, 132, dtype=BF)[..., :128], bv, t, None, None)
        _refuses("16-byte boundary", f, torch.zeros(10 * 16384 + 4, dtype=BF)[4:].view(10, 8, 16, 128), bv, t, None, None)
        _refuses("need k_scales", f, ek, ev, t, None, None)
        _refuses("need k_scales", f, ek, ev, t, es, None)
        _refuses("need k_scales", f, bk, bv, t, es, fs)
        _refuses("k_scales must be", f, ek, ev, t, es.view(torch.uint8), fs)
        _refuses("v_scales must be", f, ek, ev, t, es, fs[:5])
        _refuses("k_scales must be contiguous", f, ek, ev, t, torch.zeros(10, 8, 32, dtype=torch.uint8).view(
            torch.float8_e8m0fnu)[..., ::2], fs)
        _refuses("scales must have the same strides", f, ek, ev, t, es, torch.zeros(10, 9, 16, dtype=torch.uint8).view(
            torch.float8_e8m0fnu)[:, :8])
        _refuses("scales must be distinct", f, ek, ev, t, es, es)
        _refuses("block_tables must be", f, bk, bv, t.long(), None, None)
        _refuses("block_tables must be", f, bk, bv, t[0], None, None)
        _refuses("block_tables must be", f, bk, bv, t[:, :0], None, None)
        _refuses("block_tables must be", f, bk, bv, torch.zeros(2, 8, dtype=torch.int32)[:, ::2], None, None)
        _refuses("2\\^30", f, bk, bv, torch.empty(1, (1 << 26) + 1, dtype=torch.int32).expand(2, -1), None, None)


def test_cache_write_op(ext):
    kp, vp, _, _ = _pages(False)
    t, i = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    k, v = torch.zeros(5, 8, 128), torch.zeros(5, 8, 128)

    def f(k=k, v=v, begin=i, lengths=(2, 3), kp=kp, vp=vp, **kw):
        return ext.cache_write(k, v, kp, vp, t, begin, list(lengths), **kw)

    def refuses(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            f(**kw)

    for kind in (torch.float32, BF):
        fused = torch.zeros(5, 16, 128, dtype=kind)
        refuses("must be a GPU tensor", k=fused[:, :8], v=fused[:, 8:])
    refuses("lengths must name", lengths=(5,))
    refuses("lengths must be at least 0", lengths=(6, -1))
    refuses("lengths must be at least 0", lengths=(2 ** 31 - 1, 1))
    refuses("add up to at most 2", lengths=(2 ** 25, 1))
    refuses("k must be bfloat16 or float32", k=k.half())
    refuses("v must be Float", v=v.to(BF))
    refuses("k must have 5 rows", k=k[:4])
    refuses("the pages' 8 heads", k=k[:, :4])
    refuses("16-byte boundaries", k=torch.zeros(5, 8, 130)[..., :128])
    refuses("begin must be", begin=i.long())
    refuses("begin must be", begin=i[:1])
    refuses("no elements that overlap", kp=kp[:1].expand(10, -1, -1, -1), vp=vp[:1].expand(10, -1, -1, -1))
    refuses("no elements that overlap", kp=kp[:, :1].expand(-1, 8, -1, -1), vp=vp[:, :1].expand(-1, 8, -1, -1))
    ek, ev, es, fs = _pages(True)
    refuses("no elements that overlap", kp=ek, vp=ev, k_scales=es[:1].expand(10, -1, -1), v_scales=fs[:1].expand(10, -1, -1))


def test_cache_read_op(ext):
    kp, vp, _, _ = _pages(False)
    t, i = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    _refuses("lengths must name", ext.cache_read, kp, vp, t, i, [1, 2, 3])
    _refuses("lengths must be at least 0", ext.cache_read, kp, vp, t, i, [1, -2])
    _refuses("begin must be", ext.cache_read, kp, vp, t, i.float(), [1, 2])
    _refuses("must be a GPU tensor", ext.cache_read, kp[:1].expand(10, -1, -1, -1), vp[:1].expand(10, -1, -1, -1), t, i, [1, 2])


def test_attention_paged_op(ext):
    kp, vp, _, _ = _pages(False)
    t, n = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q, f = torch.zeros(2, 16, 128), ext.attention_paged
    for kind in (torch.float32, BF):
        _refuses("must be a GPU tensor", f, torch.zeros(2, 32, 128, dtype=kind)[:, :16], kp, vp, t, n)
    _refuses("q must be bfloat16 or float32", f, q.half(), kp, vp, t, n)
    _refuses("q must have 2 rows", f, q[:1], kp, vp, t, n)
    _refuses("q must be \\[rows, heads, 128\\]", f, q[0], kp, vp, t, n)
    _refuses("must be a multiple", f, q[:, :12], kp, vp, t, n)
    _refuses("lengths must be", f, q, kp, vp, t, n.long())
    _refuses("lengths must be", f, q, kp, vp, t, torch.zeros(4, dtype=torch.int32)[::2])
    _refuses("at most 4096", f, torch.zeros(4097, 8, 128, dtype=BF), kp, vp, t[:1].expand(4097, -1),
             torch.zeros(4097, dtype=torch.int32))
    _refuses("k_pages.*on|q must be on", f, q.to("meta"), kp, vp, t, n)
