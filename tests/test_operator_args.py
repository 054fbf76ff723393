"""Host-side tests of the operators for several sequences (``prefill_batch``, ``attention_packed``,
``beam_select``, ``beam_reorder``): bad arguments are rejected before anything is launched, by the C entry
points with hipErrorInvalidValue and by the PyTorch operators with a message. No GPU is used; arguments that
are right in all else end at "must be a GPU tensor"."""
import ctypes

import pytest
import torch

from megakernel import build as mkbuild

INVALID = 1  # hipErrorInvalidValue
vp, i32, i64, size = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
P = vp(4096)  # an aligned address that nothing reads


class Dims(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int32), ("intermediate", ctypes.c_int32),
                ("num_layers", ctypes.c_int32), ("vocab", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(mkbuild.LIB)
    lib.mk_attention_packed.argtypes = [i32, i32, vp, i64, i64, vp, i64, i64, vp, i64, i64, vp, i32, i32, vp, vp]
    lib.mk_beam_select_workspace_bytes.restype = size
    lib.mk_beam_select_workspace_bytes.argtypes = [i32, i32, i32]
    lib.mk_beam_select.argtypes = [i32, i32, i32, vp, i64, vp, vp, i32, vp, vp, vp, vp, vp, size, vp]
    lib.mk_beam_reorder.argtypes = [i32, i32, i32, i32, vp, vp, vp, vp, vp, vp]
    lib.mk_prefill_batch_workspace_bytes.restype = size
    lib.mk_prefill_batch_workspace_bytes.argtypes = [vp, i32]
    lib.mk_prefill_batch.argtypes = [vp, vp, vp, i32] + [vp] * 8 + [i64, i32, vp, vp, vp, size, vp]
    return lib


def _lengths(values):
    return (ctypes.c_int32 * max(1, len(values)))(*values)


def test_attention_packed_c(lib):
    def call(hq=16, hkv=8, q=P, qs=(2048, 128), k=P, ks=(1024, 128), v=P, vs=(1024, 128), lengths=(5, 3), fp32=0, out=P):
        arr = _lengths(lengths) if lengths is not None else None
        return lib.mk_attention_packed(hq, hkv, q, *qs, k, *ks, v, *vs, arr, len(lengths or (1,)), fp32, out, None)

    assert call(lengths=()) == 0 and call(lengths=(0, 0)) == 0  # nothing to do
    assert call(hq=0) == call(hkv=0) == call(hq=12) == call(hq=-16) == INVALID
    assert call(lengths=None) == call(lengths=(5, -1)) == INVALID
    assert call(q=None) == call(k=None) == call(v=None) == call(out=None) == INVALID
    for odd in (vp(4096 + 8),):
        assert call(q=odd) == call(k=odd) == call(v=odd) == call(out=odd) == INVALID
    assert call(qs=(2044, 128)) == call(qs=(2048, 127)) == call(qs=(-2048, 128)) == INVALID
    assert call(ks=(1020, 128)) == call(ks=(1024, 100)) == call(vs=(1020, 128)) == call(vs=(1024, -8)) == INVALID
    assert call(ks=((1 << 24) + 8, 128)) == call(vs=((1 << 24) + 8, 128)) == INVALID
    assert call(qs=(2046, 128), fp32=1) == INVALID
    assert call(lengths=(2 ** 30, 2 ** 30)) == call(lengths=(2 ** 27,)) == INVALID  # 2^31 (row, head) pairs


def test_beam_select_c(lib):
    need = lib.mk_beam_select_workspace_bytes
    assert 0 < need(4, 151936, 4) < need(8, 151936, 4) < need(8, 1 << 20, 4) and need(8, 151936, 4) % 256 == 0
    assert need(0, 100, 1) == need(4, 0, 1) == need(4, (1 << 20) + 1, 1) == need(4, 100, 0) == need(34, 100, 17) == 0

    def call(rows=8, vocab=1000, beams=4, logits=P, stride=1000, scores=P, finished=P, eos=3, outs=(P, P, P, P), ws=P,
             nbytes=1 << 30):
        return lib.mk_beam_select(rows, vocab, beams, logits, stride, scores, finished, eos, *outs, ws, nbytes, None)

    assert call(rows=0) == call(rows=7) == call(rows=65536) == call(beams=0) == call(beams=17, rows=17) == INVALID
    assert call(vocab=0) == call(vocab=(1 << 20) + 1) == call(stride=-1) == INVALID
    assert call(eos=-2) == call(eos=1000) == INVALID
    assert call(logits=None) == call(scores=None) == call(finished=None) == call(ws=None) == INVALID
    for i in range(4):
        assert call(outs=tuple(None if j == i else P for j in range(4))) == INVALID
    assert call(nbytes=need(8, 1000, 4) - 1) == call(ws=vp(4096 + 16)) == INVALID


def test_beam_reorder_c(lib):
    Q = vp(8192)

    def call(layers=28, rows=8, beams=4, max_seq=512, k=P, v=Q, parents=P, begin=P, end=P):
        return lib.mk_beam_reorder(layers, rows, beams, max_seq, k, v, parents, begin, end, None)

    assert call(layers=0) == call(max_seq=0) == call(beams=0) == call(rows=0) == call(rows=9) == INVALID
    assert call(beams=17, rows=17) == call(rows=4 * 65536) == call(max_seq=2 ** 31 - 1) == INVALID
    assert call(k=None) == call(v=None) == call(parents=None) == call(begin=None) == call(end=None) == INVALID
    assert call(k=Q) == call(k=vp(4104)) == call(v=vp(8200)) == INVALID
    assert call(beams=1) == 0  # a lone beam has nothing to move


def test_prefill_batch_c(lib):
    good = Dims(1024, 3072, 28, 151936)
    need = lib.mk_prefill_batch_workspace_bytes
    assert need(None, 5) == need(ctypes.byref(good), 0) == need(ctypes.byref(good), 262145) == 0
    sizes = [need(ctypes.byref(good), n) for n in range(1, 5000)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0  # never shrinks with the token count
    assert all(n % 256 == 0 for n in sizes)
    one = 28 * 8 * 512 * 128

    def call(dims=good, tokens=P, lengths=(5, 9), n=None, ptrs=(P,) * 8, stride=one, max_seq=512, logits=P, ws=P,
             nbytes=1 << 34):
        d = ctypes.byref(dims) if dims is not None else None
        arr = _lengths(lengths) if lengths is not None else None
        return lib.mk_prefill_batch(d, tokens, arr, len(lengths or ()) if n is None else n, *ptrs, stride, max_seq, logits,
                                    None, ws, nbytes, None)

    assert call(dims=None) == call(tokens=None) == call(lengths=None, n=1) == call(logits=None) == INVALID
    assert call(ws=None) == call(ws=vp(4096 + 128)) == INVALID
    for i in range(8):
        assert call(ptrs=tuple(None if j == i else P for j in range(8))) == INVALID
    assert call(dims=Dims(1024, 4096, 28, 151936)) == call(dims=Dims(1024, 3072, 0, 151936)) == INVALID
    assert call(dims=Dims(1024, 3072, 28, 1000)) == INVALID  # vocabulary no multiple of 16
    assert call(lengths=()) == call(lengths=(1,) * 65) == call(lengths=(5, 0)) == call(lengths=(-1,)) == INVALID
    assert call(lengths=(5, 513)) == call(lengths=(2 ** 31 - 1,), max_seq=2 ** 31 - 1) == INVALID
    for i in (6, 7):  # the caches' alignment
        assert call(ptrs=tuple(vp(4104) if j == i else P for j in range(8))) == INVALID
    assert call(stride=one - 8) == call(stride=one + 4) == call(max_seq=0) == INVALID
    assert call(nbytes=1000) == INVALID


# ---------------------------------------------------------------------------------------------
# the PyTorch operators
# ---------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def ext():
    import megakernel
    return megakernel.load()


def _refuses(match, fn, *args):
    with pytest.raises(RuntimeError, match=match):
        fn(*args)


def test_attention_packed_op(ext):
    f = ext.attention_packed
    bf = torch.bfloat16
    q, k, v = torch.zeros(8, 16, 128, dtype=bf), torch.zeros(8, 8, 128, dtype=bf), torch.zeros(8, 8, 128, dtype=bf)
    for qq in (q, q.float()):
        _refuses("must be a GPU tensor", f, qq, k, v, [5, 3])
    fused = torch.zeros(8, 32, 128, dtype=bf)
    _refuses("must be a GPU tensor", f, fused[:, :16], fused[:, 16:24], fused[:, 24:], [0, 8])
    _refuses("must be a GPU tensor", f, q[:1].as_strided((1, 16, 128), (3, 128, 1)), k[:1], v[:1], [1])  # one row: no stride
    _refuses("q must be bfloat16 or float32", f, q.half(), k, v, [8])
    _refuses("k must be BFloat16", f, q, k.float(), v, [8])
    _refuses("v must be BFloat16", f, q, k, v.half(), [8])
    _refuses("must be \\[rows, heads, 128\\]", f, q[0], k, v, [8])
    _refuses("must be \\[rows, heads, 128\\]", f, q[..., :64], k, v, [8])
    _refuses("k must be \\[rows, heads, 128\\]", f, q, k.reshape(8, -1), v, [8])
    _refuses("k must have 8 rows", f, q, k[:7], v, [8])
    _refuses("same number of heads", f, q, k, v[:, :4], [8])
    _refuses("must be a multiple", f, q[:, :12], k, v, [8])
    _refuses("contiguous in its last", f, torch.zeros(8, 16, 256, dtype=bf)[..., ::2], k, v, [8])
    _refuses("16-byte boundaries", f, torch.zeros(8 * 2052, dtype=bf).as_strided((8, 16, 128), (2052, 128, 1)), k, v, [8])
    _refuses("16-byte boundaries", f, torch.zeros(8 * 2048 + 4, dtype=bf)[4:].view(8, 16, 128), k, v, [8])
    _refuses("at most 2\\^24", f, q[:2], torch.empty((1 << 24) + 2048, dtype=bf).as_strided((2, 8, 128), ((1 << 24) + 8, 128, 1)),
             v[:2], [2])
    _refuses("add up to 7", f, q, k, v, [4, 3])
    _refuses("add up to 0", f, q, k, v, [])
    _refuses("length must be between", f, q, k, v, [9, -1])
    _refuses("k must be on meta|k must be on", f, q, k.to("meta"), v, [8])


def test_beam_select_op(ext):
    f = ext.beam_select
    x, s, d = torch.zeros(8, 100), torch.zeros(8), torch.zeros(8, dtype=torch.bool)
    _refuses("must be a GPU tensor", f, x, s, d, 4, 3)
    _refuses("must be a GPU tensor", f, x[:1].expand(8, -1), s, d, 4, -1)
    _refuses("logits must be float32", f, x.half(), s, d, 4, 3)
    _refuses("logits must be float32", f, x[0], s, d, 4, 3)
    _refuses("logits must be float32", f, x[:, ::2], s, d, 4, 3)
    _refuses("logits must be float32", f, x[:, :0], s, d, 4, 3)
    _refuses("scores must be", f, x, s.double(), d, 4, 3)
    _refuses("scores must be", f, x, s[:7], d, 4, 3)
    _refuses("scores must be", f, x, torch.zeros(16)[::2], d, 4, 3)
    _refuses("finished must be", f, x, s, d.int(), 4, 3)
    for beams in (0, 17, -1):
        _refuses("beams must be between", f, x, s, d, beams, 3)
    _refuses("multiple of beams", f, x, s, d, 3, 3)
    _refuses("multiple of beams", f, x[:0], s[:0], d[:0], 3, 3)
    for eos in (-2, 100):
        _refuses("eos must be", f, x, s, d, 4, eos)


def test_beam_reorder_op(ext):
    f = ext.beam_reorder
    k, v = (torch.zeros(4, 2, 8, 16, 128, dtype=torch.bfloat16) for _ in range(2))
    i = torch.zeros(4, dtype=torch.int32)
    _refuses("must be a GPU tensor", f, k, v, i, i, i, 2)
    _refuses("k_cache must be", f, k[0], v, i, i, i, 2)
    _refuses("must have shape", f, k, v[:, :1].contiguous(), i, i, i, 2)
    _refuses("must be contiguous", f, k[:, :, :, ::2], v, i, i, i, 2)
    _refuses("must be bfloat16", f, k.float(), v, i, i, i, 2)
    _refuses("must be distinct", f, k, k, i, i, i, 2)
    _refuses("parents must be", f, k, v, i.long(), i, i, 2)
    _refuses("begin must be", f, k, v, i, i[:3], i, 2)
    _refuses("end must be", f, k, v, i, i, torch.zeros(8, dtype=torch.int32)[::2], 2)
    _refuses("multiple of beams", f, k, v, i, i, i, 3)
    _refuses("beams must be between", f, k, v, i, i, i, 0)


def test_prefill_batch_op(ext):
    H, I, V, L, S = 1024, 3072, 512, 1, 32
    bf = torch.bfloat16
    z = lambda *s: torch.zeros(*s, dtype=bf)  # noqa: E731
    layer = [z(H), z(2048, H), z(1024, H), z(1024, H), z(128), z(128), z(H, 2048), z(H), z(I, H), z(I, H), z(H, I)]
    embed = z(V, H)

    def call(tokens=torch.zeros(9, dtype=torch.int32), lengths=(4, 5), table=embed, k=z(2, L, 8, S, 128),
             v=z(2, L, 8, S, 128), max_seq=S):
        ext.prefill_batch(tokens, list(lengths), table, table, z(H), layer, z(S, 128), z(S, 128), k, v, max_seq)

    _refuses("must be a GPU tensor", call)
    wide = [z(6, L, 8, S, 128)[::3] for _ in range(2)]
    with pytest.raises(RuntimeError, match="must be a GPU tensor"):
        call(k=wide[0], v=wide[1])

    def refuses(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            call(**kw)

    refuses("1 to 64 prompts", lengths=())
    refuses("1 to 64 prompts", lengths=(1,) * 65)
    refuses("length must be between", lengths=(9, 0))
    refuses("length must be between", lengths=(33,))
    refuses("tokens must be", lengths=(4, 4))
    refuses("tokens must be", tokens=torch.zeros(9, dtype=torch.int64))
    refuses("multiple of 16", table=z(500, H))
    refuses("k_cache must be", k=z(3, L, 8, S, 128))
    refuses("v_cache must be", v=z(1, L, 8, S, 128))
    refuses("must have shape", k=z(2, L, 8, S + 1, 128))
    refuses("must not overlap", k=z(1, L, 8, S, 128).expand(2, -1, -1, -1, -1))
    refuses("16-byte boundary", k=z(2 * L * 8 * S * 128 + 4)[4:].view(2, L, 8, S, 128))
    refuses("same strides", k=wide[0])
    refuses("cos/sin tables", max_seq=S + 1)


def test_version_tells_a_library_with_these_operators(lib, ext):
    """Libraries up to 0.25 do not have them, or have them with other results."""
    lib.mk_version.restype = ctypes.c_char_p
    version = lib.mk_version().decode()
    assert tuple(int(n) for n in version.split()[1].split(".")) >= (0, 26) and version == ext.version()
    assert all(name in version for name in ("packed attention", "several prompts", "beam selection"))
