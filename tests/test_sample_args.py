"""Host-side tests of ``sample``: bad arguments are rejected before anything is launched, by the C entry point with
hipErrorInvalidValue and by the PyTorch operator with a message. No GPU is used; arguments that are right in all else
end at "must be a GPU tensor"."""
import ctypes

import pytest
import torch

from megakernel import build as mkbuild

INVALID = 1  # hipErrorInvalidValue
vp, i32, i64, size = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
P = 4096  # an aligned address that nothing reads


def test_sample_c():
    lib = ctypes.CDLL(mkbuild.LIB)
    lib.mk_sample_workspace_bytes.restype = size
    lib.mk_sample_workspace_bytes.argtypes = [i32, i32]
    lib.mk_sample.argtypes = [i32, i32, vp, i64] + [vp] * 8 + [size, vp]
    need = lib.mk_sample_workspace_bytes
    assert need(0, 100) == need(65536, 100) == need(4, 0) == need(4, (1 << 20) + 1) == need(-1, 100) == 0
    assert 0 < need(1, 1) <= need(1, 151936) < need(64, 151936) < need(64, 1 << 20)

    def call(rows=4, vocab=1000, logits=P, stride=1000, ins=(P,) * 5, tokens=P, logprobs=P, ws=P, nbytes=1 << 40):
        return lib.mk_sample(rows, vocab, logits, stride, *ins, tokens, logprobs, ws, nbytes, None)

    assert call(rows=0) == call(rows=65536) == call(vocab=0) == call(vocab=(1 << 20) + 1) == call(stride=-1) == INVALID
    assert call(logits=None) == call(tokens=None) == call(ws=None) == INVALID
    for i in range(5):
        assert call(ins=tuple(None if j == i else P for j in range(5))) == INVALID
    assert call(nbytes=need(4, 1000) - 1) == call(ws=P + 128) == INVALID


def test_sample_op():
    import megakernel
    f = megakernel.load().sample
    x, one, k = torch.zeros(3, 100), torch.ones(3), torch.zeros(3, dtype=torch.int32)

    def refuses(match, logits=x, uniforms=one, temperature=one, top_k=k, top_p=one, min_p=one):
        with pytest.raises(RuntimeError, match=match):
            f(logits, uniforms, temperature, top_k, top_p, min_p)

    refuses("must be a GPU tensor")
    refuses("must be a GPU tensor", logits=x[:1].expand(3, -1))
    refuses("must be a GPU tensor", logits=torch.zeros(3, 200)[:, 50:150])
    for bad in (x.bfloat16(), x[0], x[:, ::2], x[:, :0], torch.empty(1, 1).expand(3, (1 << 20) + 1)):
        refuses("logits must be float32", logits=bad)
    refuses("1 to 65535 rows", logits=x[:0], uniforms=one[:0], temperature=one[:0], top_k=k[:0], top_p=one[:0], min_p=one[:0])
    refuses("1 to 65535 rows", logits=x[:1].expand(65536, -1))
    for name in ("uniforms", "temperature", "top_p", "min_p"):
        for bad in (one.double(), one[:2], torch.ones(6)[::2], one[:, None], one.to("meta")):
            refuses(f"{name} must be", **{name: bad})
    for bad in (k.long(), k[:2], one):
        refuses("top_k must be", top_k=bad)
