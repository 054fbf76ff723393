"""Packed-sequence attention (``attention_packed``) on the GPU against the formula in 64 bits.

Tolerances, derived. bf16 queries: the output's own rounding is at most 2^-8 of it, and each weight's
rounding to bf16 at most 2^-8 of the weight, which moves the output by at most 2^-8 times the weighted mean
of |v| -- bounded here by the largest |v| seen. fp32 queries: three bf16 parts hold 24 bits, so products
and sums are fp32's: the scores are off by at most 2^-22 times sum |q k| / sqrt(128) (128 terms and their
order, generously), a weight by that much of itself, and the output by twice that times the largest |v|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
D = 128


def reference(q, k, v, lengths):
    """The attention in 64 bits, on the inputs' device."""
    q, k, v = q.double(), k.double(), v.double()
    out, at = torch.zeros_like(q), 0
    g = q.shape[1] // k.shape[1]
    for n in lengths:
        r = slice(at, at + n)
        for h in range(q.shape[1]):
            s = (q[r, h].contiguous() @ k[r, h // g].t().contiguous()) / math.sqrt(D)
            s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=s.device).triu(1), -math.inf)
            out[r, h] = torch.softmax(s, 1) @ v[r, h // g].contiguous()
        at += n
    return out


def bound(q, k, v, dtype):
    vmax = v.float().abs().max().item() if v.numel() else 0.0
    if dtype == torch.bfloat16:
        return 2 * 2.0 ** -8 * vmax
    smax = (q.double().abs().amax((0, 1)) * k.double().abs().amax((0, 1))).sum().item() / math.sqrt(D)
    return (2 * 2.0 ** -22 * smax + 2.0 ** -22) * vmax


def inputs(n, hq, hkv, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = (torch.randn(n, hq, D, generator=gen, device=DEV) * scale).to(dtype)
    k = torch.randn(n, hkv, D, generator=gen, device=DEV).to(torch.bfloat16)
    v = torch.randn(n, hkv, D, generator=gen, device=DEV).to(torch.bfloat16)
    return q, k, v


def check(kernel, q, k, v, lengths):
    print(f"[packed] {q.dtype} heads {q.shape[1]}/{k.shape[1]} lengths {lengths[:12]}", flush=True)
    got = kernel.attention_packed(q, k, v, lengths)
    torch.cuda.synchronize()
    assert got.dtype == q.dtype and got.shape == q.shape
    err = (got.double() - reference(q, k, v, lengths)).abs().max().item() if q.numel() else 0.0
    assert err <= bound(q, k, v, q.dtype), err
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths", [[1], [2], [31], [64], [65], [128], [129], [300], [1000],
                                     [5, 1, 64, 0, 63, 127, 33, 0], [0, 17], [700, 3, 250]], ids=str)
def test_lengths(kernel, lengths, dtype):
    check(kernel, *inputs(sum(lengths), 16, 8, dtype, seed=len(lengths)), lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads", [(1, 1), (8, 8), (5, 1), (12, 4), (16, 2), (33, 1), (200, 1), (6, 2)], ids=str)
def test_head_layouts(kernel, heads, dtype):
    """Query heads per K/V head that divide a tile's rows, that do not, and more than it has rows."""
    lengths = [67, 1, 130]
    check(kernel, *inputs(sum(lengths), *heads, dtype, seed=heads[0]), lengths)
