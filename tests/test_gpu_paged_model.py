"""The operators of a server's step together, as a program of its own layers uses them: a small decoder whose prompts go
through ``attention_packed`` and into an 8-bit or bf16 paged cache (``cache_write``), whose tokens attend over the pages
(``attention_paged``) and are drawn by ``sample``; half-way one conversation's rows are read back (``cache_read``) and
moved to other pages. Against the same decoder in 64 bits on the values that the cache holds.

Tolerance: each of the two layers adds an attention of fp32 accuracy (2^-18 of the largest value, generously) to a
stream of magnitude about 1; projections in fp32 over 256 inputs are off by 2^-24 times the root of their number, and
the second layer's cache may round a number the other way where the first layer's difference carries it over a border: a
step of the format, 2^-3 (2^-7) of one of 128 numbers of one key, whose weight in a softmax over 20 and more keys is
small. Both decoders are therefore fed the rows that the cache holds, and logits agree to 2^-14 of their largest."""
import math

import pytest
import torch

from paged_pool import D, Pool
from test_gpu_sample import reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HQ, HKV, H, V, LAYERS, STEPS = 4, 2, 256, 1000, 2, 6


def norm(x):
    return x / x.square().mean(-1, keepdim=True).add(1e-6).sqrt()


class Decoder:
    def __init__(self, seed):
        gen = torch.Generator(device=DEV).manual_seed(seed)

        def w(*s):
            return torch.randn(*s, generator=gen, device=DEV) / math.sqrt(s[-1])

        self.embed = w(V, H) * 4
        self.layers = [(w((HQ + 2 * HKV) * D, H), w(H, HQ * D)) for _ in range(LAYERS)]

    def project(self, layer, x):
        rows = (norm(x) @ self.layers[layer][0].to(x.dtype).t()).view(len(x), HQ + 2 * HKV, D)
        return rows[:, :HQ], rows[:, HQ:HQ + HKV], rows[:, HQ + HKV:]

    def add(self, layer, x, o):
        return x + o.reshape(len(x), HQ * D) @ self.layers[layer][1].to(x.dtype).t()

    def logits(self, x):
        return norm(x) @ self.embed.to(x.dtype).t()


def attend(q, k, v, causal):
    """[rows, heads, 128] over [keys, K/V heads, 128] in 64 bits; causal: row t sees the keys up to t."""
    out = torch.empty_like(q)
    for h in range(HQ):
        s = q[:, h] @ k[:, h // (HQ // HKV)].t().contiguous() / math.sqrt(D)
        if causal:
            s.masked_fill_(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf)
        out[:, h] = torch.softmax(s, 1) @ v[:, h // (HQ // HKV)].contiguous()
    return out


@pytest.mark.parametrize("e4m3", [False, True], ids=["bf16-pages", "e4m3-pages"])
@pytest.mark.parametrize("page_size", [16, 64])
def test_a_server_of_its_own_layers(kernel, e4m3, page_size):
    model = Decoder(0)
    lengths = [23, 5, 70]
    n, rows = len(lengths), sum(lengths)
    gen = torch.Generator(device=DEV).manual_seed(1)
    tokens = torch.randint(0, V, (rows,), generator=gen, device=DEV)
    pools = [Pool(n, 128 // page_size, page_size, HKV, e4m3, DEV, "joint", seed=layer) for layer in range(LAYERS)]
    zeros = torch.zeros(n, dtype=torch.int32, device=DEV)
    starts = [sum(lengths[:i]) for i in range(n)]

    def close(got, want):
        return (got.double() - want).abs().max() <= 2.0 ** -14 * want.abs().max()

    # the prompts: attention over the rows themselves, in bf16
    x, ref = model.embed[tokens], model.embed[tokens].double()
    for layer, pool in enumerate(pools):
        q, k, v = model.project(layer, x)
        kernel.cache_write(k, v, *pool.args(), zeros, lengths, *pool.scales())
        k, v = k.bfloat16(), v.bfloat16()
        x = model.add(layer, x, kernel.attention_packed(q, k, v, lengths))
        rq, _, _ = model.project(layer, ref)
        ro = torch.cat([attend(rq[s:s + c], k[s:s + c].double(), v[s:s + c].double(), True) for s, c in zip(starts, lengths)])
        ref = model.add(layer, ref, ro)
    logits, want = model.logits(x), model.logits(ref)
    last = torch.tensor([s + c - 1 for s, c in zip(starts, lengths)], device=DEV)
    assert close(logits, want)
    logits, at = logits[last], torch.tensor(lengths, dtype=torch.int32, device=DEV)
    T, K, P, M = (torch.tensor(c, dtype=t, device=DEV) for c, t in (
        ([0.8, 0.0, 1.2], torch.float32), ([0, 0, 40], torch.int32), ([0.9, 1.0, 1.0], torch.float32),
        ([0.0, 0.0, 0.05], torch.float32)))
    for step in range(STEPS):
        numbers = torch.rand(n, generator=gen, device=DEV)
        tokens, logprobs = kernel.sample(logits, numbers, T, K, P, M)
        assert tokens.tolist() == reference(logits, numbers, T, K, P, M)[0] and (logprobs <= 0).all()
        x, ref = model.embed[tokens.long()], model.embed[tokens.long()].double()
        for layer, pool in enumerate(pools):
            q, k, v = model.project(layer, x)
            kernel.cache_write(k, v, *pool.args(), at, [1] * n, *pool.scales())
            x = model.add(layer, x, kernel.attention_paged(q, *pool.args(), at + 1, *pool.scales()))
            rq, _, _ = model.project(layer, ref)
            ro = torch.cat([attend(rq[s:s + 1], pool.rows("k", s, 0, c + 1), pool.rows("v", s, 0, c + 1), False)
                            for s, c in enumerate(at.tolist())])
            ref = model.add(layer, ref, ro)
        logits = model.logits(x)
        assert close(logits, model.logits(ref))
        at = at + 1
        if step == 2:  # the first conversation moves: its rows are read, and written where the spare pages are
            for pool in pools:
                count = at.tolist()[:1] + [0] * (n - 1)
                k, v = kernel.cache_read(*pool.args(), zeros, count, *pool.scales())
                free = sorted(set(range(pool.n)) - set(pool.tables.flatten().tolist()))
                table = pool.tables.clone()
                moved = -(-count[0] // page_size)
                assert len(free) >= moved
                table[0, :moved] = torch.tensor(free[:moved], dtype=torch.int32, device=DEV)
                pool.tables = table
                kernel.cache_write(k, v, *pool.args(), zeros, count, *pool.scales())
                again, _ = kernel.cache_read(*pool.args(), zeros, count, *pool.scales())
                assert torch.equal(again, k)
