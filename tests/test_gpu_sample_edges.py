"""``sample`` on the GPU where sums of very different sizes meet and at the ends of its filters, against its definition in
64 bits (``test_gpu_sample``). Numbers u are single precision, 2^-24 of themselves apart, and running sums are good to
2^-36 of themselves, so that nearly no u is too near a border to tell; ``apart`` leaves these few out."""
import ctypes
import math

import pytest
import torch

from megakernel import build as mkbuild
from test_gpu_sample import DEV, INF, check, rows

pytestmark = pytest.mark.gpu


def poisoned(kernel, *args):
    """check, with -7 and NaN where the outputs will lie: a token that is not written shows."""
    n = args[0].shape[0]
    for _ in range(2):
        torch.full((n,), -7, dtype=torch.int32, device=DEV)
        torch.full((n,), math.nan, device=DEV)
    return check(kernel, *args)


def poisoned_call(kernel, *args):
    n = args[0].shape[0]
    torch.full((n,), -7, dtype=torch.int32, device=DEV), torch.full((n,), math.nan, device=DEV)
    return kernel.sample(*args)


def apart(u, x, T=1.0):
    """The numbers of u whose share of the weights' sum is no nearer than 2^-34 of itself to a running sum."""
    w = torch.exp((x.double() - x.max().double()) / T)
    up = w.cumsum(0)
    goal = u.double() * up[-1]
    near = torch.searchsorted(up, goal)
    off = torch.stack([(up[(near + i).clamp(0, len(up) - 1)] - goal).abs() for i in (-1, 0)]).amin(0)
    return u[off > 2.0 ** -34 * goal]


@pytest.mark.parametrize("vocab,low,high", [(9, 0, 8), (9, 0, 1), (8192, 5, 8000), (20000, 3, 7000), (20000, 3, 19999)])
@pytest.mark.parametrize("min_p", [0.0, 1e-13])
def test_a_small_weight_before_a_large_one(kernel, vocab, low, high, min_p):
    """exp(-27.66) and 1, and every u around the first one's share."""
    x = torch.full((vocab,), -INF, device=DEV)
    x[low], x[high] = -27.660999, 0.0
    share = torch.tensor(9.705118653e-13).view(torch.int32)
    u = apart((share + torch.arange(-2000, 2000, dtype=torch.int32)).view(torch.float32).to(DEV), x)
    assert len(u) > 3900
    tokens, _ = poisoned(kernel, x.expand(len(u), -1), u, 1.0, 0, 1.0, min_p)
    assert set(tokens.tolist()) == {low, high}


@pytest.mark.parametrize("vocab", [40, 256, 3000, 50000])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (30, 1.0, 0.0), (0, 0.9999, 0.0), (0, 1.0, 1e-12)])
def test_weights_that_grow_along_the_vocabulary(kernel, vocab, k, p, m):
    """Every running sum is small against the weight behind it: factors of up to 2^20, shares down to 1e-13."""
    gen = torch.Generator().manual_seed(vocab)
    x = torch.full((vocab,), -INF)
    at = torch.randperm(vocab, generator=gen)[:30].sort().values
    x[at] = -29 + torch.linspace(0, 29, 30) + 3 * torch.randn(30, generator=gen).clamp(-1, 1)
    w = torch.exp(x.double()).cumsum(0)[at]
    border = (w / w[-1]).float()  # every border, and u on both sides of it at several distances
    step = torch.tensor([0, 1, 2, 5, 50, 500], dtype=torch.int32)
    u = (border.view(torch.int32)[:, None] + torch.cat([-step, step])).view(torch.float32).flatten()
    u = torch.cat([u[(u > 0) & (u < 1)], torch.exp(-30 * torch.rand(500, generator=gen))])
    x = x.to(DEV)
    u = apart(u.to(DEV), x)
    assert len(u) > 700
    tokens, _ = poisoned(kernel, x.expand(len(u), -1), u, 1.0, k, p, m)
    assert len(set(tokens.tolist())) > 2


def guarded(x, u, T, k, p, m):
    """The C entry on a workspace of just the bytes that it asks for, with a megabyte behind it that has to stay as it is."""
    lib = ctypes.CDLL(mkbuild.LIB)
    lib.mk_sample_workspace_bytes.restype = ctypes.c_size_t
    n, vocab = x.shape
    need = lib.mk_sample_workspace_bytes(n, vocab)
    memory = torch.full((need + (1 << 20),), 0xa5, dtype=torch.uint8, device=DEV)
    tokens, logprobs = torch.full((n,), -7, dtype=torch.int32, device=DEV), torch.full((n,), math.nan, device=DEV)
    ins = [ctypes.c_void_p(t.data_ptr()) for t in (u, rows(T, n), rows(k, n, torch.int32), rows(p, n), rows(m, n))]
    torch.cuda.synchronize()
    assert lib.mk_sample(n, vocab, ctypes.c_void_p(x.data_ptr()), ctypes.c_int64(x.stride(0)), *ins,
                         ctypes.c_void_p(tokens.data_ptr()), ctypes.c_void_p(logprobs.data_ptr()),
                         ctypes.c_void_p(memory.data_ptr()), ctypes.c_size_t(need), None) == 0
    torch.cuda.synchronize()
    assert (memory[need:] == 0xa5).all()
    return tokens, logprobs


@pytest.mark.parametrize("value", [-3.4e38, 3.3e38, -1e16, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("vocab,equal", [(300, 300), (8192, 5000), (20000, 257), (20000, 20000), (151936, 151936)])
def test_equal_logits_so_large_that_bins_have_no_numbers_of_their_own(kernel, vocab, equal, value):
    """Rows masked whole with the type's lowest value, and others whose largest logits, more than are listed, are 2^53 bins and
    more from 0."""
    gen = torch.Generator().manual_seed(vocab + equal)
    x = torch.full((5, vocab), -INF if value < 0 else 0.0)
    x[:, torch.randperm(vocab, generator=gen)[:equal]] = value
    x, u = x.to(DEV), torch.tensor([0.0, 0.3, 0.5, 0.9, 1 - 2.0 ** -24], device=DEV)
    for T, k, p, m in ((1.0, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 0, 1.0, 0.5), (1.3, 3, 0.5, 0.1), (1.0, 6000, 0.8, 1.0),
                       (1.0, 0, 1.0, 0.0), (1e-3, 257, 1.0, 0.0)):
        tokens, logprobs = check(kernel, x, u, T, k, p, m)
        for _ in range(3):
            again, lp = guarded(x, u, T, k, p, m)
            assert torch.equal(again, tokens) and torch.equal(lp.double().cpu(), logprobs)


@pytest.mark.parametrize("crowd", [300, 4000, 5000, 140000])
def test_min_p_alone_in_a_bin_of_many(kernel, crowd):
    """The bin that min_p's border falls into holds more logits than are listed, than are taken together and fewer: no other
    filter looks for a bin before it. The same answers every time."""
    gen = torch.Generator(device=DEV).manual_seed(crowd)
    x = torch.full((8, 151936), -5.0, device=DEV)
    for row in x:
        row[torch.randperm(151936, generator=gen, device=DEV)[:crowd]] = 2.02 + 0.05 * torch.rand(crowd, generator=gen, device=DEV)
    x[:, 77] = 2.07
    u = torch.rand(8, generator=gen, device=DEV)
    for m in (math.exp(2.05 - 2.07), math.exp(2.0201 - 2.07), math.exp(-7.0)):
        tokens, logprobs = check(kernel, x, u, 1.0, 0, 1.0, m)
        args = (x, u, rows(1.0, 8), rows(0, 8, torch.int32), rows(1.0, 8), rows(m, 8))
        for _ in range(20):
            again, lp = kernel.sample(*args)
            assert torch.equal(again, tokens) and torch.equal(lp.double().cpu(), logprobs)


@pytest.mark.parametrize("vocab", [2, 300, 20000, 151936, 1 << 20])
@pytest.mark.parametrize("equal", [2, 8, 5000])
def test_min_p_above_1_leaves_the_likeliest_token(kernel, vocab, equal):
    """No weight is above 1, so that of equal logits the lowest token stays alone; min_p of 1 keeps all of them."""
    gen = torch.Generator().manual_seed(vocab + equal)
    equal = min(equal, vocab)
    at = torch.randperm(vocab, generator=gen)[:equal].sort().values
    for value in (5.0, -3.4e38, 0.0):
        x = torch.full((4, vocab), -INF)
        if value == 5.0 and vocab > 2 * equal:
            x = torch.randn(4, vocab, generator=gen).clamp(max=4.0)
        x[:, at] = value
        x = x.to(DEV)
        u = torch.tensor([0.0, 0.6, 0.9, 1 - 2.0 ** -24], device=DEV)
        for T, k, p in ((1.0, 0, 1.0), (0.5, 3, 1.0), (2.0, 0, 0.9), (1.0, 100000, 0.5)):
            for m in (1.5, 1 + 2.0 ** -23, INF):
                m = torch.full((4,), m, device=DEV)
                tokens, logprobs = kernel.sample(x, u, torch.full_like(u, T), torch.full_like(u, k).int(),
                                                 torch.full_like(u, p), m)
                assert tokens.tolist() == [at[0].item()] * 4 and logprobs.tolist() == [0.0] * 4
        check(kernel, x, u, 1.0, 0, 1.0, 1.0)


@pytest.mark.parametrize("vocab", [300, 8192, 8193, 28373])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (250, 1.0, 0.0), (50, 1.0, 0.0), (8000, 0.9999999, 0.0), (0, 1.0, 1e-44)])
def test_the_smallest_weights(kernel, vocab, k, p, m):
    """u = 0 asks for the first candidate of any weight, which a weight of at least 2^-1000 of the largest is; a row of many
    that are less, whose sum is more, has an answer too."""
    steps = torch.tensor([1.0, 0.7, 3.0, 13.0, 690.0])
    x = (-steps[:, None] * torch.arange(vocab).float().flip(0)).to(DEV)
    near = torch.full((4, vocab), -INF, device=DEV)  # below 2^-1000, next to it and above, most of a chunk of them
    near[:, :vocab - 40] = torch.tensor([-694.0, -693.2, -693.0, -744.0], device=DEV)[:, None]
    near[:, vocab - 1] = 0.0
    x = torch.cat([x, near])
    n = len(x)
    T = rows(1.0, n)
    tokens, logprobs = poisoned_call(kernel, x, rows(0.0, n), T, rows(k, n, torch.int32), rows(p, n), rows(m, n))
    for r in range(n):
        z, order = torch.sort(x[r].double() - x[r].max().double(), descending=True, stable=True)
        kept = z[:k] if k > 0 else z
        if p < 1:
            w = kept.exp().cumsum(0)
            share = torch.tensor(p).double().item()  # top_p is single precision
            kept = kept[:int(torch.nonzero(w >= share * w[-1] * (1 - 2.0 ** -42))[0]) + 1]
        if m > 0:
            kept = kept[kept >= torch.tensor(m).double().log().item()]
        kept = kept[kept >= -1000 * math.log(2)]
        first = order[:len(kept)].min().item()
        assert tokens[r] == first, (r, tokens[r], first)
        want = (x[r, first].double() - x[r].max().double()).item() - kept.exp().sum().log().item()
        assert abs(logprobs[r].item() - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -22, (r, logprobs[r], want)


@pytest.mark.parametrize("vocab", [600, 20000])
@pytest.mark.parametrize("k", [257, 500])
def test_candidates_too_small_to_count(kernel, vocab, k):
    """A top_k's border among weights of exp(-488): their sum is far below every u but 0."""
    x = torch.full((4, vocab), -INF, device=DEV)
    x[:, 5:505] = -4.88 - 0.0001 * torch.arange(500, device=DEV)
    x[:, vocab - 1] = 0.0
    u = torch.tensor([0.0, 1e-38, 1e-30, 2.0 ** -24], device=DEV)
    tokens, _ = check(kernel, x, u, 0.01, k)
    assert tokens.tolist() == [5] + [vocab - 1] * 3
