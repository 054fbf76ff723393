"""``sample`` on the GPU where sums of very different sizes meet and at the ends of its filters, against its definition in
64 bits (``test_gpu_sample``). Numbers u are single precision, 2^-24 of themselves apart, and running sums are good to
2^-36 of themselves, so that nearly no u is too near a border to tell; ``apart`` leaves these few out."""
import math

import pytest
import torch

from test_gpu_sample import DEV, INF, check

pytestmark = pytest.mark.gpu


def poisoned(kernel, *args):
    """check, with -7 and NaN where the outputs will lie: a token that is not written shows."""
    n = args[0].shape[0]
    for _ in range(2):
        torch.full((n,), -7, dtype=torch.int32, device=DEV)
        torch.full((n,), math.nan, device=DEV)
    return check(kernel, *args)


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
