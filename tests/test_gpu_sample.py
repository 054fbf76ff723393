"""``sample`` on the GPU against its definition in 64 bits: tokens are whole numbers and have to be equal.

The logprobs: the reference's own rounding to fp32 is 2^-24 of them, the operator's the same, and its sums are good to
2^-42; a weight below exp(-31) of the largest is good to 2^-22 of itself (fp32's exponential, 2^-23, and its argument's
rounding), which shows in the logprob as it stands: 2^-22."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
V = 151936
INF, NAN = math.inf, math.nan


def reference(logits, uniforms, temperature, top_k, top_p, min_p):
    """(tokens, logprobs in 64 bits), row by row; rows that fail are -1 and NaN."""
    tokens, logprobs = [], []
    for r in range(logits.shape[0]):
        x = logits[r].double()
        T, k, p, m, u = (t[r].double().item() for t in (temperature, top_k, top_p, min_p, uniforms))
        if x.isnan().any() or (x == INF).any() or not (x > -INF).any() or not 0 <= T < INF or p != p or m != m or u != u:
            tokens.append(-1)
            logprobs.append(NAN)
            continue
        x, order = torch.sort(x, descending=True, stable=True)  # equal ones: the lower token first
        if T == 0:
            tokens.append(order[0].item())
            logprobs.append(0.0)
            continue
        n = int((x > -INF).sum())
        w = torch.exp((x[:n] - x[0]) / T)
        if k > 0:
            w = w[:int(k)]
        if p < 1:
            some = torch.nonzero(w.cumsum(0) >= p * w.sum() * (1 - 1e-14))
            w = w[:int(some[0]) + 1]
        w = w[w >= min(m, 1.0)]
        by, place = order[:len(w)].sort()
        w = w[place]
        up = w.cumsum(0)
        hit = torch.nonzero(up > u * up[-1] * (1 + 1e-14))
        at = int(hit[0]) if len(hit) else int(torch.nonzero(w > 0)[-1])
        tokens.append(by[at].item())
        logprobs.append((w[at].log() - up[-1].log()).item())
    return tokens, torch.tensor(logprobs, dtype=torch.float64)


def rows(values, n, kind=torch.float32):
    v = values if isinstance(values, (list, tuple)) else [values]
    return torch.tensor([v[i % len(v)] for i in range(n)], dtype=kind, device=DEV)


def check(kernel, x, u, T=1.0, k=0, p=1.0, m=0.0):
    n = x.shape[0]
    args = (x, u if torch.is_tensor(u) else rows(u, n), rows(T, n), rows(k, n, torch.int32), rows(p, n), rows(m, n))
    print(f"[sample] {n} x {x.shape[1]} T {T} k {k} p {p} m {m}", flush=True)
    tokens, logprobs = kernel.sample(*args)
    torch.cuda.synchronize()
    assert tokens.dtype == torch.int32 and logprobs.dtype == torch.float32 and tokens.shape == logprobs.shape == (n,)
    want, lp = reference(*args)
    got = tokens.tolist()
    assert got == want, [(i, g, w) for i, (g, w) in enumerate(zip(got, want)) if g != w][:8]
    lp, logprobs = lp, logprobs.double().cpu()
    assert torch.equal(lp.isnan(), logprobs.isnan())
    off = (logprobs - lp).abs()[~lp.isnan()]
    bound = (2.0 ** -24 * lp.abs() + 2.0 ** -22 * (lp < -25) + 2.0 ** -40)[~lp.isnan()]
    assert (off <= bound).all(), (off - bound).max()
    return tokens, logprobs


def logits(n, vocab, seed=0, peaks=24, scale=2.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, vocab, generator=gen, device=DEV) * scale
    if peaks:
        at = torch.randint(0, vocab, (n, peaks), generator=gen, device=DEV)
        x.scatter_add_(1, at, 6 + 3 * torch.randn(n, peaks, generator=gen, device=DEV))
    return x, torch.rand(n, generator=gen, device=DEV)


@pytest.mark.parametrize("vocab", [1, 2, 3, 100, 255, 8191, 8192, 8193, 32003, V, 1 << 20])
def test_vocabularies(kernel, vocab):
    x, u = logits(9, vocab, vocab)
    check(kernel, x, u, [1.0, 0.6, 1.4], [0, 5, 50], [1.0, 0.9], [0.0, 0.02, 0.0, 0.3])


@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (1, 1.0, 0.0), (7, 1.0, 0.0), (1000, 1.0, 0.0), (5000, 1.0, 0.0),
                                   (100000, 1.0, 0.0), (V - 1, 1.0, 0.0), (V, 1.0, 0.0), (1 << 30, 1.0, 0.0), (-3, 1.0, 0.0),
                                   (0, 0.5, 0.0), (0, 0.999, 0.0), (0, 0.9999999, 0.0), (0, 0.0, 0.0), (0, -1.0, 0.0),
                                   (0, 1e-30, 0.0), (0, 2.0, 0.0), (0, 1.0, 0.1), (0, 1.0, 1.0), (0, 1.0, 3.0), (0, 1.0, -1.0),
                                   (0, 1.0, 1e-6), (0, 1.0, 1e-30), (50, 0.9, 0.05), (20000, 0.7, 0.0), (20000, 0.99, 1e-4),
                                   (3, 0.99, 0.5), (40, 1.0, 1e-5)])
def test_filters(kernel, k, p, m):
    for peaks, T in ((24, 0.7), (0, 1.0), (24, 1.6), (0, 0.1), (3, 30.0)):
        x, u = logits(6, V, k % 1000, peaks)
        check(kernel, x, u, T, k, p, m)


def test_rows_of_all_kinds_together(kernel):
    x, u = logits(64, V, 7)
    check(kernel, x, u, [0.7, 0.6, 1.0, 0.0, 1.2, 0.9, 1.5, 0.8], [0, 20, 0, 0, 0, 1000, 40, 50],
          [0.9, 0.95, 1.0, 1.0, 1.0, 0.8, 1.0, 1.0], [0.0, 0.0, 0.0, 0.0, 0.05, 0.01, 0.1, 0.0])


def test_many_numbers_on_one_row(kernel):
    """The whole range of the random number on one row of logits, the ends too."""
    x, _ = logits(1, 5000, 3)
    u = torch.cat([torch.linspace(0, 1, 2000), torch.tensor([1 - 2.0 ** -24, 0.0, 1e-45, 1.0, 1.5, -0.5])]).to(DEV)
    for k, p, m in ((0, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.8, 0.0), (0, 1.0, 0.01)):
        tokens, _ = check(kernel, x.expand(len(u), -1), u, 1.3, k, p, m)
        assert len(set(tokens.tolist())) > 10


def test_even_weights(kernel):
    """8 equal logits: the j-th eighth of u gives the j-th, j eighths of top_p keep j, whatever else is far below."""
    at = torch.tensor([3, 99, 8191, 8192, 9000, 20000, 30000, 31999], device=DEV)
    for value, low in ((0.0, -1e4), (-3.4e38, -INF), (5.25, -INF), (3.4e38, 0.0), (-0.0, -200.0), (0.7, -INF)):
        for T in (1.0, 0.7, 1e-3, 1e30):
            if T == 1e30 and low != -INF:
                continue
            x = torch.full((8, 32000), low, device=DEV)
            x[:, at] = value
            tokens, _ = check(kernel, x, [j / 8 for j in range(8)], T)
            assert tokens.tolist()[1:] == at.tolist()[1:]  # u = 0: the first of any weight, exp(-200 / T) too
            tokens, _ = check(kernel, x, 1 - 2.0 ** -24, T, 0, [(j + 1) / 8 for j in range(8)])
            assert tokens.tolist() == at.tolist()
            tokens, _ = check(kernel, x, 1 - 2.0 ** -24, T, [j + 1 for j in range(8)])
            assert tokens.tolist() == at.tolist()


@pytest.mark.parametrize("levels", [1, 2, 5, 40])
def test_many_equal_logits(kernel, levels):
    """Borders among thousands of equal logits: the lower tokens stay."""
    gen = torch.Generator(device=DEV).manual_seed(levels)
    x = torch.randint(0, levels, (6, V), generator=gen, device=DEV).float() * 0.25 - 1
    u = torch.rand(6, generator=gen, device=DEV)
    for k, p, m in ((0, 1.0, 0.0), (10, 1.0, 0.0), (5000, 1.0, 0.0), (70001, 1.0, 0.0), (0, 0.37, 0.0), (0, 0.999, 0.0),
                    (50000, 0.5, 0.0), (0, 1.0, 0.9), (70001, 0.9, 0.5)):
        check(kernel, x, u, [1.0, 0.3, 9.0], k, p, m)


def test_zeros_of_both_signs_are_one_number(kernel):
    x = torch.full((4, 20000), -9.0, device=DEV)
    x[:, 5000:15000] = torch.where(torch.arange(10000, device=DEV) % 2 == 0, -0.0, 0.0)
    check(kernel, x, [0.1, 0.5, 0.9, 0.99], 1.0, [0, 7000, 9000, 20], [1.0, 0.9])
    tokens, _ = kernel.sample(x, rows(0.5, 4), rows(0.0, 4), rows(0, 4, torch.int32), rows(1.0, 4), rows(0.0, 4))
    assert tokens.tolist() == [5000] * 4


def test_a_crowded_bin_is_narrowed(kernel):
    """More logits than are sorted at once within one bin, none of them equal, some in the tail."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.rand(6, V, generator=gen, device=DEV) * 1e-3 + 2.0
    x[3:] -= 1000
    x[3:, 77] = 5.0
    u = torch.rand(6, generator=gen, device=DEV)
    for T in (1.0, 0.01, 25.0):
        for k, p, m in ((9000, 1.0, 0.0), (1, 1.0, 0.0), (0, 0.3, 0.0), (100000, 0.8, 0.0), (0, 1.0, 0.9998), (0, 1.0, 1e-44),
                        (140000, 1.0, 1e-40), (9000, 0.5, 0.99999)):
            check(kernel, x, u, T, k, p, m)


@pytest.mark.parametrize("above", [0, 6000])
def test_min_p_in_a_crowded_bin(kernel, above):
    """A border in a bin of which min_p leaves some logits, too many to be listed, and not many more; with 6,000 spread over the
    bin above, that bin's and its own logits are more than are told apart by their bins alone."""
    gen = torch.Generator(device=DEV).manual_seed(above + 1)
    top = 2.14 if above else 2.07  # bins of x log2(e) 11: 32 up to 2.0797, 33 up to 2.1427
    x = 2.02 + 0.03 * torch.rand(6, V, generator=gen, device=DEV)
    for c in range(3):
        x[:, 40000 * c:40000 * c + 1200] = 2.06 + 0.009 * torch.rand(6, 1200, generator=gen, device=DEV)
    if above:
        x[:, 100000:100000 + above] = 2.09 + 0.049 * torch.rand(6, above, generator=gen, device=DEV)
    x[:, 8191::8192] = top
    x[:, V - 1] = top
    u = torch.tensor([0.0, 0.2, 0.5, 0.7, 0.9, 0.9999], device=DEV)
    for k in (0, 50, 150, 1000, 3000, 3617, 7000, 9000, 9621, 100000):
        for threshold in (2.055, 2.065, 2.0695, 2.08, 2.03):
            if threshold < top:
                check(kernel, x, u, 1.0, k, 1.0, math.exp(threshold - top))


def test_temperatures(kernel):
    x, u = logits(12, 40000, 5)
    check(kernel, x, u, [0.0, 1e-45, 1e-30, 1e-3, 0.05, 0.5, 3.0, 100.0, 1e6, 1e30, 3.4e38, 0.01], [0, 300])
    x = x * 1e36
    check(kernel, x, u, [0.0, 1e-45, 1e30, 1e36, 5e36, 1e38, 3.4e38], [0, 300], [1.0, 1.0, 0.8])


def test_minus_infinity_is_never_drawn(kernel):
    x, u = logits(8, 30000, 2)
    x[:, ::2] = -INF
    x[4:, :29000] = -INF
    check(kernel, x, u, [1.0, 5.0], [0, 20000, 400], [1.0, 1.0, 1.0, 0.9])
    one = torch.full((4, 20000), -INF, device=DEV)
    one[torch.arange(4), torch.tensor([0, 8191, 8192, 19999])] = torch.tensor([1.0, -3e38, 3e38, 0.0], device=DEV)
    tokens, logprobs = check(kernel, one, [0.0, 0.5, 0.999, 1.0], [1.0, 0.0], [0, 3], [0.5, 1.0], [0.5, 0.0])
    assert tokens.tolist() == [0, 8191, 8192, 19999] and (logprobs == 0).all()


def test_rows_that_fail(kernel):
    x, u = logits(16, 20000, 4)
    x[0, 12345], x[1, 19999], x[2] = NAN, INF, -INF
    x[3, 0], x[3, 5] = INF, NAN
    T, k, p, m = rows(1.0, 16), rows(50, 16, torch.int32), rows(0.9, 16), rows(0.01, 16)
    T[4], T[5], T[6], T[7] = -1.0, NAN, INF, -INF
    u[8], p[9], m[10] = NAN, NAN, NAN
    T[11], x[11, 3] = 0.0, NAN
    tokens, logprobs = kernel.sample(x, u, T, k, p, m)
    want, lp = reference(x, u, T, k, p, m)
    assert tokens.tolist() == want and want[:12] == [-1] * 12 and min(want[12:]) >= 0
    assert torch.equal(logprobs.isnan().cpu(), lp.isnan())


def test_strides_and_rows_at_any_element(kernel):
    wide = torch.full((5, 20011), NAN, device=DEV)
    x, u = logits(5, 20000, 9)
    for first in (0, 1, 2, 3, 7):
        view = wide[:, first:first + 20000]
        view.copy_(x)
        tokens, _ = check(kernel, view, u, 0.9, 30, 0.95, 0.01)
        wide.fill_(NAN)


def test_many_rows_at_once(kernel):
    x, u = logits(1500, 1000, 11)
    check(kernel, x, u, [0.7, 1.3], [0, 10, 200], [0.9, 1.0, 0.5, 0.99], [0.0, 0.0, 0.1, 0.0, 0.01])


def test_offsets_past_32_bits(kernel):
    """Rows that start more than 2^31 elements into the logits."""
    n = 3
    stride = (1 << 30) + 4096
    flat = torch.empty(2 * stride + V, device=DEV)
    view = flat.as_strided((n, V), (stride, 1))
    x, u = logits(n, V, 12)
    view.copy_(x)
    check(kernel, view, u, 0.8, 40, 0.9, 0.0)


def test_the_same_answers_on_any_stream_and_at_once(kernel):
    x, u = logits(16, V, 13)
    args = (x, u, rows([0.8, 1.2], 16), rows([0, 50], 16, torch.int32), rows([0.9, 1.0], 16), rows([0.0, 0.01], 16))
    first, lp = kernel.sample(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        streams[i % 2].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i % 2]):
            outs.append(kernel.sample(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(t, first) and torch.equal(p, lp) for t, p in outs)


def test_captured_and_replayed(kernel):
    x, u = logits(7, V, 14)
    T, k, p, m = rows([0.8, 1.2, 0.0], 7), rows([0, 50], 7, torch.int32), rows([0.9, 1.0], 7), rows([0.0, 0.01], 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernel.sample(x, u, T, k, p, m)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, logprobs = kernel.sample(x, u, T, k, p, m)
    for i in range(4):
        new, fresh = logits(7, V, 20 + i)
        x.copy_(new)
        u.copy_(fresh)
        T.copy_(T.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        want, _ = reference(x, u, T, k, p, m)
        assert tokens.tolist() == want
        eager, lp = kernel.sample(x, u, T, k, p, m)
        assert torch.equal(eager, tokens) and torch.equal(lp, logprobs)


def test_the_argmax_is_the_batched_decodes_choice_of_logits(kernel):
    """Temperature 0 is torch's argmax, the lowest token of equal ones."""
    x, u = logits(5, V, 15)
    x[1, 400], x[1, 9000], x[1, 140000] = 50.0, 50.0, 50.0
    tokens, _ = check(kernel, x, u, 0.0, [0, 3], 0.5, 0.5)
    assert tokens.tolist() == x.argmax(1).tolist() and tokens[1] == 400
