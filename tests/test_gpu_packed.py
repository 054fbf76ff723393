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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths", [[2048], [3000, 17], [900] * 5, [1 + 13 * i for i in range(60)],
                                     [3 + i % 61 for i in range(150)], [40] * 300, [301] * 40,
                                     [1900] + [64 + 9 * i for i in range(50)] + [5] * 70,
                                     [450], [800, 3, 64, 65], [1500], [1000, 700], [300] * 5, [600, 599, 601]],
                         ids=lambda v: f"{len(v)}x{v[0]}")
def test_every_split_of_the_work(kernel, lengths, dtype):
    """32 rows to a workgroup (the lengths above), 64 (up to 512 workgroups of those) and four key groups or two,
    128 and two or one, with all blocks in turn and with the first sequences' one after another, and more sequences
    than one launch takes."""
    check(kernel, *inputs(sum(lengths), 16, 8, dtype, seed=7), lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_random_lengths_again_and_again(kernel, dtype):
    """Waves of a workgroup run apart by different amounts; a place in LDS that is written too early shows as a
    wrong row in some of these."""
    gen = torch.Generator().manual_seed(11)
    for _ in range(30):
        lengths = torch.randint(1, 420, (int(torch.randint(1, 6, (1,), generator=gen)),), generator=gen).tolist()
        check(kernel, *inputs(sum(lengths), 16, 8, dtype, seed=sum(lengths)), lengths)


def test_strided_operands(kernel):
    """q, k and v as slices of one projection's rows, in another order, and keys shared by expansion."""
    lengths = [70, 200, 1]
    n = sum(lengths)
    rows = torch.randn(n, 40, D, device=DEV).to(torch.bfloat16)
    check(kernel, rows[:, 24:], rows[:, 8:16], rows[:, :8], lengths)
    heads_first = torch.randn(16, n, D, device=DEV).to(torch.bfloat16).transpose(0, 1)
    check(kernel, heads_first, rows[:, 8:16], rows[:, :8], lengths)
    check(kernel, heads_first.float()[:, ::2], rows[:, 8:12], rows[:, ::10], lengths)
    one = torch.randn(n, 1, D, device=DEV).to(torch.bfloat16).expand(n, 8, D)
    check(kernel, heads_first, one, rows[:, :8], lengths)


def test_key_rows_far_apart(kernel):
    """Rows 2^18 elements apart: offsets inside the operands pass 2^31 bytes."""
    n = 4500
    big = torch.zeros(n * (1 << 18) + 2 * D, dtype=torch.bfloat16, device=DEV)
    k, v = (big.as_strided((n, 1, D), (1 << 18, D, 1), o) for o in (0, D))
    q, kk, vv = inputs(n, 2, 1, torch.bfloat16, seed=3)
    k.copy_(kk)
    v.copy_(vv)
    check(kernel, q, k, v, [n - 100, 100])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_one_sharp_key_and_large_scores(kernel, dtype):
    """Scores in the hundreds: the running maximum grows tile by tile, and all weight ends on one key."""
    lengths = [300, 90]
    q, k, v = inputs(390, 4, 2, dtype, seed=5)
    k *= torch.linspace(0.1, 6, 390, device=DEV).to(torch.bfloat16)[:, None, None]
    check(kernel, q * 4, k, v, lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("step", [0.02, 0.5, -0.02, -0.5], ids=str)
def test_scores_that_rise_or_fall_along_the_keys(kernel, step, dtype):
    """A maximum that grows a little with every tile, or by a lot, from very low scores or from high ones; queries
    of one wave whose maxima move differently."""
    for lengths in ([150], [1500], [500] * 20):
        q, k, v = inputs(sum(lengths), 16, 8, dtype, seed=5, scale=0.1)
        u = torch.zeros(D, device=DEV)
        u[::4] = 1.0
        at = torch.cat([torch.arange(n, device=DEV) for n in lengths]).float()
        k = (k.float() * 0.1 + (step * (at - 300.0)).view(-1, 1, 1) * u).to(torch.bfloat16)
        q = (q.float() + u * (torch.arange(len(at), device=DEV) % 5 - 1.0).view(-1, 1, 1) / 4).to(dtype)
        check(kernel, q, k, v, lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths", [[200], [40, 130, 64], [700, 500], [300] * 5, [700] * 8, [1300, 1250, 900],
                                     [250] * 30], ids=lambda v: f"{len(v)}x{v[0]}")
def test_values_that_a_token_may_not_see_do_not_reach_it(kernel, lengths, dtype):
    """Infinities and NaN in some value rows: tokens before them, and other sequences, are as without them;
    tokens from them on get the infinity or NaN that the formula gives, in those dimensions alone."""
    n = sum(lengths)
    q, k, v = inputs(n, 6, 2, dtype, seed=9)
    want = check(kernel, q, k, v, lengths)
    bad = v.clone()
    starts = [sum(lengths[:i]) for i in range(len(lengths))]
    marks = []  # (sequence, its first marked token, K/V head, dim, value)
    for s, (at, length) in enumerate(zip(starts, lengths)):
        for j, (t, value) in enumerate(((length // 3, math.inf), (length - 1, math.nan), (length // 2, -math.inf))):
            head, dim = j % 2, 5 + 40 * j + s
            bad[at + t, head, dim] = value
            marks.append((s, t, head, dim, value))
    got = kernel.attention_packed(q, k, bad, lengths)
    expect = want.clone()
    for s, t, head, dim, value in marks:
        r = slice(starts[s] + t, starts[s] + lengths[s])
        expect[r, 3 * head:3 * head + 3, dim] = value
    fine = torch.isfinite(expect)
    assert torch.equal(got[fine], want[fine])
    assert torch.equal(torch.isnan(got), torch.isnan(expect))
    assert torch.equal(got[~fine & ~torch.isnan(expect)], expect[~fine & ~torch.isnan(expect)])


def test_a_nan_key_or_query_stays_with_the_rows_that_see_it(kernel):
    lengths = [100, 150]
    q, k, v = inputs(250, 2, 1, torch.bfloat16, seed=10)
    want = kernel.attention_packed(q, k, v, lengths)
    k[170] = math.nan
    q[20, 1] = math.nan
    got = kernel.attention_packed(q, k, v, lengths)
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[170:] = True
    nan[20, 1] = True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])


def test_a_sequence_does_not_depend_on_its_batch(kernel):
    """Rows of a sequence alone, at another place and among others, in launches of the same kind: bit for bit."""
    lengths = [130, 77, 64]
    q, k, v = inputs(sum(lengths), 16, 8, torch.bfloat16, seed=12)
    whole = kernel.attention_packed(q, k, v, lengths)
    at = 0
    for n in lengths:
        r = slice(at, at + n)
        assert torch.equal(kernel.attention_packed(q[r], k[r], v[r], [n]), whole[r])
        at += n


def test_empty_call(kernel):
    q, k, v = inputs(0, 16, 8, torch.bfloat16)
    assert kernel.attention_packed(q, k, v, []).shape == (0, 16, 128)
    assert kernel.attention_packed(q, k, v, [0, 0]).shape == (0, 16, 128)


def test_on_another_stream_and_in_a_graph(kernel):
    lengths = [300, 20, 129]
    q, k, v = inputs(sum(lengths), 16, 8, torch.bfloat16, seed=13)
    want = kernel.attention_packed(q, k, v, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernel.attention_packed(q, k, v, lengths)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = kernel.attention_packed(q, k, v, lengths)
    for seed in (14, 15, 16):
        for old, new in zip((q, k, v), inputs(sum(lengths), 16, 8, torch.bfloat16, seed=seed)):
            old.copy_(new)
        held.zero_()
        eager = kernel.attention_packed(q, k, v, lengths)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, eager)


SPLITS = [[200], [40, 130, 64], [700, 500], [300] * 5, [700] * 8, [1300, 1250, 900], [250] * 30]


def keys_with_infinities(lengths, dtype, seed):
    """Inputs whose dimension 7 is positive in every query; some keys (never a sequence's first) hold -infinity
    there, which leaves them no weight, and one sequence's last holds +infinity: NaN for the row that sees it."""
    n = sum(lengths)
    q, k, v = inputs(n, 6, 2, dtype, seed=seed)
    q[:, :, 7] = q[:, :, 7].abs() + 0.25
    starts = [sum(lengths[:i]) for i in range(len(lengths))]
    for j, (at, length) in enumerate(zip(starts, lengths)):
        for t in (1 + j % 3, length // 3, length // 2, length - 2):
            k[at + t, j % 2, 7] = -math.inf
    k[starts[-1] + lengths[-1] - 1, 1, 7] = math.inf
    return q, k, v


def check_where_finite(got, want, limit):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    err = (got.double() - want)[fine].abs().max().item()
    assert err <= limit, err


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths", SPLITS, ids=lambda v: f"{len(v)}x{v[0]}")
def test_infinite_keys(kernel, lengths, dtype):
    """A score of -infinity has no weight, one of +infinity or NaN (a query's 0 on an infinite key) makes its row
    NaN, and no other row knows of it."""
    q, k, v = keys_with_infinities(lengths, dtype, seed=21)
    q[lengths[0] - 1, 0, 7] = 0.0  # a row that meets infinite keys with a 0
    print(f"[packed] {dtype} infinite keys, lengths {lengths[:12]}", flush=True)
    got = kernel.attention_packed(q, k, v, lengths)
    limit = bound(q, k.masked_fill(torch.isinf(k), 0), v, dtype)
    want = reference(q, k, v, lengths)
    assert torch.isnan(want[lengths[0] - 1, 0]).all() and torch.isnan(want[-1, 3:]).all()
    check_where_finite(got, want, limit)


def test_fp32_queries_up_to_the_largest_number(kernel):
    """fp32 holds numbers above bf16's largest, which a first bf16 part cannot: the formula's scores are ordinary,
    on keys as small as bf16's."""
    lengths = [90, 300]
    q, k, v = inputs(390, 4, 2, torch.float32, seed=22)
    q[::3, :, 9] = 3.4e38
    q[1::3, 1, 9] = -3.402e38
    k[:, :, 9] = (k[:, :, 9].sign() * 2.0 ** -126).to(torch.bfloat16)
    got = kernel.attention_packed(q, k, v, lengths)
    assert (got.double() - reference(q, k, v, lengths)).abs().max().item() <= bound(q, k, v, torch.float32)


def fragments(rows, cols, hi, lo):
    """A bf16 hi/lo pair of matrices out of 16 x 32 blocks of 1 KB: lane m % 16 + 16 (k % 32 / 8) of a block holds 8
    consecutive columns."""
    m, c = torch.arange(rows, device=DEV)[:, None], torch.arange(cols, device=DEV)[None]
    at = (((m // 16) * (cols // 32) + c // 32) * 64 + (c // 8 % 4) * 16 + m % 16) * 8 + c % 8
    return hi[at].double() + lo[at].double()


@pytest.mark.parametrize("lengths", SPLITS, ids=lambda v: f"{len(v)}x{v[0]}")
def test_infinite_keys_for_the_prefills_queries(lengths):
    """The form that prefill_batch runs (bf16 hi/lo queries over the caches, by the library's internal entry). Weights
    and output are held as two bf16 numbers, off by 2^-16 of the largest |v| together; the scores' fp32 sums of 16
    products are off by at most 2^-20 of sum |q k| / sqrt(128), the output by twice that times the largest |v|."""
    import ctypes
    from megakernel import build as mkbuild

    class Prefill(ctypes.Structure):
        _fields_ = [(n, ctypes.c_void_p) for n in ("qh", "ql", "k_cache", "v_cache", "oh", "ol")] + [
            ("frag", ctypes.c_int), ("layer", ctypes.c_int), ("max_seq", ctypes.c_int), ("seq_stride", ctypes.c_int64),
            ("lengths", ctypes.c_void_p), ("num_seqs", ctypes.c_int)]

    n, hq, hkv, T = sum(lengths), 16, 8, max(lengths)
    q, k, v = inputs(n, hq, hkv, torch.float32, seed=23)
    q[:, :, 7] = q[:, :, 7].abs() + 0.25
    qh = q.to(torch.bfloat16)
    ql = (q - qh.float()).to(torch.bfloat16)
    caches = torch.full((2, len(lengths), hkv, T, D), math.nan, dtype=torch.bfloat16, device=DEV)
    at = 0
    for i, length in enumerate(lengths):
        for t in (1 + i % 3, length // 3, length // 2, length - 2):
            k[at + t, i % 8, 7] = -math.inf
        for dst, src in zip(caches, (k, v)):
            dst[i, :, :length] = src[at:at + length].transpose(0, 1)
        at += length
    oh, ol = (torch.zeros((n + 15) // 16 * 16 * hq * D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    host = (ctypes.c_int32 * len(lengths))(*lengths)
    call = Prefill(qh.data_ptr(), ql.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr(), oh.data_ptr(), ol.data_ptr(),
                   1, 0, T, hkv * T * D, ctypes.addressof(host), len(lengths))
    lib = ctypes.CDLL(mkbuild.LIB)
    run = lib["_Z21mkp_attention_prefillRK15MkPackedPrefillP12ihipStream_t"]
    run.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    print(f"[packed] hi/lo infinite keys, lengths {lengths[:12]}", flush=True)
    assert run(ctypes.addressof(call), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    want = reference(qh.float() + ql.float(), k, v, lengths)
    finite = k.masked_fill(torch.isinf(k), 0)
    smax = (q.double().abs().amax((0, 1)) * finite.double().abs().amax((0, 1))).sum().item() / math.sqrt(D)
    limit = (2 * 2.0 ** -20 * smax + 2 * 2.0 ** -16) * v.float().abs().max().item()
    check_where_finite(fragments(n, hq * D, oh, ol).view(n, hq, D), want, limit)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths", SPLITS, ids=lambda v: f"{len(v)}x{v[0]}")
def test_very_low_scores_behind_keys_without_weight(kernel, lengths, dtype):
    """Every sequence begins with keys of score -infinity, up to more than a tile of them, and goes on with scores
    around -150: the first finite maximum is far below 0. (fp32 queries: one term makes most of a score, and each of
    the up to 24 products added to it rounds at its size: 6 times the bound's 2^-22.)"""
    n = sum(lengths)
    q, k, v = inputs(n, 6, 2, dtype, seed=24, scale=0.1)
    q[:, :, 7], q[:, :, 8] = 1.0, 40.0
    k[:, :, 8] = -42.0
    at = 0
    for j, length in enumerate(lengths):
        k[at:at + min(1 + 47 * (j % 4), length - 1) if j else at + 130, :, 7] = -math.inf
        at += length
    print(f"[packed] {dtype} low scores, lengths {lengths[:12]}", flush=True)
    got = kernel.attention_packed(q, k, v, lengths)
    limit = (6 if dtype == torch.float32 else 1) * bound(q, k.masked_fill(torch.isinf(k), 0), v, dtype)
    check_where_finite(got, reference(q, k, v, lengths), limit)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths", SPLITS, ids=lambda v: f"{len(v)}x{v[0]}")
@pytest.mark.parametrize("rise", [600.0, 0.5], ids=["sharp key", "rising scores"])
def test_an_infinite_value_with_a_weight_too_small_to_hold(kernel, lengths, dtype, rise):
    """A weight is positive however small: an infinite value that a token sees reaches it, also where fp32 holds the
    weight as 0 (scores behind it that are hundreds higher), wherever its key lies in the tiles. (fp32 queries: 6 times the bound's
    2^-22, as one term makes most of a score and up to 24 products are added to it.)"""
    n = sum(lengths)
    q, k, v = inputs(n, 6, 2, dtype, seed=25)
    starts = [sum(lengths[:i]) for i in range(len(lengths))]
    q[:, :, 8] = 8.0
    k[:, :, 8] = 0.0
    marks = []
    for s, (at, length) in enumerate(zip(starts, lengths)):
        if rise > 100:
            k[at + length // 2:at + length, :, 8] = rise
        else:
            k[at:at + length, :, 8] = (rise * torch.arange(length, device=DEV)).to(torch.bfloat16)[:, None]
        for j, (t, value) in enumerate(((0, math.inf), (length // 4, -math.inf), (length // 3, math.nan))):
            v[at + t, j % 2, 11 + 40 * j] = value
            marks.append((slice(at + t, at + length), j % 2, 11 + 40 * j, value))
    print(f"[packed] {dtype} infinite values of no weight, lengths {lengths[:12]}", flush=True)
    got = kernel.attention_packed(q, k, v, lengths)
    finite = v.masked_fill(~torch.isfinite(v), 0)
    want = reference(q, k, finite, lengths)
    for r, head, dim, value in marks:
        want[r, 3 * head:3 * head + 3, dim] = value
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), want[inf])
    limit = (6 if dtype == torch.float32 else 1) * bound(q, k, finite, dtype)
    check_where_finite(got.masked_fill(inf, 0), want.masked_fill(inf, 0), limit)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_a_row_whose_keys_all_have_no_weight(kernel, dtype):
    """Nothing but scores of -infinity: 0 / 0, in the dimensions of an infinite value too."""
    q, k, v = inputs(300, 6, 2, dtype, seed=28)
    q[:, :, 7] = 1.0
    k[:70, :, 7] = -math.inf
    v[3, :, 20] = math.inf
    got = kernel.attention_packed(q, k, v, [300])
    assert torch.isnan(got[:70]).all()
    assert torch.isfinite(got[70:, :, :20]).all() and torch.isfinite(got[70:, :, 21:]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_a_sequence_among_others_differs_by_summation_order_alone(kernel, dtype):
    """A prompt alone and in batches that other instances of the kernel take: each within the bound of the formula,
    no other sequence's values in it (theirs are infinite here)."""
    n = 130
    q, k, v = inputs(n, 16, 8, dtype, seed=26)
    want, limit = reference(q, k, v, [n]), bound(q, k, v, dtype)
    for others in ([], [20], [600, 700], [900] * 6, [2500], [300] * 40):
        m = sum(others)
        q2, k2, v2 = inputs(m, 16, 8, dtype, seed=27)
        v2[:] = math.inf
        got = kernel.attention_packed(torch.cat([q2, q]), torch.cat([k2, k]), torch.cat([v2, v]), others + [n])
        err = (got[m:].double() - want).abs().max().item()
        assert err <= limit, (others, err)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lengths", SPLITS + [[2500], [900] * 24], ids=lambda v: f"{len(v)}x{v[0]}")
def test_the_same_call_gives_the_same_bits(kernel, lengths, dtype):
    q, k, v = inputs(sum(lengths), 16, 8, dtype, seed=29)
    want = kernel.attention_packed(q, k, v, lengths)
    for _ in range(5):
        assert torch.equal(kernel.attention_packed(q, k, v, lengths), want)
