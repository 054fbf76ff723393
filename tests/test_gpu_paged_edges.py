"""``attention_paged`` and the paged cache on the GPU where shares of the work, scales and rows end in unusual places, against
the definitions in 64 bits (``paged_pool``; the tolerances are derived in ``test_gpu_paged``)."""
import math

import pytest
import torch

from paged_pool import E8, D, Pool, attention
from test_gpu_paged import DEV, KINDS, PAGES, check, ints, queries, write_and_check

pytestmark = pytest.mark.gpu


@KINDS
@PAGES
@pytest.mark.parametrize("lengths", [[300, 0, 1, 513, 64], [1024], [31] * 9, [1] * 700], ids=["ragged", "one", "tiles", "many"])
def test_attention_where_a_wave_has_one_tile(kernel, dtype, e4m3, lengths):
    """Each wave of a workgroup ends with a piece of its own, as early as one can. What calls left in memory is NaN, so that a
    piece that is not joined, or one that was not made, shows."""
    pool = Pool(len(lengths), 64, 16, 8, e4m3, DEV, seed=len(lengths))
    q, n = queries(len(lengths), 16, dtype), ints(lengths)
    first = check(kernel, pool, q, lengths)
    for _ in range(10):
        for size in (33024 + 2 * 512 * 2 * 130 * 4, q.numel() * q.element_size()):  # the workspace's bytes and the output's
            torch.full((size // 4,), float("nan"), device=DEV)
        assert torch.equal(kernel.attention_paged(q, *pool.args(), n, *pool.scales()), first)


def milliseconds(call):
    """The least of eight measured runs of ten calls."""
    best = float("inf")
    for _ in range(8):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(10):
            call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) / 10)
    return best


@pytest.mark.parametrize("capacity", [512, 1024])
def test_attention_takes_no_longer_for_what_is_behind_the_last_key(kernel, capacity):
    """fp32 queries, 8-bit pages: a scale of NaN behind the last key makes NaN of scores that nobody asks for. None of them is
    made again (when they were, calls like these took about twice as long)."""
    gen = torch.Generator().manual_seed(capacity)
    lengths = [8 * int(n) + 1 for n in torch.randint(8, capacity // 8 - 1, (256,), generator=gen)]
    pool = Pool(256, capacity // 64, 64, 8, True, DEV)
    q, n = queries(256, 16, torch.float32), ints(lengths)
    call = lambda: kernel.attention_paged(q, *pool.args(), n, *pool.scales())  # noqa: E731
    expected, before = call(), milliseconds(call)
    for s, length in enumerate(lengths):
        for scales in (pool.ks, pool.vs):
            scales.view(torch.uint8)[pool.tables[s, length // 64].item(), :, length % 64:] = 255
    assert torch.equal(call(), expected)
    after = milliseconds(call)
    assert after < 1.3 * before, (before, after)


@KINDS
@pytest.mark.parametrize("hq,hkv,seqs", [(16, 8, 300), (40, 2, 110), (5, 1, 900), (16, 8, 4096)])
def test_attention_of_few_sequences_among_free_places(kernel, dtype, hq, hkv, seqs):
    """More pairs of sequence and head than the join takes one by one, most of them without keys, some lengths out of range."""
    pool = Pool(8, 130, 16, hkv, False, DEV, seed=seqs)
    used = {0: 2000, 1: 1, 2: 1500, seqs // 2: 700, seqs - 2: 2080, seqs - 1: 33}
    lengths = [0] * seqs
    table = pool.tables[:1].repeat(seqs, 1)
    for i, (s, n) in enumerate(used.items()):
        lengths[s] = n
        table[s] = pool.tables[i]
    pool.tables = table
    q = queries(seqs, hq, dtype)
    got = check(kernel, pool, q, lengths)
    bad = list(lengths)
    bad[3], bad[seqs // 3], bad[seqs - 3] = -1, 2081, 2 ** 31 - 1
    again = kernel.attention_paged(q, *pool.args(), ints(bad))
    out = torch.tensor([n != m for n, m in zip(lengths, bad)], device=DEV)
    assert again[out].isnan().all() and torch.equal(again[~out], got[~out])


def test_attention_of_a_long_sequence_among_many_places(kernel):
    """The heads of a sequence of many keys are joined side by side, however many places there are besides (one after the other,
    512 places took three times as long as 64)."""
    pool = Pool(1, 256, 16, 8, False, DEV)
    took = []
    for seqs in (64, 512):
        q, n = queries(seqs, 16, torch.float32), ints([4000] + [0] * (seqs - 1))
        tables = pool.tables.repeat(seqs, 1)
        took.append(milliseconds(lambda: kernel.attention_paged(q, pool.k, pool.v, tables, n)))
    assert took[1] < 1.8 * took[0], took


def test_scales_that_cache_write_does_not_make(kernel):
    """Bytes 0 .. 9 and 255 of the scales: powers of two down to 2^-127, and rows of NaN whatever their values are."""
    numbers = torch.arange(256, dtype=torch.uint8, device=DEV).view(2, D)
    units = torch.tensor([*range(12), 255], dtype=torch.uint8, device=DEV)
    pool = Pool(len(units), 2, 32, 2, True, DEV, fill=False)
    at = pool.tables[:, 0].long()
    for pages, scales in ((pool.k, pool.ks), (pool.v, pool.vs)):
        pages.view(torch.uint8)[at, :, 3] = numbers
        scales.view(torch.uint8)[at, :, 3] = units[:, None]
    k, v = kernel.cache_read(*pool.args(), ints([3] * len(units)), [1] * len(units), *pool.scales())
    expected = numbers.view(torch.float8_e4m3fn).double() * torch.exp2(units.double() - 127)[:, None, None]
    expected[-1] = math.nan
    for x in (k, v):
        assert torch.equal(x.isnan(), expected.isnan())
        # bf16's rounding, and its numbers below 2^-126, 2^-133 apart
        assert ((x.double() - expected).abs() <= 2.0 ** -134).logical_or(expected.isnan()).all()


@KINDS
@pytest.mark.parametrize("entries", [8, 64])
@pytest.mark.parametrize("page_size", [4, 8, 64])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_of_rows_whose_scale_is_nan(kernel, dtype, entries, page_size, sign):
    """A scale of 255 is a row of NaN, however its finite values and the query would add up."""
    pool = Pool(3, entries * 64 // page_size, page_size, 2, True, DEV)
    lengths = [300, 45, 64]
    q = queries(3, 8, dtype).abs() * sign
    plain = check(kernel, pool, q, lengths)
    for which in "kv":
        pages, scales = (pool.k, pool.ks) if which == "k" else (pool.v, pool.vs)
        for s, p, head in ((0, 123, 1), (1, 44, 0), (2, 0, 1)):
            page, row = pool.tables[s, p // page_size].item(), p % page_size
            kept = pages.view(torch.uint8)[page, head, row].clone(), scales.view(torch.uint8)[page, head, row].item()
            pages.view(torch.uint8)[page, head, row] = 0x38  # 1
            for byte in (255, 127):
                scales.view(torch.uint8)[page, head, row] = byte
                got = kernel.attention_paged(q, *pool.args(), ints(lengths), *pool.scales())
                hit = torch.zeros_like(got, dtype=torch.bool)
                hit[s, 4 * head:4 * head + 4] = True
                assert torch.equal(got[~hit], plain[~hit])
                assert got[hit].isnan().all() if byte == 255 else got[hit].isfinite().all()
            pages.view(torch.uint8)[page, head, row], scales.view(torch.uint8)[page, head, row] = kept


def loose_scales(pool, first, between):
    """pool's scales as slices of wider ones: `first` bytes before each head's, `between` bytes in all besides them."""
    made = []
    for scales in (pool.ks, pool.vs):
        n, h, p = scales.shape
        wide = torch.full((n, h, p + between), 255, dtype=torch.uint8, device=DEV)
        wide[..., first:first + p] = scales.view(torch.uint8)
        made.append(wide[..., first:first + p].view(E8))
    pool.ks, pool.vs = made


@KINDS
@pytest.mark.parametrize("page_size", [8, 16, 64])
@pytest.mark.parametrize("first,between", [(0, 1), (1, 3), (4, 8), (0, 8), (3, 20)])
def test_scales_at_any_byte(kernel, dtype, page_size, first, between):
    """Scales whose 8 bytes of 8 rows are not one aligned number, and (0, 8) ones that are, with others between the heads."""
    lengths = [70, 0, 1, 500, 33]
    for capacity in (512, 1024):
        pool = Pool(len(lengths), capacity // page_size, page_size, 8, True, DEV, seed=page_size)
        q = queries(len(lengths), 16, dtype)
        plain = check(kernel, pool, q, lengths)
        loose_scales(pool, first, between)
        got = check(kernel, pool, q, lengths)
        assert torch.equal(got, plain)
    rows = torch.randn(60, 8, D, generator=torch.Generator(device=DEV).manual_seed(first), device=DEV).to(dtype)
    at = [(0, 5 + i) for i in range(40)] + [(3, 100 + i) for i in range(20)]
    write_and_check(kernel, pool, rows, rows.flip(0), ints([5, 0, 0, 100, 0]), [40, 0, 0, 20, 0], at)
    k, _ = kernel.cache_read(*pool.args(), ints([5, 0, 0, 100, 0]), [40, 0, 0, 20, 0], *pool.scales())
    assert torch.equal(k.double(), torch.cat([pool.rows("k", 0, 5, 40), pool.rows("k", 3, 100, 20)]))


@KINDS
@PAGES
@pytest.mark.parametrize("heads", [9, 16, 17, 40])
def test_cache_of_more_than_8_heads(kernel, dtype, e4m3, heads):
    """More rows to a position than a wave has in flight."""
    pool = Pool(3, 4, 16, heads, e4m3, DEV, "rows", seed=heads)
    lengths, begin = [20, 0, 7], [3, 0, 60]
    rows = torch.randn(27, 2 * heads, D, generator=torch.Generator(device=DEV).manual_seed(heads), device=DEV)
    rows = (rows * torch.exp2(torch.arange(2 * heads, device=DEV) % 13 - 6)[:, None]).to(dtype)
    at = [(s, b + i) if b + i < 64 else None for s, (b, n) in enumerate(zip(begin, lengths)) for i in range(n)]
    write_and_check(kernel, pool, rows[:, :heads], rows[:, heads:], ints(begin), lengths, at)
    k, v = kernel.cache_read(*pool.args(), ints([0, 0, 60]), [23, 0, 4], *pool.scales())
    for got, which in ((k, "k"), (v, "v")):
        assert torch.equal(got.double(), torch.cat([pool.rows(which, 0, 0, 23), pool.rows(which, 2, 60, 4)]))


@KINDS
@PAGES
@pytest.mark.parametrize("capacity", [512, 1024])
def test_attention_whose_last_key_is_not_finite(kernel, dtype, e4m3, capacity):
    """The last key of a tile that ends there stands in for those behind it, which have no weight: an infinite or NaN value of
    its reaches its own elements alone, a key of NaN its head's, a key of -infinity nothing."""
    pool = Pool(3, capacity // 16, 16, 2, e4m3, DEV)
    lengths = [201, 33, 1]
    q = queries(3, 8, dtype).abs()
    plain = check(kernel, pool, q, lengths)
    bads = [(0x7f, math.nan)] if e4m3 else [(None, math.nan), (None, math.inf), (None, -math.inf)]
    for s, n in enumerate(lengths):
        page, row = pool.tables[s, (n - 1) // 16].item(), (n - 1) % 16
        for byte, bad in bads:
            for pages in (pool.v, pool.k):
                place = pages.view(torch.uint8)[page, 1, row, 9:10] if e4m3 else pages[page, 1, row, 9:10]
                kept = place.clone()
                place.fill_(byte if e4m3 else bad)
                got = kernel.attention_paged(q, *pool.args(), ints(lengths), *pool.scales())
                hit = torch.zeros_like(got, dtype=torch.bool)
                if pages is pool.v:
                    hit[s, 4:, 9] = True
                else:
                    hit[s, 4:] = True
                assert torch.equal(got[~hit], plain[~hit])
                if pages is pool.k and bad == -math.inf and n > 1:  # no weight: as without it
                    check(kernel, pool, q, lengths)
                else:
                    assert not got[hit].isfinite().any()
                place.copy_(kept)


@PAGES
def test_attention_of_bf16_queries_is_rounded_once(kernel, e4m3):
    """Scores and weights of 24 bits, a score off by about 2^-22: outputs of many keys, errors of either sign like the sum's own
    terms, are off by about 2^-22 of themselves before they are rounded, next to steps of 2^-8 to 2^-7. So about 2^-13 of them
    round to the other side of 64 bits' result; four times as many are allowed. (Weights of 16 bits: sixteen
    times as many of bf16 pages.)"""
    lengths = [2000, 1333, 900, 513] * 4
    pool = Pool(len(lengths), 2048 // 64, 64, 8, e4m3, DEV)
    q = queries(len(lengths), 16, torch.bfloat16)
    got = check(kernel, pool, q, lengths)
    exact, _ = attention(pool, q, lengths)
    other = (got != exact.to(torch.bfloat16)).double().mean().item()
    print(f"[paged] the other side: {other:.2e}")
    assert other < 2.0 ** -11
