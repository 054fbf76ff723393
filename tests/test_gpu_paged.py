"""The paged cache of many sequences (``cache_write``, ``cache_read``, ``attention_paged``) on the GPU against the
definitions in 64 bits (``paged_pool``).

Writing and reading are exact: a number's rounding is fixed by its definition. Tolerances of the attention,
derived. A score is off by at most 2^-22 of the sum of its products' magnitudes, S (128 terms and their order, three
bf16 parts hold 24 bits), a weight by that much of itself, and the output by twice that times the largest |v|:
2^-21 S |v|. The sums over the keys take at most 11 additions per 32 keys one after the other (8 weights, 3 products)
and 64 where they are joined, each rounded by 2^-24 at most and either way: four times the root of their number.
bf16 queries: a weight in two bf16 parts is off by at most 2^-16 of itself, the output's rounding by 2^-8 of it."""
import math

import pytest
import torch

from oracle.spec import SHAPES
from paged_pool import D, Pool, attention, stored, values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float32
KINDS = pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
PAGES = pytest.mark.parametrize("e4m3", [False, True], ids=["bf16-pages", "e4m3-pages"])


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def queries(seqs, hq, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(seqs, hq, D, generator=gen, device=DEV) * scale).to(dtype)


def check(kernel, pool, q, lengths, expected=None):
    print(f"[paged] {q.dtype} e4m3 {pool.e4m3} page {pool.ps} heads {q.shape[1]}/{pool.h} lengths {lengths[:12]} "
          f"of {pool.tables.shape[1] * pool.ps}", flush=True)
    got = kernel.attention_paged(q, *pool.args(), ints(lengths), *pool.scales())
    torch.cuda.synchronize()
    assert got.dtype == q.dtype and got.shape == q.shape and got.is_contiguous()
    ref, off = attention(pool, q, lengths) if expected is None else expected
    worst = ((got.double() - ref).abs() / off.clamp(min=1e-30)).nan_to_num(nan=math.inf).max().item() if q.numel() else 0
    assert worst <= 1, worst
    return got


# ---------------------------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------------------------
def write_and_check(kernel, pool, k, v, begin, lengths, positions):
    """One call, and every place of the pool after it; positions[r] = (sequence, position) of row r, or None."""
    before = [(p.clone(), s.clone() if s is not None else None) for p, s in ((pool.k, pool.ks), (pool.v, pool.vs))]
    kernel.cache_write(k, v, *pool.args(), begin, lengths, *pool.scales())
    torch.cuda.synchronize()
    tables = pool.tables.tolist()
    rows = [(r, tables[p[0]][p[1] // pool.ps], p[1] % pool.ps) for r, p in enumerate(positions) if p is not None]
    for x, (pages, scales), (old, olds) in ((k, (pool.k, pool.ks), before[0]), (v, (pool.v, pool.vs), before[1])):
        expected = values(old, olds)
        if rows:
            r, page, at = (torch.tensor(c, device=DEV) for c in zip(*rows))
            expected[page, :, at] = stored(x[r], pool.e4m3)
        got = values(pages, scales)
        assert torch.equal(got.isnan(), expected.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), expected.nan_to_num(nan=0.0))
        if scales is not None:  # the bytes of rows that were not written
            kept = torch.ones(pages.shape[:3], dtype=torch.bool, device=DEV).permute(0, 2, 1).contiguous()
            if rows:
                kept[page, at] = False
            kept = kept.permute(0, 2, 1)
            assert torch.equal(pages.view(torch.uint8)[kept], old.view(torch.uint8)[kept])
            assert torch.equal(scales.view(torch.uint8)[kept], olds.view(torch.uint8)[kept])


@KINDS
@PAGES
@pytest.mark.parametrize("page_size,heads,layout", [(1, 8, "plain"), (8, 5, "joint"), (16, 8, "rows"), (64, 1, "plain"),
                                                    (512, 3, "joint"), (4096, 2, "plain")])
def test_cache(kernel, dtype, e4m3, page_size, heads, layout):
    entries = max(2, 700 // page_size + 1)
    pool = Pool(5, entries, page_size, heads, e4m3, DEV, layout, seed=page_size)
    begin, lengths = [0, 3, entries * page_size - 1, 129, 17], [31, 0, 1, 400, 5]
    total = sum(lengths)
    gen = torch.Generator(device=DEV).manual_seed(1)
    rows = torch.randn(total, 2 * heads, D, generator=gen, device=DEV)
    rows *= torch.exp2(torch.randint(-20, 20, (total, 2 * heads, 1), generator=gen, device=DEV).float())
    rows = rows.to(dtype)
    k, v = rows[:, :heads], rows[:, heads:]
    at = [(s, b + i) for s, (b, n) in enumerate(zip(begin, lengths)) for i in range(n)]
    write_and_check(kernel, pool, k, v, ints(begin), lengths, at)
    first, count = [1, 0, 5, 100, 0], [30, 3, 0, 429, 22]
    kk, vv = kernel.cache_read(*pool.args(), ints(first), count, *pool.scales())
    for got, which in ((kk, "k"), (vv, "v")):
        assert got.dtype == BF and got.shape == (sum(count), heads, D)
        expected = torch.cat([pool.rows(which, s, f, n) for s, (f, n) in enumerate(zip(first, count))])
        assert torch.equal(got.double(), expected)


@KINDS
def test_cache_rounds_to_even_at_every_border(kernel, dtype):
    """Every e4m3 number, every middle between two and the numbers next to the middles, in units of several
    powers of two; the largest magnitudes' own borders (448 times a power of two)."""
    numbers = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    numbers = numbers[numbers.isfinite()].unique()
    middle = (numbers[1:] + numbers[:-1]) / 2
    near = torch.cat([numbers, middle, torch.nextafter(middle, middle + 1), torch.nextafter(middle, middle - 1)])
    near = torch.cat([near, near.new_zeros(-len(near) % 127)]).view(-1, 127)
    rows = torch.cat([near, torch.full((len(near), 1), 448.0)], 1)  # the unit: 1
    tops = torch.tensor([448.0, math.nextafter(448.0, 1e9), 447.99, 449.0, 1.0, 0.5, 256.0, 255.9, 0.0, 1e-30, 3e38])
    more = torch.randn(len(tops), D, generator=torch.Generator().manual_seed(0)).clamp(-3, 3) / 4
    more = more / more.abs().amax(1, keepdim=True) * tops.double()[:, None].float()
    more[:, 5] = tops
    rows = torch.cat([rows, more])
    rows = torch.cat([rows * 2.0 ** e for e in (0, -7, 5)])
    rows = rows[rows.isfinite().all(1)].to(dtype).to(DEV)
    heads = 4
    rows = torch.cat([rows, rows.new_zeros(-len(rows) % heads, D)]).view(-1, heads, D)
    for e4m3 in (True, False):
        pool = Pool(1, len(rows) // 16 + 1, 16, heads, e4m3, DEV)
        write_and_check(kernel, pool, rows, -rows, ints([0]), [len(rows)], [(0, i) for i in range(len(rows))])


@KINDS
@PAGES
def test_cache_infinities_nan_and_the_smallest_numbers(kernel, dtype, e4m3):
    rows = torch.randn(7, 4, D, generator=torch.Generator().manual_seed(0))
    rows[0, 0, 5], rows[0, 1, 127], rows[1, 2, 0], rows[1, 3] = math.inf, math.nan, -math.inf, math.nan
    rows[2] = 0.0
    rows[3] *= 2.0 ** -130  # numbers of bf16 and fp32 below the normal ones
    rows[4] *= 2.0 ** -118
    rows[5, 0], rows[5, 1], rows[5, 2] = 3.3e38, -3.3e38, 1e-45
    rows[6, 0, :64] = 0.0
    rows = rows.to(dtype).to(DEV)
    pool = Pool(1, 1, 8, 4, e4m3, DEV)
    write_and_check(kernel, pool, rows, rows.flip(0), ints([0]), [7], [(0, i) for i in range(7)])
    k, v = kernel.cache_read(*pool.args(), ints([0]), [7], *pool.scales())
    expected = pool.rows("k", 0, 0, 7).to(BF).double()  # 3.3e38 is stored as 256 * 2^120, in bf16 an infinity
    assert torch.equal(k.double().nan_to_num(nan=7.5), expected.nan_to_num(nan=7.5))
    assert torch.equal(v.double().nan_to_num(nan=7.5), expected.flip(0).nan_to_num(nan=7.5))


@PAGES
def test_cache_places_out_of_range_are_left_out(kernel, e4m3):
    pool = Pool(4, 3, 16, 2, e4m3, DEV)
    pool.tables[1, 1], pool.tables[2, 0], pool.tables[2, 1] = -1, pool.n, 2 ** 31 - 1
    begin, lengths = [-3, 10, 0, 40], [10, 20, 48, 30]
    total = sum(lengths)
    k = torch.randn(total, 2, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    at = []
    for s, (b, n) in enumerate(zip(begin, lengths)):
        for p in range(b, b + n):
            inside = 0 <= p < 48 and not (s == 1 and 16 <= p < 32) and not (s == 2 and p < 32)
            at.append((s, p) if inside else None)
    write_and_check(kernel, pool, k, -k, ints(begin), lengths, at)
    first, count = [-2, 8, 30, 47], [5, 30, 6, 3]
    kk, vv = kernel.cache_read(*pool.args(), ints(first), count, *pool.scales())
    r = 0
    for s, (b, n) in enumerate(zip(first, count)):
        for p in range(b, b + n):
            inside = 0 <= p < 48 and not (s == 1 and 16 <= p < 32) and not (s == 2 and p < 32)
            if inside:
                assert torch.equal(kk[r].double(), pool.rows("k", s, p, 1)[0])
                assert torch.equal(vv[r].double(), pool.rows("v", s, p, 1)[0])
            else:
                assert kk[r].isnan().all() and vv[r].isnan().all()
            r += 1
    extreme = ints([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 5, -1])
    write_and_check(kernel, pool, k[:40], k[:40], extreme, [10, 10, 10, 1 + 9], [None] * 31 + [(3, i) for i in range(9)])


@PAGES
def test_cache_of_many_sequences(kernel, e4m3):
    """More than one launch takes, among them sequences without rows, first and last too."""
    seqs = 391
    pool = Pool(seqs, 2, 8, 3, e4m3, DEV)
    gen = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 6, (seqs,), generator=gen).tolist()
    lengths[0] = lengths[1] = lengths[128] = lengths[255] = lengths[256] = lengths[-1] = 0
    begin = torch.randint(0, 10, (seqs,), generator=gen).tolist()
    k = torch.randn(sum(lengths), 3, D, generator=gen).to(DEV)
    at = [(s, b + i) for s, (b, n) in enumerate(zip(begin, lengths)) for i in range(n)]
    write_and_check(kernel, pool, k, k * 3, ints(begin), lengths, at)
    kk, vv = kernel.cache_read(*pool.args(), ints(begin), lengths, *pool.scales())
    assert torch.equal(kk.double(), stored(k, e4m3)) and torch.equal(vv.double(), stored(k * 3, e4m3))
    # no rows at all
    kk, vv = kernel.cache_read(*pool.args(), ints(begin), [0] * seqs, *pool.scales())
    assert kk.shape == vv.shape == (0, 3, D)
    write_and_check(kernel, pool, k[:0], k[:0], ints(begin), [0] * seqs, [])


@KINDS
@PAGES
def test_cache_of_more_rows_than_the_caches_hold(kernel, dtype, e4m3):
    """More than 32 MiB of rows (read past the L2s)."""
    pool = Pool(2, 150, 64, 8, e4m3, DEV, "rows")
    n = (33 << 20) // (8 * 2 * D * (2 if dtype == BF else 4)) + 1
    lengths = [n - 700, 700]
    rows = torch.randn(n, 16, D, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(dtype)
    at = [(s, 9 + i) for s, c in enumerate(lengths) for i in range(c)]
    write_and_check(kernel, pool, rows[:, :8], rows[:, 8:], ints([9, 9]), lengths, at)


# ---------------------------------------------------------------------------------------------
# the attention
# ---------------------------------------------------------------------------------------------
@KINDS
@PAGES
@pytest.mark.parametrize("page_size", [1, 2, 4, 8, 16, 32, 64, 512])
def test_attention_lengths_and_pages(kernel, dtype, e4m3, page_size):
    lengths = [1, 0, 2, 31, 32, 33, 300, 129, 7, 512]
    for capacity in (512, 1024):  # a workgroup to a unit; the units' tiles shared out
        pool = Pool(len(lengths), capacity // page_size, page_size, 8, e4m3, DEV, seed=page_size)
        check(kernel, pool, queries(len(lengths), 16, dtype), lengths)


@KINDS
@PAGES
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (5, 1), (16, 2), (16, 1), (17, 1), (40, 2), (99, 3), (128, 128)])
def test_attention_head_layouts(kernel, dtype, e4m3, hq, hkv):
    lengths = [70, 1, 0, 190]
    for page_size, entries in ((16, 12), (32, 40)):
        pool = Pool(4, entries, page_size, hkv, e4m3, DEV, seed=hq)
        check(kernel, pool, queries(4, hq, dtype, seed=hq), lengths)


@KINDS
@PAGES
@pytest.mark.parametrize("lengths", [[5000], [3000, 1, 4097, 33], [20000], [2048] * 16, [0, 0, 700, 0], [0, 0, 0]],
                         ids=["5000", "ragged", "20000", "16x2048", "empty-around", "empty"])
def test_attention_long_and_ragged(kernel, dtype, e4m3, lengths):
    for page_size, layout in ((64, "plain"), (16, "joint")):
        pool = Pool(len(lengths), max(16, max(lengths) // page_size + 2), page_size, 8, e4m3, DEV, layout)
        check(kernel, pool, queries(len(lengths), 16, dtype), lengths)


@KINDS
@PAGES
def test_attention_of_many_short_sequences(kernel, dtype, e4m3):
    gen = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 40, (1500,), generator=gen).tolist()
    lengths[700] = 900
    pool = Pool(1500, 60, 16, 2, e4m3, DEV)
    check(kernel, pool, queries(1500, 4, dtype), lengths)
    pool = Pool(4096, 1, 32, 1, e4m3, DEV)
    lengths = torch.randint(0, 33, (4096,), generator=gen).tolist()
    check(kernel, pool, queries(4096, 1, dtype), lengths)


@KINDS
@PAGES
@pytest.mark.parametrize("layout", ["joint", "rows"])
def test_attention_strides(kernel, dtype, e4m3, layout):
    pool = Pool(3, 20, 32, 4, e4m3, DEV, layout)
    rows = queries(3, 16, dtype)
    check(kernel, pool, rows[:, 2:10], [600, 33, 5])  # a slice of a projection's rows
    wide = torch.zeros(3, 8, 2 * D, dtype=dtype, device=DEV)[..., :D].copy_(rows[:, :8])
    check(kernel, pool, wide, [1, 640, 320])
    check(kernel, pool, rows[:1, :8].expand(3, -1, -1), [600, 33, 5])  # one token's queries for all
    pool.tables = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)[:, 7:27].copy_(pool.tables)
    check(kernel, pool, rows[:, :8], [600, 33, 5])


@KINDS
@PAGES
def test_attention_large_scores(kernel, dtype, e4m3):
    pool = Pool(2, 40, 16, 4, e4m3, DEV)
    check(kernel, pool, queries(2, 8, dtype, scale=30.0), [600, 64])
    check(kernel, pool, queries(2, 8, dtype, scale=1e-20), [600, 64])
    check(kernel, pool, queries(2, 8, dtype) * 0, [600, 64])


@KINDS
@PAGES
@pytest.mark.parametrize("page_size", [8, 64])
def test_attention_does_not_look_behind_the_last_key(kernel, dtype, e4m3, page_size):
    """NaN in every row that no sequence's length reaches, and garbage in the table's entries behind it."""
    lengths = [37, 0, 300, 1]
    for entries in (512 // page_size, 1024 // page_size):
        pool = Pool(4, entries, page_size, 8, e4m3, DEV)
        q = queries(4, 16, dtype)
        expected = check(kernel, pool, q, lengths)
        used = torch.zeros(pool.n, page_size, dtype=torch.bool, device=DEV)
        for s, n in enumerate(lengths):
            at = torch.arange(n, device=DEV)
            used[pool.tables[s].long()[at // page_size], at % page_size] = True
        for pages, scales in ((pool.k, pool.ks), (pool.v, pool.vs)):
            if scales is None:
                pages.permute(0, 2, 1, 3)[~used] = math.nan
            else:
                pages.view(torch.uint8).permute(0, 2, 1, 3)[~used] = 0x7f
                scales.view(torch.uint8).permute(0, 2, 1)[~used] = 255
        for s, n in enumerate(lengths):
            left = pool.tables[s, -(-n // page_size):]
            left.copy_(ints([-1, 2 ** 31 - 1, pool.n, -2 ** 31])[torch.arange(len(left), device=DEV) % 4])
        got = kernel.attention_paged(q, *pool.args(), ints(lengths), *pool.scales())
        assert torch.equal(got, expected)


@KINDS
@PAGES
@pytest.mark.parametrize("page_size,entries", [(16, 20), (16, 80), (64, 8), (64, 40)])
def test_attention_reports_pages_and_lengths_out_of_range(kernel, dtype, e4m3, page_size, entries):
    capacity = page_size * entries
    lengths = [300, 65, capacity, 33, 200, 0]
    pool = Pool(6, entries, page_size, 8, e4m3, DEV)
    q = queries(6, 16, dtype)
    expected = check(kernel, pool, q, lengths)
    for s, (place, entry) in enumerate([(0, -1), (64 // page_size, pool.n), (entries - 1, 2 ** 31 - 1)]):
        kept = pool.tables[s, place].item()
        pool.tables[s, place] = entry
        got = kernel.attention_paged(q, *pool.args(), ints(lengths), *pool.scales())
        pool.tables[s, place] = kept
        for i in range(6):
            if i == s:
                assert got[i].isnan().all()
            else:
                assert torch.equal(got[i], expected[i])
    bad = [-1, 65, capacity + 1, 2 ** 31 - 1, -2 ** 31, 0]
    got = kernel.attention_paged(q, *pool.args(), ints(bad), *pool.scales())
    for i in (0, 2, 3, 4):
        assert got[i].isnan().all()
    ref, off = attention(pool, q, [0, 65, 0, 0, 0, 0])  # its neighbours' tiles are gone: the same up to rounding
    assert ((got[1].double() - ref[1]).abs() <= off[1]).all()
    assert (got[5] == 0).all()


@KINDS
@pytest.mark.parametrize("entries", [20, 80])
def test_attention_infinities_and_nan_among_what_is_seen(kernel, dtype, entries):
    """bf16 pages. A value that is not finite reaches its element of every query of its head and sequence, and
    nothing else; a key that makes a score -infinity weighs nothing, one that makes +infinity or NaN makes NaN."""
    pool = Pool(3, entries, 16, 2, False, DEV)
    lengths = [200, 290, 64]
    q = queries(3, 8, dtype)
    q[..., 3] = q[..., 3].abs() + 0.1
    plain = check(kernel, pool, q, lengths)

    def place(s, p):
        return pool.tables[s, p // 16].item(), p % 16

    for bad in (math.inf, -math.inf, math.nan):
        page, at = place(1, 77)
        kept = pool.v[page, 1, at, 9].item()
        pool.v[page, 1, at, 9] = bad
        got = kernel.attention_paged(q, *pool.args(), ints(lengths))
        pool.v[page, 1, at, 9] = kept
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[1, 4:, 9] = True
        assert not got[hit].isfinite().any() and torch.equal(got[~hit], plain[~hit])
    # a key of -infinity where the queries are positive: no weight
    page, at = place(0, 150)
    kept = pool.k[page, 0, at, 3].item()
    pool.k[page, 0, at, 3] = -math.inf
    got = check(kernel, pool, q, lengths)
    assert torch.equal(got[1:], plain[1:]) and torch.equal(got[0, 4:], plain[0, 4:])
    for bad in (math.inf, math.nan):
        pool.k[page, 0, at, 3] = bad
        got = kernel.attention_paged(q, *pool.args(), ints(lengths))
        assert got[0, :4].isnan().all() and torch.equal(got[0, 4:], plain[0, 4:]) and torch.equal(got[1:], plain[1:])
    pool.k[page, 0, at, 3] = kept
    # all scores -infinity: NaN
    at = torch.arange(64, device=DEV)
    pool.k[pool.tables[2].long()[at // 16], 1, at % 16, 3] = -math.inf
    got = kernel.attention_paged(q, *pool.args(), ints(lengths))
    assert got[2, 4:].isnan().all() and torch.equal(got[2, :4], plain[2, :4])
    # a query that is not finite
    q[0, 5, 2] = math.nan
    got = kernel.attention_paged(q, *pool.args(), ints(lengths))
    assert got[0, 5].isnan().all() and torch.equal(got[0, [0, 1, 2, 3, 4, 6, 7]], plain[0, [0, 1, 2, 3, 4, 6, 7]])


@KINDS
def test_attention_of_failed_rows_in_8_bit_pages(kernel, dtype):
    pool = Pool(2, 80, 16, 2, True, DEV)
    lengths = [500, 500]
    plain = check(kernel, pool, queries(2, 4, dtype), lengths)
    row = torch.full((1, 2, D), math.inf, device=DEV)
    good = pool.rows("v", 0, 123, 1).float()
    kernel.cache_write(pool.rows("k", 0, 123, 1).float(), row, *pool.args(), ints([123, 0]), [1, 0], *pool.scales())
    got = kernel.attention_paged(queries(2, 4, dtype), *pool.args(), ints(lengths), *pool.scales())
    assert got[0].isnan().all() and torch.equal(got[1], plain[1])
    kernel.cache_write(row, good, *pool.args(), ints([123, 0]), [1, 0], *pool.scales())
    got = kernel.attention_paged(queries(2, 4, dtype), *pool.args(), ints(lengths), *pool.scales())
    assert got[0].isnan().all() and torch.equal(got[1], plain[1])


def test_every_8_bit_number_in_every_unit(kernel):
    """Attention of one key is its value: all 256 bytes, all units that cache_write makes, as the kernel reads them."""
    bytes_ = torch.arange(256, dtype=torch.uint8, device=DEV).view(2, D)
    units = torch.arange(10, 248, dtype=torch.uint8, device=DEV)
    for page_size in (16, 32):
        pool = Pool(len(units), 1, page_size, 2, True, DEV, fill=False)
        pool.v.view(torch.uint8)[pool.tables[:, 0].long(), :, 0] = bytes_
        pool.vs.view(torch.uint8)[pool.tables[:, 0].long(), :, 0] = units[:, None]
        out = kernel.attention_paged(torch.zeros(len(units), 2, D, device=DEV), *pool.args(), ints([1] * len(units)),
                                     *pool.scales())
        k, v = kernel.cache_read(*pool.args(), ints([0] * len(units)), [1] * len(units), *pool.scales())
        expected = bytes_.view(torch.float8_e4m3fn).float().double() * torch.exp2(units.double() - 127)[:, None, None]
        expected = expected.to(BF).double()  # exact but for 2^128 and more
        assert torch.equal(v.double().nan_to_num(nan=0.25), expected.nan_to_num(nan=0.25)) and (k == 0).all()
        fine = expected.isfinite()
        assert torch.equal(out.double()[fine], expected[fine]) and not out[~fine].isfinite().any()


@PAGES
def test_places_past_32_bits(kernel, e4m3):
    """Pages more than 2^32 bytes (and elements) into the pool."""
    n, ps, h = (1 << 16) + 700, 64, 8
    kind = torch.uint8 if e4m3 else torch.bfloat16
    k, v = (torch.empty(n, h, ps, D, dtype=kind, device=DEV) for _ in range(2))
    pool = Pool(2, 10, ps, h, e4m3, DEV, fill=False)
    pool.k, pool.v, pool.n = (k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), n) if e4m3 else (k, v, n)
    if e4m3:
        pool.ks, pool.vs = (torch.empty(n, h, ps, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
                            for _ in range(2))
    pool.tables = (n - 1 - torch.arange(20, device=DEV).view(2, 10) * 31).int()
    rows = torch.randn(900, h, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    kernel.cache_write(rows, rows * 0.5, *pool.args(), ints([0, 0]), [600, 300], *pool.scales())
    kk, vv = kernel.cache_read(*pool.args(), ints([0, 0]), [600, 300], *pool.scales())
    assert torch.equal(kk.double(), stored(rows, e4m3)) and torch.equal(vv.double(), stored(rows * 0.5, e4m3))
    check(kernel, pool, queries(2, 16, FP), [600, 300])


@KINDS
@PAGES
def test_the_same_call_gives_the_same_bits_on_any_stream(kernel, dtype, e4m3):
    lengths = [4000, 77, 1500]
    pool = Pool(3, 256, 16, 8, e4m3, DEV)
    q, n = queries(3, 16, dtype), ints(lengths)
    first = check(kernel, pool, q, lengths)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):  # two at once
        streams[i % 2].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i % 2]):
            outs.append(kernel.attention_paged(q, *pool.args(), n, *pool.scales()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


@PAGES
def test_a_captured_step_replays_on_new_lengths_and_tables(kernel, e4m3):
    """A decode step's calls in a graph: the new row written, the attention, and the lengths counted up."""
    for capacity in (512, 2048):
        pool = Pool(5, capacity // 16, 16, 8, e4m3, DEV)
        at = ints([100, 0, 37, 15, 400])
        k, v = torch.zeros(5, 8, D, device=DEV), torch.zeros(5, 8, D, device=DEV)
        q = torch.zeros(5, 16, D, device=DEV)

        def step():
            kernel.cache_write(k, v, *pool.args(), at, [1] * 5, *pool.scales())
            return kernel.attention_paged(q, *pool.args(), at + 1, *pool.scales())

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        gen = torch.Generator(device=DEV).manual_seed(0)
        for i in range(4):
            for t in (k, v, q):
                t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
            at += 1
            if i == 2:  # other pages
                pool.tables.copy_(pool.tables.flip(1))
            graph.replay()
            torch.cuda.synchronize()
            lengths = (at + 1).tolist()
            got = out.clone()
            ref, off = attention(pool, q, lengths)
            assert ((got.double() - ref).abs() <= off).all()
            assert torch.equal(got, step())


def test_pages_of_a_paged_prefill(kernel):
    """A layer of prefill_paged's pools is a paged cache: it reads back as the contiguous prefill's cache."""
    shape = SHAPES["qwen3-0.6b"]
    H, I, V, L, S, n = shape.hidden, shape.intermediate, 512, 2, 128, 77
    gen = torch.Generator(device=DEV).manual_seed(0)

    def w(*s):
        return (torch.randn(*s, generator=gen, device=DEV) * 0.02).to(BF)

    one = lambda m: torch.ones(m, dtype=BF, device=DEV)  # noqa: E731
    layers = []
    for _ in range(L):
        layers += [one(H), w(2048, H), w(1024, H), w(1024, H), one(128), one(128), w(H, 2048), one(H), w(I, H), w(I, H), w(H, I)]
    embed = w(V, H)
    angle = torch.arange(S, device=DEV)[:, None] * 1e6 ** (-(torch.arange(D, device=DEV) % 64) / 64)
    cos, sin = angle.cos().to(BF), angle.sin().to(BF)
    tokens = torch.randint(0, V, (n,), device=DEV, dtype=torch.int32, generator=gen)
    flat = [torch.zeros(L, 8, S, D, dtype=BF, device=DEV) for _ in range(2)]
    kernel.prefill(tokens, embed, embed, one(H), layers, cos, sin, *flat, 0, S)
    pages = [torch.zeros(L, 11, 8, 16, D, dtype=BF, device=DEV) for _ in range(2)]
    table = ints([[7, 0, 3, 10, 9, 1, 2, 5]])
    kernel.prefill_paged(tokens, embed, embed, one(H), layers, cos, sin, *pages, table[0], 0, S)
    for layer in range(L):
        k, v = kernel.cache_read(pages[0][layer], pages[1][layer], table, ints([0]), [n])
        assert torch.equal(k, flat[0][layer, :, :n].transpose(0, 1)) and torch.equal(v, flat[1][layer, :, :n].transpose(0, 1))
        pool = Pool(1, 8, 16, 8, False, DEV, fill=False)
        pool.k, pool.v, pool.tables = pages[0][layer], pages[1][layer], table
        check(kernel, pool, queries(1, 16, FP), [n])
