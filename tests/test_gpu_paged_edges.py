"""``attention_paged`` and the paged cache on the GPU where shares of the work, scales and rows end in unusual places, against
the definitions in 64 bits (``paged_pool``; the tolerances are derived in ``test_gpu_paged``)."""
import pytest
import torch

from paged_pool import Pool
from test_gpu_paged import DEV, KINDS, PAGES, check, ints, queries

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
