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
