"""GPU tier of attention over the paged cache: where prefixes and requests end inside a key tile, tables that name nothing
there, and what masked and missing keys hold.  Batch, check and the tolerance are test_paged_gpu's."""
import math

import pytest
import torch

from test_paged_gpu import BF16, DEV, F16, Batch, check, ints

pytestmark = pytest.mark.gpu

KINDS = [(64, F16), (64, BF16), (128, F16), (128, BF16), (256, F16), (256, BF16)]


@pytest.mark.parametrize("D,dtype", KINDS)
@pytest.mark.parametrize("prefix", [8192 + 5, 2048 + 33, 1024 + 17, 16])
def test_many_rows_behind_a_prefix_that_ends_inside_a_tile(fa, D, dtype, prefix):
    """A prompt chunk and as many single tokens, on pages shorter than a key tile; nothing in the tables behind the last page
    (Batch fills them with -7).  The same keys on pages longer than a tile give the same bits."""
    for new, held in [([150, 3], [150 + 371, 40]), ([1] * 140, [1 + i % 37 for i in range(140)])]:
        got = {}
        for page in (16, 128):
            b = Batch(fa, new, held, prefix, 2, 1, D, page, dtype, seed=50)
            g = torch.Generator(device=DEV).manual_seed(51)
            for pages, n in [(b.prefix, prefix)] + list(zip(b.table, held)):
                k, v = torch.randn(2, n, 1, D, dtype=dtype, device=DEV, generator=g)
                slots = torch.tensor(pages, device=DEV).repeat_interleave(page)[:n] * page + torch.arange(n, device=DEV) % page
                fa.cache_write(k, v, b.cache, slots.int())
            got[page] = check(fa, b)
        assert torch.equal(got[16], got[128])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_missing_pages_here_and_there(fa, D):
    """Pages that are none at both ends of the runs of 64 entries in which the kernel reads a table, and after a tile's first half."""
    for holes in ([0], [63], [64], [62, 65, 191], [300], list(range(128, 192)), list(range(0, 400, 2))):
        b = Batch(fa, [130, 1], [130 + 3000, 900], 400 * 16 + 5, 2, 1, D, 16, BF16, seed=52)
        for t in (b.prefix, b.table[0], b.table[1]):
            for i in holes:
                if i < len(t):
                    t[i] = -1
        check(fa, b)
        check(fa, b, causal=False)


def test_long_contexts_beside_so_many_rows_that_none_is_divided(fa):
    """22 000 tokens and more of 64 heads: the workspace has one part of own keys, or, without a prefix, none."""
    check(fa, Batch(fa, [1, 32999], [40001, 50], 0, 64, 4, 64, 16, F16, seed=53), causal=False)
    check(fa, Batch(fa, [3, 21997], [20000, 60], 500, 64, 4, 64, 16, BF16, seed=54), causal=False)
    b = Batch(fa, [2, 33000], [30000, 40], 0, 64, 8, 128, 16, BF16, seed=55)
    assert fa.lib().fa_shared_prefix_workspace(33002, 2, 64, 8, 128, 0, 1 << 20) == 4 * 33002 * 64
    check(fa, b, causal=False)
