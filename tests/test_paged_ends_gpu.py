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


def test_refused_requests_in_a_step(fa):
    """Of five requests the second and the fourth find no page: told apart by their lengths, nothing of them stored, the rows of the
    others as if they were alone, and their own as if their tokens were the last keys held."""
    page, Hq, Hkv, D = 16, 4, 2, 64
    held, new, fits = [16, 30, 5, 32, 3], [10, 20, 11, 1, 1], [True, False, True, False, True]
    b = Batch(fa, new, [h + n * ok for h, n, ok in zip(held, new, fits)], 50, Hq, Hkv, D, page, BF16, seed=56)
    owned = [-(-h // page) for h in held]
    table = ints([t[:n] + [-1] * (4 - n) for t, n in zip(b.table, owned)])
    free = ints([b.table[0][1]])  # one page, which the first request takes
    plan = fa.cache_plan(ints(held), ints(new), table, free, ints([1]), page, sum(new))
    assert plan.counts.tolist() == [0, 2] and plan.q_start.tolist() == b.start
    grown = (plan.k_len - ints(held)).tolist()
    assert [g == n for g, n in zip(grown, new)] == fits and plan.k_len.tolist() == b.held
    stored = [s >= 0 for s in plan.slots.tolist()]
    assert stored == sum(([ok] * n for ok, n in zip(fits, new)), [])
    k, v = torch.randn(2, sum(new), Hkv, D, dtype=BF16, device=DEV)
    before = b.cache.k.clone()
    fa.cache_write(k, v, b.cache, plan.slots)
    assert (before != b.cache.k).any(-1).sum() == Hkv * sum(stored)
    got = fa.attention_shared_prefix(b.q, b.cache, plan.q_start, plan.k_len, table, ints(b.prefix), 50)
    b.table = table.tolist()
    want, tol = b.expected()
    assert bool(((got.double() - want).abs() <= tol).all())
    keep = torch.tensor(stored, device=DEV)
    b.new, b.held, b.table = ([x for x, ok in zip(y, fits) if ok] for y in (b.new, b.held, b.table))
    b.q, b.start = b.q[keep], [0, 10, 21, 22]
    want, tol = b.expected()
    assert bool(((got[keep].double() - want).abs() <= tol).all())
