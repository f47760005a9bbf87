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


def put(b, pages, key, head, column, value):
    b.cache.v[pages[key // b.page], head, key % b.page, column] = value


@pytest.mark.parametrize("D,dtype", KINDS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_specials_in_values_reach_the_rows_that_see_them(fa, D, dtype, bad):
    """In V alone, in tiles that are masked for some rows of a wave: the rows that see the key have it in its column, all other
    elements keep their bits.  A prompt's own keys, the cut tile of a prefix that many rows stack up against, a few rows."""
    # 150 tokens of two heads a K/V head behind a prefix and 75 keys of their own
    b = Batch(fa, [150], [225], 37, 4, 2, D, 16, dtype, seed=57)
    clean = check(fa, b)
    put(b, b.table[0], 75 + 90, 0, 5, bad)
    put(b, b.table[0], 75 + 120, 0, 5, -bad)
    put(b, b.table[0], 75 + 149, 1, D - 1, bad)
    got = b.call(fa)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[90:, :2, 5] = True
    hit[149:, 2:, D - 1] = True
    assert torch.equal(got[~hit], clean[~hit])
    seen = torch.cat([got[90:120, :2, 5].flatten(), got[149, 2:, D - 1]])
    assert bool(seen.isnan().all()) if math.isnan(bad) else bool((seen == bad).all())
    assert bool(got[120:, :2, 5].isnan().all())  # (inf - inf)

    # 140 single tokens; the prefix' last key, and what lies behind it on its last page
    for count in (140, 12):
        b = Batch(fa, [1] * count, [1 + i % 40 for i in range(count)], 1000 + 5, 4, 2, D, 16, dtype, seed=58)
        clean = check(fa, b)
        put(b, b.prefix, 1004, 1, 7, bad)
        put(b, b.prefix, 960, 0, 8, bad)
        put(b, b.prefix, 1005, 0, slice(None), bad)
        put(b, b.table[3], b.held[3] - 1, 1, 9, bad)
        got = b.call(fa)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[:, 2:, 7] = True
        hit[:, :2, 8] = True
        hit[3, 2:, 9] = True
        assert torch.equal(got[~hit], clean[~hit])
        assert bool(got[hit].isnan().all()) if math.isnan(bad) else bool((got[hit] == bad).all())


@pytest.mark.parametrize("D,dtype", KINDS)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_page_0_is_nothing_where_no_page_is_named(fa, D, dtype, bad):
    """Page 0, which the kernels read where a table names no page and behind the last key, full of NaN or infinities; nobody's own."""
    for new, held, prefix in [([1, 9, 2], [100, 90, 40], 200 + 21), ([150, 3], [150 + 471, 40], 1024 + 17), ([1] * 140, [1 + i % 37 for i in range(140)], 517)]:
        b = Batch(fa, new, held, prefix, 2, 1, D, 16, dtype, seed=59)
        used = set(b.prefix + sum(b.table, []))
        spare = min(p for p in range(1, b.cache.n_pages) if p not in used)
        b.prefix, b.table = [spare if p == 0 else p for p in b.prefix], [[spare if p == 0 else p for p in t] for t in b.table]
        clean = check(fa, b)
        b.cache.k[0] = b.cache.v[0] = bad
        assert torch.equal(b.call(fa), clean)
        b.prefix[3], b.prefix[7], b.table[1][1] = -1, b.cache.n_pages, -2 ** 31
        b.table[0][2 % len(b.table[0])] = 2 ** 31 - 1
        check(fa, b)
        check(fa, b, causal=False)


def test_a_batch_in_several_calls(fa):
    """Each call with its own entries of q_start and k_len and its own rows of the table writes its own rows of one output."""
    b = Batch(fa, [1, 0, 3, 1, 140, 2, 1, 1, 5], [9, 4, 70, 33, 500, 2, 129, 64, 300], 333, 4, 2, 128, 16, BF16, seed=60, pad=4)
    q_start, k_len, table, prefix = ints(b.start), ints(b.held), ints(b.table), ints(b.prefix)
    out = torch.full_like(b.q, 3.5)
    for lo, hi in ((4, 7), (0, 4), (7, 9)):
        before = out.clone()
        fa.attention_shared_prefix(b.q, b.cache, q_start[lo:hi + 1], k_len[lo:hi], table[lo:hi], prefix, 333, out=out)
        mine = torch.zeros(b.q.shape[0], dtype=torch.bool, device=DEV)
        mine[b.start[lo]:b.start[hi]] = True
        assert torch.equal(out[~mine], before[~mine])
    want, tol = b.expected()
    n = b.start[-1]
    assert bool(((out.double() - want).abs() <= tol)[:n].all()) and bool((out[n:] == 3.5).all())
