"""GPU tier of the paged-cache operators (cache_plan, cache_write, attention_shared_prefix) against plain implementations:
Python integers for the tables, float64 for attention."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ attention

def make_cache(fa, n_pages, heads, page, D, dtype, layout="hnd", seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if layout == "pool":  # K and V of a page beside each other
        both = torch.randn(n_pages, 2, heads, page, D, dtype=dtype, device=DEV, generator=g)
        return fa.PagedCache(both[:, 0], both[:, 1])
    shape = (n_pages, heads, page, D) if layout == "hnd" else (n_pages, page, heads, D)
    k, v = (torch.randn(shape, dtype=dtype, device=DEV, generator=g) for _ in range(2))
    if layout == "nhd":
        k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    return fa.PagedCache(k, v)


class Batch:
    """Requests with new[b] tokens and held[b] keys (the new ones among them) behind prefix_len shared keys."""

    def __init__(self, fa, new, held, prefix_len, Hq, Hkv, D, page, dtype, layout="hnd", seed=0, pad=0, scale=None):
        rng = random.Random(seed)
        pages, prefix_pages = [-(-h // page) for h in held], -(-prefix_len // page)
        ids = list(range(sum(pages) + prefix_pages + 3))
        rng.shuffle(ids)
        self.cache = make_cache(fa, len(ids), Hkv, page, D, dtype, layout, seed)
        self.prefix = ids[:prefix_pages]
        at, self.table = prefix_pages, []
        for n in pages:
            self.table.append(ids[at:at + n] + [-7] * (max(pages) + 1 - n))
            at += n
        self.start = [0]
        for n in new:
            self.start.append(self.start[-1] + n)
        self.new, self.held, self.prefix_len, self.page = new, held, prefix_len, page
        g = torch.Generator(device=DEV).manual_seed(seed + 1)
        self.q = torch.randn(self.start[-1] + pad, Hq, D, dtype=dtype, device=DEV, generator=g)
        self.scale = scale

    def call(self, fa, causal=True, **kw):
        return fa.attention_shared_prefix(self.q, self.cache, ints(self.start), ints(self.held), ints(self.table),
                                          prefix_table=ints(self.prefix) if self.prefix_len else None, prefix_len=self.prefix_len,
                                          causal=causal, scale=self.scale, **kw)

    def keys(self, c, pages, n, h):
        """Rows of the keys a list of pages names, and which of them exist."""
        ok = torch.tensor([0 <= p < self.cache.n_pages for p in pages], device=DEV, dtype=torch.bool).repeat_interleave(self.page)[:n]
        at = torch.tensor([min(max(p, 0), self.cache.n_pages - 1) for p in pages], device=DEV, dtype=torch.long)
        rows = c[at, h].reshape(-1, c.shape[-1])[:n].double()
        return rows, ok

    def expected(self, causal=True):
        """(output in float64, bound of the kernel's error): see tolerance() below."""
        T, Hq, D = self.q.shape
        g = Hq // self.cache.heads
        out = torch.zeros(T, Hq, D, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(out)
        scale = D ** -0.5 if self.scale is None else self.scale
        for b, (n, held) in enumerate(zip(self.new, self.held)):
            own = self.table[b][: -(-held // self.page)]
            for h in range(self.cache.heads):
                if n == 0 or self.prefix_len + held == 0:
                    continue
                parts = []
                for c in (self.cache.k, self.cache.v):
                    a, ok_a = self.keys(c, self.prefix, self.prefix_len, h)
                    o, ok_o = self.keys(c, own, held, h)
                    parts.append(torch.cat([a, o]))
                k, v = parts
                ok = torch.cat([ok_a, ok_o])
                q = self.q[self.start[b]:self.start[b + 1], h * g:(h + 1) * g].double()
                pos = torch.arange(k.shape[0], device=DEV)
                last = self.prefix_len + held - (n - torch.arange(n, device=DEV) if causal else torch.ones(n, device=DEV))
                seen = (ok & ((pos < self.prefix_len) | (pos <= last[:, None])))[:, None, :].expand(n, g, -1)
                k = torch.where(ok[:, None], k, 0.0)
                scores = torch.where(seen, (q.reshape(n * g, D) @ k.t()).reshape(n, g, -1) * scale, -math.inf)
                m = scores.amax(-1, keepdim=True)
                p = torch.where(seen, torch.exp(scores - torch.where(m == -math.inf, 0.0, m)), 0.0)
                l = p.sum(-1, keepdim=True)
                # a masked place takes no part whatever it holds: values are read where some row sees them
                rows = torch.where(ok[:, None], v, 0.0)
                if not bool(rows.isfinite().all()):
                    o = torch.stack([torch.stack([(p[i, j][seen[i, j]][:, None] * rows[seen[i, j]]).sum(0) for j in range(g)]) for i in range(n)])
                    a = torch.full_like(o, math.inf)
                else:
                    o = (p.reshape(n * g, -1) @ rows).reshape(n, g, D)
                    a = (p.reshape(n * g, -1) @ rows.abs()).reshape(n, g, D)
                safe = torch.where(l == 0, 1.0, l)
                o, a = torch.where(l == 0, 0.0, o / safe), torch.where(l == 0, 0.0, a / safe)
                size = (q.abs().reshape(n * g, D) @ k.abs().t()).reshape(n, g, -1).amax(-1, keepdim=True) * abs(scale)
                out[self.start[b]:self.start[b + 1], h * g:(h + 1) * g] = o
                tol[self.start[b]:self.start[b + 1], h * g:(h + 1) * g] = tolerance(self.q.dtype, o, a, size, D, k.shape[0], rows)
        return out, tol


def tolerance(dtype, o, a, size, D, n, v):
    """Bound of |kernel - exact| for output o, a = sum p|v| / sum p, size = largest sum |q k| scale of the row.  u: half a
    step of dtype relative to the value, e = 2^-24.
      P rounded to dtype                            u a       (its sum is taken before the rounding)
      the output rounded                            u |o|
      scores in fp32: D products and additions, scale, log2(e), maximum taken off: (D + 8) e size in the exponent, which
        moves every p by as much; exp2 itself 2 e;  both in P and in its sum:       2 ((D + 8) size + 4) e a
      sums of n terms in fp32, 16 a step, and up to 64 parts joined:               2 (n / 16 + 80) e a
      fp16 only: p below 2^-14 is rounded by half its smallest step, 2^-25 (the largest p is at least 1):  n 2^-25 mean|v|"""
    e, u = 2.0 ** -24, torch.finfo(dtype).eps / 2
    t = u * (a + o.abs()) * (1 + 2 ** -8) + 2 * ((D + 8) * size + 4 + n / 16 + 80) * e * a
    if dtype == F16:
        t = t + n * 2.0 ** -25 * v.abs().mean() + 2.0 ** -24
    return t + 1e-30


def check(fa, batch, causal=True, **kw):
    got = batch.call(fa, causal, **kw)
    want, tol = batch.expected(causal)
    n = batch.start[-1]
    err = (got.double() - want).abs()[:n]
    bad = ~(err <= tol[:n])
    assert not bool(bad.any()), (int(bad.sum()), float(err.max()), float((err / tol[:n]).max()), bad.nonzero()[0].tolist())
    return got


SHAPES = [
    # new tokens, own keys, prefix, Hq, Hkv, D, page, dtype, layout
    ([1], [1], 0, 1, 1, 128, 16, F16, "hnd"),
    ([1], [1], 1, 4, 1, 64, 16, BF16, "hnd"),
    ([1, 1, 1], [1, 16, 17], 15, 8, 2, 128, 16, BF16, "nhd"),
    ([1] * 5, [63, 64, 65, 127, 130], 64, 8, 8, 64, 32, F16, "pool"),
    ([1] * 9, [1, 2, 300, 40, 5, 60, 70, 8, 129], 1000, 20, 4, 128, 16, F16, "hnd"),
    ([1] * 33, [10 * i + 1 for i in range(33)], 513, 16, 2, 128, 64, BF16, "nhd"),
    ([1] * 7, [40] * 7, 333, 6, 2, 256, 16, F16, "hnd"),
    ([4] * 6, [4, 5, 20, 64, 65, 200], 100, 16, 4, 256, 32, BF16, "hnd"),
    ([5, 3, 0, 1, 8], [5, 100, 50, 1, 8], 65, 7, 1, 128, 16, F16, "pool"),
    ([130, 1, 40], [130, 77, 300], 200, 8, 2, 128, 128, BF16, "hnd"),
    ([257], [257], 0, 4, 4, 64, 16, F16, "nhd"),
    ([33, 64, 1], [500, 64, 65], 0, 12, 4, 128, 16, BF16, "hnd"),
    ([100, 200], [100, 900], 1500, 4, 1, 256, 64, F16, "nhd"),
    ([1] * 130, [3] * 130, 40, 3, 3, 64, 16, BF16, "hnd"),
    ([1, 1], [5000, 1], 7001, 8, 1, 128, 256, F16, "hnd"),
    ([300, 2, 300], [300, 2, 700], 129, 10, 2, 64, 32, BF16, "pool"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_shapes(fa, case, causal):
    new, held, prefix, Hq, Hkv, D, page, dtype, layout = SHAPES[case]
    check(fa, Batch(fa, new, held, prefix, Hq, Hkv, D, page, dtype, layout, seed=case), causal)


@pytest.mark.parametrize("seed", range(12))
def test_drawn_shapes(fa, seed):
    rng = random.Random(100 + seed)
    Hkv, g, D = rng.choice([1, 2, 3, 8]), rng.randint(1, 9), rng.choice([64, 128, 256])
    B = rng.randint(1, 20)
    new = [rng.choice([0, 1, 1, 1, 2, rng.randint(1, 60)]) for _ in range(B)]
    held = [n + rng.choice([0, rng.randint(0, 30), rng.randint(0, 600)]) for n in new]
    check(fa, Batch(fa, new, held, rng.choice([0, rng.randint(1, 100), rng.randint(100, 3000)]), Hkv * g, Hkv, D, rng.choice([16, 32, 64, 128]),
                    rng.choice([F16, BF16]), rng.choice(["hnd", "nhd", "pool"]), seed=seed), rng.random() < 0.7)


@pytest.mark.parametrize("D,dtype", [(64, F16), (64, BF16), (128, F16), (128, BF16), (256, F16), (256, BF16)])
@pytest.mark.parametrize("rows", [15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 257])
def test_row_counts(fa, rows, D, dtype):
    """Around the sizes where the kernel's forms change: one request's rows, and as many single tokens stacked up."""
    check(fa, Batch(fa, [rows], [rows + 21], 83, 1, 1, D, 16, dtype, seed=rows))
    check(fa, Batch(fa, [1] * rows, [1 + i % 5 for i in range(rows)], 150, 1, 1, D, 16, dtype, seed=rows + 1))


def test_many_requests(fa):
    """More than one round of 64 and of 128 lengths; idle requests and long ones among them."""
    rng = random.Random(4)
    new = [rng.choice([0, 1, 1, 1, 2]) for _ in range(700)]
    new[77], new[300], new[699] = 140, 33, 200
    check(fa, Batch(fa, new, [n + rng.randint(0, 40) for n in new], 90, 2, 1, 64, 16, BF16, seed=20))
    new = [1] * 4000
    b = Batch(fa, new, [1 + i % 3 for i in range(4000)], 20, 1, 1, 64, 16, F16, seed=21)
    got = b.call(fa)
    some = [0, 1, 63, 64, 127, 128, 1999, 3998, 3999]
    b.new, b.held, b.table = [1] * len(some), [b.held[i] for i in some], [b.table[i] for i in some]
    b.q, b.start = b.q[some], list(range(len(some) + 1))
    want, tol = b.expected()
    assert bool(((got[some].double() - want).abs() <= tol).all())
    with pytest.raises(fa.FlashAttentionError):
        Batch(fa, [0] * 4001, [1] * 4001, 0, 1, 1, 64, 16, F16, pad=1).call(fa)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_ranges(fa, D):
    """Keys of one request, and a prefix, over many parts and many runs of 64 page entries, some of which name no page."""
    check(fa, Batch(fa, [1], [40001], 0, 2, 1, D, 16, F16, seed=22))
    check(fa, Batch(fa, [3], [20000], 30011, 8, 1, D, 32, BF16, seed=23))
    b = Batch(fa, [1, 140], [3000, 5000], 9000, 2, 1, D, 16, F16, seed=24)
    for t in (b.prefix, b.table[0], b.table[1]):
        for i in range(3, len(t), 71):
            t[i] = -1
    check(fa, b)


def test_ends_of_the_ranges(fa):
    """128 query heads on one K/V head, 100 K/V heads, the largest pages."""
    check(fa, Batch(fa, [1, 2, 0, 1], [1, 70, 5, 300], 200, 128, 1, 128, 16, F16, seed=30))
    check(fa, Batch(fa, [1, 3], [1, 70], 45, 100, 100, 64, 16, BF16, seed=31))
    check(fa, Batch(fa, [1, 20], [5000, 33], 66000, 4, 2, 64, 65536, F16, seed=32))
    check(fa, Batch(fa, [3, 150], [9, 4000], 2000, 2, 1, 256, 4096, BF16, seed=33))


def test_long_context_beside_very_many_rows(fa):
    """The workspace of many rows has room for few parts: the one token's 40 001 keys still count, each once."""
    check(fa, Batch(fa, [1, 19999], [40001, 50], 0, 32, 4, 64, 16, F16, seed=39), causal=False)


def test_tables_without_columns_and_empty_calls(fa):
    b = Batch(fa, [1, 3], [0, 0], 77, 4, 2, 128, 16, BF16, seed=40)
    want, tol = b.expected()
    none = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    for held in ([0, 0], [5, 900]):  # (the table names no page: clamped to no keys)
        got = fa.attention_shared_prefix(b.q, b.cache, ints(b.start), ints(held), none, ints(b.prefix), 77)
        assert bool(((got.double() - want).abs() <= tol).all())
    assert not fa.attention_shared_prefix(b.q, b.cache, ints(b.start), ints([5, 9]), none).any()
    assert fa.attention_shared_prefix(b.q[:0], b.cache, ints([0, 0, 0]), ints([5, 9]), none, ints(b.prefix), 77).shape == (0, 4, 128)
    assert not fa.attention_shared_prefix(b.q, b.cache, ints([0]), ints([]), none[:0], ints(b.prefix), 77).any()
    plan = fa.cache_plan(ints([3]), ints([2]), ints([[1]]), ints([]), ints([0]), 16, 0)  # no room for a token: refused
    assert plan.k_len.tolist() == [3] and plan.counts.tolist() == [0, 1] and plan.slots.numel() == 0


def test_strides_of_axes_of_one(fa):
    """One token, one head, one page: the stride of such an axis may be anything."""
    b = Batch(fa, [1], [9], 0, 1, 1, 64, 16, F16, seed=41)
    want = b.call(fa)
    b.q = torch.as_strided(b.q, b.q.shape, (3, 5, 1))
    assert torch.equal(b.call(fa, out=torch.as_strided(torch.zeros(64, dtype=F16, device=DEV), (1, 1, 64), (1, 1, 1))), want)
    k, v = b.cache.k[:1], b.cache.v[:1]
    odd = [torch.as_strided(x, x.shape, (7, 3, 64, 1)) for x in (k, v)]
    b.cache = fa.PagedCache(*odd)
    b.table = [[0]]
    want, tol = b.expected()
    assert bool(((b.call(fa).double() - want).abs() <= tol).all())
    rows = torch.as_strided(torch.randn(64, dtype=F16, device=DEV), (1, 1, 64), (1, 1, 1))
    fa.cache_write(rows, rows, b.cache, ints([4]))
    assert torch.equal(b.cache.k[0, 0, 4], rows[0, 0])


def test_calls_at_once(fa):
    """Two batches of different sizes on two streams, a handle and a stream object, with nothing between the calls."""
    a = Batch(fa, [1] * 40, [50 * i + 1 for i in range(40)], 6000, 8, 2, 128, 16, F16, seed=34)
    b = Batch(fa, [200, 1], [900, 3000], 3000, 4, 1, 128, 16, F16, seed=35)
    want = [x.call(fa) for x in (a, b)]
    args = [(x.q, x.cache, ints(x.start), ints(x.held), ints(x.table), ints(x.prefix), x.prefix_len) for x in (a, b)]
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [fa.attention_shared_prefix(*args[i % 2], stream=(s[0], s[1].cuda_stream)[i % 2]) for i in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(got))


def test_output_over_the_queries_is_refused(fa):
    b = Batch(fa, [1], [9], 20, 2, 1, 64, 16, F16, seed=36)
    with pytest.raises(fa.FlashAttentionError):
        b.call(fa, out=b.q)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_scores_and_other_scales(fa, dtype):
    b = Batch(fa, [1, 20, 3], [50, 70, 3], 300, 8, 2, 128, 16, dtype, seed=5, scale=1.7)
    check(fa, b)
    b.scale = 1e-3
    check(fa, b)


def test_requests_without_keys_or_tokens(fa):
    """No prefix: a request without keys gives 0; tokens ahead of the request's keys see nothing."""
    b = Batch(fa, [2, 0, 1, 4], [0, 30, 20, 2], 0, 4, 2, 128, 16, F16, seed=3)
    out = b.call(fa)
    assert bool((out[:2] == 0).all()) and bool((out[3:5] == 0).all())
    want, tol = b.expected()
    assert bool(((out.double() - want).abs() <= tol)[2:].all())
    # nothing but idle requests: no row is written
    b = Batch(fa, [0, 0], [16, 5], 40, 4, 2, 64, 16, BF16, seed=3, pad=3)
    out = torch.full_like(b.q, 7.0)
    assert b.call(fa, out=out) is out and bool((out == 7).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_of_no_request_keep_their_bytes(fa, D):
    b = Batch(fa, [1, 3, 40], [9, 3, 60], 70, 6, 2, D, 16, F16, seed=4, pad=37)
    out = torch.full_like(b.q, 3.5)
    check(fa, b, out=out)
    assert bool((out[b.start[-1]:] == 3.5).all())
    assert bool((check(fa, b)[b.start[-1]:] == 0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_places_may_hold_anything(fa, D, dtype, bad):
    """Behind the last key of a page, on pages that nobody names, and in keys that later tokens alone see."""
    b = Batch(fa, [1, 5, 70], [17, 40, 90], 100, 4, 2, D, 16, dtype, seed=6)
    want, tol = b.expected()
    named = torch.zeros(b.cache.n_pages, 1, 16, dtype=torch.bool, device=DEV)
    for pages, n in [(b.prefix, b.prefix_len)] + list(zip(b.table, b.held)):
        for i in range(n):
            named[pages[i // 16], 0, i % 16] = True
    for c in (b.cache.k, b.cache.v):
        c[(~named).expand(-1, c.shape[1], -1)] = bad
    got = b.call(fa)
    assert bool(((got.double() - want).abs() <= tol).all())
    # the last key of every request: only its last token sees it
    for t, n in zip(b.table, b.held):
        b.cache.k[t[(n - 1) // 16], :, (n - 1) % 16] = bad
        b.cache.v[t[(n - 1) // 16], :, (n - 1) % 16] = bad
    got = b.call(fa)
    last = torch.zeros(b.start[-1], dtype=torch.bool, device=DEV)
    last[[s - 1 for s in b.start[1:]]] = True
    assert bool(((got.double() - want).abs() <= tol)[~last].all())
    assert not bool(got[last].isfinite().any(-1).any()) or not math.isnan(bad)


@pytest.mark.parametrize("D", [64, 128])
def test_visible_specials_come_out(fa, D):
    """A NaN score makes the row NaN; an infinite value comes out with its sign, in its column alone."""
    b = Batch(fa, [1, 6], [20, 33], 50, 4, 2, D, 16, F16, seed=8)
    clean = b.call(fa)
    row = 33 - 3  # the fourth token's own key: tokens 3, 4, 5 of request 1 see it
    page, r = b.table[1][row // 16], row % 16
    b.cache.v[page, 0, r, 5] = math.inf
    b.cache.v[page, 1, r, 7] = -math.inf
    got = b.call(fa)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[1 + 3:, :2, 5] = True
    hit[1 + 3:, 2:, 7] = True
    assert bool((got[1 + 3:, :2, 5] == math.inf).all()) and bool((got[1 + 3:, 2:, 7] == -math.inf).all())
    assert torch.equal(got[~hit], clean[~hit])
    b.cache.k[page, 0, r, 0] = math.nan
    got = b.call(fa)
    assert bool(got[1 + 3:, :2].isnan().all()) and bool(got[:1 + 3].isfinite().all()) and not bool(got[:, 2:].isnan().any())
    # in the prefix, everybody sees it
    b.cache.v[b.prefix[1], 1, 3, 9] = math.nan
    got = b.call(fa)
    assert bool(got[:, 2:, 9].isnan().all()) and not bool(got[:, 2:, 10].isnan().any())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_entries_that_name_no_page(fa, dtype):
    """Their keys take no part, whatever page 0 holds; a request all of whose pages are gone gives 0."""
    b = Batch(fa, [1, 9, 2, 1], [100, 90, 40, 30], 200, 8, 2, 128, 16, dtype, seed=9)
    b.prefix[3] = -1
    b.prefix[7] = b.cache.n_pages
    b.table[0][2], b.table[1][0], b.table[1][4] = 2 ** 31 - 1, -2 ** 31, -1
    used = set(b.prefix + sum(b.table, []))
    if 0 not in used:
        b.cache.v[0] = math.nan
    check(fa, b)
    check(fa, b, causal=False)
    b.prefix_len, b.table[3] = 0, [-1] * len(b.table[3])
    assert bool((check(fa, b)[-1] == 0).all())


def test_strided_queries_and_outputs(fa):
    """q as a slice of a fused projection, the output in a wider buffer, both with a head axis that is not the last but one."""
    b = Batch(fa, [1, 7, 30], [11, 7, 55], 90, 8, 2, 128, 16, BF16, seed=10)
    T = b.q.shape[0]
    fused = torch.randn(T, 8 + 2 + 2, 128, dtype=BF16, device=DEV)
    fused[:, :8] = b.q
    b.q = fused[:, :8]
    wide = torch.zeros(8, T, 136, dtype=BF16, device=DEV)
    out = wide[:, :, :128].transpose(0, 1)
    check(fa, b, out=out)
    assert bool((wide[:, :, 128:] == 0).all())
    with pytest.raises(fa.FlashAttentionError):
        b.q = torch.zeros(T, 8, 129, dtype=BF16, device=DEV)[:, :, 1:]
        b.call(fa)


def test_a_request_longer_than_the_bound_is_still_whole(fa):
    b = Batch(fa, [1, 3], [700, 90], 40, 8, 2, 128, 16, F16, seed=11)
    check(fa, b, max_k_len=64)
    check(fa, b, max_k_len=0)
    check(fa, b, max_k_len=10 ** 9)


def test_lengths_beyond_the_table_are_clamped(fa):
    b = Batch(fa, [1, 2], [64, 50], 20, 4, 2, 64, 16, F16, seed=12)
    want = b.call(fa)
    b.table = [t[:4] for t in b.table]
    got = fa.attention_shared_prefix(b.q, b.cache, ints([0, 1, 3 + 1000]), ints([10 ** 9, 50]), ints(b.table), ints(b.prefix), 20)
    assert torch.equal(got[0], want[0])


def test_offsets_past_32_bits(fa):
    """A cache of 2^33 elements, its pages used at both ends."""
    n_pages, heads, page, D = 32768 + 3, 8, 256, 128
    k = torch.empty(n_pages, heads, page, D, dtype=F16, device=DEV)
    v = torch.empty(n_pages, heads, page, D, dtype=F16, device=DEV)
    b = Batch(fa, [1, 3], [300, 290], 600, 8, 8, D, page, F16, seed=13)
    ids = sorted(set(b.prefix + [p for t, h in zip(b.table, b.held) for p in t[: -(-h // page)]]))
    far = {p: (n_pages - 1 - i if i % 2 else i) for i, p in enumerate(ids)}
    for p, f in far.items():
        k[f], v[f] = b.cache.k[p], b.cache.v[p]
    b.cache = fa.PagedCache(k, v)
    b.prefix = [far[p] for p in b.prefix]
    b.table = [[far.get(p, -1) for p in t] for t in b.table]
    check(fa, b)
    rows = torch.randn(2, heads, D, dtype=F16, device=DEV)
    slots = ints([(n_pages - 2) * page + 255, 5])
    fa.cache_write(rows, rows, b.cache, slots)
    assert torch.equal(k[n_pages - 2, :, 255], rows[0]) and torch.equal(v[0, :, 5], rows[1])


def test_same_bits_twice_and_on_another_stream(fa):
    b = Batch(fa, [1] * 17, [40 * i + 1 for i in range(17)], 2000, 8, 2, 128, 32, BF16, seed=14)
    first = b.call(fa)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.zeros_like(b.q) for _ in range(4)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        b.call(fa, out=o, **({"stream": side} if i % 2 else {}))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    with torch.cuda.stream(side):
        assert torch.equal(b.call(fa), first)
    o, ms = b.call(fa, timed=True)
    assert torch.equal(o, first) and ms > 0


def test_captured_and_replayed_with_other_lengths(fa):
    """Two graphs of one step at a time, replayed in turn over lengths that change between the replays, beside eager calls."""
    b = Batch(fa, [1, 1, 4], [300, 9, 100], 500, 8, 2, 128, 16, F16, seed=15, pad=2)
    q_start, k_len, table, prefix = ints(b.start), ints(b.held), ints(b.table), ints(b.prefix)
    graphs = []
    for _ in range(2):
        out = torch.zeros_like(b.q)
        call = lambda: fa.attention_shared_prefix(b.q, b.cache, q_start, k_len, table, prefix, 500, out=out)  # noqa: B023, E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append((g, out))
    for step in range(4):
        held, start = [300 - step, 9 + step, 100 - 30 * step], [0, 1, 2, 6 - step]
        k_len.copy_(ints(held))
        q_start.copy_(ints(start))
        eager = fa.attention_shared_prefix(b.q, b.cache, q_start, k_len, table, prefix, 500)
        for g, out in graphs:
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        b.held, b.start, b.new = held, start, [1, 1, 4 - step]
        want, tol = b.expected()
        assert bool(((eager.double() - want).abs() <= tol).all())
        for _, out in graphs:
            assert torch.equal(out, eager)


# ------------------------------------------------------------------------------------------------ the cache

def plan_in_python(held, new, table, stack, page, max_tokens):
    """The step as a program would write it down: the same lists, updated."""
    pages = lambda x: -(-x // page)  # noqa: E731
    width = len(table[0])
    start, t = [0], 0
    for n in new:
        t += max(n, 0)
        start.append(t)
    after, slots, refused, needed = [], [-1] * max_tokens, 0, 0
    new = [max(n, -h) for n, h in zip(new, held)]
    for b, (h, n) in enumerate(zip(held, new)):
        if n < 0:
            stack += table[b][pages(h + n):pages(h)]
    have = len(stack)
    for b, (h, n) in enumerate(zip(held, new)):
        wide = h + n > width * page or (n > 0 and start[b + 1] > max_tokens)
        need = 0 if wide else max(0, pages(h + n) - pages(h))
        needed += need
        if wide or (need and needed > have):
            refused += 1
            after.append(h)
            continue
        for j in range(pages(h), pages(h) + need):
            table[b][j] = stack.pop()
        for i in range(max(n, 0)):
            slots[start[b] + i] = table[b][(h + i) // page] * page + (h + i) % page
        after.append(h + n)
    return start, after, slots, [len(stack), refused]


def run_plan(fa, held, new, table, stack, cap, page, max_tokens, out=None):
    free = ints(stack + [-9] * (cap - len(stack)))
    t = ints(table)
    p = fa.cache_plan(ints(held), ints(new), t, free, ints([len(stack)]), page, max_tokens, out=out)
    return p, t, free


@pytest.mark.parametrize("seed", range(24))
def test_plan_against_python(fa, seed):
    rng = random.Random(seed)
    B, page, width = rng.choice([1, 2, 7, 64, 300, 1500]), rng.choice([16, 32, 256]), rng.randint(1, 40)
    room = page * width
    held = [rng.choice([0, rng.randint(0, room), room]) for _ in range(B)]
    new = [rng.choice([0, 1, 1, 1, 3, rng.randint(0, room), -1, -rng.randint(0, room), -h]) for h in held]
    pages = [-(-h // page) for h in held]
    ids = list(range(sum(pages) + rng.choice([0, 3, B * width])))
    rng.shuffle(ids)
    table, at = [], 0
    for n in pages:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    stack = ids[at:]
    cap = len(ids) + 2
    tokens = sum(max(n, 0) for n in new)
    max_tokens = rng.choice([tokens, tokens + 70, max(0, tokens - 5)])
    p, t, free = run_plan(fa, held, new, table, stack, cap, page, max_tokens)
    n_before = len(stack)
    start, after, slots, counts = plan_in_python(held, new, table, stack, page, max_tokens)
    assert p.counts.tolist() == counts
    assert p.q_start.tolist() == start and p.k_len.tolist() == after
    assert p.slots.tolist() == slots
    got = t.tolist()
    for b in range(B):  # entries that name keys held; what lies behind is the program's own
        n = -(-after[b] // page)
        assert got[b][:n] == table[b][:n], b
    assert free.tolist()[:counts[0]] == stack[:counts[0]]
    assert n_before <= cap


def test_plan_ends_of_the_range(fa):
    big = 2 ** 31 - 1
    # lengths that are no lengths, sums past 31 bits, an empty list, no room for tokens
    p, t, _ = run_plan(fa, [-5, big, 0, 3], [1, big, big, -big], [[-1] * 2] * 4, [4], 1, 16, 0)
    assert p.k_len.tolist() == [0, 32, 0, 0] and p.counts.tolist() == [1, 3]
    assert p.q_start.tolist() == [0, 1, big, big, big]
    # 5120 requests, one token each; one more is refused
    B = 5120
    p, t, _ = run_plan(fa, [0] * B, [1] * B, [[-1]] * B, list(range(B)), B, 16, B)
    assert p.counts.tolist() == [0, 0] and p.slots.tolist() == [16 * (B - 1 - i) for i in range(B)]
    with pytest.raises(fa.FlashAttentionError):
        run_plan(fa, [0] * (B + 1), [1] * (B + 1), [[-1]] * (B + 1), [], 0, 16, 0)
    # a count that is none is taken as the nearest that is
    one = ints([1])
    for count, left in ((-3, 0), (99, 1)):
        p = fa.cache_plan(ints([0]), one, ints([[-1]]), ints([5, 6]), ints([count]), 16, 1)
        assert p.counts.tolist() == ([0, 1] if count < 0 else [left, 0])
    # free pages that are none have no slots
    p = fa.cache_plan(ints([0, 0]), ints([2, 1]), ints([[-1], [-1]]), ints([big, -4]), ints([2]), 16, 4)
    assert p.slots.tolist() == [-1] * 4 and p.counts.tolist() == [0, 0]


def test_plan_refuses_what_it_cannot_update(fa):
    k = ints([1, 2])
    with pytest.raises(fa.FlashAttentionError):
        p = fa.make_cache_plan(2, 4, DEV)
        fa.cache_plan(p.k_len, k, ints([[0], [1]]), ints([2, 3]), ints([2]), 16, out=p)
    with pytest.raises(ValueError):
        fa.cache_plan(k, ints([1]), ints([[0], [1]]), ints([2, 3]), ints([2]), 16, 4)
    with pytest.raises(ValueError):
        fa.cache_plan(k, k.long(), ints([[0], [1]]), ints([2, 3]), ints([2]), 16, 4)


@pytest.mark.parametrize("dtype,D,layout,heads", [(F16, 64, "hnd", 3), (BF16, 128, "nhd", 8), (F16, 256, "pool", 1), (BF16, 128, "hnd", 5)])
@pytest.mark.parametrize("T", [1, 7, 300])
def test_write(fa, dtype, D, layout, heads, T):
    cache = make_cache(fa, 30, heads, 16, D, dtype, layout)
    fused = torch.randn(T, 2 * heads + 1, D, dtype=dtype, device=DEV)
    k, v = fused[:, :heads], fused[:, heads:2 * heads]
    slots = torch.randperm(30 * 16, device=DEV)[:T].int()
    slots[::5] = torch.tensor([-1, 30 * 16, 2 ** 31 - 1, -2 ** 31], device=DEV, dtype=torch.int32).repeat(T)[:len(slots[::5])]
    want_k, want_v = cache.k.clone(), cache.v.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < 30 * 16:
            want_k[s // 16, :, s % 16], want_v[s // 16, :, s % 16] = k[t], v[t]
    fa.cache_write(k, v, cache, slots)
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)


def test_write_refusals(fa):
    cache = make_cache(fa, 2, 2, 16, 64, F16)
    rows = torch.zeros(3, 2, 64, dtype=F16, device=DEV)
    for bad in (rows.bfloat16(), rows[:, :1], rows[..., :32], rows.cpu()):
        with pytest.raises(ValueError):
            fa.cache_write(bad, bad, cache, ints([0, 1, 2]))
    with pytest.raises(ValueError):
        fa.cache_write(rows, rows, cache, ints([0, 1]))
    fa.cache_write(rows[:0], rows[:0], cache, ints([]))


def test_a_run_of_steps(fa):
    """Requests come with prompts, decode, drop drafted tokens, finish and give their pages to others: after every step
    attention equals that over each request's own dense keys.  Plan, write and attention on the GPU, nothing on the host in between."""
    torch.manual_seed(3)
    B, page, width, Hq, Hkv, D, dtype, prefix_len = 6, 16, 8, 8, 2, 128, BF16, 75
    n_pages = 5 + 30
    cache = make_cache(fa, n_pages, Hkv, page, D, dtype, "hnd")
    shared_k, shared_v = torch.randn(2, prefix_len, Hkv, D, dtype=dtype, device=DEV)
    fa.cache_write(shared_k, shared_v, cache, torch.arange(prefix_len, device=DEV, dtype=torch.int32))
    prefix = ints(list(range(5)))
    table, free = torch.full((B, width), -1, dtype=torch.int32, device=DEV), ints(list(range(5, n_pages)))
    plans = [fa.make_cache_plan(B, 128, DEV) for _ in range(2)]
    k_len, count = ints([0] * B), ints([30])
    dense = [[torch.empty(0, Hkv, D, dtype=dtype, device=DEV)] * 2 for _ in range(B)]
    steps = [[40, 1, 0, 0, 17, 0], [1, 1, 30, 0, 1, 0], [1, 5, 1, 16, 1, 0], [-41, 1, 1, 1, -3, 64], [33, -4, 1, 1, 1, 1], [1, 1, -32, 1, 1, 1],
             [0, 0, 100, 0, 0, 0], [1, 1, 1, 1, 1, 1]]
    for i, new in enumerate(steps):
        p = fa.cache_plan(k_len, ints(new), table, free, count, page, out=plans[i % 2])
        T = p.slots.numel()
        q, k, v = (torch.randn(T, h, D, dtype=dtype, device=DEV) for h in (Hq, Hkv, Hkv))
        fa.cache_write(k, v, cache, p.slots)
        out = fa.attention_shared_prefix(q, cache, p.q_start, p.k_len, table, prefix, prefix_len)
        k_len, count = p.k_len, p.counts[:1]
        assert p.counts[1].item() == 0
        at = 0
        for b, n in enumerate(new):
            held = dense[b][0].shape[0]
            dense[b] = [torch.cat([x[: held + min(n, 0)], y[at:at + max(n, 0)]]) for x, y in zip(dense[b], (k, v))]
            assert p.k_len[b].item() == held + n
            if n > 0:
                kk, vv = (torch.cat([s, x]).double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1) for s, x in zip((shared_k, shared_v), dense[b]))
                qq = q[at:at + n].double().transpose(0, 1)
                s = qq @ kk.transpose(1, 2) / D ** 0.5
                L = kk.shape[1]
                s.masked_fill_(torch.arange(L, device=DEV) > L - n + torch.arange(n, device=DEV)[:, None], -math.inf)
                w = s.softmax(-1)
                o, a = (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1)
                size = (qq.abs() @ kk.abs().transpose(1, 2)).amax() / D ** 0.5
                assert bool(((out[at:at + n].double() - o).abs() <= tolerance(dtype, o, a, size, D, L, vv)).all()), (i, b)
            at += max(n, 0)
        assert bool((out[at:] == 0).all())


def test_a_captured_run_of_steps(fa):
    """Two steps (the two sets of tables in turn) in one graph: plan, write, attention.  Replayed with other lengths each time it
    leaves what the same calls leave in a twin of the cache."""
    torch.manual_seed(5)
    B, page, width, Hq, Hkv, D, T = 5, 16, 8, 4, 2, 64, 24
    n_new, rows = [ints([0] * B) for _ in range(2)], [torch.randn(3, T, Hq, D, dtype=F16, device=DEV) for _ in range(2)]

    def state():
        cache = make_cache(fa, 40, Hkv, page, D, F16, seed=37)
        table, free = torch.full((B, width), -1, dtype=torch.int32, device=DEV), ints(list(range(4, 40)))
        plans = [fa.make_cache_plan(B, T, DEV) for _ in range(2)]
        plans[1].k_len.copy_(ints([0] * B))
        plans[1].counts.copy_(ints([36, 0]))
        outs = [torch.zeros(T, Hq, D, dtype=F16, device=DEV) for _ in range(2)]
        return cache, table, free, plans, outs

    prefix = ints([0, 1, 2, 3])

    def steps(cache, table, free, plans, outs):
        for i in range(2):
            held = plans[1 - i]
            p = fa.cache_plan(held.k_len, n_new[i], table, free, held.counts[:1], page, out=plans[i])
            q, k, v = rows[i]
            fa.cache_write(k[:, :Hkv], v[:, :Hkv], cache, p.slots)
            fa.attention_shared_prefix(q, cache, p.q_start, p.k_len, table, prefix, 60, out=outs[i])

    eager, captured = state(), state()
    steps(*eager)  # (adds nothing)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(*captured)
    for new in ([[3, 1, 0, 16, 2], [1, 1, 1, 1, 1]], [[1, -2, 20, 0, 1], [1, 4, 1, -17, 1]], [[-4, 1, 1, 17, 1], [20, 1, 1, 1, 1]], [[0] * 5, [1] * 5]):
        for i in range(2):
            n_new[i].copy_(ints(new[i]))
            rows[i].normal_()
        for o in eager[4] + captured[4]:
            o.zero_()
        graph.replay()
        steps(*eager)
        torch.cuda.synchronize()
        for a, b in zip(eager[3] + [eager[1:3]] + [eager[4]], captured[3] + [captured[1:3]] + [captured[4]]):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert torch.equal(eager[0].k, captured[0].k) and torch.equal(eager[0].v, captured[0].v)
        assert captured[3][1].counts[1].item() == 0 and captured[4][1].any()  # (the first step of the last replay adds no token)


def test_plan_and_write_on_another_stream_and_timed(fa):
    cache, side = make_cache(fa, 8, 2, 16, 64, F16, seed=38), torch.cuda.Stream()
    k, table, free = torch.randn(20, 2, 64, dtype=F16, device=DEV), torch.full((2, 4), -1, dtype=torch.int32, device=DEV), ints(list(range(8)))
    held, new, count = ints([0, 0]), ints([17, 3]), ints([8])
    torch.cuda.synchronize()
    plan, ms = fa.cache_plan(held, new, table, free, count, 16, 20, stream=side, timed=True)
    assert ms > 0
    assert fa.cache_write(k, k, cache, plan.slots, stream=side.cuda_stream, timed=True) > 0
    side.synchronize()
    at = plan.slots.long()
    assert torch.equal(cache.k[at // 16, :, at % 16], k) and torch.equal(cache.v[at // 16, :, at % 16], k) and plan.k_len.tolist() == [17, 3]
