// Index arithmetic of the paged K/V cache: which page a key lies in, where a cache row is in memory, how a launch is divided
// into workgroups and how many it can need.  Plain functions of whole numbers for host and device: the kernels take every bound
// from here, and the CPU tests run the same code (tests/cpp/paged_*_check.cpp).
//
// A cache is [n_pages][Hkv][page_size][D] with any strides of the first three axes (so token-major pages are a
// permuted view); a page holds 2^log2_page keys, 16 at least.  An entry of a block table outside [0, n_pages) names no
// page: its keys take no part in attention, its rows are not written.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define FA_HD __host__ __device__ __forceinline__
#else
#define FA_HD inline
#endif

namespace fa {

constexpr int kMinLog2Page = 4, kMaxLog2Page = 16;
constexpr int key_tile(int D) { return D == 64 ? 64 : 32; }  // keys of an attention tile
constexpr int kMaxPlanRequests = 5120;  // four numbers per request in a workgroup's LDS, five requests per thread

// Element strides of one cache tensor.
struct CacheStrides {
    int64_t page, head, row;
};

FA_HD bool page_ok(int page, int n_pages) { return (unsigned)page < (unsigned)n_pages; }
FA_HD int64_t cache_offset(const CacheStrides& s, int page, int head, int row) {
    return (int64_t)page * s.page + (int64_t)head * s.head + (int64_t)row * s.row;
}
FA_HD int clamp_int(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
FA_HD int pages_for(int64_t keys, int log2_page) { return (int)((keys + (1 << log2_page) - 1) >> log2_page); }

// The page that holds keys key .. key + 15 of a walk over `keys` keys (key a multiple of 16), -1 where the table's entry names
// none.  Keys behind the last one are hidden by the rows' limits whatever is read in their place: they are read from page 0, and
// what the table holds there, or whether it goes on, does not matter.  (`keys` is at most what the table names.)
FA_HD int page_of_keys(const int* table, int key, int keys, int log2_page, int n_pages) {
    if (key >= keys) return 0;
    const int page = table[key >> log2_page];
    return page_ok(page, n_pages) ? page : -1;
}
// The kernels read a table 64 groups of 16 keys (a run) at a time, and keep which of a run's groups lie on no page (bit i: group i of
// the run) for the run that the transfers have reached and for the one before it: the computation is less than a run behind them.
// Those of the `per` groups (a divisor of 64) of tile `tile`, looked at when tile + ahead is the last tile transferred.
FA_HD unsigned pageless_groups(uint64_t before, uint64_t run, int tile, int ahead, int per) {
    const int group = tile * per, reached = ((tile + ahead) * per) & ~63;
    return (unsigned)((group >= reached ? run : before) >> (group & 63)) & ((1u << per) - 1);
}

// Slot of a key in page `page`: -1 where the page is none or the number passes 31 bits.
FA_HD int slot_of(int page, int row, int log2_page) {
    const int64_t s = ((int64_t)page << log2_page) + row;
    return page < 0 || s > 0x7fffffffLL ? -1 : (int)s;
}

// a / b for 0 <= a < 2^31, 1 <= b, from a reciprocal r of b that is good to 1 ulp (v_rcp_f32): the first quotient is off by
// 2^-22 of itself and one at most, the second by one.
FA_HD int div_by(int a, int b, float r) {
    const float f = (float)a * r;
    int q = f >= 2147483520.0f ? 2147483520 : (int)f;
    unsigned m = (unsigned)a - (unsigned)q * (unsigned)b;
    q += (int)((float)(int)m * r);
    const int e = (int)((unsigned)a - (unsigned)q * (unsigned)b);
    return e < 0 ? q - 1 : e >= b ? q + 1 : q;
}
// a / b for 0 <= a < 2^31, 1 <= b, by a reciprocal that rcp(b) gives to 1 ulp.
template <typename Rcp>
FA_HD int quick_div(int a, int b, Rcp rcp) { return div_by(a, b, rcp(b)); }

// How a launch of shared-prefix attention is divided into workgroups, from the requests' lengths.
//   A request with fewer than 128 rows (new tokens x g) is short: its rows are stacked up with those of the other short
// requests against the prefix (items of kind P: one K/V head, a row tile of the stack, a range of the prefix) and alone against
// its own keys (O: one head, a row tile of the request, a range of its keys).  A longer request fills row tiles of its own,
// which walk prefix and own keys in one go (J: one head, 128 of its rows, a range of both): nothing is gained by stacking.
//   Ranges take about the same time each, up to half more or less: the launch's key tiles over the workgroups that the chip
// holds, a tile of many rows counted as kManyCost tiles of few (1 and 3 measured no better), `least` key tiles (256 keys) at
// least: a workgroup's start and end cost 13 - 20 thousand cycles, as much as some 500 keys, and each part is written, read and
// joined again (128: 32 requests behind 8 192 keys 28.7 us, 256: 28.1).
constexpr int kRowTile = 128, kManyCost = 2, kMaxParts = 64;
struct DivisionRule {
    int heads, slots, two_per_unit;         // K/V heads; workgroups that the chip holds at a time; whether two share a compute unit
    int few_rows, few_tile, log2_few_tile;  // up to this many rows take the form for few, so many at a time
    int max_prefix_parts, max_own_parts;    // parts of one row's sum
    int least;                              // key tiles of a range
};
FA_HD int row_tiles(int64_t rows) { return (int)((rows + kRowTile - 1) / kRowTile); }
FA_HD int steps_for(float work, int heads, int slots, int least) {
    const float per = work * (float)heads / (float)slots;
    const int n = (int)(per < 1e9f ? per : 1e9f) + 1;
    return n < least ? least : n;
}
// Up to few_rows rows are taken few_tile at a time (each tile reads the keys again, from the L2: cheaper than the form for
// many rows, in which one wave of four would compute), more 128 at a time.
FA_HD int tile_rows(const DivisionRule& d, int rows) { return rows <= d.few_rows ? d.few_tile : kRowTile; }
FA_HD int tiles_of(const DivisionRule& d, int rows) {
    return rows <= d.few_rows ? (rows + d.few_tile - 1) >> d.log2_few_tile : row_tiles(rows);
}
// Ranges of a row tile's `tiles` key tiles: tiles / steps, rounded, from 1 to `most`.
template <typename Rcp>
FA_HD int range_count(int tiles, int steps, int most, Rcp rcp) {
    const int n = quick_div(tiles + (steps >> 1), steps, rcp);
    return n < 1 || most < 1 ? 1 : n < most ? n : most;
}

// Key tiles of all row tiles of a launch, per K/V head, in either form.
struct LaunchWork {
    float few = 0.0f, many = 0.0f;
    FA_HD void add_request(const DivisionRule& d, int rows, int own_tiles, int prefix_tiles) {
        if (rows >= kRowTile)
            many += (float)row_tiles(rows) * (float)(own_tiles + prefix_tiles);
        else if (rows > d.few_rows)
            many += (float)own_tiles;
        else
            few += (float)tiles_of(d, rows) * (float)own_tiles;
    }
};
struct SharedPlan {
    int stacked;       // rows of the short requests, per K/V head
    int prefix_tiles;  // key tiles of the prefix
    int prefix_parts;  // ranges of the prefix that P items walk
    int p_items;
    int steps_few, steps_many;  // key tiles of a range
};
// `w`: the requests' own work (LaunchWork::add_request of each).
template <typename Rcp>
FA_HD SharedPlan shared_plan_of(const DivisionRule& d, LaunchWork w, int stacked, int prefix_tiles, Rcp rcp) {
    SharedPlan s;
    s.stacked = stacked, s.prefix_tiles = prefix_tiles;
    const int p_tiles = tiles_of(d, stacked);
    const bool p_few = stacked <= d.few_rows;
    (p_few ? w.few : w.many) += (float)p_tiles * (float)prefix_tiles;
    s.steps_few = steps_for(w.few + (float)kManyCost * w.many, d.heads, d.slots, d.least);
    const int half_steps = (s.steps_few + kManyCost - 1) / kManyCost;
    s.steps_many = half_steps < d.least ? d.least : half_steps;
    s.prefix_parts = 0;
    if (prefix_tiles > 0 && p_tiles > 0) {
        s.prefix_parts = range_count(prefix_tiles, p_few ? s.steps_few : s.steps_many, d.max_prefix_parts, rcp);
        // Two workgroups to a unit: with more P items than units some units hold two, which take nearly twice as long, and the
        // requests' own items, which wait for memory, find no unit to share with one that computes.
        const int units = p_tiles * d.heads, half = d.slots >> 1;
        if (d.two_per_unit && units * s.prefix_parts > half && units * s.prefix_parts <= d.slots) {
            const int n = quick_div(half, units, rcp);
            s.prefix_parts = n < 1 ? 1 : n;
        }
    }
    s.p_items = p_tiles * s.prefix_parts * d.heads;
    return s;
}
// Ranges of a request's keys, and its items.
template <typename Rcp>
FA_HD int request_parts(const DivisionRule& d, const SharedPlan& s, int rows, int own_tiles, Rcp rcp) {
    return rows >= kRowTile ? range_count(s.prefix_tiles + own_tiles, s.steps_many, d.max_prefix_parts + d.max_own_parts, rcp)
                            : range_count(own_tiles, rows <= d.few_rows ? s.steps_few : s.steps_many, d.max_own_parts, rcp);
}
template <typename Rcp>
FA_HD int request_items(const DivisionRule& d, const SharedPlan& s, int rows, int own_tiles, Rcp rcp) {
    return tiles_of(d, rows) * request_parts(d, s, rows, own_tiles, rcp) * d.heads;
}
// Item x of units x tiles: eight units at a time, tile by tile, so that the row tiles that read the same keys (one unit: a
// K/V head and a range) follow each other on one XCD (workgroup ids congruent mod 8 share one and its L2).
template <typename Rcp>
FA_HD void unit_and_tile(int x, int units, int tiles, int& unit, int& tile, Rcp rcp) {
    const int full = units >> 3, per = 8 * tiles, q = quick_div(x, per, rcp);
    const int grp = q < full ? q : full, r = x - grp * per, w = grp < full ? 8 : units & 7;
    tile = quick_div(r, w, rcp);
    unit = grp * 8 + (r - tile * w);
}
// Part `part` of `parts` of the key tiles first .. last: where it begins, and how many it has.
template <typename Rcp>
FA_HD void range_of(int first, int last, int part, int parts, int& u0, int& n_tiles, Rcp rcp) {
    const int each = quick_div(last - first, parts, rcp), over = last - first - each * parts;
    u0 = first + part * each + (part < over ? part : over);
    n_tiles = each + (part < over ? 1 : 0);
}

// What the host, which does not know the lengths, decides of a launch: the bounds that the workspace and the grid are made for.
//   Workgroups: with x = tiles / steps a row tile has max(1, floor(x + 1/2)) ranges at most, i.e. fewer than x beyond the first,
// and all x together are at most `slots`; another `slots` and the half are room for the rounding of the sum.  So blocks_bound
// holds for any lengths.
FA_HD int64_t request_tiles_bound(int64_t rows, int requests) { return rows / kRowTile + requests; }  // row tiles of a batch
FA_HD int64_t blocks_bound(int64_t prefix_row_tiles, int64_t request_row_tiles, int heads, int slots) {
    return heads * (prefix_row_tiles + request_row_tiles) + 5 * (int64_t)slots / 2 + 1;
}
constexpr int64_t part_bytes(int D) { return (D + 2) * (int64_t)sizeof(float); }  // of one row: O, the maximum and the sum
struct LaunchBounds {
    DivisionRule rule;
    int64_t blocks;  // items of any lengths
    int parts_kept;  // parts of every row that the workspace holds
    int parts() const { return rule.max_prefix_parts + rule.max_own_parts; }
};
// Two workgroups share a compute unit at D = 64 and 128 (64 KiB of LDS, at most 256 registers), one has it at D = 256.
inline LaunchBounds launch_bounds_of(int T, int B, int Hkv, int g, int D, int prefix_len, int max_k_len, int cus) {
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    auto within = [](int64_t x, int64_t lo, int64_t hi) { return (int)(x < lo ? lo : x > hi ? hi : x); };
    const int64_t rows = (int64_t)T * g;
    LaunchBounds b;
    DivisionRule& d = b.rule;
    d.heads = Hkv, d.slots = cus * (D == 256 ? 1 : 2), d.two_per_unit = D != 256;
    d.log2_few_tile = D == 64 ? 5 : 4, d.few_tile = 1 << d.log2_few_tile, d.few_rows = 2 * d.few_tile;
    d.least = 256 / key_tile(D);
    // enough parts to fill the chip twice over from the prefix alone, or from a few requests' own keys.  (A part has about 256 keys
    // at least, so 128 keys a part bound their number, a part that is up to half shorter included.)
    d.max_prefix_parts = prefix_len > 0 ? within(up(2 * d.slots, up(rows, 128) * Hkv), 1, within(up(prefix_len, 128), 1, kMaxParts)) : 0;
    d.max_own_parts = within(up(2 * d.slots, (int64_t)B * Hkv), 4, kMaxParts);
    d.max_own_parts = within(up(max_k_len, 128), 1, d.max_own_parts);
    // Every part is room for all rows.  With many rows few requests can want many parts (the launch's work is divided over the
    // workgroups, and the row tiles alone fill them several times over), so 1 GiB bounds them, one of own keys at least; only a
    // request of few rows and a long context beside very many other rows would take more.  A row of one part goes to the output
    // at once, so a launch whose rows all have one needs no room for it: it is left out where it would pass the bound.
    const int64_t per_part = rows * Hkv * part_bytes(D), most_bytes = 1 << 30;
    const int held = within(most_bytes / per_part - d.max_prefix_parts, 1, kMaxParts);
    if (d.max_own_parts > held) d.max_own_parts = held;
    b.parts_kept = b.parts() == 1 && per_part > most_bytes ? 0 : b.parts();
    // (a batch or a request of few rows has two tiles at most, where 128 rows would be one)
    const int64_t p_tiles = prefix_len > 0 ? row_tiles(rows) + 1 : 0, r_tiles = request_tiles_bound(rows, B) + B;
    const int64_t most = Hkv * (p_tiles * d.max_prefix_parts + r_tiles * b.parts()), sum = blocks_bound(p_tiles, r_tiles, Hkv, d.slots);
    b.blocks = most < sum ? most : sum;
    return b;
}

// 2^32 / g rounded up: R / g is the high word of R times this for R g < 2^32 (g = 1 apart, which needs none).
FA_HD unsigned group_reciprocal(int g) { return (unsigned)((((uint64_t)1 << 32) + g - 1) / g); }

// One request's step, from its lengths alone.  keys held (clamped to what a table row names), keys after the step,
// pages before and after; `wide`: the step asks for more than the row of the table can name.
struct PlanRow {
    int held, after, have, want;
    bool wide;
    FA_HD int released() const { return have > want ? have - want : 0; }
    FA_HD int needed() const { return want > have ? want - have : 0; }
};
FA_HD PlanRow plan_row(int k_len, int n_new, int width, int log2_page) {
    PlanRow r;
    const int64_t room = (int64_t)width << log2_page;
    r.held = k_len < 0 ? 0 : (int64_t)k_len > room ? (int)room : k_len;
    int64_t after = (int64_t)r.held + n_new;
    r.wide = after > room;
    if (after < 0) after = 0;
    if (r.wide) after = r.held;
    r.after = (int)after;
    r.have = pages_for(r.held, log2_page);
    r.want = pages_for(r.after, log2_page);
    return r;
}

// Index of the last entry <= x of a[0 .. n) (ascending, a[0] <= x): the request that owns position x of a running sum.
template <typename A>
FA_HD int owner_of(const A& a, int n, int x) {
    int lo = 0, hi = n;  // a[lo] <= x, a[hi] > x
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

}  // namespace fa
