// Index arithmetic of the paged K/V cache: which page a key lies in, where a cache row is in memory, how many workgroups a
// launch can need.  Plain functions of whole numbers for host and device: the kernels take every bound
// from here, and the CPU tests run the same code (tests/cpp/paged_index_check.cpp).
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
// Which 16-key groups lie on no page (bit i: group from + i), of the run of 64 that the transfers have reached and of the one
// before it: the computation is less than a run behind them.
struct PagelessGroups {
    uint64_t before = 0, run = 0;
    int from = 0;
    FA_HD void next_run(int first, uint64_t pageless) {
        before = run;
        run = pageless;
        from = first;
    }
    FA_HD bool any() const { return (before | run) != 0; }
    // of the `count` groups from `group` on (count divides 64 and group)
    FA_HD unsigned of(int group, int count) const { return (unsigned)((group >= from ? run : before) >> (group & 63)) & ((1u << count) - 1); }
};

// Slot of a key in page `page`: -1 where the page is none or the number passes 31 bits.
FA_HD int slot_of(int page, int row, int log2_page) {
    const int64_t s = ((int64_t)page << log2_page) + row;
    return page < 0 || s > 0x7fffffffLL ? -1 : (int)s;
}

// How a launch of shared-prefix attention is divided.  Row tiles of 128 rows (few rows: less) walk `tiles` key tiles each, in
// tiles / steps ranges, rounded, of about `steps_for` key tiles: all key tiles of the launch (`work`, per K/V head) over the
// workgroups that the chip holds (`slots`).  With x = tiles / steps a row tile has max(1, floor(x + 1/2)) ranges at most,
// i.e. fewer than x beyond the first, and all x together are at most `slots`; another `slots` and the half are room for the
// rounding of the sum.  So blocks_bound holds for any lengths.
constexpr int kRowTile = 128;
FA_HD int row_tiles(int64_t rows) { return (int)((rows + kRowTile - 1) / kRowTile); }
FA_HD int steps_for(float work, int heads, int slots, int least) {
    const float per = work * (float)heads / (float)slots;
    const int n = (int)(per < 1e9f ? per : 1e9f) + 1;
    return n < least ? least : n;
}
// Row tiles of a batch of `requests` with `rows` rows in all, and its workgroups.
FA_HD int64_t request_tiles_bound(int64_t rows, int requests) { return rows / kRowTile + requests; }
FA_HD int64_t blocks_bound(int64_t prefix_row_tiles, int64_t request_row_tiles, int heads, int slots) {
    return heads * (prefix_row_tiles + request_row_tiles) + 5 * (int64_t)slots / 2 + 1;
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
