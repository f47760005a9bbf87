// Index arithmetic of the paged K/V cache: which page a key lies in, where a cache row is in memory, which request a
// tile of query rows belongs to.  Plain functions of whole numbers for host and device: the kernels take every bound
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
constexpr int kMaxPlanRequests = 5120;  // three sums per request in a workgroup's LDS: 61 of the 64 KB a launch may ask for

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

// Slot of a key in page `page`: -1 where the page is none or the number passes 31 bits.
FA_HD int slot_of(int page, int row, int log2_page) {
    const int64_t s = ((int64_t)page << log2_page) + row;
    return page < 0 || s > 0x7fffffffLL ? -1 : (int)s;
}

// Rows of request b (its new tokens times the query heads that share a K/V head) in tiles of 2^log2_rows: tile x of the
// batch is tile x - first_row_tile(b) of the request with the largest first_row_tile(b) <= x.  The sums
// floor(rows before b / tile) + b leave every request room for its own tiles, whatever the lengths; tiles past a
// request's last row are empty.
FA_HD int first_row_tile(int q_start_b, int b, int group, int log2_rows) {
    return (int)(((int64_t)q_start_b * group) >> log2_rows) + b;
}
FA_HD int row_tiles_bound(int tokens, int requests, int group, int log2_rows) {
    return (int)(((int64_t)tokens * group) >> log2_rows) + requests;
}

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
