// The index arithmetic of the paged-cache kernels (csrc/fa_paged_index.hpp), run on the CPU: every bound the kernels
// rely on, over the values that could break it.  Exit status 0 and "ok" when all hold.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../flash-attention_amd/csrc/fa_paged_index.hpp"

static void need(bool ok, const char* what, long a = 0, long b = 0, long c = 0) {
    if (ok) return;
    std::printf("FAILED: %s (%ld, %ld, %ld)\n", what, a, b, c);
    std::exit(1);
}

// tiles / steps, rounded, from 1 to `most`: what the kernels do by reciprocals (div_by, checked below)
static int parts_for(int tiles, int steps, int most) {
    return std::max(1L, std::min(((long)tiles + steps / 2) / steps, (long)most));
}

int main() {
    using namespace fa;
    // table entries: inside [0, n_pages) or no page at all
    const int odd[] = {INT_MIN, -2, -1, 0, 1, 6, 7, 8, INT_MAX};
    for (int page : odd) need(page_ok(page, 7) == (page >= 0 && page < 7), "page_ok", page);
    // slots: 31 bits or -1
    for (int page : odd)
        for (int log2p = kMinLog2Page; log2p <= kMaxLog2Page; ++log2p)
            for (int row : {0, (1 << log2p) - 1}) {
                const long want = (long)page * (1L << log2p) + row;
                need(slot_of(page, row, log2p) == (page < 0 || want > INT_MAX ? -1 : (int)want), "slot_of", page, log2p, row);
            }
    // offsets past 32 bits
    const CacheStrides s{(int64_t)65536 * 8 * 256, 256, 2048};
    need(cache_offset(s, 100000, 7, 65535) == 100000LL * 65536 * 8 * 256 + 7 * 256 + 65535LL * 2048, "cache_offset");
    // a request's step, at the ends of every range
    for (int log2p : {4, 6, 16})
        for (int width : {1, 3, 16384})
            for (int k : {INT_MIN, -1, 0, 1, 15, 16, 17, 65536, INT_MAX})
                for (int n : {INT_MIN, -65537, -16, -1, 0, 1, 16, 65536, INT_MAX}) {
                    if (((int64_t)width << log2p) > (1 << 30)) continue;
                    const PlanRow r = plan_row(k, n, width, log2p);
                    const int64_t room = (int64_t)width << log2p;
                    need(r.held >= 0 && r.held <= room && r.after >= 0 && r.after <= room, "plan_row lengths", k, n, width);
                    need(r.have >= 0 && r.have <= width && r.want >= 0 && r.want <= width, "plan_row pages", k, n, width);
                    need(r.wide == ((int64_t)r.held + n > room), "plan_row wide", k, n, width);
                    if (r.wide) need(r.needed() == 0 && r.released() == 0, "a step that is too wide takes nothing", k, n, width);
                    need((int64_t)r.have << log2p >= r.held && (r.have == 0 || (int64_t)(r.have - 1) << log2p < r.held), "pages of held", k, n, width);
                }
    // owners in a running sum, empty ones among them
    const std::vector<int> len = {0, 3, 0, 0, 1, 5, 0, 2, 0};
    std::vector<int> sum = {0};
    for (int l : len) sum.push_back(sum.back() + l);
    for (int x = 0; x < sum.back(); ++x) {
        const int b = owner_of(sum, (int)len.size(), x);
        need(sum[b] <= x && x < sum[b + 1], "owner_of", x, b);
    }
    // division by a reciprocal that is off by 1 ulp either way
    const int tops[] = {0, 1, 2, 3, 7, 127, 128, 1000, 65535, 1 << 20, (1 << 24) + 1, (1 << 25) - 1, 1 << 30, INT_MAX - 1, INT_MAX};
    for (int bb = 1; bb < 70000; bb += bb < 300 ? 1 : 977)
        for (int a : tops)
            for (int near : {-1, 0, 1}) {
                const long x = (long)a / bb * bb + near;  // around the multiples, where a quotient goes wrong
                for (long n : {(long)a, x}) {
                    if (n < 0 || n > INT_MAX) continue;
                    const float r = 1.0f / bb;
                    for (float q : {r, std::nextafterf(r, 0.0f), std::nextafterf(r, 2.0f)})
                        need(div_by((int)n, bb, q) == n / bb, "div_by", n, bb, div_by((int)n, bb, q));
                }
            }
    for (int g = 2; g <= 128; ++g)
        for (int i = 0; i < 4000; ++i) {
            const unsigned top = (1u << 25) - 1, R = i < 2000 ? (unsigned)i * 16777u % (top + 1) / g * g + (i & 1 ? g - 1 : 0) : top - (i - 2000);
            if ((uint64_t)R * g >= (uint64_t)1 << 32) continue;
            need((unsigned)(((uint64_t)R * group_reciprocal(g)) >> 32) == R / g, "group_reciprocal", R, g);
        }
    // workgroups of a launch: never more than the grid made from the bound, whatever the lengths
    std::srand(1);
    for (int trial = 0; trial < 20000; ++trial) {
        const int B = 1 + std::rand() % 40, heads = 1 + std::rand() % 9, g = 1 + std::rand() % 20, slots = std::rand() % 2 ? 512 : 256;
        const int prefix = std::rand() % 3 ? std::rand() % 3000 : std::rand() % 3, least = 1 + std::rand() % 4;
        const int most_prefix = 1 + std::rand() % 64, most_own = 1 + std::rand() % 64;
        std::vector<int> rows(B), own(B);
        long stacked = 0, total = 0;
        float few = 0, many = 0;
        const int few_tile = std::rand() % 2 ? 16 : 32, few_rows = 2 * few_tile;
        auto tiles = [&](long r) { return r <= few_rows ? (int)((r + few_tile - 1) / few_tile) : row_tiles(r); };
        for (int b = 0; b < B; ++b) {
            rows[b] = g * (std::rand() % 3 ? std::rand() % 4 : std::rand() % 300);
            own[b] = std::rand() % 4 ? std::rand() % 40 : std::rand() % 5000;
            total += rows[b];
            if (rows[b] < 128) stacked += rows[b];
            (rows[b] <= few_rows ? few : many) += (float)tiles(rows[b]) * (own[b] + (rows[b] < 128 ? 0 : prefix));
        }
        (stacked <= few_rows ? few : many) += (float)tiles(stacked) * prefix;
        const int steps_few = steps_for(few + 2 * many, heads, slots, least), half = (steps_few + 1) / 2, steps_many = half < least ? least : half;
        need(steps_few >= least, "steps", trial);
        // the stacked rows' ranges may be made as many as the slots
        const int units = heads * tiles(stacked);
        int p_parts = parts_for(prefix, stacked <= few_rows ? steps_few : steps_many, most_prefix);
        if (units > 0 && units * p_parts < slots) p_parts = std::max(p_parts, std::min(slots / units, most_prefix));
        long items = prefix > 0 ? (long)units * p_parts : 0;
        for (int b = 0; b < B; ++b)
            items += (long)heads * tiles(rows[b]) *
                     (rows[b] < 128 ? parts_for(own[b], rows[b] <= few_rows ? steps_few : steps_many, most_own)
                                    : parts_for(prefix + own[b], steps_many, most_prefix + most_own));
        const long bound = blocks_bound(prefix > 0 ? row_tiles(total) + 1 : 0, request_tiles_bound(total, B) + B, heads, slots);
        need(items <= bound, "blocks", trial, items, bound);
    }
    std::printf("ok\n");
    return 0;
}
