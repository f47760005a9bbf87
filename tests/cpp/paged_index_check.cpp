// The index arithmetic of the paged-cache kernels (csrc/fa_paged_index.hpp), run on the CPU: every bound the kernels
// rely on, over the values that could break it.  Exit status 0 and "ok" when all hold.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../flash-attention_amd/csrc/fa_paged_index.hpp"

static void need(bool ok, const char* what, long a = 0, long b = 0, long c = 0) {
    if (ok) return;
    std::printf("FAILED: %s (%ld, %ld, %ld)\n", what, a, b, c);
    std::exit(1);
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
    // workgroups of a launch: never more than the grid made from the bound, whatever the lengths
    std::srand(1);
    for (int trial = 0; trial < 20000; ++trial) {
        const int B = 1 + std::rand() % 40, heads = 1 + std::rand() % 9, g = 1 + std::rand() % 20, slots = std::rand() % 2 ? 512 : 256;
        const int prefix = std::rand() % 3 ? std::rand() % 3000 : std::rand() % 3, least = 1 + std::rand() % 4;
        const int most_prefix = 1 + std::rand() % 64, most_own = 1 + std::rand() % 64;
        std::vector<int> rows(B), own(B);
        long stacked = 0, total = 0;
        float work = 0;
        for (int b = 0; b < B; ++b) {
            rows[b] = g * (std::rand() % 3 ? std::rand() % 4 : std::rand() % 300);
            own[b] = std::rand() % 4 ? std::rand() % 40 : std::rand() % 5000;
            total += rows[b];
            if (rows[b] < 128) stacked += rows[b];
            work += (float)row_tiles(rows[b]) * (own[b] + (rows[b] < 128 ? 0 : prefix));
        }
        work += (float)row_tiles(stacked) * prefix;
        const int steps = steps_for(work, heads, slots, least);
        need(steps >= least, "steps", trial);
        long items = prefix > 0 ? (long)heads * row_tiles(stacked) * parts_for(prefix, steps, most_prefix) : 0;
        for (int b = 0; b < B; ++b)
            items += (long)heads * row_tiles(rows[b]) *
                     (rows[b] < 128 ? parts_for(own[b], steps, most_own) : parts_for(prefix + own[b], steps, most_prefix + most_own));
        const long bound = blocks_bound(prefix > 0 ? row_tiles(total) : 0, request_tiles_bound(total, B), heads, slots);
        need(items <= bound, "blocks", trial, items, bound);
    }
    std::printf("ok\n");
    return 0;
}
