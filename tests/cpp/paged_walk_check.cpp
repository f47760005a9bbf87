// How the attention kernels walk a block table (csrc/fa_paged_index.hpp), run on the CPU: the page of each group of 16 keys, and
// the account of groups on no page, at the distance at which the kernels' transfers run ahead of the computation.
#include <algorithm>
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
    const int n_pages = 1000;
    // every key that counts: its table entry; behind the last key: page 0, whatever the table holds there
    for (int log2p : {4, 5, 6, 8})
        for (int keys = 0; keys < 300; ++keys)
            for (int behind : {-1, n_pages, INT_MIN, INT_MAX, 7}) {
                std::vector<int> table;
                for (int i = 0; i < pages_for(keys, log2p); ++i) table.push_back(i % 5 == 3 ? -1 - i : 10 + i);
                table.resize(table.size() + 40, behind);
                for (int key = 0; key < keys + 128; key += 16) {
                    const int e = table[key >> log2p], want = key >= keys ? 0 : e < 0 ? -1 : e;
                    need(page_of_keys(table.data(), key, keys, log2p, n_pages) == want, "page_of_keys", key, keys, log2p);
                }
            }
    const int edge[] = {0, n_pages - 1, n_pages, -1, INT_MAX};
    for (int i = 0; i < 5; ++i) need(page_of_keys(edge, 16 * i, 80, 4, n_pages) == (i < 2 ? edge[i] : -1), "entries at the ends", i);

    // a walk: tile t + 3 is transferred before tile t is computed and tile t + 1 is looked at
    std::srand(2);
    for (int trial = 0; trial < 3000; ++trial) {
        const int per = trial % 2 ? 2 : 4, tiles = 1 + std::rand() % 200, groups = tiles * per;
        const int keys = 16 * groups - std::rand() % (16 * per);  // the last tile is cut anywhere
        std::vector<int> table(groups, -1);                        // nothing behind the last page
        for (int i = 0; i < pages_for(keys, 4); ++i) table[i] = i;
        const int holes = trial % 3 ? std::rand() % 4 : 0;
        for (int i = 0; i < holes; ++i) table[std::rand() % pages_for(keys, 4)] = -1;
        auto pageless_at = [&](int g) { return g < groups && page_of_keys(table.data(), 16 * g, keys, 4, n_pages) < 0; };
        uint64_t before = 0, run = 0;
        auto transfer = [&](int t) {
            if (t * per % 64 != 0) return;
            before = run, run = 0;
            for (int i = 0; i < 64; ++i) run |= (uint64_t)pageless_at(t * per + i) << i;
        };
        auto look = [&](int t) {
            unsigned want = 0;
            for (int i = 0; i < per; ++i) want |= (unsigned)pageless_at(t * per + i) << i;
            need(pageless_groups(before, run, t, 2, per) == want, "groups of a tile", trial, t, want);
            if (holes == 0) need((before | run) == 0, "a prefix' or a request's end is no missing page", trial, t, keys);
            bool near = false;
            for (int g = std::max(0, t * per - 192); g < t * per + 192; ++g) near = near || pageless_at(g);
            if (!near) need((before | run) == 0, "a missing page far away", trial, t);
        };
        for (int t = 0; t < 3 && t < tiles; ++t) transfer(t);
        look(0);
        for (int t = 0; t < tiles; ++t) {
            transfer(t + 3);
            if (t + 1 < tiles) look(t + 1);
        }
    }
    std::printf("ok\n");
    return 0;
}
