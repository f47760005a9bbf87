// How a launch of shared-prefix attention is divided (csrc/fa_paged_index.hpp), run on the CPU with the functions that the host
// and the kernels call: the grid holds every item whatever the lengths, no row has more parts than the workspace, and the items
// cover every row tile's keys once.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include <vector>

#include "../../flash-attention_amd/csrc/fa_paged_index.hpp"

static void need(bool ok, const char* what, long a = 0, long b = 0, long c = 0) {
    if (ok) return;
    std::printf("FAILED: %s (%ld, %ld, %ld)\n", what, a, b, c);
    std::exit(1);
}
// a reciprocal that is off by up to 1 ulp either way, as the hardware's may be
struct Rcp {
    int off;
    float operator()(int b) const {
        const float r = 1.0f / b;
        return off < 0 ? std::nextafterf(r, 0.0f) : off > 0 ? std::nextafterf(r, 2.0f) : r;
    }
};
static int any_of(std::initializer_list<int> v) { return v.begin()[std::rand() % v.size()]; }
static int about(int top) { return (int)std::exp(std::log(top + 1.0) * std::rand() / RAND_MAX); }  // 1 .. top, small ones as often as large

int main() {
    using namespace fa;
    std::srand(3);
    long walked = 0;
    for (int trial = 0; trial < 60000; ++trial) {
        const int D = any_of({64, 128, 256}), TK = key_tile(D), B = trial % 50 ? about(60) : about(4000), Hkv = any_of({1, 2, 3, 8, 100}), g = any_of({1, 2, 4, 7, 16, 128});
        const int prefix_len = any_of({0, 1, 31, 32, 33, 1000, about(100000), about(1 << 30)}), cus = any_of({256, 256, 304, 64});
        const int longest = any_of({1, 100, 3000, about(1 << 20), about(1 << 30)}), few_tokens = any_of({1, 1, 5, 400});
        std::vector<int> tokens(B), keys(B);
        long T = 0;
        for (int b = 0; b < B; ++b) {
            tokens[b] = std::rand() % 8 ? std::rand() % (few_tokens + 1) : std::rand() % 2000 / (1 + B / 40);
            keys[b] = std::rand() % 2 ? about(longest) : std::rand() % 300;
            T += tokens[b];
        }
        T += std::rand() % 3 * (std::rand() % 500);  // rows of no request
        if (T == 0 || T * Hkv * g > 0x7fffffffL / 64) continue;
        // the host's bound on the requests' keys may be true, or far too low or high
        const LaunchBounds bounds = launch_bounds_of((int)T, B, Hkv, g, D, prefix_len, any_of({longest, 0, 1 << 30}), cus);
        const DivisionRule& d = bounds.rule;
        const Rcp rcp{std::rand() % 3 - 1};
        need(d.max_prefix_parts <= kMaxParts && d.max_own_parts <= kMaxParts && (d.max_prefix_parts > 0) == (prefix_len > 0) && d.max_own_parts > 0, "parts", trial);
        const int64_t held = (int64_t)bounds.parts_kept * T * Hkv * g * part_bytes(D);
        need(held <= 1 << 30 || (bounds.parts_kept == 2 && d.max_prefix_parts == 1), "bytes of the parts", trial, held, bounds.parts_kept);
        need(bounds.parts_kept == bounds.parts() || (bounds.parts_kept == 0 && bounds.parts() == 1), "parts that are written have room", trial);
        // the kernels' division
        const int prefix_tiles = (prefix_len + TK - 1) / TK;
        auto own_tiles = [&](int b) { return (keys[b] + TK - 1) / TK; };
        LaunchWork work;
        int stacked = 0;
        for (int b = 0; b < B; ++b) {
            if (tokens[b] * g < kRowTile) stacked += tokens[b];
            work.add_request(d, tokens[b] * g, own_tiles(b), prefix_tiles);
        }
        const SharedPlan s = shared_plan_of(d, work, stacked * g, prefix_tiles, rcp);
        need(s.prefix_parts <= d.max_prefix_parts && s.steps_few >= d.least && s.steps_many >= d.least, "prefix", trial, s.prefix_parts, s.steps_many);
        long items = s.p_items;
        for (int b = 0; b < B; ++b) {
            const int rows = tokens[b] * g, parts = request_parts(d, s, rows, own_tiles(b), rcp);
            need(parts >= 1 && (rows >= kRowTile ? parts <= bounds.parts() : parts <= d.max_own_parts), "parts of a row", trial, b, parts);
            items += request_items(d, s, rows, own_tiles(b), rcp);
        }
        need(items <= bounds.blocks && bounds.blocks <= 0x7fffffffL, "the grid holds every item", trial, items, bounds.blocks);
        if (items > 30000 || trial % 8) continue;
        // every item, as the kernel finds it from its number: each row tile of each head, its keys once, in order of its parts
        auto walk = [&](int first_item, int tiles, int parts, int rows, int first, int last) {
            std::vector<int> seen(Hkv * parts * tiles);
            need(tiles == (rows + tile_rows(d, rows) - 1) / tile_rows(d, rows), "row tiles", trial, tiles, rows);
            for (int x = 0; x < Hkv * parts * tiles; ++x) {
                int unit, tile;
                unit_and_tile(x, Hkv * parts, tiles, unit, tile, rcp);
                need(unit >= 0 && unit < Hkv * parts && tile >= 0 && tile < tiles, "unit and tile", trial, unit, tile);
                const int head = quick_div(unit, parts, rcp);
                need(head >= 0 && head < Hkv && unit - head * parts >= 0 && unit - head * parts < parts, "head and part", trial, head);
                need(!seen[unit * tiles + tile]++, "an item twice", trial, first_item + x);
            }
            int at = first;
            for (int part = 0; part < parts; ++part) {
                int u0, n;
                range_of(first, last, part, parts, u0, n, rcp);
                need(u0 == at && n >= 0, "ranges follow one another", trial, part, u0);
                at += n;
            }
            need(at == last, "ranges end with the keys", trial, at, last);
        };
        if (s.p_items) walk(0, tiles_of(d, s.stacked), s.prefix_parts, s.stacked, 0, prefix_tiles);
        int at = s.p_items;
        for (int b = 0; b < B; ++b) {
            const int rows = tokens[b] * g, first = rows >= kRowTile ? 0 : prefix_tiles;
            if (rows) walk(at, tiles_of(d, rows), request_parts(d, s, rows, own_tiles(b), rcp), rows, first, prefix_tiles + std::rand() % (own_tiles(b) + 1));
            at += request_items(d, s, rows, own_tiles(b), rcp);
        }
        need(at == items, "items", trial, at, items);
        ++walked;
    }
    need(walked > 1000, "launches walked", walked);
    std::printf("ok\n");
    return 0;
}
