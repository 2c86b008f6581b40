// Host replay of how packed prompts' items are dealt out and cut along their keys (test only, plain C++): for every
// number of items and several lengths of prefix, each item is taken once, whole or part by part, each part's results have
// a place of their own inside the workspace, and each cut item's place for the join is stored to by one turn,
// whatever rounds a workgroup looks up at the same time. Prints the cuts of each number of whole rounds, then "ok", or
// the first violation and exits 1.
#include <stdio.h>
#include <algorithm>
#include <vector>
#include "packed_cut.hpp"

using namespace cdna4::packed;

static int fail(const char* what, int items, int G, int tiles, int x) {
    printf("%s: items %d, workgroups %d, tiles %d, at %d\n", what, items, G, tiles, x);
    return 1;
}

int main() {
    static const int tile_counts[] = {0, 1, 15, 16, 17, 24, 31, 39, 62, 64, 100, 128, 255, 256, 512, 625, 2048, 33000000};
    static const int chips[][2] = {{256, 2}, {256, 3}, {248, 2}, {32, 3}, {8, 2}};   // CUs, workgroups per CU
    long cuts[4] = {0, 0, 0, 0};
    for (auto& chip : chips)
        for (int qt = 1; qt <= 2; ++qt)
            for (int tiles : tile_counts) {
                const int G = chip[0] * chip[1];
                for (int items = 0; items <= 4 * G; items += items < 64 || items % G < 32 || G < 100 ? 1 : 7) {
                    const Cut cut = cut_items(items, G, tiles, chip[1], qt);
                    std::vector<int> whole(items), parts(items), stores(G), results(G);
                    // as the kernel: the four waves look four rounds up together, and go on while there are items
                    for (int p = 0; p < G; ++p)
                        for (int round = 0; round < cut.rounds + 8; ++round) {
                            const Turn t = turn_of(cut, round, p, G);
                            const bool there = t.idx < items;
                            if (t.place >= 0) {
                                if (t.place >= cut.tail || !there || t.idx - cut.rounds * G != t.place) return fail("place of another item", items, G, tiles, p);
                                ++stores[t.place];
                            }
                            if (!there) continue;
                            if (t.idx < 0) return fail("item below 0", items, G, tiles, t.idx);
                            if (t.part < 0) { ++whole[t.idx]; continue; }
                            if (t.part >= G || t.part != t.y * cut.tail + t.idx - cut.rounds * G) return fail("part's place", items, G, tiles, t.part);
                            if (t.y < 0 || t.y >= cut.each) return fail("part", items, G, tiles, t.y);
                            ++results[t.part];
                            ++parts[t.idx];
                        }
                    if (cut.tail && (cut.each < 2 || cut.each > kMaxParts || cut.tail > G / 2 || cut.each * cut.tail > G || tiles < cut.each))
                        return fail("cut", items, G, tiles, cut.each);
                    for (int i = 0; i < items; ++i) {
                        const bool tail = cut.tail && i >= cut.rounds * G;
                        if (whole[i] != (tail ? 0 : 1) || parts[i] != (tail ? cut.each : 0)) return fail("item not taken once", items, G, tiles, i);
                    }
                    for (int e = 0; e < cut.tail; ++e)
                        if (stores[e] != 1) return fail("place not stored to once", items, G, tiles, e);
                    for (int r = 0; r < cut.each * cut.tail; ++r)
                        if (results[r] != 1) return fail("part's results not stored once", items, G, tiles, r);
                    if (cut.tail) ++cuts[std::min(cut.rounds, 3)];
                }
            }
    printf("%ld %ld %ld %ld\nok\n", cuts[0], cuts[1], cuts[2], cuts[3]);
    return 0;
}
