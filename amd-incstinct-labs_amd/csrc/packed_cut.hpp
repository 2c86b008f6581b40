// How the packed prompts' items (prefill_packed.hip: blocks of queries times groups of heads, most keys first) are
// dealt out to the workgroups of one round of the chip, and when the last of them are cut along their keys:
// constexpr functions shared by the kernel, its launcher and a host-side replay (tests/native/packed_cut_check.cpp) that
// checks that every item is taken once, or every part of it once. Plain C++: clang compiles constexpr functions for
// host and device alike.
//
// Behind a long prefix all items take about as long, so the rounds of the chip's workgroups count: the items past
// the last full round, where they are few, are cut into `each` parts along their keys, one to a workgroup, and
// packed_join joins the parts. Part y of the tail's item e goes to workgroup y tail + e: the items of one kv head stay on
// one XCD, whose L2 their prefix comes through.
#pragma once

namespace cdna4 {
namespace packed {

constexpr int kMinTiles = 16;   // tiles of an item that is cut
constexpr int kMaxParts = 32;   // of an item
struct Cut { int rounds, tail, each; };   // rounds of whole items before the cut ones; tail 0: none is cut

// Whether and how the items past the last full round of G workgroups (per_cu to a CU) of 64 qt rows behind `tiles` tiles
// are cut, by estimated times in eighths of a tile's (0.7 us at D = 128): a workgroup that has its CU to itself
// takes 8 per tile, all that fit it together 13 (two) or 19 (three); the join costs five tiles for its launch and a
// sixth per part and 64 rows for the results' way through memory (512 parts of 128 rows: 68 MB). Measured at 32/8 heads,
// D 128, bf16: one sequence of 64 tokens behind 8,192 keys 93-95 -> 27 us, four of 16 behind 32,768 348-355 -> 56-59, ten of
// 200 behind 8,192 (560 items on 512 workgroups) 359-369 -> 268-275; cut all the same, six of 70 behind 2,048 30.5 -> 48.
constexpr Cut cut_items(int items, int G, int tiles, int per_cu, int qt) {
    const int rounds = items / G, tail = items - rounds * G, cus = G / per_cu;
    const int full = per_cu == 2 ? 13 : 19;
    Cut best{rounds, 0, 0};
    if (tail == 0 || tiles < kMinTiles) return best;
    int most = 1;   // parts of an item, about the root of its tiles
    while (most < kMaxParts && (most + 1) * (most + 1) <= tiles) ++most;
    long long time = (long long)tiles * (tail > cus ? full : 8);
    for (int k = 0; k < 2; ++k) {   // to one workgroup per CU, or to as many as fit
        int each = (k ? G : cus) / tail;
        if (each > most) each = most;
        if (each < 2) continue;
        const long long t = (long long)tiles * (each * tail > cus ? full : 8) / each + 40 + each * tail * qt / 6;
        if (t < time) {
            time = t;
            best = Cut{rounds, tail, each};
        }
    }
    return best;
}

// What workgroup p of G takes in a round: item idx (past every list: none), whole (part -1) or its y-th part, whose results
// go to place `part` of the parts'; place >= 0: the place among the cut items where the join finds the item. Each
// place has one turn that stores to it: other rounds of the same workgroup, found by other waves at the same time, must
// not.
struct Turn { int idx, y, part, place; };
constexpr int kNoItem = 0x7fffffff;
constexpr Turn turn_of(const Cut& cut, int round, int p, int G) {
    if (cut.tail == 0 || round < cut.rounds) return Turn{round * G + ((round & 1) ? G - 1 - p : p), 0, -1, -1};
    const int y = p / cut.tail;
    if (round > cut.rounds || y >= cut.each) return Turn{kNoItem, 0, -1, -1};
    return Turn{cut.rounds * G + p - y * cut.tail, y, p, y == 0 ? p : -1};
}

}  // namespace packed
}  // namespace cdna4
