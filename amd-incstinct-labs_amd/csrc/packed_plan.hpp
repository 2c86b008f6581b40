// The plan of a packed prompt call (prefill_packed.hip): block size, how items are handed out, workspace. Plain C++, shared by
// the launcher and a host-side sweep (tests/native/packed_plan_check.cpp).
#pragma once
#include <stddef.h>
#include <algorithm>

#include "cdna4_attn.h"
#include "packed_cut.hpp"

namespace cdna4 {
namespace packed {

// How fa_packed's workgroups get their items: dealt out, from a list, or dealt out and cut along their keys
enum { kDealt, kFromList, kDealtCut };

// Workgroups of fa_packed that a CU holds (registers and LDS).
template <int D, int QT> constexpr int resident() { return D == 64 ? 3 : 2; }

constexpr int kTileKeys = 64;             // keys of a K/V tile
constexpr int kLevels = 1024;             // block indices that a workgroup holds: sequences of 32,768 tokens and more
constexpr int kListSeqs = 2048;           // sequences of the listing kernel's LDS
constexpr size_t kListHeadBytes = 1280;   // the queues' ends
constexpr size_t kItemBytes = 16;
constexpr long long kMaxItems = 1LL << 30;

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

struct PackedPlan {
    int rows, hp, qt, order;
    long long grid, items, cut, parts;   // cut: items that may be cut, parts: their parts
    size_t ws_bytes;
};

template <int D>
PackedPlan plan_packed(const cdna4_packed_cfg& c, bool with_ws, int device_cus) {
    PackedPlan p{};
    // Query heads of one kv head side by side, up to one per wave: a block then has 128, 64 or 32 tokens, its
    // waves end at the same key or nearly so (with 128 tokens they pass the last two tiles as a staircase), and
    // short sequences fill it.
    const int G = c.nQHeads / c.nKVHeads;
    p.hp = G % 4 == 0 ? 2 : G % 2 == 0 ? 1 : 0;
    // sum of ceil(len / rows) is at most total / rows + the sequences that are not empty
    auto items = [&](int rows) { return (long long)(c.nQHeads >> p.hp) * (c.total / rows + std::min(c.batch, c.total)); };
    const long long cus = device_cus & ~7;
    const long long slots = resident<D, 2>() * cus;   // resident workgroups: the grid is one round of them
    // Blocks of half as many rows for calls of about one round of blocks and less, whose time is that of their
    // longest block: one sequence of 1,024 tokens, 32/8 heads D 128, 21.4 against 25.7 us; above that they read K and V
    // more often and fill the matrix cores less: four of 512-1,024 (808 blocks of 128) 40.0 against 34.8 us. Half a
    // block per sequence is taken for the last ones.
    p.qt = (long long)(c.nQHeads >> p.hp) * (2LL * c.total / (128 >> p.hp) + std::min(c.batch, c.total)) <= 4 * cus ? 1 : 2;
    p.order = kDealt;
    // Behind a prefix, items may be cut along their keys (cut_items) where the blocks that the call probably has, or
    // the most it can have, would be. Whole blocks where long shares leave them their better use of K and V: one
    // sequence of 512 tokens behind 8,192 keys 82 against 88 us. That choice is for cut calls alone: a call that is not
    // cut needs no workspace and runs the same blocks with and without one.
    bool cut = false;
    if (with_ws && c.prefix >= kMinTiles * kTileKeys && items(128 >> p.hp) < 2 * slots && ((long long)c.total << p.hp) / 64 < kLevels) {
        const int tiles = c.prefix / kTileKeys, seqs = std::min(c.batch, c.total);
        auto blocks = [&](int rows) { return (long long)(c.nQHeads >> p.hp) * (2LL * c.total / rows + seqs) / 2; };
        const long long n = blocks(128 >> p.hp);
        const int qt = ((long long)c.total << p.hp) >= 128LL * seqs && n <= slots / 2 && n * tiles >= 32 * slots ? 2 : p.qt;
        const int round = (int)(qt == 2 ? slots : resident<D, 1>() * cus), rows = (64 * qt) >> p.hp;
        for (long long x : {blocks(rows), items(rows)})
            if (cut_items((int)x, round, tiles, (int)(round / cus), qt).tail > 0) cut = true;
        if (cut) {
            p.order = kDealtCut;
            p.qt = qt;
        }
    }
    p.rows = (p.qt == 2 ? 128 : 64) >> p.hp;
    p.items = items(p.rows);
    const long long round = p.qt == 2 ? slots : resident<D, 1>() * cus;
    p.grid = cut ? round : std::min(p.items, round);
    if (cut) {
        p.cut = std::min(p.items, round / 2);
        p.parts = std::min(round, kMaxParts * p.cut);
        p.ws_bytes = 256 + align256(p.cut * kItemBytes) + (size_t)p.parts * (64 * p.qt) * (D + 2) * sizeof(float);
    } else if (with_ws && D == 128 && p.qt == 2 && p.items >= 2 * slots && c.batch <= kListSeqs && p.items <= kMaxItems) {
        p.order = kFromList;
        p.ws_bytes = kListHeadBytes + (size_t)p.items * kItemBytes;
    }
    return p;
}

}  // namespace packed
}  // namespace cdna4
