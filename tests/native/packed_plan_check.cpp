// Host sweep of the packed prompts' plan (test only, plain C++): where the plan asks for no workspace, a call without one
// runs the same plan; where it cuts items along their keys or lists them, the workspace holds what the kernels store; and
// rows, items and grid fit each other. Prints how many plans of each order it saw, then "ok", or the first violation and
// exits 1.
#include <stdio.h>
#include <vector>
#include "packed_plan.hpp"

using namespace cdna4;
using namespace packed;

static long long seen[3];

static int fail(const char* what, const cdna4_packed_cfg& c, int cus) {
    printf("%s: D %d heads %d/%d batch %d total %d prefix %d, %d CUs\n", what, c.D, c.nQHeads, c.nKVHeads, c.batch, c.total, c.prefix, cus);
    return 1;
}

template <int D>
static int check(const cdna4_packed_cfg& c, int cus) {
    const PackedPlan p = plan_packed<D>(c, true, cus), n = plan_packed<D>(c, false, cus);
    ++seen[p.order];
    if (n.ws_bytes != 0 || n.order != kDealt) return fail("workspace without one", c, cus);
    if ((p.ws_bytes == 0) != (p.order == kDealt)) return fail("order", c, cus);
    if (p.ws_bytes == 0 && (p.qt != n.qt || p.rows != n.rows || p.hp != n.hp || p.grid != n.grid || p.items != n.items))
        return fail("no workspace, and another plan without one", c, cus);
    if (p.order == kFromList && (p.qt != n.qt || p.rows != n.rows || p.grid != n.grid))
        return fail("listed, and other blocks without a list", c, cus);
    for (const PackedPlan& x : {p, n}) {
        const int G = c.nQHeads / c.nKVHeads;
        const long long round = (x.qt == 2 ? resident<D, 2>() : resident<D, 1>()) * (cus & ~7);
        if ((x.qt != 1 && x.qt != 2) || x.rows != (64 * x.qt) >> x.hp || G % (1 << x.hp)) return fail("rows", c, cus);
        if (x.grid < 1 || x.grid > round || (x.order != kDealt && x.grid != round)) return fail("grid", c, cus);
        if (x.items < (long long)(c.nQHeads >> x.hp) * ((c.total + x.rows - 1) / x.rows)) return fail("items", c, cus);
    }
    if (p.order == kFromList && p.ws_bytes < kListHeadBytes + (size_t)p.items * kItemBytes) return fail("list's workspace", c, cus);
    if (p.order == kDealtCut) {
        const long long rows = 64 * p.qt;
        if (((c.total << p.hp) + 63) / 64 > kLevels) return fail("cut with more levels than are held", c, cus);
        if (p.ws_bytes < 256 + (size_t)p.cut * kItemBytes + (size_t)(p.parts * rows) * (D + 2) * 4) return fail("cut items' workspace", c, cus);
        for (long long items = 0; items <= p.items; items += items < 64 ? 1 : 13) {   // whatever the lengths turn out to be
            const Cut cut = cut_items((int)items, (int)p.grid, c.prefix / kTileKeys, (int)(p.grid / (cus & ~7)), p.qt);
            if (cut.tail > p.cut || (long long)cut.each * cut.tail > p.parts) return fail("more parts than places", c, cus);
        }
    }
    return 0;
}

int main() {
    static const int heads[][2] = {{1, 1}, {3, 1}, {8, 1}, {12, 12}, {16, 4}, {20, 10}, {32, 8}, {40, 8}, {64, 8}};
    static const int batches[] = {1, 2, 5, 24, 200, 2048, 2049};
    static const int prefixes[] = {0, 1, 1000, 1024, 1100, 2048, 4096, 5000, 8192, 8960, 16384, 40000};
    static const int chips[] = {256, 252, 32};
    std::vector<int> totals;
    for (int t = 1; t <= 70000; t += t < 40 ? 1 : t < 2400 ? 9 : t / 6) totals.push_back(t);
    for (int t : {200, 512, 791, 1008, 32768, 65536}) totals.push_back(t);
    for (int cus : chips)
        for (auto& h : heads)
            for (int batch : batches)
                for (int prefix : prefixes)
                    for (int total : totals) {
                        cdna4_packed_cfg c{64, h[0], h[1], batch, total, 0, prefix, 0};
                        if (check<64>(c, cus)) return 1;
                        c.D = 128;
                        if (check<128>(c, cus)) return 1;
                    }
    printf("%lld %lld %lld\nok\n", seen[kDealt], seen[kFromList], seen[kDealtCut]);
    return 0;
}
