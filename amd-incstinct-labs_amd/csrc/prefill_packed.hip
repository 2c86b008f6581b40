// Prompt attention over packed sequences for gfx950: prompts of different lengths one after another in
// token-major Q, K, V, causal within each, optionally behind a prefix of keys that all of them see.
//
// Token i of sequence s (rows cu[s] .. cu[s+1] - 1) sees the P prefix keys and its sequence's tokens 0 .. i:
//   O = sum_j 2^(c q.k_j - m) v_j / sum_j 2^(c q.k_j - m),  c = log2(e) / sqrt(D), m a running maximum.
// The kernels are the prompt kernels' tile machinery (attn_tile.hpp, attn_pipe.hpp) over one key axis per
// sequence, prefix keys 0 .. P - 1 and then the sequence's own, with no padding where they meet: key k lies
// in the prefix cache or in the packed rows, and the tile that holds both takes its addresses per lane.
//
// Lengths are read on the device (a captured call replays on other lengths): a workgroup finds its items,
// blocks of queries of one sequence and group of heads, from cu alone, or takes them from a list that a launch
// before it has made (packed_plan.hpp: which way when; packed_cut.hpp: how they are dealt out). Blocks are ordered by their
// index in the sequence, the last ones (the most keys) first: a longest-first schedule whatever the lengths are.
//
// A weight is rounded to the inputs' 16-bit type for the P.V product, whose matrix instructions take no wider operand at
// their rate, and the sum of a row adds the rounded weights, in fp32, so that both sides of the quotient weigh alike.
// Maxima, sums and O are fp32. Against an fp32 product that costs the relative error of the output, which its own
// rounding dominates, a factor of 1.0-1.2 in bf16 and 1.2-1.4 in fp16 (0.0016 -> 0.0019, 0.00021 -> 0.00029); bf16 weights
// of the keys that rows of few keys see carry a second term (attn_tile.hpp, kLoKeys).
//
// Bound by the matrix cores: four prompts of 2,011-8,192 tokens, 32/8 heads D 128 bf16, 919-967 us in a graph by machine
// (1,170-1,230 TFLOP/s, matrix cores 65 % busy), 24 of 33-2,048 145-152 us (840-880 TFLOP/s: a block's start and end take a
// quarter of its time), 16 of 90-1,024, 12 heads D 64 fp16, 24 us (the longest block's 16 tiles one after another).
#include <type_traits>
#include <algorithm>

#include "attn_tile.hpp"
#include "attn_stream.hpp"
#include "attn_block.hpp"
#include "packed_plan.hpp"

namespace cdna4 {
namespace {

using namespace tile;
using namespace pipe;
using namespace packed;
using block::Keys;
using wave::xlane::allreduce;
using wave::xlane::Max;
using wave::xlane::Sum;

struct PackedArgs {
    const uint16_t *Q, *K, *V, *Kp, *Vp;
    uint16_t* O;
    const int* cu;
    long long q_rs, q_hs, k_rs, k_hs, o_rs, o_hs;   // row (token) and head strides, elements
    long long p_hs;                                  // head stride of the prefix (rows are D elements apart)
    int nQH, G, batch, total, prefix;
    int hp;       // log2 of the query heads per workgroup
    int single;   // 1: a workgroup per item, at most
    struct ListHead* head;   // the work list, if there is one
    int4* items;
    Cut* split;                // cut items, if any can be: how, their places, the parts' results
    int4* cut;
    float *part_ml, *part_o;   // [part][rows][2], [part][rows][D]
    int max_items;           // blocks times groups of heads that the sequences can have; the list's room
    int copy32;   // 1: a step's rows span < 4 GiB (32-bit copy offsets)
    float sc;     // log2(e) / sqrt(D)
};

// ---- work items ----------------------------------------------------------------------------------
// Rows of sequence s; cu outside 0 .. total or decreasing is cut to it, so that no contents of cu lead
// outside the tensors.
__device__ __forceinline__ void seq_rows(const PackedArgs& a, int s, int& start, int& len) {
    start = min(max(a.cu[s], 0), a.total);
    len = min(max(a.cu[s + 1], start), a.total) - start;   // cut before the difference, which then cannot wrap
}

// The list of blocks, block index descending and sequences ascending within one index. With n_s the blocks of
// sequence s, f(d) = sum_s max(0, n_s - d) blocks have an index of d or more, so entry idx of the list has
// the largest index d with f(d) > idx, and is the (idx - f(d + 1))-th sequence with more than d blocks. A
// workgroup forms f once, in LDS: a histogram of the n_s, summed twice from the top (the sequences with more
// than d blocks, then their blocks).
constexpr int kSeqs = 512;      // sequences held; the rows of others are read again
struct Items {
    int f[kLevels];
    int2 seq[kSeqs];   // first row, rows
    int levels;
};

__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }   // the same in every lane

__device__ __forceinline__ int blocks_of(const PackedArgs& a, const Items& it, int s, int rows_log2) {
    int start, len;
    if (s >= a.batch) return 0;
    if (s < kSeqs) len = it.seq[s].y;
    else seq_rows(a, s, start, len);
    return (len + (1 << rows_log2) - 1) >> rows_log2;
}

// hist: kLevels + 1 words of LDS, free until the barrier at the end.
__device__ __forceinline__ void list_items(const PackedArgs& a, int rows_log2, Items& it, int* hist, int tid) {
    for (int i = tid; i <= kLevels; i += 256) hist[i] = 0;
    __syncthreads();
    for (int s = tid; s < a.batch; s += 256) {
        int start, len;
        seq_rows(a, s, start, len);
        if (s < kSeqs) it.seq[s] = make_int2(start, len);
        const int n = (len + (1 << rows_log2) - 1) >> rows_log2;
        if (n > 0) {
            atomicAdd(&hist[min(n, kLevels)], 1);
            atomicMax(&hist[0], n);   // entry 0 is not a count
        }
    }
    __syncthreads();
    if (tid < 64) {
        const int levels = scalar(hist[0]);
        if (tid == 0) it.levels = levels;
        int more = 0, f = 0;   // of the levels above
        for (int d0 = (min(levels, kLevels) - 1) & ~63; d0 >= 0; d0 -= 64) {
            const int d = d0 + 63 - tid;
            const int g = wave::xlane::scan_inclusive(d < kLevels ? hist[d + 1] : 0, Sum{}) + more;
            const int x = wave::xlane::scan_inclusive(g, Sum{}) + f;
            it.f[d] = x;
            more = __builtin_amdgcn_readlane(g, 63);
            f = __builtin_amdgcn_readlane(x, 63);
        }
    }
    __syncthreads();
}

// Entry idx of the list; false past its end.
__device__ __forceinline__ bool find_item(const PackedArgs& a, int rows_log2, const Items& it, int idx, int lane, int& start,
                                          int& len, int& blk) {
    const int levels = scalar(it.levels);
    if (levels == 0) return false;
    int f_above;
    if (levels <= kLevels) {
        if (idx >= scalar(it.f[0])) return false;
        constexpr int kStep = kLevels / 64;
        const int seg = kStep * (__popcll(__builtin_amdgcn_ballot_w64(kStep * lane < levels && it.f[kStep * lane] > idx)) - 1);
        const int d = seg + lane;
        blk = seg + __popcll(__builtin_amdgcn_ballot_w64(lane < kStep && d < levels && it.f[min(d, kLevels - 1)] > idx)) - 1;
        f_above = blk + 1 < levels ? scalar(it.f[blk + 1]) : 0;
    } else {   // longer than the levels held: f by bisection, each from all sequences
        auto f = [&](int d) {
            int x = 0;
            for (int s = lane; s < a.batch; s += 64) x += max(blocks_of(a, it, s, rows_log2) - d, 0);
            return scalar(allreduce(x, Sum{}));
        };
        if (idx >= f(0)) return false;
        int lo = 0, hi = levels;   // f(lo) > idx >= f(hi)
        f_above = 0;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1, x = f(mid);
            if (x > idx) lo = mid;
            else { hi = mid; f_above = x; }
        }
        blk = lo;
    }
    int r = idx - f_above, seq = 0;
    for (int s0 = 0; s0 < a.batch; s0 += 64) {
        const bool has = blocks_of(a, it, s0 + lane, rows_log2) > blk;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(has);
        const int c = __popcll(mask);
        if (r < c) {
            const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
            const uint64_t here = __builtin_amdgcn_ballot_w64(has && before == r);
            seq = s0 + (here ? __builtin_ctzll(here) : 0);
            break;
        }
        r -= c;
    }
    if (seq < kSeqs) {
        const int2 sl = it.seq[seq];
        start = sl.x;
        len = sl.y;
    } else {
        seq_rows(a, seq, start, len);
    }
    start = scalar(start);
    len = scalar(len);
    return (blk << rows_log2) < len;   // always, but for counts of overlapping sequences that pass 32 bits
}

// ---- work lists -----------------------------------------------------------------------------------
// Many items (several rounds of the chip's workgroups) are listed by a launch of one workgroup and handed out
// while the kernel runs. Eight queues, one per XCD, so that the blocks of one sequence and kv head, which read
// the same K and V, run on one XCD at about the same time and find them in its L2; longest sequences first, the
// last blocks of a sequence first; a workgroup whose queue is empty takes from the others. Against the list
// in LDS (longest blocks of all sequences first, dealt out in turn): 64 prompts of 512 tokens, 32/8 heads
// D 128, read their 134 MB of K and V again for every block index there, 258 us against 224 in this order; four of
// 2,011-8,192 tokens 945 against 925 us.
struct ListHead {
    int next[8][32];   // of the queue's entries, a cache line each
    int begin[8], end[8];
    int pad[48];
};
static_assert(sizeof(ListHead) == kListHeadBytes && sizeof(int4) == kItemBytes, "the plan's sizes");

// Heads (nh per entry) of the sequence at place q that go to queue x: cnt of them, the c-th is head(c).
struct QueueHeads {
    int first, step, cnt;
    __device__ __forceinline__ QueueHeads(int q, int nh, int x) {
        if ((nh & 7) == 0) {   // neighbouring heads, which share K and V
            cnt = nh >> 3;
            first = x * cnt;
            step = 1;
        } else {               // the sequences' heads in turn
            first = (x - q * nh) & 7;
            step = 8;
            cnt = first < nh ? (nh - first + 7) >> 3 : 0;
        }
    }
};

__global__ __launch_bounds__(1024) void packed_list(PackedArgs a, int per_queue) {
    __shared__ int hist[kLevels + 1];
    __shared__ int2 seq[kListSeqs];            // by place: longest first
    __shared__ int blocks[kListSeqs];
    __shared__ int pre[8][kListSeqs + 1];      // entries of the queue before place q
    __shared__ int placed;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int rows_log2 = block::rows_log2<2>() - a.hp, nh = a.nQH >> a.hp;
    for (int i = tid; i <= kLevels; i += 1024) hist[i] = 0;
    __syncthreads();
    int2 mine[kListSeqs / 1024];
    int n[kListSeqs / 1024];
#pragma unroll
    for (int k = 0; k < kListSeqs / 1024; ++k) {
        const int s = k * 1024 + tid;
        n[k] = 0;
        if (s < a.batch) {
            seq_rows(a, s, mine[k].x, mine[k].y);
            n[k] = (mine[k].y + (1 << rows_log2) - 1) >> rows_log2;
            if (n[k] > 0) {
                atomicAdd(&hist[min(n[k], kLevels)], 1);
                atomicMax(&hist[0], min(n[k], kLevels));   // entry 0 is not a count
            }
        }
    }
    __syncthreads();
    if (wave == 0) {   // hist[i] becomes the places before the sequences of i blocks
        int more = 0;
        for (int d0 = (hist[0] - 1) & ~63; d0 >= 0; d0 -= 64) {
            const int i = d0 + 64 - lane, h = hist[i];
            const int g = wave::xlane::scan_inclusive(h, Sum{}) + more;
            hist[i] = g - h;
            more = __builtin_amdgcn_readlane(g, 63);
        }
        if (lane == 0) placed = more;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kListSeqs / 1024; ++k) {
        if (n[k] == 0) continue;
        const int q = atomicAdd(&hist[min(n[k], kLevels)], 1);   // equal counts in any order: no result depends on it
        seq[q] = mine[k];
        blocks[q] = n[k];
    }
    __syncthreads();
    const int nseq = placed;
    if (wave < 8) {
        // Sequences of a wrong cu may overlap and have more blocks than the list has room for (a.max_items, up to
        // 2^30): sums in 64 bits, cut to it.
        long long sum = 0;
        const long long most = a.max_items;
        for (int q0 = 0; q0 < nseq; q0 += 64) {
            const int q = q0 + lane;
            const long long v = q < nseq ? (long long)blocks[q] * QueueHeads(q, nh, wave).cnt : 0;
            const long long g = wave::xlane::scan_inclusive(v, Sum{}) + sum;
            if (q < nseq) pre[wave][q] = (int)min(g - v, most);
            sum = __shfl(g, 63);
        }
        if (lane == 0) pre[wave][nseq] = (int)min(sum, most);
    }
    __syncthreads();
    int begin[8];
    begin[0] = 0;
#pragma unroll
    for (int x = 1; x < 8; ++x) begin[x] = min(begin[x - 1] + pre[x - 1][nseq], a.max_items);
    if (tid == 0) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const int len = min(pre[x][nseq], a.max_items - begin[x]);
            a.head->begin[x] = begin[x];
            a.head->end[x] = begin[x] + len;
            a.head->next[x][0] = begin[x] + min(len, per_queue);   // the workgroups' first items
        }
    }
    // one thread per entry: its queue from the eight lengths, its sequence by bisection
    const int all = min(begin[7] + pre[7][nseq], a.max_items);
    for (int i = tid; i < all; i += 1024) {
        int x = 0;
#pragma unroll
        for (int y = 1; y < 8; ++y) x += i >= begin[y];
        int e = i;
#pragma unroll
        for (int y = 1; y < 8; ++y) e = x == y ? i - begin[y] : e;
        int lo = 0, hi = nseq;   // pre[lo] <= e < pre[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[x][mid] <= e) lo = mid;
            else hi = mid;
        }
        const QueueHeads qh(lo, nh, x);
        e -= pre[x][lo];
        const int d = e / qh.cnt, c = e - d * qh.cnt;
        const int2 sl = seq[lo];
        a.items[i] = make_int4(sl.x, sl.y, (blocks[lo] - 1 - d) << rows_log2, (qh.first + c * qh.step) << a.hp);
    }
}

// Entry idx of the list for a workgroup that takes one item: f by bisection, from the block counts that the
// lanes hold (sequences lane, lane + 64, ..: kHeld in registers, others read again). False past the list's end.
constexpr int kHeld = 4;
__device__ __forceinline__ bool packed_item(const PackedArgs& a, int rows_log2, int idx, int lane, int& start, int& len,
                                            int& blk) {
    int n[kHeld];
    auto blocks = [&](int s) {
        int st, ln;
        if (s >= a.batch) return 0;
        seq_rows(a, s, st, ln);
        return (ln + (1 << rows_log2) - 1) >> rows_log2;
    };
    int most = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        n[i] = 0;
        if (64 * i < a.batch) n[i] = blocks(64 * i + lane);
        most = max(most, n[i]);
        sum += n[i];
    }
    for (int s = 64 * kHeld; s < a.batch; s += 64) {
        const int x = blocks(s + lane);
        most = max(most, x);
        sum += x;
    }
    if (idx >= scalar(allreduce(sum, Sum{}))) return false;
    auto above = [&](int d) {
        int x = 0;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) x += max(n[i] - d, 0);
        for (int s = 64 * kHeld; s < a.batch; s += 64) x += max(blocks(s + lane) - d, 0);
        return scalar(allreduce(x, Sum{}));
    };
    int lo = 0, hi = scalar(allreduce(most, Max{})), f_hi = 0;   // f(lo) > idx >= f(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1, f = above(mid);
        if (f > idx) lo = mid;
        else { hi = mid; f_hi = f; }
    }
    blk = lo;
    int r = idx - f_hi, seq = -1;   // the r-th sequence with more than blk blocks
    auto pick = [&](int s0, int cnt) {
        const uint64_t mask = __builtin_amdgcn_ballot_w64(cnt > blk);
        const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
        const uint64_t here = __builtin_amdgcn_ballot_w64(cnt > blk && before == r);
        if (here != 0 && seq < 0) seq = s0 + __builtin_ctzll(here);
        r -= __popcll(mask);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) pick(64 * i, n[i]);
    for (int s = 64 * kHeld; s < a.batch && seq < 0; s += 64) pick(s, blocks(s + lane));
    seq_rows(a, max(seq, 0), start, len);
    start = scalar(start);
    len = scalar(len);
    return (blk << rows_log2) < len;   // always, but for counts of overlapping sequences that pass 32 bits
}

// Head of workgroup i within one entry's nQH workgroups. Workgroups go to the XCDs round-robin: with nQH a
// multiple of 8 each XCD takes nQH / 8 neighbouring query heads, which share K and V heads in its L2.
__device__ __forceinline__ int item_head(int i, int nQH) {
    return (nQH & 7) ? i : (i & 7) * (nQH >> 3) + (i >> 3);
}

// O^T / l of 16 queries as 16-bit rows: lane (li, g) holds elements 16 dt + 4 g + e of query li. A swap between
// neighbouring rows of lanes gives each lane eight neighbouring elements, so that a store writes 64 contiguous
// bytes per query instead of 32, in half the instructions.
template <int D, bool kBf16>
__device__ __forceinline__ void store_rows(const f32x4 (&o)[D / 16], float l, uint16_t* row, int g, bool valid) {
    typedef uint32_t u32x4_8 __attribute__((ext_vector_type(4), aligned(8)));   // O is 8-byte aligned
    const float inv = l > 0.f ? 1.f / l : 1.f;
    uint16_t* dst = row + (g & 1) * 16 + (g >> 1) * 8;
#pragma unroll
    for (int dt = 0; dt < D / 16; dt += 2) {
        u32x4_8 w;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t even = pack2<kBf16>(o[dt][2 * x] * inv, o[dt][2 * x + 1] * inv);
            const uint32_t odd = pack2<kBf16>(o[dt + 1][2 * x] * inv, o[dt + 1][2 * x + 1] * inv);
            const auto r = __builtin_amdgcn_permlane16_swap(even, odd, false, false);
            w[x] = r[0];
            w[2 + x] = r[1];
        }
        if (valid) *(u32x4_8*)(dst + dt * 16) = w;
    }
}

// ---- 128 rows per workgroup, two workgroups per CU -------------------------------------------------
// Four waves of 32 queries share 64-key K/V tiles in LDS, two slots each for K and V (64 KiB at D = 128), so
// that two workgroups fit a CU: while one waits for its first tiles, masks its diagonal or stores, the other
// has the matrix cores. The grid is one round of them; workgroup p takes entries p, 2 G - 1 - p, 2 G + p, ..
// of the list times the heads (G workgroups), which evens out what a round's order costs, and loads the next
// item's queries and first tiles before it stores its results: an item of one tile took 12.4 us as a
// workgroup of its own, of which 2.4 to find it, 3.0 for the first loads and 2.9 for the stores.
template <int D, int QT, bool kBf16, bool kPrefix, int kOrder>
__global__ __launch_bounds__(256, (resident<D, QT>())) void fa_packed(PackedArgs a) {
    constexpr bool kListed = kOrder == kFromList, kCut = kOrder == kDealtCut;
    constexpr int ND = D / 32, NDT = D / 16;
    __shared__ __attribute__((aligned(16))) uint16_t lds[block::lds_elems<D>()];
    static_assert((kLevels + 1) * 4 <= (int)sizeof(lds), "the histogram fits the tiles' LDS");
    const int lane = (int)(threadIdx.x & 63u);
    const int wave = scalar((int)(threadIdx.x >> 6));
    const int li = lane & 15, g = lane >> 4;
    // The workgroup's waves serve 1 << hp query heads of one kv head, a block's rows >> hp tokens each
    const int hp = a.hp, rows_log2 = block::rows_log2<QT>() - hp, nh = a.nQH >> hp;
    const int P = kPrefix ? a.prefix : 0;
    struct Item {
        int start, len, q0, h0;   // len 0: none
        int t0, t1, part;         // its tiles of keys, part >= 0: where its results go for packed_join
    };
    __shared__ int4 next_s[4];
    __shared__ int4 piece_s[kCut ? 4 : 1];
    auto all_tiles = [&](int q0, int len) { return (P + min(q0 + (1 << rows_log2), len) + kBc - 1) / kBc; };
    auto item_at = [&](int round) {
        const int4 x = next_s[kListed ? 0 : round & 3];
        Item it{scalar(x.x), scalar(x.y), scalar(x.z), scalar(x.w), 0, 0, -1};
        if (kCut) {
            const int4 y = piece_s[round & 3];
            it.t0 = scalar(y.x);
            it.t1 = scalar(y.y);
            it.part = scalar(y.z);
        } else {
            it.t1 = all_tiles(it.q0, it.len);
        }
        return it;
    };
    // Listed: the first item is the workgroup's place in its XCD's queue, the others are claimed by wave 0 ahead
    // of an item's last tiles.
    int queue = (int)blockIdx.x & 7, claimed = -1;   // of wave 0
    auto claim = [&]() {
        if (!kListed || wave != 0) return;
        claimed = -1;
        for (int k = 0; k < 8; ++k) {
            int i = 0;
            if (lane == 0) i = atomicAdd(&a.head->next[queue][0], 1);
            i = scalar(i);
            if (i < scalar(a.head->end[queue])) {
                claimed = i;
                break;
            }
            queue = (queue + 1) & 7;
        }
    };
    auto publish = [&]() {
        if (kListed && wave == 0 && lane == 0) next_s[0] = claimed >= 0 ? a.items[claimed] : make_int4(0, 0, 0, 0);
    };
    // Not listed: each wave finds the item of another of the next four rounds.
    struct NoItems {};
    __shared__ std::conditional_t<kListed, NoItems, Items> items;
    Cut cut{0, 0, 0};
    auto find = [&](int round) {
        if constexpr (!kListed) {
            const Turn turn = turn_of(cut, round, (int)blockIdx.x, (int)gridDim.x);
            const int entry = turn.idx / nh;
            int start = 0, len = 0, blk = 0;
            // overlapping sequences of a wrong cu can have more items than lengths that add up to the tokens: no more
            const bool ok = turn.idx < a.max_items && find_item(a, rows_log2, items, entry, lane, start, len, blk);
            const int4 x = make_int4(start, ok ? len : 0, blk << rows_log2, item_head(turn.idx - entry * nh, nh) << hp);
            if (lane == 0) next_s[round & 3] = x;
            if constexpr (kCut) {
                const int n = all_tiles(x.z, x.y);   // no fewer than the prefix has, so no part is empty
                if (lane == 0) {
                    piece_s[round & 3] = turn.part >= 0 ? make_int4(n * turn.y / cut.each, n * (turn.y + 1) / cut.each, turn.part, 0)
                                                        : make_int4(0, n, -1, 0);
                    if (turn.place >= 0) a.cut[turn.place] = x;   // one wave of one workgroup for each place
                }
            }
        }
    };
    if constexpr (kListed) {
        if (wave == 0) {
            const int i = scalar(a.head->begin[queue]) + ((int)blockIdx.x >> 3);
            if (i < scalar(a.head->end[queue])) claimed = i;
            else claim();
            publish();
        }
    } else if (!a.single) {
        list_items(a, rows_log2, items, (int*)lds, (int)threadIdx.x);
        if constexpr (kCut) {
            cut = cut_items(scalar(items.levels) ? min(scalar(items.f[0]) * nh, a.max_items) : 0, (int)gridDim.x, P / kBc, resident<D, QT>(), QT);
            if (blockIdx.x == 0 && threadIdx.x == 0) *a.split = cut;
        }
        find(wave);
    }
    const block::Offsets own = block::own_offsets<D>(a.k_rs, wave, lane);
    u32x4 qb[QT][ND];
    // keys from a part's first on: all that are left for an item's last part, whose tiles end with the block
    auto keys_of = [&](const Item& it) {
        const int left = P + it.len - it.t0 * kBc;
        return kCut && it.t1 < all_tiles(it.q0, it.len) ? (it.t1 - it.t0) * kBc : left;
    };
    auto keys = [&](const Item& it, const uint16_t* own, const uint16_t* pre) {
        const int kvh = it.h0 / a.G;
        const uint16_t* o = own + it.start * a.k_rs + kvh * a.k_hs;
        const uint16_t* p = pre + kvh * a.p_hs;
        if (!kCut) return Keys<kPrefix>{o, p, a.k_rs, P, P + it.len, a.copy32};
        const int k0 = it.t0 * kBc;   // the axis of a part begins at its first key
        return Keys<kPrefix>{o + max(k0 - P, 0) * a.k_rs, p + (long long)min(k0, P) * D, a.k_rs, max(P - k0, 0), keys_of(it), a.copy32};
    };
    const int dq = (wave & ((4 >> hp) - 1)) * QT * 16, dh = wave >> (2 - hp);   // of this wave in the block
    auto load = [&](const Item& it) {   // the queries and the first tiles
        const uint16_t* Qh = a.Q + it.start * a.q_rs + (it.h0 + dh) * a.q_hs;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int q = min(it.q0 + dq + t * 16 + li, it.len - 1);
#pragma unroll
            for (int c = 0; c < ND; ++c) qb[t][c] = *(const u32x4*)(Qh + q * a.q_rs + c * 32 + g * 8);
        }
        block::first_copies<D, kPrefix>(keys(it, a.K, a.Kp), keys(it, a.V, a.Vp), it.t1 - it.t0, own, lds, wave, lane);
    };
    Item it;
    if (!kListed && a.single) {   // no list to form: every wave finds the one item
        const int entry = (int)blockIdx.x / nh;
        int blk;
        if (!packed_item(a, rows_log2, entry, lane, it.start, it.len, blk)) return;
        it.q0 = blk << rows_log2;
        it.h0 = item_head((int)blockIdx.x - entry * nh, nh) << hp;
        it.t0 = 0;
        it.t1 = all_tiles(it.q0, it.len);
        it.part = -1;
    } else {
        __syncthreads();
        it = item_at(0);
        if (it.len == 0) return;
    }
    load(it);
    for (int round = 1;; ++round) {
        const int qw0 = it.q0 + dq, S = keys_of(it), ntiles = it.t1 - it.t0, P0 = P - it.t0 * kBc;
        const int wave_end = min(qw0 + QT * 16, it.len);                  // one past this wave's last query
        int nch = wave_end > qw0 ? (P0 + wave_end + 31) / 32 : 0;          // the wave's chunks; 0: no queries
        if (kCut) nch = max(min(nch, 2 * ntiles), 0);
        // Main tiles: chunks 2t + 1 and 2t + 2 lie below the workgroup's first query, and the copies of
        // V (t + 1) and K (t + 2) are whole tiles that exist.
        int t_main = P0 + it.q0 >= 95 ? (P0 + it.q0 - 95) / 64 + 1 : 0;
        t_main = min(t_main, min(ntiles - 2, S / kBc - 2));
        if (!a.copy32) t_main = 0;
        f32x4 o[QT][NDT], lacc[QT];
        float m[QT];
        block::attend<D, QT, kBf16, kPrefix, true>(keys(it, a.K, a.Kp), keys(it, a.V, a.Vp), block::Shape{S, ntiles, nch, P0 + qw0, t_main},
                                               qb, o, lacc, m, own, lds, a.sc, wave, lane);
        uint16_t* Oh = a.O + it.start * a.o_rs + (it.h0 + dh) * a.o_hs;
        const int len = it.len, part = it.part;
        // What lies between two items is short and holds the matrix cores up: ahead of the CU's other waves
        __builtin_amdgcn_s_setprio(3);
        bool more = kListed || !a.single;
        if (more) {
            if (kListed) { claim(); publish(); }
            else if ((round & 3) == 0) find(round + wave);
            __syncthreads();   // every wave is done with the tiles; the next items are there
            it = item_at(round);
            more = it.len > 0;
            if (more) load(it);
        }
        if (kCut && part >= 0) {
#pragma unroll
            for (int x = 0; x < QT; ++x) {
                const size_t row = (size_t)part * (64 * QT) + (wave * QT + x) * 16 + li;
                float* dst = a.part_o + row * D + g * 4;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) *(f32x4*)(dst + dt * 16) = o[x][dt];
                if (g == 0) *(float2*)(a.part_ml + row * 2) = make_float2(m[x], lacc[x][0]);
            }
        } else {
#pragma unroll
            for (int x = 0; x < QT; ++x) {
                const int q = qw0 + x * 16 + li;
                store_rows<D, kBf16>(o[x], lacc[x][0], Oh + q * a.o_rs, g, q < len);
            }
        }
        if (!more) break;
        __builtin_amdgcn_s_setprio(0);
    }
}

// The rows of the cut items: o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p over an item's parts, D / 4 lanes per row.
template <int D, int QT, bool kBf16>
__global__ __launch_bounds__(256) void packed_join(PackedArgs a) {
    constexpr int kRows = 64 * QT, kLanes = D / 4, kStep = 256 / kLanes;
    const Cut cut = *a.split;
    const int e = (int)blockIdx.x / (kRows / kStep);
    if (e >= cut.tail) return;
    const int4 it = a.cut[e];   // first row, rows, first query, first head
    const int r = (int)blockIdx.x % (kRows / kStep) * kStep + (int)threadIdx.x / kLanes, d = 4 * ((int)threadIdx.x % kLanes);
    const int wave = r / (16 * QT), hp = a.hp;
    const int q = it.z + (wave & ((4 >> hp) - 1)) * (16 * QT) + r % (16 * QT), head = it.w + (wave >> (2 - hp));
    if (q >= it.y) return;
    const int n = cut.each;
    const size_t step = (size_t)cut.tail * kRows;   // rows from one part to the next
    const float* ml = a.part_ml + ((size_t)e * kRows + r) * 2;
    const float* po = a.part_o + ((size_t)e * kRows + r) * D + d;
    constexpr int kFlight = 8;
    float M = kInitM, L = 0.f;
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < n; i0 += kFlight) {   // parts in flight; those past the last re-read it, weighted 0
        f32x4 v[kFlight];
        float2 s[kFlight];
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
            const size_t x = min(i0 + i, n - 1);
            s[i] = *(const float2*)(ml + x * step * 2);
            v[i] = *(const f32x4*)(po + x * step * D);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < kFlight; ++i) top = fmaxf(top, s[i].x);
        const float old = __builtin_amdgcn_exp2f(M - top);
        M = top;
        L *= old;
        acc *= old;
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
            const float w = i0 + i < n ? __builtin_amdgcn_exp2f(s[i].x - M) : 0.f;
            L = fmaf(w, s[i].y, L);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] = fmaf(w, v[i][k], acc[k]);
        }
    }
    const float inv = L > 0.f ? 1.f / L : 1.f;
    uint2 o;
    o.x = pack2<kBf16>(acc[0] * inv, acc[1] * inv);
    o.y = pack2<kBf16>(acc[2] * inv, acc[3] * inv);
    *(uint2*)(a.O + (it.x + q) * a.o_rs + head * a.o_hs + d) = o;
}

}  // namespace

namespace {

// Every call reads cu in each of its workgroups, and a block's keys and the blocks are counted in 32 bits.
constexpr int kMaxBatch = 1 << 20;

bool valid_cfg(const cdna4_packed_cfg& c) {
    if (c.D != 64 && c.D != 128) return false;
    if (c.nQHeads < 1 || c.nKVHeads < 1 || c.nQHeads % c.nKVHeads) return false;
    if (c.batch < 0 || c.batch > kMaxBatch || c.total < 0 || c.max_seq < 0 || c.max_seq > c.total || c.prefix < 0) return false;
    if (c.total > 0x7fffffff - 1024 || c.prefix > 0x7fffffff - 1024 - c.total) return false;
    return c.stride_prefix == 0 || c.stride_prefix >= c.prefix;
}

int check_packed(const cdna4_packed_cfg* cfg, const cdna4_packed_strides* st, const void* Q, const void* K, const void* V,
                 const void* Kp, const void* Vp, const void* O, const int* cu, int dtype) {
    if (!cfg || !st || !valid_cfg(*cfg)) return CDNA4_ERR_INVALID_VALUE;
    const cdna4_packed_cfg& c = *cfg;
    if (dtype != CDNA4_F16 && dtype != CDNA4_BF16) return CDNA4_ERR_INVALID_VALUE;
    const long long in[4] = {st->q_row, st->q_head, st->kv_row, st->kv_head};
    for (long long x : in)
        if (x < 0 || (x & 7)) return CDNA4_ERR_INVALID_VALUE;
    const long long out[2] = {st->o_row, st->o_head};
    for (long long x : out)
        if (x < 0 || (x & 3)) return CDNA4_ERR_INVALID_VALUE;
    if (st->q_row < c.D || st->kv_row < c.D || st->o_row < c.D || (c.nQHeads > 1 && st->o_head < c.D)) return CDNA4_ERR_INVALID_VALUE;
    if (c.batch == 0 || c.total == 0) return 0;
    if (!Q || !K || !V || !O || !cu || ((uintptr_t)cu & 3u)) return CDNA4_ERR_INVALID_VALUE;
    if ((((uintptr_t)Q | (uintptr_t)K | (uintptr_t)V) & 15u) || ((uintptr_t)O & 7u)) return CDNA4_ERR_INVALID_VALUE;
    if (c.prefix > 0 && (!Kp || !Vp || (((uintptr_t)Kp | (uintptr_t)Vp) & 15u))) return CDNA4_ERR_INVALID_VALUE;
    return 0;
}

template <int D, bool kBf16>
int launch_packed(const cdna4_packed_cfg& c, const cdna4_packed_strides& st, const void* Q, const void* K, const void* V,
                  const void* Kp, const void* Vp, void* O, const int* cu, void* ws, hipStream_t s) {
    const PackedPlan p = plan_packed<D>(c, ws != nullptr, device_cus());
    if (p.items > kMaxItems) return CDNA4_ERR_INVALID_VALUE;
    PackedArgs a;
    a.Q = (const uint16_t*)Q; a.K = (const uint16_t*)K; a.V = (const uint16_t*)V; a.O = (uint16_t*)O;
    a.Kp = (const uint16_t*)Kp; a.Vp = (const uint16_t*)Vp;
    a.cu = cu;
    a.q_rs = st.q_row; a.q_hs = st.q_head; a.k_rs = st.kv_row; a.k_hs = st.kv_head; a.o_rs = st.o_row; a.o_hs = st.o_head;
    a.p_hs = (long long)(c.stride_prefix ? c.stride_prefix : c.prefix) * D;
    a.nQH = c.nQHeads; a.G = c.nQHeads / c.nKVHeads; a.batch = c.batch; a.total = c.total; a.prefix = c.prefix; a.hp = p.hp; a.single = p.order == kDealt && p.grid == p.items;
    a.copy32 = 256 * st.kv_row * 2 < (1LL << 32) ? 1 : 0;
    a.sc = kLog2e / sqrtf((float)D);
    const unsigned grid = (unsigned)p.grid;
    a.head = nullptr;
    a.items = nullptr;
    a.max_items = (int)p.items;   // up to kMaxItems
    a.split = nullptr;
    a.cut = nullptr;
    a.part_ml = a.part_o = nullptr;
    if constexpr (D == 128) {
        if (p.order == kFromList) {
            a.head = (ListHead*)ws;
            a.items = (int4*)(a.head + 1);
            packed_list<<<1, 1024, 0, s>>>(a, (int)(grid >> 3));
            if (c.prefix) fa_packed<D, 2, kBf16, true, kFromList><<<grid, 256, 0, s>>>(a);
            else fa_packed<D, 2, kBf16, false, kFromList><<<grid, 256, 0, s>>>(a);
            return launch_status();
        }
    }
    if (p.order == kDealtCut) {
        a.split = (Cut*)ws;
        a.cut = (int4*)((char*)ws + 256);
        a.part_o = (float*)((char*)a.cut + align256(p.cut * kItemBytes));
        a.part_ml = a.part_o + (size_t)p.parts * (64 * p.qt) * D;
        const unsigned join = (unsigned)(p.cut * (64 * p.qt) / (1024 / D));
        if (p.qt == 2) {
            fa_packed<D, 2, kBf16, true, kDealtCut><<<grid, 256, 0, s>>>(a);
            packed_join<D, 2, kBf16><<<join, 256, 0, s>>>(a);
        } else {
            fa_packed<D, 1, kBf16, true, kDealtCut><<<grid, 256, 0, s>>>(a);
            packed_join<D, 1, kBf16><<<join, 256, 0, s>>>(a);
        }
        return launch_status();
    }
    if (p.qt == 2) {
        if (c.prefix) fa_packed<D, 2, kBf16, true, kDealt><<<grid, 256, 0, s>>>(a);
        else fa_packed<D, 2, kBf16, false, kDealt><<<grid, 256, 0, s>>>(a);
    } else {
        if (c.prefix) fa_packed<D, 1, kBf16, true, kDealt><<<grid, 256, 0, s>>>(a);
        else fa_packed<D, 1, kBf16, false, kDealt><<<grid, 256, 0, s>>>(a);
    }
    return launch_status();
}

}  // namespace
}  // namespace cdna4

using namespace cdna4;

extern "C" int cdna4_attn_prefill_packed(const void* Q, const void* K, const void* V, const void* K_prefix,
                                         const void* V_prefix, void* O, const int* cu_seqlens, const cdna4_packed_cfg* cfg,
                                         const cdna4_packed_strides* strides, int dtype, void* workspace,
                                         size_t ws_bytes, cdna4_stream_t stream) {
    if (int e = check_packed(cfg, strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, dtype)) return e;
    if (cfg->batch == 0 || cfg->total == 0) return 0;
    if (workspace && (((uintptr_t)workspace & 15u) || ws_bytes < cdna4_attn_prefill_packed_workspace_size(cfg))) return CDNA4_ERR_INVALID_VALUE;
    if (int e = check_device()) return e;
    hipStream_t s = (hipStream_t)stream;
    const bool bf = dtype == CDNA4_BF16;
    if (cfg->D == 128)
        return bf ? launch_packed<128, true>(*cfg, *strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, workspace, s)
                  : launch_packed<128, false>(*cfg, *strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, workspace, s);
    return bf ? launch_packed<64, true>(*cfg, *strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, workspace, s)
              : launch_packed<64, false>(*cfg, *strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, workspace, s);
}

extern "C" size_t cdna4_attn_prefill_packed_workspace_size(const cdna4_packed_cfg* cfg) {
    cdna3_plan_info info;
    return cdna4_attn_prefill_packed_plan(cfg, CDNA4_F16, &info) == 0 ? info.workspace : 0;
}

extern "C" int cdna4_attn_prefill_packed_plan(const cdna4_packed_cfg* cfg, int dtype, cdna3_plan_info* out) {
    if (!cfg || !out) return CDNA4_ERR_INVALID_VALUE;
    const cdna4_packed_cfg& c = *cfg;
    if (!valid_cfg(c) || c.batch < 1 || c.total < 1 || (dtype != CDNA4_F16 && dtype != CDNA4_BF16)) return CDNA4_ERR_INVALID_VALUE;
    const PackedPlan p = c.D == 128 ? plan_packed<128>(c, true, device_cus()) : plan_packed<64>(c, true, device_cus());
    if (p.items > kMaxItems) return CDNA4_ERR_INVALID_VALUE;
    out->kernel = CDNA4_KERNEL_PACKED;
    out->waves = block::kWaves;
    out->rows = p.rows;
    out->grid = p.grid;
    out->partials = 1;
    out->workspace = p.ws_bytes;
    return 0;
}
