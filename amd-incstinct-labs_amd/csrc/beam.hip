// Beam search's selection (gfx950): the n best continuations of each group of beams over beams x vocabulary.
//
//   score = cum[row] + x_v - log sum_u e^(x_u) = cum[row] + (x_v - M) - log S,  M = max x, S = sum_u e^(x_u - M)
//
// Within a row the order of the scores is that of the logits, so one pass over them finds both a row's (M, S) and its n best.
// Launch 1: a wave takes a range of a row. Its lanes hold the running (m, s) of what they read, and the range's best keys so
// far sorted over the lanes (n <= 64), key = (logit's order, lowest token first) in 64 bits. What is above the n-th best key of
// the list, or of a first bound for it, is inserted one by one: random logits need that about n ln(range / n) times; of equal ones, or
// a mask of a finite value, the first step's some hundred times, the others' never (45-48 us for the batch below, 26 of random ones); logits that
// rise from token to token more in every step (200).
// Launch 2: a workgroup takes a group: (M, S) and the n best of each row from its ranges, scores in fp64, the n best of those.
// 256 rows of 100,003 bf16 logits, n = 16 (51 MB): 18-19 us, of which the reads alone take 14 (3.7 TB/s; all waves start at once and have 12 KB
// each) and the insertions most of the rest, and 6.6 in the second launch, a chain of loads, ranks and fp64 functions. Four rows of
// 32,000: 5.2 + 4.5.
#include <algorithm>
#include <math.h>
#include <type_traits>

#include "common.hpp"
#include "wave_primitives/detail/xlane.hpp"

namespace cdna4 {
namespace {

using wave::xlane::allreduce;
using wave::xlane::Max;
using wave::xlane::Min;
using wave::xlane::Sum;

typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));   // rows of odd length start anywhere

constexpr int kMost = 64;      // beams of a group, continuations of a group
constexpr int kValues = 32;    // logits of a lane at a time
template <int kDtype> constexpr int vec() { return kDtype == CDNA4_F32 ? 4 : 8; }   // logits of a load: 16 bytes
constexpr int kStep = 64 * kValues;                                                   // logits of a wave at a time
constexpr float kLowest = -3.402823466e38f, kLargest = 3.402823466e38f;

struct RangeSum { double s; float m; int pad; };   // sum of e^(x - m) over a range

struct BeamArgs {
    cdna4_beam_args p;
    int parts, range;        // ranges of a row, logits of a range (a multiple of 8)
    uint64_t* keys;          // [rows][n][parts], 0: none
    RangeSum* sums;          // [rows][parts]
};

// A finite float's order as an unsigned number above 0, and back.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t o) {
    return f32_from_bits(o ^ (o >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float x, int token) {
    // -0 and 0 are one value
    return (uint64_t)order_of(x + 0.f) << 32 | (uint32_t)~token;
}

__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}

// The list's lanes hold keys in descending order; a new key takes its place and moves those below by one lane.
__device__ __forceinline__ uint64_t insert(uint64_t list, uint64_t key, int lane) {
    const int at = __popcll(__builtin_amdgcn_ballot_w64(list > key));
    constexpr int kWaveShr1 = 0x138;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)list, kWaveShr1, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(list >> 32), kWaveShr1, 0xf, 0xf, false);
    return lane < at ? list : lane == at ? key : (uint64_t)hi << 32 | lo;
}

// The n-th largest of the lanes' values: the least of those that fewer than n are above. 700 cycles; bit by bit from the top, a
// ballot each, it took 3,000.
__device__ __forceinline__ uint32_t nth_largest(uint32_t v, int n) {
    int above = 0;
#pragma unroll
    for (int l = 0; l < 64; ++l) above += (uint32_t)__builtin_amdgcn_readlane((int)v, l) > v ? 1 : 0;
    return allreduce(above < n ? v : 0xffffffffu, Min{});
}

// Keys of a lane into the list, those whose order reaches `least` and that of the n-th best so far, one by one.
// top: the order of the lane's largest; key_at(k): its k-th key; reaches(b): a test of whether the k-th is of order b or more. Of
// kCount keys the first `count` are looked at, a multiple of 8. behind: all of them are of higher tokens than the list's, so that equal
// logits come after n of those.
template <int kCount, class KeyAt, class Reaches>
__device__ __forceinline__ uint64_t merge(uint64_t list, int n, uint32_t least, uint32_t top, KeyAt key_at, Reaches reaches, int lane, int count = kCount,
                                          bool behind = false) {
    const uint64_t nth = read_lane(list, n - 1);
    const uint32_t bound = max(max(least, (uint32_t)(nth >> 32) + (behind ? 1u : 0u)), order_of(kLowest));
    const uint64_t lanes = __builtin_amdgcn_ballot_w64(top >= bound);
    if (!lanes) return list;
    const auto test = reaches(bound);
    auto take = [&](auto many) {
#pragma unroll
        for (int k = 0; k < kCount; ++k) {
            if (k % 8 == 0 && k >= count) break;
            uint64_t need = __builtin_amdgcn_ballot_w64(test(k));
            if (!need) continue;
            const uint64_t key = key_at(k);
            if constexpr (decltype(many)::value) need &= __builtin_amdgcn_ballot_w64(key > read_lane(list, n - 1));
            while (need) {   // a key that is none of the n best goes behind them, or past the last lane
                list = insert(list, read_lane(key, __builtin_ctzll(need)), lane);
                need &= need - 1;
            }
        }
    };
    // Where most lanes have some, equal or rising logits may be nearly all that they have: each of the lanes' keys is then held against the
    // list as it has become. 256 flat rows of 100,003, n = 16, take 48 us so, 823 without; looking at every time took 26.4 us of random rows for 25.5.
    if (__popcll(lanes) > 32) take(std::true_type{});
    else take(std::false_type{});
    return list;
}

__device__ __forceinline__ float logit(const cdna4_beam_args& p, int dtype, size_t at) {
    if (dtype == CDNA4_F32) return ((const float*)p.logits)[at];
    const uint32_t b = ((const uint16_t*)p.logits)[at];
    return dtype == CDNA4_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// NaN as -inf, +inf as the largest value.
__device__ __forceinline__ float cleaned(float x) { return x != x ? -INFINITY : fminf(x, kLargest); }

__device__ __forceinline__ bool has_own(const cdna4_beam_args& p, int row) {   // continuations from its logits
    const float c = p.cum[row];
    return !(p.done && p.done[row]) && c > -INFINITY && c < INFINITY;
}

// e^d for d <= 0. The constant's rounding (1.3e-8 of it) moves a sum by 1.3e-8 times the mean of -d, alike in all rows.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269502f); }

template <int kDtype>
__global__ __launch_bounds__(256) void beam_ranges(BeamArgs a) {
    constexpr int kVec = vec<kDtype>(), kLoads = kValues / kVec;
    const int lane = (int)(threadIdx.x & 63u);
    const long long item = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int row = (int)(item / a.parts), part = (int)(item % a.parts);
    if (row >= a.p.groups * a.p.beams) return;
    const bool own = has_own(a.p, row);   // waited for behind the first logits
    const int n = a.p.n, V = a.p.V;
    const size_t base = (size_t)row * a.p.logits_stride;
    // Ranges begin at multiples of 16 bytes, the first one up to a load before the row (51 MB of bf16 rows of odd length are read in 14 us
    // so, in 17 with loads that are not aligned). A vocabulary below a load is read one by one.
    const bool vectors = V >= kVec;
    const int back = vectors ? (int)(((uintptr_t)a.p.logits / (16 / kVec) + base) % kVec) : 0;
    const int begin = part * a.range - back, end = min(begin + a.range, V);
    // Where a workgroup's four ranges are one row's, its waves share a bound: n logits of theirs, a quarter in each, are no less than
    // the least of the waves' (n / 4)-th best so far. What the others have published may be old: a bound that is too low.
    __shared__ volatile uint32_t quarter[4];
    const bool shared = (a.parts & 3) == 0;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    float m = kLowest, s = 0.f;
    uint64_t list = 0;
    // A load that begins before the row or ends past the range is moved into it; the lane has those of its logits that were in its place.
    u32x4_u raw[kLoads];   // of the next step
    auto place = [&](int i0, int u) { return begin + i0 + (u * 64 + lane) * kVec; };
    auto first_of = [&](int i0, int u) { return max(min(place(i0, u), end - kVec), 0); };
    auto load = [&](int i0) {
        if (!vectors) return;
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const size_t at = base + first_of(i0, u);
            if constexpr (kDtype == CDNA4_F32) raw[u] = *(const u32x4_u*)((const float*)a.p.logits + at);
            else raw[u] = *(const u32x4_u*)((const uint16_t*)a.p.logits + at);
        }
    };
    // Logits that are NaN or +inf make the sum NaN: the range is then read once more with a look at each.
    load(0);
    if (!own) return;   // all waves of a shared row
    for (bool careful = false;; careful = true) {
        m = kLowest;
        s = 0.f;
        list = 0;
        if (careful) load(0);
        uint32_t least = 0;
        for (int i0 = 0; i0 == 0 || begin + i0 < end; i0 += kStep) {   // once also where the range is empty
            float x[kValues];
            int from[kLoads];   // the token of each load's first logit
            const bool more = begin + i0 + kStep <= end, edge = !more || begin + i0 < 0;
            // Logits of the step, lane by lane, in eights: a range's last step has fewer, and what a wave does goes by them.
            const int count = max(min(kValues, ((end - begin - i0 + 64 * kVec - 1) / (64 * kVec) * kVec + 7) & ~7), 8);
            const bool look = careful || !vectors;
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kLoads; ++u) {
                from[u] = vectors ? first_of(i0, u) : place(i0, u);
                if (u * kVec >= count) continue;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const uint32_t w = raw[u][kDtype == CDNA4_F32 ? e : e / 2];
                    x[u * kVec + e] = kDtype == CDNA4_F32 ? f32_from_bits(w)
                                    : kDtype == CDNA4_BF16 ? f32_from_bits(e & 1 ? w & 0xffff0000u : w << 16)
                                                           : f16_bits_to_f32(e & 1 ? w >> 16 : w & 0xffffu);
                }
                if (look) {
#pragma unroll
                    for (int e = 0; e < kVec; ++e) {
                        float& y = x[u * kVec + e];
                        if (!vectors) y = from[u] + e < V ? logit(a.p, kDtype, base + from[u] + e) : -INFINITY;
                        y = cleaned(y);
                    }
                }
                if (edge) {
                    const int own0 = place(i0, u), own1 = min(own0 + kVec, end);
#pragma unroll
                    for (int e = 0; e < kVec; ++e)
                        if (from[u] + e < own0 || from[u] + e >= own1) x[u * kVec + e] = -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < kVec; ++e) top = fmaxf(top, x[u * kVec + e]);
            }
            if (more) load(i0 + kStep);   // clamped to the end where the range ends with this step
            if (top > m) {
                s *= exp_of(m - top);
                m = top;
            }
#pragma unroll
            for (int u = 0; u < kLoads; ++u) {
                if (u * kVec >= count) continue;
#pragma unroll
                for (int e = 0; e < kVec; ++e) s += exp_of(x[u * kVec + e] - m);
            }
            const uint32_t top_order = order_of(cleaned(top) + 0.f);
            const bool share = shared && !careful;
            if (i0 == 0) {
                least = nth_largest(top_order, share ? (n + 3) / 4 : n);
                if (share) {
                    if (lane == 0) quarter[wave] = least;
                    __syncthreads();   // every wave of the workgroup comes here once: a row's four
                }
            }
            if (share) least = min(min(quarter[0], quarter[1]), min(quarter[2], quarter[3]));
            list = merge<kValues>(list, n, least, top_order,
                                  [&](int k) { return key_of(x[k], from[k / kVec] + k % kVec); },
                                  [&](uint32_t b) { return [&x, f = of_order(b)](int k) { return x[k] >= f; }; }, lane, count, i0 > 0);
            if (share) {
                const uint32_t best = (uint32_t)(read_lane(list, (n + 3) / 4 - 1) >> 32);
                if (lane == 0 && best > quarter[wave]) quarter[wave] = best;
            }
        }
        if (careful || !__builtin_amdgcn_ballot_w64(s != s)) break;
    }
    const float M = allreduce(m, Max{});
    const double S = allreduce((double)s * (double)exp_of(m - M), Sum{});
    if (lane < n) a.keys[((size_t)row * n + lane) * a.parts + part] = list;   // the ranges' best ones side by side
    if (lane == 0) a.sums[(size_t)row * a.parts + part] = RangeSum{S, M, 0};
}

__global__ __launch_bounds__(1024) void beam_join(BeamArgs a) {
    // Candidates that can be among the group's n best: no less, rounded to fp32, than the n-th largest of a sample that has the best of
    // each row, two to a lane where they are more than 64.
    __shared__ double score[kMost * kMost];
    __shared__ int token[kMost * kMost], place[kMost * kMost];   // place: row n + place in the row's list
    __shared__ uint32_t sample[2 * 64];
    __shared__ uint64_t best[16][64];   // of each wave
    __shared__ int filled;
    const int lane = (int)(threadIdx.x & 63u), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int waves = (int)blockDim.x >> 6, n = a.p.n, beams = a.p.beams, row0 = (int)blockIdx.x * beams;
    if (threadIdx.x == 0) filled = 0;
    const int each = max((n + beams - 1) / beams, 64 / beams);   // of a row in the sample: 128 in all at most
    for (int i = beams * each + (int)threadIdx.x; i < 128; i += (int)blockDim.x) sample[i] = 0;
    double held[kMost / 16];   // a wave has up to four rows (16 waves)
    int said[kMost / 16], where[kMost / 16];
#pragma unroll 1
    for (int b = wave; b < beams; b += waves) {
        const int row = row0 + b;
        // all that the row needs is on its way at once; what a row without continuations of its own left there is not used
        const float cum = a.p.cum[row];
        const int ended = a.p.done ? a.p.done[row] : 0;
        const RangeSum* sums = a.sums + (size_t)row * a.parts;
        const RangeSum first = sums[min(lane, a.parts - 1)];
        const uint64_t* keys = a.keys + (size_t)row * a.parts * n;
        const int all = a.parts * n;
        uint64_t key[4];
        auto load = [&](int i0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) key[k] = keys[min(i0 + 64 * k + lane, all - 1)];
        };
        load(0);
        double sc = -INFINITY;
        int tok = -1, rank = lane, i0 = 0;   // rank: a lane's place in the row
        uint64_t mine = 0;
        const bool fine = cum > -INFINITY && cum < INFINITY;
        if (ended) {
            if (lane == 0 && fine) {
                sc = cum;
                tok = a.p.eos;
            }
        } else if (fine) {
            rank = 0;
            float M = first.m;
            for (int i = lane + 64; i < a.parts; i += 64) M = fmaxf(M, sums[i].m);
            M = allreduce(M, Max{});
            double S = lane < a.parts ? first.s * exp((double)first.m - (double)M) : 0.0;
            for (int i = lane + 64; i < a.parts; i += 64) S += sums[i].s * exp((double)sums[i].m - (double)M);
            S = allreduce(S, Sum{});
            // The keys that reach the n-th best of the lanes' largest, a few more than n as a rule: each lane takes one and counts
            // those before it. Where they are more than 64 (equal logits), or the row's keys more than a load, into a list one by one.
            auto tops = [&]() {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (64 * k + lane >= all - i0) key[k] = 0;
                return (uint32_t)(max(max(key[0], key[1]), max(key[2], key[3])) >> 32);
            };
            const uint32_t least = max(nth_largest(tops(), n), order_of(kLowest));
            int count = 0;
            if (all <= 256) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t in = __builtin_amdgcn_ballot_w64((uint32_t)(key[k] >> 32) >= least);
                    const int at = count + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0u));
                    if ((in >> lane & 1) && at < 64) best[wave][at] = key[k];
                    count += __popcll(in);
                }
            }
            if (all <= 256 && count <= 64) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the other lanes' keys
                __builtin_amdgcn_wave_barrier();
                mine = lane < count ? best[wave][lane] : 0;
#pragma unroll 4
                for (int j = 0; j < count; ++j) rank += best[wave][j] > mine ? 1 : 0;
            } else {
                for (;;) {
                    // a range's keys stand in descending order, `parts` apart: none here, none from here on
                    const uint32_t nth = max(least, (uint32_t)(read_lane(mine, n - 1) >> 32));
                    if (a.parts <= 256 && !__builtin_amdgcn_ballot_w64(tops() >= nth)) break;
                    mine = merge<4>(mine, n, least, tops(), [&](int k) { return key[k]; },
                                    [&](uint32_t b) { return [&key, b](int k) { return (uint32_t)(key[k] >> 32) >= b; }; }, lane);
                    i0 += 256;
                    if (i0 >= all) break;
                    load(i0);
                }
                rank = lane;
            }
            if (mine) {
                sc = (double)cum + ((double)of_order((uint32_t)(mine >> 32)) - (double)M) - log(S);
                tok = (int)~(uint32_t)mine;
            }
        }
        for (int i = lane; i < each; i += 64) sample[b * each + i] = 0;
        __builtin_amdgcn_wave_barrier();
        if (tok >= 0 && rank < each) sample[b * each + rank] = order_of((float)sc + 0.f);
        held[b / waves] = sc;   // of the rows that this wave has
        said[b / waves] = rank < n ? tok : -1;
        where[b / waves] = b * n + rank;
    }
    __syncthreads();
    const uint32_t least = nth_largest(max(sample[lane], sample[lane + 64]), n);
    for (int b = wave; b < beams; b += waves) {
        const bool in = said[b / waves] >= 0 && order_of((float)held[b / waves] + 0.f) >= least;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(in);
        int at = 0;
        if (lane == 0) at = atomicAdd(&filled, __popcll(mask));
        at = __builtin_amdgcn_readfirstlane(at) + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
        if (in) {
            score[at] = held[b / waves];
            token[at] = said[b / waves];
            place[at] = where[b / waves];
        }
    }
    __syncthreads();
    // A candidate's place is the number of those before it, by score, then by row and place in the row's list: eight lanes count.
    const int all = filled, sub = (int)threadIdx.x & 7;
    for (int i = (int)threadIdx.x >> 3; i < all; i += (int)blockDim.x >> 3) {
        const double sc = score[i];
        const int pl = place[i];
        int rank = 0;
#pragma unroll 4
        for (int j = sub; j < all; j += 8) {
            const double o = score[j];
            rank += o > sc || (o == sc && place[j] < pl) ? 1 : 0;
        }
        rank += wave::xlane::dpp_full<wave::xlane::kQuadXor1>(rank);
        rank += wave::xlane::dpp_full<wave::xlane::kQuadXor2>(rank);
        rank += wave::xlane::dpp_full<wave::xlane::kRowHalfMirror>(rank);
        if (sub == 0 && rank < n) {
            const size_t at = (size_t)blockIdx.x * n + rank;
            a.p.scores[at] = (float)sc;
            a.p.parents[at] = row0 + pl / n;
            a.p.tokens[at] = token[i];
        }
    }
    for (int i = all + (int)threadIdx.x; i < n; i += (int)blockDim.x) {   // places that nothing fills
        const size_t at = (size_t)blockIdx.x * n + i;
        a.p.scores[at] = -INFINITY;
        a.p.parents[at] = -1;
        a.p.tokens[at] = -1;
    }
}

// Ranges of a row: enough of them for sixteen waves per CU, none shorter than 1,024 logits.
struct BeamPlan { int parts, range; size_t ws_bytes; };

bool plan_beam(long long rows, int V, int beams, int n, BeamPlan& p) {
    if (rows < 0 || rows >= 1 << 24 || V < 1 || V > 0x7fffffff - 65536 || beams < 1 || beams > kMost || n < 1 || n > kMost) return false;
    // four waves of a workgroup on one row, unless it is short: they share a bound
    p.parts = 1;
    if (V >= 4096) p.parts = (int)std::max(4LL, std::min<long long>(V / 1024, rows ? 16LL * device_cus() / rows : 1) & ~3LL);
    p.range = (int)(((long long)V + 7 + p.parts - 1) / p.parts + 7) & ~7;   // from up to 7 before the row; the last ranges may be empty
    p.ws_bytes = (size_t)rows * p.parts * (n * sizeof(uint64_t) + sizeof(RangeSum)) + 16;
    return (rows * p.parts + 3) / 4 * 256 <= 0xffffffffLL;
}

int check_beam(const cdna4_beam_args* a, int dtype) {
    if (!a) return CDNA4_ERR_INVALID_VALUE;
    if (dtype != CDNA4_F32 && dtype != CDNA4_F16 && dtype != CDNA4_BF16) return CDNA4_ERR_INVALID_VALUE;
    if (a->groups < 0 || a->logits_stride < a->V) return CDNA4_ERR_INVALID_VALUE;
    if (a->done && (a->eos < 0 || a->eos >= a->V)) return CDNA4_ERR_INVALID_VALUE;
    if (a->groups == 0) return 0;
    const uintptr_t el = dtype == CDNA4_F32 ? 3u : 1u;
    if (!a->logits || ((uintptr_t)a->logits & el)) return CDNA4_ERR_INVALID_VALUE;
    const void* words[5] = {a->cum, a->scores, a->parents, a->tokens, a->done};
    for (int i = 0; i < 5; ++i)
        if ((i < 4 && !words[i]) || ((uintptr_t)words[i] & 3u)) return CDNA4_ERR_INVALID_VALUE;
    // a group's scores in the place of its own cum alone: other groups' workgroups read theirs meanwhile
    if (a->scores == a->cum && a->n != a->beams) return CDNA4_ERR_INVALID_VALUE;
    return 0;
}

}  // namespace
}  // namespace cdna4

using namespace cdna4;

extern "C" size_t cdna4_beam_select_workspace_size(int rows, int V, int beams, int n) {
    BeamPlan p;
    return plan_beam(rows, V, beams, n, p) ? p.ws_bytes : 0;
}

extern "C" int cdna4_beam_select(const cdna4_beam_args* args, int dtype, void* workspace, size_t ws_bytes, cdna4_stream_t stream) {
    if (int e = check_beam(args, dtype)) return e;
    const cdna4_beam_args& p = *args;
    BeamPlan plan;
    if (!plan_beam((long long)p.groups * p.beams, p.V, p.beams, p.n, plan)) return CDNA4_ERR_INVALID_VALUE;
    if (p.groups == 0) return 0;
    if (!workspace || ((uintptr_t)workspace & 15u) || ws_bytes < plan.ws_bytes) return CDNA4_ERR_INVALID_VALUE;
    if (int e = check_device()) return e;
    hipStream_t s = (hipStream_t)stream;
    BeamArgs a;
    a.p = p;
    a.parts = plan.parts;
    a.range = plan.range;
    a.sums = (RangeSum*)workspace;
    a.keys = (uint64_t*)(a.sums + (size_t)p.groups * p.beams * plan.parts);
    const unsigned grid = ceil_div((size_t)p.groups * p.beams * plan.parts, 4);
    if (dtype == CDNA4_F32) beam_ranges<CDNA4_F32><<<grid, 256, 0, s>>>(a);
    else if (dtype == CDNA4_BF16) beam_ranges<CDNA4_BF16><<<grid, 256, 0, s>>>(a);
    else beam_ranges<CDNA4_F16><<<grid, 256, 0, s>>>(a);
    if (int e = launch_status()) return e;
    const int waves = std::max(4, std::min(16, p.beams));
    beam_join<<<(unsigned)p.groups, 64 * waves, 0, s>>>(a);
    return launch_status();
}
