// Decode attention over a paged KV cache (gfx950): nq queries per sequence, the last nq tokens', over the sequence's pages, whose
// rows are 16-bit or MXFP4.
//
//   o[b][i][h] = sum_j 2^(c q.k_j - m) v_j / sum_j 2^(c q.k_j - m),  j < lens[b] - nq + 1 + i,  c = log2(e) / sqrt(D)
//
// The G query heads of a kv head, times the nq queries, are the rows of one matrix product, kRT tiles of 16 rows at most ("row
// block"); a row block and a sequence's keys are one item, its keys are cut into chunks of 32. Two forms:
//   - Short tables (choose_waves): a workgroup of one to eight waves per item, joined in LDS, one launch.
//   - Others: all chunks of all items lie on one axis, items of a sequence side by side, and every wave takes an equal share of
//     it: lengths are read on the device, and what a wave has to do does not depend on how they differ. A share that holds all
//     chunks of an item writes the output; of an item that shares cut, each leaves (m, l, O), and a second launch joins them,
//     o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p.
// Weights go into P.V as two terms of the inputs' 16-bit type, 16 (bf16) or 22 bits of each, and are added up as they go, in fp32: an
// output is then off by its own rounding. With one term its error is 1.1 to 1.4 times that, over any number of keys, and the time the same
// within 2 %: 148.4 against 148.6 us (128 sequences of 500-4,096 in bf16), 39.8 against 40.5 (two row tiles), 53.7 against 54.7 and
// 24.9 against 23.9 (MXFP4; there the branch that gave only the first keys a second term spilled registers). MXFP4 values are decoded to
// the 16-bit type exactly.
// More than 32 rows of a kv head (nq G) are items of their own, and each reads the keys again: 16 sequences of 8,000 16-bit keys of one
// head (66 MB), D 128, in the first launch: 20 rows 20.5 us, 32 rows 21.2, 64 rows 27.6 (134 MB read), 160 rows 56.5 (333 MB).
// Bound by HBM where there are keys enough: 128 sequences of 500-4,096 bf16 keys, 32/8 heads, D 128 (902 MB) 141-145 us in the first launch,
// 6.3 TB/s, and 4.4 in the join; three of 30,000-131,072 in MXFP4 (267 MB) 47-54 and 6.2-7.4. A share's start (its place 1.1 us, its pages'
// entries 0.5, its first keys 1.4: three loads behind one another) and the join's are most of a short call: 64 sequences of 20-4,000
// in MXFP4 (57 MB) take 19-21 + 4.5 us, where a wave has five chunks of 1.5 us each (half of the waves end 11.4 us after the first one's start,
// 95 % after 13.6, the last, with many short sequences, after 18). One launch of four sequences of up to 545 keys, 12 heads, D 64: 5.8.
#include <algorithm>
#include <math.h>

#include "attn_stream.hpp"
#include "paged.hpp"

namespace cdna4 {
namespace {

using namespace tile;
using namespace paged;
using wave::xlane::allreduce;
using wave::xlane::Max;
using wave::xlane::Sum;

constexpr int kKeys = 32;         // keys of a chunk
constexpr int kMinChunks = 2;     // a share's chunks at least
constexpr int kMaxParts = 512;    // shares that an item is cut into, but for the two at its ends

struct PagedArgs {
    const uint16_t* q;
    const char *K, *V;
    const int *tables, *lens;
    uint16_t* o;
    long long* head;      // [0]: chunks of a share; [1 + b]: chunks before sequence b
    float *part_ml, *part_o;   // [share][2][rows][2], [share][2][rows][D]: of the item that begins before the share, of its last
    long long table_stride;
    int nQH, HK, G, nq, batch, rows;   // rows of a row block
    int HB, items;                     // row blocks per kv head, items per sequence
    int page, lp, pages, max_len;
    uint32_t head_bytes, page_bytes;   // of a pool's page: one head's, all heads' (below 2^31)
    int shares;
    float sc;
};

__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long scalar(long long x) {
    return (long long)((uint64_t)(uint32_t)scalar((int)(x >> 32)) << 32 | (uint32_t)scalar((int)x));
}
// No branch, and nothing for the compiler to know of the lanes past the batch: with a branch here it follows "0 there" through ballots
// into loops of their own for these lanes, which then take no part in the wave's copies. tests/test_paged_waves.py follows the masks
// through the compiled kernels.
__device__ __forceinline__ int length_of(const PagedArgs& a, int b) {
    int len = min(max(a.lens[min(b, a.batch - 1)], 0), a.max_len);
    len = b < a.batch ? len : 0;
    asm volatile("" : "+v"(len));
    return len;
}
__device__ __forceinline__ int chunks_of(int len) { return (len + kKeys - 1) / kKeys; }

// Quotients of numbers that are nearly always below 2^32, where a division takes a third of the time.
__device__ __forceinline__ long long quotient(long long x, long long y) {
    if (((uint64_t)x | (uint64_t)y) >> 32 == 0) return (long long)((uint32_t)x / (uint32_t)y);
    return x / y;
}

// Where a wave stands: sequence b of len keys, `before` chunks of one item in the sequences before it.
struct Place { int b, len; long long before; };

// Lengths of 64 sequences, one per lane, from sequence `first` on.
struct Window {
    int first, len;
    __device__ __forceinline__ void load(const PagedArgs& a, int f, int lane) {
        first = f;
        len = length_of(a, f + lane);
    }
};

// What a share holds: chunks begin .. end - 1 of the axis, the first of them in sequence `at`.
struct Share { long long per, begin, end; Place at; };

// Equal shares of all chunks, but none below kMinChunks, and no item in more than about kMaxParts: each lane counts the chunks of a
// run of sequences, a scan over the lanes finds the one in whose run the share begins, and so on within that run.
__device__ __forceinline__ Share share_of(const PagedArgs& a, int share, Window& w, int lane) {
    int lo = 0, n = a.batch, most = 0;
    long long x = 0, before = 0;
    Share s{0, 0, 0, Place{0, 0, 0}};
    for (bool first = true;; first = false) {
        const int step = (n + 63) / 64;   // sequences of a lane
        long long c = 0;
        if (step == 1) {
            w.load(a, lo, lane);
            if (lane < n) c = chunks_of(w.len);
            most = max(most, (int)c);
        } else {
            for (int i = 0; i < step; ++i) {
                const int at = lane * step + i, m = at < n ? chunks_of(length_of(a, lo + at)) : 0;
                c += m;
                most = max(most, m);
            }
        }
        const long long upto = wave::xlane::scan_inclusive(c, Sum{}) + before;
        if (first) {
            const long long all = scalar(__shfl(upto, 63)) * a.items;
            most = scalar(allreduce(most, Max{}));
            s.per = max(quotient(all + a.shares - 1, a.shares), (long long)max(kMinChunks, (most + kMaxParts - 1) / kMaxParts));
            s.begin = share * s.per;
            s.end = min(s.begin + s.per, all);
            if (s.begin >= s.end) return s;
            x = quotient(s.begin, a.items);
        }
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > x));   // some lane's is: x lies below the run's end
        before = scalar(__shfl(upto - c, l));
        lo += l * step;
        if (step == 1) {
            s.at = Place{lo, __builtin_amdgcn_readlane(w.len, l), before};
            return s;
        }
        n = min(step, n - l * step);
    }
}

// Pages of a sequence, 64 table entries at a time, one per lane; entries past its rows are not read.
struct Pages {
    int first, ids;
    __device__ __forceinline__ void load(const PagedArgs& a, int b, int len, int f, int lane) {
        first = f;
        const int* table = a.tables + b * a.table_stride;
        ids = min(max(table[min(f + lane, (len - 1) >> a.lp)], 0), a.pages - 1);
    }
};

// Where the 16 rows of a head from key k on begin in the pools, k the same in every lane and its entry among the loaded ones. Rows past
// the last one lie in its page or, past that, in some page of the sequence: they are read and come to nothing.
__device__ __forceinline__ size_t rows_at(const PagedArgs& a, const Pages& pg, int k, int kvh, int row_bytes) {
    const uint32_t id = (uint32_t)__builtin_amdgcn_readlane(pg.ids, (k >> a.lp) - pg.first);
    return (size_t)id * a.page_bytes + ((uint32_t)kvh * a.head_bytes + (uint32_t)((k & (a.page - 1)) * row_bytes));
}

// One chunk's K and V rows into a ring stage (K first), 16-bit rows. A chunk lies in one page, or, with pages of 16 rows, in two: the copies
// take their bases from the scalar unit, and a lane's offset within them differs from copy to copy by the swizzle alone.
template <int D, bool kNT>
__device__ __forceinline__ void copy_chunk(const PagedArgs& a, const Pages& pg, int kb, int kvh, uint16_t* stage, int lane) {
    constexpr int CPR = D / 8, NI = kKeys * CPR / 64, kRows = 64 / CPR;   // copies of K, rows of a copy
    uint16_t* const vstage = stage + kKeys * D;
    size_t at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) at[h] = rows_at(a, pg, scalar(kb) + 16 * h, scalar(kvh), 2 * D);
    const int r = lane / CPR, c = lane % CPR;
    const uint32_t ko = (uint32_t)(r * 2 * D + (c ^ swz_k<D>(r)) * 16), vo = (uint32_t)(r * 2 * D + (c ^ swz_v<D>(r)) * 16);
#pragma unroll
    for (int j = 0; j < NI; ++j)
        stream::dma16_s<kNT>(a.K + at[j / (NI / 2)] + j % (NI / 2) * 1024, ko ^ (uint32_t)(swz_k<D>(j * kRows) << 4), stage + j * 512);
#pragma unroll
    for (int j = 0; j < NI; ++j)
        stream::dma16_s<kNT>(a.V + at[j / (NI / 2)] + j % (NI / 2) * 1024, vo ^ (uint32_t)(swz_v<D>(j * kRows) << 4), vstage + j * 512);
}

// V rows of a chunk from the `live`-th on, which may hold anything: zeros, since their weights of zero do not undo what is not finite.
template <int D>
__device__ __forceinline__ void clear_rows(uint16_t* vstage, int live, int lane) {
#pragma unroll
    for (int j = 0; j < kKeys * D / 512; ++j)
        if ((j * 64 + lane) / (D / 8) >= live) *(u32x4*)(vstage + (j * 64 + lane) * 8) = u32x4{0u, 0u, 0u, 0u};
}

// MXFP4 rows in registers. K: lane (li, g) holds its g-th quarter of the rows that it has in the two K operand tiles, D / 4
// values that lie in one block; operand c is 8 of them, so query operands take the same D / 4 g + 8 c. V: blocks of 32 values,
// lane by lane in the order of memory.
template <int D>
struct Codes {
    static constexpr int KW = D / 32;            // dwords of a quarter row
    static constexpr int VB = kKeys * D / 2048;  // blocks of V per lane
    uint32_t k[2][KW];
    u32x4 v[VB];
    uint32_t ks[2], vs[VB];
};

template <int D, bool kNT>
__device__ __forceinline__ void load_codes(const PagedArgs& a, const Pages& pg, int kb, int kvh, Codes<D>& x, int lane) {
    const int li = lane & 15, g = lane >> 4;
    constexpr int KW = Codes<D>::KW, VB = Codes<D>::VB, BPR = D / 32;   // blocks of a row
    auto get = [&](auto* p) {
        if constexpr (kNT) return __builtin_nontemporal_load(p);
        else return *p;
    };
    using KV = uint32_t __attribute__((ext_vector_type(KW)));
    // the first row of each half of the chunk: its codes, its scales
    size_t at[2], sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = scalar(kb) + 16 * h;
        const size_t head = rows_at(a, pg, k, scalar(kvh), 0);
        const uint32_t row = (uint32_t)(k & (a.page - 1));
        at[h] = head + row * (D / 2);
        sc[h] = head + ((uint32_t)a.page * (D / 2) + row * BPR);
    }
    // K rows 8 (li / 4) + li % 4 + 4 u: lanes li < 8 in the first half of the chunk
    const int kr = 8 * (li >> 2 & 1) + (li & 3);
    const char *kc = a.K + (li < 8 ? at[0] : at[1]), *ksc = a.K + (li < 8 ? sc[0] : sc[1]);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const KV w = get((const KV*)(kc + ((kr + 4 * u) * (D / 2) + g * (D / 8))));
#pragma unroll
        for (int i = 0; i < KW; ++i) x.k[u][i] = w[i];
        x.ks[u] = *(const uint8_t*)(ksc + ((kr + 4 * u) * BPR + g * BPR / 4));
    }
    // V rows (64 j + lane) / BPR: copy j of D 128 is half j, lanes below 32 of D 64 are the first half
#pragma unroll
    for (int j = 0; j < VB; ++j) {
        const int r = (64 * j + lane) / BPR;
        const bool second = VB == 2 ? j == 1 : lane >= 32;
        const char *vc = a.V + (second ? at[1] : at[0]), *vsc = a.V + (second ? sc[1] : sc[0]);
        x.v[j] = get((const u32x4*)(vc + ((r & 15) * (D / 2) + lane % BPR * 16)));
        x.vs[j] = *(const uint8_t*)(vsc + ((r & 15) * BPR + lane % BPR));
    }
}

template <bool kBf16>
__device__ __forceinline__ u32x4 decode8(uint32_t c, float scale) {
    return u32x4{decode2<kBf16, 0>(c, scale), decode2<kBf16, 1>(c, scale), decode2<kBf16, 2>(c, scale), decode2<kBf16, 3>(c, scale)};
}

// Scores that a row must not see are masked by the row's own limit.
template <int RT>
__device__ __forceinline__ bool check_limits(f32x4 (&s)[RT][2], const float (&m)[RT], float (&lm)[RT], int kb, const int (&limit)[RT],
                                             bool mask, float sc, int g) {
    if (mask) {
        asm volatile("");   // a branch of its own: the compiler has put the masks of every chunk into its arithmetic
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (kb + g * 8 + u * 4 + e >= limit[t]) s[t][u][e] = -INFINITY;
    }
    bool need = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float v = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) v = fmaxf(v, s[t][u][e]);
        lm[t] = v;
        need |= v * sc > m[t] + kTau;
    }
    return need;
}

// Weights p = 2^(s sc - m) as two 16-bit terms each, hi = round(p), lo = round(p - hi) (p - hi is exact in fp32), packed into the B
// operands of the P.V product.
template <int RT, bool kBf16>
__device__ __forceinline__ void two_terms(const f32x4 (&s)[RT][2], const float (&m)[RT], u32x4 (&hi)[RT], u32x4 (&lo)[RT], float sc) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[t][x >> 1][(x & 1) * 2], sc, -m[t]));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[t][x >> 1][(x & 1) * 2 + 1], sc, -m[t]));
            const uint32_t h = pack2<kBf16>(p0, p1);
            hi[t][x] = h;
            if constexpr (kBf16) lo[t][x] = pack2<true>(p0 - f32_from_bits(h << 16), p1 - f32_from_bits(h & 0xffff0000u));
            else lo[t][x] = pack2<false>(p0 - f16_bits_to_f32(h & 0xffffu), p1 - f16_bits_to_f32(h >> 16));
        }
}

// Waves that a CU holds: 16-bit rows as many as have a ring in its LDS, MXFP4 as the registers allow.
constexpr int waves_per_cu(int D, int RT, bool fp4) { return fp4 ? (RT == 2 ? 8 : D == 128 ? 12 : 16) : D == 128 ? 4 : 8; }

// LDS of a wave, elements. 16 bits: a ring of two chunks of K and V. MXFP4: one chunk of V as 16-bit values.
template <int D> constexpr int stage_elems() { return 2 * kKeys * D; }
template <int D, bool kFp4> constexpr int wave_lds() { return kFp4 ? kKeys * D : 2 * stage_elems<D>(); }

// A row block in a wave: queries, running maxima, sums and outputs. Row r of a kv head: query r / G, head kvh G + r % G.
template <int D, int RT, bool kBf16, bool kFp4>
struct RowBlock {
    static constexpr int ND = D / 32, NDT = D / 16;
    using Queries = u32x4[RT][ND];
    const PagedArgs& a;
    const int lane, li, g, R;
    const LdsOffsets off;
    Queries q;
    int limit[RT];
    f32x4 o[RT][NDT], lacc[RT];
    float m[RT];

    __device__ __forceinline__ RowBlock(const PagedArgs& args, int l)
        : a(args), lane(l), li(l & 15), g(l >> 4), R(args.nq * args.G), off(lds_offsets<D>(l & 15, l >> 4)) {}

    __device__ __forceinline__ size_t row_of(int b, int kvh, int r) const {
        const int i = r / a.G;
        return (((size_t)b * a.nq + i) * a.nQH + (size_t)kvh * a.G + (r - i * a.G)) * D;
    }
    __device__ __forceinline__ void load_q(int b, int kvh, int hb, Queries& to) const {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const uint16_t* src = a.q + row_of(b, kvh, min(hb * RT * 16 + t * 16 + li, R - 1));   // rows past the last repeat it, unused
#pragma unroll
            for (int c = 0; c < ND; ++c) to[t][c] = *(const u32x4*)(src + (kFp4 ? g * (D / 4) + c * 8 : c * 32 + g * 8));
        }
    }
    __device__ __forceinline__ void ready() {   // the compiler waits for the queries here
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            if constexpr (ND == 4) asm volatile("" : "+v"(q[t][0]), "+v"(q[t][1]), "+v"(q[t][2]), "+v"(q[t][3]));
            else asm volatile("" : "+v"(q[t][0]), "+v"(q[t][1]));
        }
    }
    __device__ __forceinline__ void begin(int len, int hb) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = hb * RT * 16 + t * 16 + li;
            limit[t] = r < R ? len - a.nq + 1 + r / a.G : len;
            m[t] = kInitM;
            lacc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < NDT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // scores of a chunk to weights, weights times V
    __device__ __forceinline__ void weigh(f32x4 (&s)[RT][2], int kb, int len, const char* Vt) {
        float lm[RT];
        const bool need = check_limits<RT>(s, m, lm, kb, limit, kb + kKeys > len - a.nq + 1, a.sc, g);
        if (__builtin_amdgcn_ballot_w64(need)) rescale_rows<D, RT>(lm, m, o, lacc, a.sc);
        u32x4 hi[RT], lo[RT];
        two_terms<RT, kBf16>(s, m, hi, lo, a.sc);
        const uint32_t one2 = kBf16 ? 0x3F803F80u : 0x3C003C00u;   // two 16-bit 1.0
        const u32x4 ones{one2, one2, one2, one2};
#pragma unroll
        for (int t = 0; t < RT; ++t) lacc[t] = mfma<kBf16>(ones, lo[t], mfma<kBf16>(ones, hi[t], lacc[t]));
#pragma unroll
        for (int d = 0; d < NDT; ++d) {
            const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(Vt + off.vd(d))));
            const u32x2 v1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(Vt + off.vd(d) + 4 * D * 2)));
            const u32x4 va{v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
            for (int t = 0; t < RT; ++t) o[t][d] = mfma<kBf16>(va, lo[t], mfma<kBf16>(va, hi[t], o[t][d]));
        }
    }
    // A chunk of 16-bit rows that is in a ring stage.
    __device__ __forceinline__ void use(uint16_t* stage, int kb, int len) {
        if (kb + kKeys > len) clear_rows<D>(stage + kKeys * D, len - kb, lane);
        f32x4 s[RT][2];
        qk_chunk<D, RT, kBf16>((const char*)stage, off, q, s, 0);
        weigh(s, kb, len, (const char*)(stage + kKeys * D));
    }
    // A chunk of codes; V's values go to LDS, where the P.V product reads them transposed.
    __device__ __forceinline__ void use(const Codes<D>& x, int kb, int len, uint16_t* vlds) {
#pragma unroll
        for (int j = 0; j < Codes<D>::VB; ++j) {
            const int r = (64 * j + lane) / ND, blk = lane % ND;
            // rows past the last: values of next to nothing whatever they hold, since their weights of zero do not undo what is not
            // finite; here and not at the load, which would wait for it
            uint32_t scale = x.vs[j];
            if (kb + kKeys > len && kb + r >= len) scale = 0;
            const float f = f32_from_bits(scale << 23);
#pragma unroll
            for (int i = 0; i < 4; ++i) *(u32x4*)(vlds + r * D + ((4 * blk + i) ^ swz_v<D>(r)) * 8) = decode8<kBf16>(x.v[j][i], f);
        }
        f32x4 s[RT][2];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) s[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float f = f32_from_bits(x.ks[u] << 23);
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                const u32x4 ka = decode8<kBf16>(x.k[u][i], f);
#pragma unroll
                for (int t = 0; t < RT; ++t) s[t][u] = mfma<kBf16>(ka, q[t][i], s[t][u]);
            }
        }
        weigh(s, kb, len, (const char*)vlds);
    }
    __device__ __forceinline__ void store(int b, int kvh, int hb) const {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = hb * RT * 16 + t * 16 + li;
            if (r >= R) continue;
            const float inv = lacc[t][0] > 0.f ? 1.f / lacc[t][0] : 1.f;
            uint16_t* dst = a.o + row_of(b, kvh, r) + g * 4;
#pragma unroll
            for (int d = 0; d < NDT; ++d) {
                ((uint32_t*)(dst + d * 16))[0] = pack2<kBf16>(o[t][d][0] * inv, o[t][d][1] * inv);
                ((uint32_t*)(dst + d * 16))[1] = pack2<kBf16>(o[t][d][2] * inv, o[t][d][3] * inv);
            }
        }
    }
    // (m, l, O) as they are: rows `first` on of ml and out, up to `rows` of them
    __device__ __forceinline__ void store_part(float* ml, float* out, size_t first, int rows) const {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            if (t * 16 + li >= rows) continue;
            const size_t idx = first + t * 16 + li;
            float* dst = out + idx * D + g * 4;
#pragma unroll
            for (int d = 0; d < NDT; ++d) *(f32x4*)(dst + d * 16) = o[t][d];
            if (g == 0) *(float2*)(ml + idx * 2) = make_float2(m[t], lacc[t][0]);
        }
    }
};

template <int D> constexpr int copies() { return 2 * kKeys * (D / 8) / 64; }   // of a chunk's K and V

// What a wave does next: chunks c0 .. c1 - 1 of an item's n, and the pages they begin in.
struct Segment { int b, len, kvh, hb, c0, c1, n; Pages pg; };

// The entries of chunk c's pages, loaded if they are not.
__device__ __forceinline__ void pages_for(const PagedArgs& a, Segment& s, int c, int lane) {
    const int last = ((c + 1) * kKeys - 1) >> a.lp;
    if (last - s.pg.first >= 64) s.pg.load(a, s.b, s.len, (c * kKeys) >> a.lp, lane);
}

// ---- equal shares of all keys -----------------------------------------------------------------------
template <int D, int RT, bool kBf16, bool kFp4, bool kNT>
__global__ __launch_bounds__(64, (waves_per_cu(D, RT, kFp4) + 3) / 4) void paged_parts(PagedArgs a) {
    __shared__ __attribute__((aligned(16))) uint16_t lds[wave_lds<D, kFp4>()];
    const int lane = (int)threadIdx.x, share = (int)blockIdx.x;
    Window w;
    const Share sh = share_of(a, share, w, lane);
    if (share == 0 && lane == 0) a.head[0] = sh.per;
    if (sh.begin >= sh.end) return;

    // The share's segments one after another; their table entries are loaded as they are found.
    // The same in every lane, as all that follows from it; the compiler is told, and keeps it in scalar registers.
    int left = scalar((int)(sh.end - sh.begin));   // chunks from the next segment on
    Place pl{scalar(sh.at.b), scalar(sh.at.len), scalar(sh.at.before)};
    int item, c_next;
    {
        const int n = chunks_of(pl.len);
        const long long in_seq = sh.begin - pl.before * a.items;
        item = scalar((int)quotient(in_seq, n));
        c_next = scalar((int)(in_seq - (long long)item * n));
    }
    auto next_segment = [&](Segment& s) {
        const int n = chunks_of(pl.len);
        s.b = pl.b;
        s.len = pl.len;
        s.kvh = item / a.HB;
        s.hb = item - s.kvh * a.HB;
        s.n = n;
        s.c0 = c_next;
        s.c1 = min(n, c_next + left);
        if (item == 0 && c_next == 0 && lane == 0) a.head[1 + pl.b] = pl.before;
        s.pg.load(a, s.b, s.len, (s.c0 * kKeys) >> a.lp, lane);
        left -= s.c1 - s.c0;
        c_next = 0;
        if (left > 0 && ++item == a.items) {   // on to the next sequence that has keys
            item = 0;
            pl.before += n;
            int l = pl.b + 1 - w.first;
            for (;;) {
                const uint64_t more = l < 64 ? __builtin_amdgcn_ballot_w64(w.len > 0 && lane >= l) : 0;
                if (more) {
                    l = scalar((int)__builtin_ctzll(more));
                    pl.b = scalar(w.first + l);
                    pl.len = __builtin_amdgcn_readlane(w.len, l);
                    break;
                }
                if (w.first + 64 >= a.batch) {   // not reached: chunks are left
                    left = 0;
                    break;
                }
                w.load(a, w.first + 64, lane);
                l = 0;
            }
        }
    };
    RowBlock<D, RT, kBf16, kFp4> rb(a, lane);
    Segment cur, nxt;
    bool more;   // nxt is there
    auto finish = [&]() {
        if (cur.c0 == 0 && cur.c1 == cur.n) rb.store(cur.b, cur.kvh, cur.hb);
        else rb.store_part(a.part_ml, a.part_o, ((size_t)share * 2 + (cur.c0 == 0 ? 1 : 0)) * a.rows, min(a.rows, rb.R - cur.hb * RT * 16));
    };
    next_segment(cur);
    if constexpr (kFp4) {
        // The next segment's pages are loaded a segment ahead, its first codes while the last ones of this are used.
        Codes<D> x, y;   // in turn: the next chunk's codes are on their way while one is used
        load_codes<D, kNT>(a, cur.pg, cur.c0 * kKeys, cur.kvh, x, lane);
        for (;;) {
            rb.load_q(cur.b, cur.kvh, cur.hb, rb.q);
            more = left > 0;
            if (more) next_segment(nxt);
            rb.begin(cur.len, cur.hb);
            auto ahead = [&](Codes<D>& z, int c) {
                if (c < cur.c1) {
                    pages_for(a, cur, c, lane);
                    load_codes<D, kNT>(a, cur.pg, c * kKeys, cur.kvh, z, lane);
                } else if (more) {
                    load_codes<D, kNT>(a, nxt.pg, nxt.c0 * kKeys, nxt.kvh, z, lane);
                }
            };
            bool in_y;   // where the next segment's codes are
            for (int c = cur.c0;; c += 2) {
                ahead(y, c + 1);
                rb.use(x, c * kKeys, cur.len, lds);
                in_y = c + 1 >= cur.c1;
                if (in_y) break;
                ahead(x, c + 2);
                rb.use(y, (c + 1) * kKeys, cur.len, lds);
                if (c + 2 >= cur.c1) break;
            }
            finish();
            if (!more) break;
            if (in_y) x = y;
            cur = nxt;
        }
    } else {
        // The copies go on across segments: the next one's first chunk is on its way while the last chunk of this is used, so
        // its pages and queries are loaded a segment ahead.
        typename RowBlock<D, RT, kBf16, kFp4>::Queries qn;
        auto look_ahead = [&]() {
            more = left > 0;
            if (!more) return;
            next_segment(nxt);
            rb.load_q(nxt.b, nxt.kvh, nxt.hb, qn);
        };
        rb.load_q(cur.b, cur.kvh, cur.hb, rb.q);
        copy_chunk<D, kNT>(a, cur.pg, cur.c0 * kKeys, cur.kvh, lds, lane);
        rb.begin(cur.len, cur.hb);
        look_ahead();
        rb.ready();
        for (int c = cur.c0, st = 0;; st ^= 1) {
            uint16_t* const there = lds + (st ^ 1) * stage_elems<D>();
            const bool last = c + 1 == cur.c1;
            if (!last) {
                pages_for(a, cur, c + 1, lane);
                copy_chunk<D, kNT>(a, cur.pg, (c + 1) * kKeys, cur.kvh, there, lane);
                asm volatile("s_waitcnt vmcnt(%0)" : : "n"(copies<D>()) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
                if (more) copy_chunk<D, kNT>(a, nxt.pg, nxt.c0 * kKeys, nxt.kvh, there, lane);
            }
            rb.use(lds + st * stage_elems<D>(), c * kKeys, cur.len);
            if (!last) {
                ++c;
                continue;
            }
            finish();
            if (!more) break;
            cur = nxt;
            c = cur.c0;
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) rb.q[t][i] = qn[t][i];
            rb.begin(cur.len, cur.hb);
            look_ahead();
        }
    }
}

// ---- one workgroup per item -------------------------------------------------------------------------
// Short caches (choose_waves): W waves take an item's chunks in equal runs and join their results in LDS; one launch.
template <int D, int RT, bool kBf16, bool kFp4, int W>
__global__ __launch_bounds__(64 * W) void paged_whole(PagedArgs a) {
    constexpr int kRing = wave_lds<D, kFp4>(), kRows = 16 * RT;
    constexpr int kBytes = W == 1 ? kRing * 2 : std::max(W * kRing * 2, W * kRows * (D + 2) * 4);
    __shared__ __attribute__((aligned(16))) char smem[kBytes];
    const int lane = (int)(threadIdx.x & 63u), wave = scalar((int)(threadIdx.x >> 6));
    uint16_t* const lds = (uint16_t*)smem + wave * kRing;
    Segment s;
    s.b = (int)(blockIdx.x / (unsigned)a.items);
    const int item = (int)(blockIdx.x % (unsigned)a.items);
    s.kvh = item / a.HB;
    s.hb = item - s.kvh * a.HB;
    RowBlock<D, RT, kBf16, kFp4> rb(a, lane);
    rb.load_q(s.b, s.kvh, s.hb, rb.q);
    {   // the length and the first 64 entries at once; entries past the last row's are not used for a row that is
        int ids = a.tables[s.b * a.table_stride + min(lane, (a.max_len >> a.lp) - 1)], len = a.lens[s.b];
        asm volatile("" : "+v"(ids), "+v"(len));
        s.len = scalar(min(max(len, 0), a.max_len));
        s.pg.first = 0;
        s.pg.ids = min(max(ids, 0), a.pages - 1);
    }
    s.n = chunks_of(s.len);
    s.c0 = s.n * wave / W;
    s.c1 = s.n * (wave + 1) / W;
    rb.begin(s.len, s.hb);
    if (s.c0 < s.c1) {
        if constexpr (kFp4) {
            // Chunks in pairs, the next one's codes always on their way (past the last, that one's once more): where ways with and without
            // loads meet, the compiler waits for all that may be on its way.
            Codes<D> x, y;
            auto load = [&](int c, Codes<D>& to) {
                pages_for(a, s, c, lane);
                load_codes<D, false>(a, s.pg, c * kKeys, s.kvh, to, lane);
            };
            load(s.c0, x);
            int c = s.c0;
            for (; c + 1 < s.c1; c += 2) {
                load(c + 1, y);
                rb.use(x, c * kKeys, s.len, lds);
                load(min(c + 2, s.c1 - 1), x);
                rb.use(y, (c + 1) * kKeys, s.len, lds);
            }
            if (c < s.c1) rb.use(x, c * kKeys, s.len, lds);
        } else {
            pages_for(a, s, s.c0, lane);
            copy_chunk<D, false>(a, s.pg, s.c0 * kKeys, s.kvh, lds, lane);
            rb.ready();
            for (int c = s.c0, st = 0; c < s.c1; ++c, st ^= 1) {
                if (c + 1 < s.c1) {
                    pages_for(a, s, c + 1, lane);
                    copy_chunk<D, false>(a, s.pg, (c + 1) * kKeys, s.kvh, lds + (st ^ 1) * stage_elems<D>(), lane);
                    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(copies<D>()) : "memory");
                } else {
                    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
                }
                rb.use(lds + st * stage_elems<D>(), c * kKeys, s.len);
            }
        }
    }
    if constexpr (W == 1) {
        rb.store(s.b, s.kvh, s.hb);
        return;
    }
    __syncthreads();   // every wave is done with its ring: the results over them
    const int rows = min(kRows, rb.R - s.hb * kRows);
    float* const po = (float*)smem;
    float* const pml = po + W * kRows * D;
    rb.store_part(pml, po, wave * kRows, rows);
    __syncthreads();
    for (int x = (int)threadIdx.x; x < rows * (D / 4); x += 64 * W) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float M = kInitM, L = 0.f;
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < W; ++k) M = fmaxf(M, pml[(k * kRows + r) * 2]);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float2 ml = *(const float2*)(pml + (k * kRows + r) * 2);
            const float wt = __builtin_amdgcn_exp2f(ml.x - M);
            L = fmaf(wt, ml.y, L);
            acc += *(const f32x4*)(po + (k * kRows + r) * D + d) * wt;
        }
        const float inv = L > 0.f ? 1.f / L : 1.f;
        uint16_t* dst = a.o + rb.row_of(s.b, s.kvh, s.hb * kRows + r) + d;
        ((uint32_t*)dst)[0] = pack2<kBf16>(acc[0] * inv, acc[1] * inv);
        ((uint32_t*)dst)[1] = pack2<kBf16>(acc[2] * inv, acc[3] * inv);
    }
}

// A workgroup per row of q: from the parts that its item's shares left, D / 4 lanes for a part; zeros where
// the sequence has no keys.
template <int D, bool kBf16, int kThreads>
__global__ __launch_bounds__(kThreads) void paged_join(PagedArgs a) {
    constexpr int kLanes = D / 4, kGroups = kThreads / kLanes, kFlight = kThreads == 64 ? 4 : 8;
    __shared__ __attribute__((aligned(16))) f32x4 acc_s[kGroups][kLanes];
    __shared__ float2 ml_s[kGroups];
    const int R = a.nq * a.G;
    const int b = (int)(blockIdx.x / (a.HK * R)), kvh = (int)(blockIdx.x / R % a.HK), rr = (int)(blockIdx.x % R);
    const int r = rr % a.rows, item = kvh * a.HB + rr / a.rows;
    const int n = chunks_of(length_of(a, b));
    const long long per = a.head[0], before = a.head[1 + b];   // of no meaning where n is 0
    int parts = 0;
    long long first = 0;
    if (n > 0) {
        const long long begin = before * a.items + (long long)item * n;
        first = quotient(begin, per);
        parts = (int)(quotient(begin + n - 1, per) - first) + 1;
        if (parts == 1) return;   // written by its share
    }
    const int grp = (int)threadIdx.x / kLanes, d = (int)threadIdx.x % kLanes * 4;
    // the first part begins its item, the others go on with it
    auto place = [&](int i) { return ((size_t)(first + i) * 2 + (i == 0 ? 1 : 0)) * a.rows + r; };
    float M = kInitM, L = 0.f;
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    for (int i0 = grp; i0 < parts; i0 += kGroups * kFlight) {   // parts in flight
        float2 ml[kFlight];
        f32x4 v[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            ml[k] = make_float2(kInitM, 0.f);
            v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (i0 + k * kGroups < parts) {
                const size_t idx = place(i0 + k * kGroups);
                ml[k] = *(const float2*)(a.part_ml + idx * 2);
                v[k] = *(const f32x4*)(a.part_o + idx * D + d);
            }
        }
        float top = M;
#pragma unroll
        for (int k = 0; k < kFlight; ++k) top = fmaxf(top, ml[k].x);
        const float old = __builtin_amdgcn_exp2f(M - top);
        M = top;
        L *= old;
        acc *= old;
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const float w = __builtin_amdgcn_exp2f(ml[k].x - M);
            L = fmaf(w, ml[k].y, L);
            acc += v[k] * w;
        }
    }
    acc_s[grp][d / 4] = acc;
    if (d == 0) ml_s[grp] = make_float2(M, L);
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) M = fmaxf(M, ml_s[k].x);
    L = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kGroups; ++k) {
        const float w = __builtin_amdgcn_exp2f(ml_s[k].x - M);
        L = fmaf(w, ml_s[k].y, L);
        acc += acc_s[k][d / 4] * w;
    }
    const float inv = L > 0.f ? 1.f / L : 1.f;
    uint16_t* dst = a.o + (((size_t)b * a.nq + rr / a.G) * a.nQH + (size_t)kvh * a.G + rr % a.G) * D + d;
    ((uint32_t*)dst)[0] = pack2<kBf16>(acc[0] * inv, acc[1] * inv);
    ((uint32_t*)dst)[1] = pack2<kBf16>(acc[2] * inv, acc[3] * inv);
}

// ---- plan -----------------------------------------------------------------------------------------
struct PagedPlan {
    int G, RT, HB, items, rows, shares;
    int waves;   // of a workgroup per item, 0: equal shares
    size_t head_bytes, ml_bytes, ws_bytes;
};

// Eight waves of 16-bit rows at D 128 are more than the LDS has room for, of MXFP4 and two row tiles more than the registers.
constexpr int most_waves(int D, int RT, bool fp4) { return D == 64 || (fp4 && RT == 1) ? 8 : 4; }

// One launch for short caches: the waves per item that end soonest, a round of the chip's waves taken for five chunks' time and those
// that a wave has; 0: equal shares. Their second launch and the walk over the lengths cost 7-10 us, which up to eight chunks a
// wave, and of 16-bit rows sixteen over its rounds or four to an item, do not: 16 sequences, 32/8 heads D 128, of 120 keys 5.0 against
// 16 us, of 1,000 13 against 19; 64 of 1,000 41 against 47, 256 of 250 41 against 49, 4,000 of 120 377 against 423. Beyond, the
// shares' even ends win: 128 of 1,000 (32 chunks) 95 against 87 us. In MXFP4, where a share's waves have fewer registers, 128 of 1,000 29
// against 37, 1,600 of 500 183 against 190. Those are calls that find the Infinity Cache as the one before left it. Behind other work that
// fills it, one launch wins up to about 70 MB (16 of 1,000 27 against 32, in MXFP4 9.9 against 16 and 64 of 1,000 30 against 38) and loses
// above (64 of 1,000 82 against 52, 256 of 250 83 against 54, in MXFP4 128 of 1,000 56 against 42), but for many short ones (4,000 of 120
// 425 against 472); tables with more room than the sequences need (max_pages) take the shares.
int choose_waves(long long items, int max_len, int D, int RT, bool fp4, long long resident) {
    const int chunks = (max_len + kKeys - 1) / kKeys;
    int best = 0;
    long long least = 0;
    for (int w = 1; w <= most_waves(D, RT, fp4); w *= 2) {
        const int each = (chunks + w - 1) / w;
        const long long rounds = (items * w + resident - 1) / resident, t = rounds * (5 + each);
        if (each > 8 || rounds > 1024 || (!fp4 && chunks > 4 && rounds * each > 16)) continue;   // fewer than 2^32 threads in any case
        if (best == 0 || t < least) { best = w; least = t; }
    }
    return best;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

bool plan_paged(const cdna4_paged_cache& k, const cdna4_paged_decode_cfg& c, PagedPlan& p) {
    p = {};
    if (!valid_cache(k)) return false;
    if (c.nQHeads < 1 || c.nQHeads % k.nKVHeads || c.nq < 1 || c.nq > 16) return false;
    if (c.batch < 0 || c.batch >= 1 << 24) return false;
    const long long qrows = (long long)c.batch * c.nq * c.nQHeads;
    if (c.nQHeads > 1 << 20 || qrows >= 1LL << 24) return false;   // a launch has fewer than 2^32 threads: 256 per row of q
    p.G = c.nQHeads / k.nKVHeads;
    const int R = p.G * c.nq;
    p.RT = R > 16 ? 2 : 1;
    p.HB = (R + 16 * p.RT - 1) / (16 * p.RT);
    p.items = k.nKVHeads * p.HB;
    p.rows = std::min(R, 16 * p.RT);
    p.shares = device_cus() * waves_per_cu(k.D, p.RT, k.format == CDNA4_KV_MXFP4);
    const long long items = (long long)c.batch * p.items;   // below 2^24, as the rows of q
    const int max_len = k.max_pages * k.page;
    if (items * ((max_len + kKeys - 1) / kKeys) > ((long long)p.shares << 30)) return false;   // a share's chunks are an int
    p.waves = choose_waves(items, max_len, k.D, p.RT, k.format == CDNA4_KV_MXFP4, p.shares);
    if (p.waves) return true;   // no workspace
    p.head_bytes = align256(((size_t)c.batch + 1) * sizeof(long long));
    p.ml_bytes = align256((size_t)p.shares * 2 * p.rows * 2 * sizeof(float));
    p.ws_bytes = p.head_bytes + p.ml_bytes + (size_t)p.shares * 2 * p.rows * k.D * sizeof(float);
    return true;
}

template <int D, int RT, bool kBf16, bool kFp4>
void launch_parts(const PagedArgs& a, bool nt, hipStream_t s) {
    if (nt) paged_parts<D, RT, kBf16, kFp4, true><<<a.shares, 64, 0, s>>>(a);
    else paged_parts<D, RT, kBf16, kFp4, false><<<a.shares, 64, 0, s>>>(a);
}

template <int D, int RT, bool kBf16, bool kFp4>
int launch_whole(const PagedArgs& a, int waves, hipStream_t s) {
    const unsigned grid = (unsigned)(a.batch * a.items);
    switch (waves) {
        case 1: paged_whole<D, RT, kBf16, kFp4, 1><<<grid, 64, 0, s>>>(a); break;
        case 2: paged_whole<D, RT, kBf16, kFp4, 2><<<grid, 128, 0, s>>>(a); break;
        case 4: paged_whole<D, RT, kBf16, kFp4, 4><<<grid, 256, 0, s>>>(a); break;
        default:
            if constexpr (most_waves(D, RT, kFp4) == 8) paged_whole<D, RT, kBf16, kFp4, 8><<<grid, 512, 0, s>>>(a);
    }
    return launch_status();
}

template <int D, bool kBf16>
int launch_paged(const PagedArgs& a, const PagedPlan& p, bool fp4, hipStream_t s) {
    if (p.waves) {
        if (p.RT == 2) return fp4 ? launch_whole<D, 2, kBf16, true>(a, p.waves, s) : launch_whole<D, 2, kBf16, false>(a, p.waves, s);
        return fp4 ? launch_whole<D, 1, kBf16, true>(a, p.waves, s) : launch_whole<D, 1, kBf16, false>(a, p.waves, s);
    }
    // Pools of more than half the Infinity Cache are read past it (stream::dma16): K and V of 157 MB 40.6 against 44.0 us, of 267 MB
    // 48.3 against 54.6; those of 58 MB that it holds 23.6 against 21.8.
    const bool nt = 2.0 * a.pages * a.HK * a.page * row_bytes(D, fp4) > 128.0 * 1024 * 1024;
    if (p.RT == 2) {
        if (fp4) launch_parts<D, 2, kBf16, true>(a, nt, s);
        else launch_parts<D, 2, kBf16, false>(a, nt, s);
    } else {
        if (fp4) launch_parts<D, 1, kBf16, true>(a, nt, s);
        else launch_parts<D, 1, kBf16, false>(a, nt, s);
    }
    if (int e = launch_status()) return e;
    const unsigned rows = (unsigned)((size_t)a.batch * a.nq * a.nQH);
    // By the parts that an item has on the average: one, 4.7 against 6.8 us with 128 threads and 9.3 with 256 (4,096 rows); six, 4.4
    // against 5.3 and 6.5 (2,048 rows); 128, 6.6 with 256 threads against 8.2 and 16.8 (96 rows). Many rows fill the chip without.
    const long long items = (long long)a.batch * a.items;
    if (a.shares < 4 * items) paged_join<D, kBf16, 64><<<rows, 64, 0, s>>>(a);
    else if (a.shares < 32 * items || rows > 8u * (unsigned)device_cus()) paged_join<D, kBf16, 128><<<rows, 128, 0, s>>>(a);
    else paged_join<D, kBf16, 256><<<rows, 256, 0, s>>>(a);
    return launch_status();
}

}  // namespace
}  // namespace cdna4

using namespace cdna4;

extern "C" size_t cdna4_attn_decode_paged_workspace_size(const cdna4_paged_cache* cache, const cdna4_paged_decode_cfg* cfg) {
    PagedPlan p;
    return cache && cfg && plan_paged(*cache, *cfg, p) ? p.ws_bytes : 0;
}

extern "C" int cdna4_attn_decode_paged(const void* q, const void* K_pages, const void* V_pages, const int* tables, const int* lens,
                                       void* o, const cdna4_paged_cache* cache, const cdna4_paged_decode_cfg* cfg, int dtype,
                                       void* workspace, size_t ws_bytes, cdna4_stream_t stream) {
    if (!cache || !cfg || (dtype != CDNA4_F16 && dtype != CDNA4_BF16)) return CDNA4_ERR_INVALID_VALUE;
    PagedPlan p;
    if (!plan_paged(*cache, *cfg, p)) return CDNA4_ERR_INVALID_VALUE;
    if (cfg->batch == 0) return 0;
    if (!q || !o || ((uintptr_t)q & 15u) || ((uintptr_t)o & 3u)) return CDNA4_ERR_INVALID_VALUE;
    if (!K_pages || !V_pages || (((uintptr_t)K_pages | (uintptr_t)V_pages) & 15u)) return CDNA4_ERR_INVALID_VALUE;
    if (!tables || !lens || (((uintptr_t)tables | (uintptr_t)lens) & 3u)) return CDNA4_ERR_INVALID_VALUE;
    if (p.ws_bytes && (!workspace || ((uintptr_t)workspace & 15u) || ws_bytes < p.ws_bytes)) return CDNA4_ERR_INVALID_VALUE;
    if (int e = check_device()) return e;
    PagedArgs a;
    a.q = (const uint16_t*)q; a.K = (const char*)K_pages; a.V = (const char*)V_pages;
    a.tables = tables; a.lens = lens;
    a.o = (uint16_t*)o;
    a.head = (long long*)workspace;
    a.part_ml = (float*)((char*)workspace + p.head_bytes);
    a.part_o = (float*)((char*)workspace + p.head_bytes + p.ml_bytes);
    a.table_stride = table_stride(*cache);
    a.nQH = cfg->nQHeads; a.HK = cache->nKVHeads; a.G = p.G; a.nq = cfg->nq; a.batch = cfg->batch; a.rows = p.rows;
    a.HB = p.HB; a.items = p.items;
    a.page = cache->page; a.lp = log2_of(cache->page); a.pages = cache->pages; a.max_len = cache->max_pages * cache->page;
    a.head_bytes = (uint32_t)(cache->page * paged::row_bytes(cache->D, cache->format == CDNA4_KV_MXFP4));
    a.page_bytes = (uint32_t)cache->nKVHeads * a.head_bytes;
    a.shares = p.shares;
    a.sc = kLog2e / sqrtf((float)cache->D);
    hipStream_t s = (hipStream_t)stream;
    const bool bf = dtype == CDNA4_BF16, fp4 = cache->format == CDNA4_KV_MXFP4;
    if (cache->D == 128) return bf ? launch_paged<128, true>(a, p, fp4, s) : launch_paged<128, false>(a, p, fp4, s);
    return bf ? launch_paged<64, true>(a, p, fp4, s) : launch_paged<64, false>(a, p, fp4, s);
}

extern "C" int cdna4_attn_decode_paged_plan(const cdna4_paged_cache* cache, const cdna4_paged_decode_cfg* cfg, int dtype, cdna3_plan_info* out) {
    PagedPlan p;
    if (!cache || !cfg || !out || (dtype != CDNA4_F16 && dtype != CDNA4_BF16) || !plan_paged(*cache, *cfg, p)) return CDNA4_ERR_INVALID_VALUE;
    out->kernel = CDNA4_KERNEL_DECODE_PAGED;
    out->waves = p.waves ? p.waves : 1;
    out->rows = p.rows;
    out->partials = p.waves ? 1 : p.shares;
    out->grid = p.waves ? (long long)cfg->batch * p.items : p.shares;
    out->workspace = p.ws_bytes;
    return 0;
}
