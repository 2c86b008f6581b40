// Decode attention over a paged KV cache (gfx950): nq queries per sequence, the last nq tokens', over the sequence's pages, whose
// rows are 16-bit or MXFP4.
//
//   o[b][i][h] = sum_j 2^(c q.k_j - m) v_j / sum_j 2^(c q.k_j - m),  j < lens[b] - nq + 1 + i,  c = log2(e) / sqrt(D)
//
// The G query heads of a kv head, times the nq queries, are the rows of one matrix product, kRT tiles of 16 rows at most ("row
// block"); a row block and a sequence's keys are one item, its keys are cut into chunks of 32. All chunks of all items lie on
// one axis, items of a sequence side by side, and every wave takes an equal share of it: lengths are read on the device, and
// what a wave has to do does not depend on how they differ. A share that holds all chunks of an item writes the output;
// of an item that shares cut, each leaves (m, l, O), and a second launch joins them,
// o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p.
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
constexpr int kMaxParts = 64;     // shares that an item is cut into, but for the two at its ends

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
    int shares;
    float sc;
};

__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long scalar(long long x) {
    return (long long)((uint64_t)(uint32_t)scalar((int)(x >> 32)) << 32 | (uint32_t)scalar((int)x));
}
__device__ __forceinline__ int length_of(const PagedArgs& a, int b) { return b < a.batch ? min(max(a.lens[b], 0), a.max_len) : 0; }
__device__ __forceinline__ int chunks_of(int len) { return (len + kKeys - 1) / kKeys; }

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

// Finds the sequence that holds chunk x of the axis of one item (0 <= x < all): each level narrows the sequences to a lane's.
__device__ __forceinline__ Place find(const PagedArgs& a, long long x, Window& w, int lane) {
    int lo = 0, n = a.batch;
    long long before = 0;
    for (;;) {
        const int step = (n + 63) / 64;   // sequences of a lane
        if (step == 1) {
            w.load(a, lo, lane);
            const long long c = lane < n ? chunks_of(w.len) : 0;
            const long long upto = wave::xlane::scan_inclusive(c, Sum{}) + before;
            const uint64_t here = __builtin_amdgcn_ballot_w64(upto > x);
            const int l = here ? __builtin_ctzll(here) : 63;
            return Place{lo + l, __builtin_amdgcn_readlane(w.len, l), scalar(__shfl(upto - c, l))};
        }
        long long c = 0;
        for (int i = 0; i < step; ++i) {
            const int at = lane * step + i;
            if (at < n) c += chunks_of(length_of(a, lo + at));
        }
        const long long upto = wave::xlane::scan_inclusive(c, Sum{}) + before;
        const uint64_t here = __builtin_amdgcn_ballot_w64(upto > x);
        const int l = here ? __builtin_ctzll(here) : 63;
        before = scalar(__shfl(upto - c, l));
        lo += l * step;
        n = min(step, n - l * step);
        if (n < 1) { lo = 0; n = 1; }   // not reached: x lies below the last lane's sum
    }
}

// Chunks of a share: equal shares of all, but none below kMinChunks, and no item in more than about kMaxParts.
__device__ __forceinline__ long long share_of(const PagedArgs& a, long long& all, int lane) {
    long long c = 0;
    int most = 0;
    for (int b = lane; b < a.batch; b += 64) {
        const int n = chunks_of(length_of(a, b));
        c += n;
        most = max(most, n);
    }
    all = scalar(allreduce(c, Sum{})) * a.items;
    most = scalar(allreduce(most, Max{}));
    const long long even = (all + a.shares - 1) / a.shares;
    return max(even, (long long)max(kMinChunks, (most + kMaxParts - 1) / kMaxParts));
}

// Pages of a sequence, 64 table entries at a time, one per lane; entries past its rows are not read.
struct Pages {
    const int* table;
    int first, ids, most;   // most: entries with rows
    __device__ __forceinline__ void load(const PagedArgs& a, int f, int lane) {
        first = f;
        ids = min(max(table[min(f + lane, most - 1)], 0), a.pages - 1);
    }
};

// The address of key k's row of one head in lane-by-lane form; the row's page is in the loaded entries.
__device__ __forceinline__ size_t row_at(const PagedArgs& a, const Pages& pg, int k, int kvh, int head_bytes, int rbytes) {
    const int id = __shfl(pg.ids, (k >> a.lp) - pg.first);
    return ((size_t)id * a.HK + kvh) * head_bytes + (size_t)(k & (a.page - 1)) * rbytes;
}

// Copies one chunk's K or V rows into a ring stage; rows past the last re-read it (masked).
template <int D, bool kIsK>
__device__ __forceinline__ void copy_chunk(const PagedArgs& a, const Pages& pg, int kb, int len, int kvh, uint16_t* stage, int lane) {
    constexpr int CPR = D / 8, NI = kKeys * CPR / 64;
    const int head_bytes = a.page * 2 * D;
    const char* pool = kIsK ? a.K : a.V;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int p = j * 64 + lane, r = p / CPR;
        const size_t at = row_at(a, pg, min(kb + r, len - 1), kvh, head_bytes, 2 * D);
        stream::dma16<false>(pool + at + ((p % CPR) ^ swz<D, kIsK>(r)) * 16, stage + j * 512);
    }
}

// Scores that a row must not see are masked by the row's own limit.
template <int RT>
__device__ __forceinline__ bool check_limits(f32x4 (&s)[RT][2], const float (&m)[RT], float (&lm)[RT], int kb, const int (&limit)[RT],
                                             bool mask, float sc, int g) {
    bool need = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float v = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (mask && kb + g * 8 + u * 4 + e >= limit[t]) s[t][u][e] = -INFINITY;
                v = fmaxf(v, s[t][u][e]);
            }
        lm[t] = v;
        need |= v * sc > m[t] + kTau;
    }
    return need;
}

template <int D, int RT, bool kBf16, bool kFp4>
__global__ __launch_bounds__(64) void paged_parts(PagedArgs a) {
    constexpr int ND = D / 32, NDT = D / 16, kStage = kKeys * D;
    __shared__ __attribute__((aligned(16))) uint16_t lds[4 * kStage];
    const int lane = (int)threadIdx.x, li = lane & 15, g = lane >> 4, share = (int)blockIdx.x;
    long long all;
    const long long per = share_of(a, all, lane);
    if (share == 0 && lane == 0) a.head[0] = per;
    long long at = share * per;
    const long long end = min(at + per, all);
    if (at >= end) return;
    Window w;
    Place pl = find(a, at / a.items, w, lane);
    const LdsOffsets off = lds_offsets<D>(li, g);
    const size_t slot0 = (size_t)share * 2 * a.rows;
    while (at < end) {
        const int n = chunks_of(pl.len);
        const long long in_seq = at - pl.before * a.items;
        const int item = (int)(in_seq / n), c0 = (int)(in_seq % n), c1 = (int)min((long long)n, c0 + (end - at));
        if (item == 0 && c0 == 0 && lane == 0) a.head[1 + pl.b] = pl.before;
        const int kvh = item / a.HB, hb = item % a.HB;
        // row r of the item: query r / G, head kvh G + r % G
        const int R = a.nq * a.G;
        int limit[RT];
        u32x4 qb[RT][ND];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = hb * RT * 16 + t * 16 + li, i = r / a.G;
            limit[t] = pl.len;
#pragma unroll
            for (int c = 0; c < ND; ++c) qb[t][c] = u32x4{0u, 0u, 0u, 0u};
            if (r < R) {
                limit[t] = pl.len - a.nq + 1 + i;
                const uint16_t* q = a.q + (((size_t)pl.b * a.nq + i) * a.nQH + (size_t)kvh * a.G + r % a.G) * D;
#pragma unroll
                for (int c = 0; c < ND; ++c) qb[t][c] = *(const u32x4*)(q + c * 32 + g * 8);
            }
        }
        Pages pg;
        pg.table = a.tables + pl.b * a.table_stride;
        pg.most = (pl.len + a.page - 1) >> a.lp;
        f32x4 o[RT][NDT], lacc[RT];
        float m[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            m[t] = kInitM;
            lacc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < NDT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        pg.load(a, (c0 * kKeys) >> a.lp, lane);
        for (int c = c0; c < c1; ++c) {
            const int kb = c * kKeys;
            if (((min(kb + kKeys, pl.len) - 1) >> a.lp) - pg.first >= 64) pg.load(a, kb >> a.lp, lane);
            __syncthreads();
            if constexpr (kFp4) {
                const int head_bytes = a.page * (D / 2 + D / 32);
                // 16 codes to a lane: half a block
#pragma unroll
                for (int kv = 0; kv < 2; ++kv)
#pragma unroll
                    for (int j = 0; j < kKeys * D / 16 / 64; ++j) {
                        const int p = j * 64 + lane, r = p / (D / 16), x = p % (D / 16);
                        const int k = min(kb + r, pl.len - 1);
                        const char* pool = (kv ? a.V : a.K) + row_at(a, pg, 0 + k, kvh, head_bytes, 0) - 0;
                        const char* headp = pool;
                        const int row = k & (a.page - 1);
                        const uint2 c2 = *(const uint2*)(headp + row * (D / 2) + x * 8);
                        const float f = f32_from_bits((uint32_t)*(const uint8_t*)(headp + a.page * (D / 2) + row * (D / 32) + x / 2) << 23);
                        u32x4 lo{decode2<kBf16, 0>(c2.x, f), decode2<kBf16, 1>(c2.x, f), decode2<kBf16, 2>(c2.x, f), decode2<kBf16, 3>(c2.x, f)};
                        u32x4 hi{decode2<kBf16, 0>(c2.y, f), decode2<kBf16, 1>(c2.y, f), decode2<kBf16, 2>(c2.y, f), decode2<kBf16, 3>(c2.y, f)};
                        uint16_t* dst = lds + kv * kStage + r * D;
                        const int z = kv ? swz_v<D>(r) : swz_k<D>(r);
                        *(u32x4*)(dst + ((2 * x) ^ z) * 8) = lo;
                        *(u32x4*)(dst + ((2 * x + 1) ^ z) * 8) = hi;
                    }
            } else {
                copy_chunk<D, true>(a, pg, kb, pl.len, kvh, lds, lane);
                copy_chunk<D, false>(a, pg, kb, pl.len, kvh, lds + kStage, lane);
                asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
            }
            __syncthreads();
            const char *Kt = (const char*)lds, *Vt = (const char*)(lds + kStage);
            f32x4 s[RT][2];
            qk_chunk<D, RT, kBf16>(Kt, off, qb, s, 0);
            float lm[RT];
            const bool need = check_limits<RT>(s, m, lm, kb, limit, kb + kKeys > pl.len - a.nq + 1, a.sc, g);
            if (__builtin_amdgcn_ballot_w64(need)) rescale_rows<D, RT>(lm, m, o, lacc, a.sc);
            u32x4 pb[RT];
            softmax_chunk<RT, kBf16>(s, m, pb, a.sc);
            pv_chunk<D, RT, kBf16>(Vt, off, pb, o, lacc, 0);
            if constexpr (kBf16) {
                if (kb < kLoKeys) {
                    softmax_lo_chunk<RT>(s, m, pb, a.sc);
                    pv_chunk<D, RT, true>(Vt, off, pb, o, lacc, 0);
                }
            }
        }
        const bool whole = c0 == 0 && c1 == n;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r16 = t * 16 + li, r = hb * RT * 16 + r16;
            if (r >= R) continue;
            if (whole) {
                const float inv = lacc[t][0] > 0.f ? 1.f / lacc[t][0] : 1.f;
                uint16_t* dst = a.o + (((size_t)pl.b * a.nq + r / a.G) * a.nQH + (size_t)kvh * a.G + r % a.G) * D + g * 4;
#pragma unroll
                for (int d = 0; d < NDT; ++d) {
                    ((uint32_t*)(dst + d * 16))[0] = pack2<kBf16>(o[t][d][0] * inv, o[t][d][1] * inv);
                    ((uint32_t*)(dst + d * 16))[1] = pack2<kBf16>(o[t][d][2] * inv, o[t][d][3] * inv);
                }
            } else {
                const size_t idx = slot0 + (c0 == 0 ? a.rows : 0) + r16;
                float* dst = a.part_o + idx * D + g * 4;
#pragma unroll
                for (int d = 0; d < NDT; ++d) *(f32x4*)(dst + d * 16) = o[t][d];
                if (g == 0) *(float2*)(a.part_ml + idx * 2) = make_float2(m[t], lacc[t][0]);
            }
        }
        at += c1 - c0;
        if (at < end && c1 == n && item + 1 == a.items) {   // on to the next sequence that has keys
            pl.before += n;
            int l = pl.b + 1 - w.first;
            for (;;) {
                const uint64_t more = l < 64 ? __builtin_amdgcn_ballot_w64(w.len > 0 && lane >= l) : 0;
                if (more) {
                    l = __builtin_ctzll(more);
                    pl.b = w.first + l;
                    pl.len = __builtin_amdgcn_readlane(w.len, l);
                    break;
                }
                if (w.first + 64 >= a.batch) return;   // not reached: chunks are left
                w.load(a, w.first + 64, lane);
                l = 0;
            }
        }
    }
}

// A workgroup per sequence and item: its rows from the parts that its shares left, zeros where the sequence has no keys.
template <int D, bool kBf16>
__global__ __launch_bounds__(256) void paged_join(PagedArgs a) {
    const int b = (int)(blockIdx.x / a.items), item = (int)(blockIdx.x % a.items), hb = item % a.HB, kvh = item / a.HB;
    const int n = chunks_of(length_of(a, b));
    long long first = 0, parts = 0;
    if (n > 0) {
        const long long per = a.head[0], begin = a.head[1 + b] * a.items + (long long)item * n;
        first = begin / per;
        parts = (begin + n - 1) / per - first + 1;
        if (parts == 1) return;   // written by its share
    }
    const int R = a.nq * a.G, rows = min(a.rows, R - hb * a.rows);
    for (int x = (int)threadIdx.x; x < rows * (D / 4); x += 256) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float M = kInitM, L = 0.f;
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
        for (long long i = 0; i < parts; ++i) {
            // the first part begins its item, the others go on with it
            const size_t idx = ((size_t)(first + i) * 2 + (i == 0 ? 1 : 0)) * a.rows + r;
            const float2 ml = *(const float2*)(a.part_ml + idx * 2);
            const f32x4 v = *(const f32x4*)(a.part_o + idx * D + d);
            const float top = fmaxf(M, ml.x), w0 = __builtin_amdgcn_exp2f(M - top), w1 = __builtin_amdgcn_exp2f(ml.x - top);
            M = top;
            L = L * w0 + ml.y * w1;
            acc = acc * w0 + v * w1;
        }
        const float inv = L > 0.f ? 1.f / L : 1.f;
        const int rr = hb * a.rows + r;
        uint16_t* dst = a.o + (((size_t)b * a.nq + rr / a.G) * a.nQH + (size_t)kvh * a.G + rr % a.G) * D + d;
        ((uint32_t*)dst)[0] = pack2<kBf16>(acc[0] * inv, acc[1] * inv);
        ((uint32_t*)dst)[1] = pack2<kBf16>(acc[2] * inv, acc[3] * inv);
    }
}

// ---- plan -----------------------------------------------------------------------------------------
struct PagedPlan {
    int G, RT, HB, items, rows, shares;
    size_t head_bytes, ml_bytes, ws_bytes;
};

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

bool plan_paged(const cdna4_paged_cache& k, const cdna4_paged_decode_cfg& c, PagedPlan& p) {
    if (!valid_cache(k)) return false;
    if (c.nQHeads < 1 || c.nQHeads % k.nKVHeads || c.nq < 1 || c.nq > 16) return false;
    if (c.batch < 0 || c.batch >= 1 << 24) return false;
    const long long qrows = (long long)c.batch * c.nq * c.nQHeads;
    if (c.nQHeads > 1 << 20 || qrows > (1LL << 26) - 4) return false;
    p.G = c.nQHeads / k.nKVHeads;
    const int R = p.G * c.nq;
    p.RT = R > 16 ? 2 : 1;
    p.HB = (R + 16 * p.RT - 1) / (16 * p.RT);
    p.items = k.nKVHeads * p.HB;
    p.rows = std::min(R, 16 * p.RT);
    if ((long long)c.batch * p.items * 256 > 0xffffffffLL) return false;
    p.shares = device_cus() * (k.D == 64 ? 10 : 5);
    p.head_bytes = align256(((size_t)c.batch + 1) * sizeof(long long));
    p.ml_bytes = align256((size_t)p.shares * 2 * p.rows * 2 * sizeof(float));
    p.ws_bytes = p.head_bytes + p.ml_bytes + (size_t)p.shares * 2 * p.rows * k.D * sizeof(float);
    return true;
}

template <int D, bool kBf16>
int launch_paged(const PagedArgs& a, const PagedPlan& p, bool fp4, hipStream_t s) {
    if (p.RT == 2) {
        if (fp4) paged_parts<D, 2, kBf16, true><<<p.shares, 64, 0, s>>>(a);
        else paged_parts<D, 2, kBf16, false><<<p.shares, 64, 0, s>>>(a);
    } else {
        if (fp4) paged_parts<D, 1, kBf16, true><<<p.shares, 64, 0, s>>>(a);
        else paged_parts<D, 1, kBf16, false><<<p.shares, 64, 0, s>>>(a);
    }
    if (int e = launch_status()) return e;
    paged_join<D, kBf16><<<(unsigned)((size_t)a.batch * a.items), 256, 0, s>>>(a);
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
    if (!workspace || ((uintptr_t)workspace & 15u) || ws_bytes < p.ws_bytes) return CDNA4_ERR_INVALID_VALUE;
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
    out->waves = 1;
    out->rows = p.rows;
    out->partials = p.shares;
    out->grid = p.shares;
    out->workspace = p.ws_bytes;
    return 0;
}
