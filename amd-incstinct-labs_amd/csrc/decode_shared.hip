// Decode attention of a batch that shares a prefix (gfx950): one query token per sequence over the prefix's
// keys, which lie in the cache once, and over the sequence's own keys, whose number differs by sequence.
//
//   o[b][h] = sum_j 2^(c q.k_j - M) v_j / sum_j 2^(c q.k_j - M) over the prefix and own keys, c = log2(e) / sqrt(D)
//
// The keys of a row are cut into parts; each part leaves (m, l, O) with its own maximum m, and a second
// launch joins the parts of a row, o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p.
//   * Prefix parts: the G query heads of a kv head of all sequences are the rows of one matrix product, so
//     the prefix is read once for the batch (per 128 rows) instead of once per sequence. A workgroup takes 128
//     rows and a range of prefix keys (attn_block.hpp).
//   * Own parts: a workgroup takes a range of one sequence's own keys for up to 16 query heads of a kv head, its
//     waves streaming parts of the range (attn_stream.hpp); the lengths are read on the device.
// Both kinds run in one launch, prefix parts first: those of a large batch are bound by the matrix
// cores and own parts by HBM, and the two workgroups that a CU holds then often are one of each.
//
// Weights are rounded to the inputs' 16-bit type for the P.V products and summed as rounded, in fp32, as in the prompt
// kernels (prefill_packed.hip); the parts' maxima, sums and O stay fp32 through the join. The output's relative error, its own
// rounding with it, is 1.2-1.4 times that of fp32 products (bf16 0.0017 -> 0.0020-0.0023, fp16 0.00021 -> 0.00029).
//
// Measured, 32/8 heads D 128, in a graph: 256 sequences of 64-2,048 own keys behind 16,384, bf16, 144 us (the parts 134 at 5.1
// TB/s, bound by HBM, the join 8); 64 of 20-1,000 behind 8,192, fp16, 29.7 us; few rows by two dependent launches, 7-10 us.
// Without a prefix, 64 of 2,048 87 us (6.2 TB/s), 64 of 64-4,096 in caches of 4,096 50 us (the longest decide); the prefix
// alone, 64 rows of 8,192 keys, 23 us.
#include <algorithm>
#include <math.h>

#include "attn_block.hpp"

namespace cdna4 {
namespace {

using namespace tile;
using wave::xlane::allreduce;
using wave::xlane::Max;
using wave::xlane::Sum;

constexpr int kBlockRows = 1 << block::rows_log2<2>();   // rows of a prefix part's workgroup

struct SharedArgs {
    const uint16_t *q, *Kp, *Vp, *K, *V;
    uint16_t* o;
    const int* lens;
    float* part_ml;   // [batch][nQH][PT][2]
    float* part_o;    // [batch][nQH][PT][D]
    long long p_hs, kv_hs;     // elements between kv heads of the prefix and of the own keys
    int nQH, nKVH, G, HB, batch, prefix, max_own;
    int blocks, kpp, Pp;       // row blocks per kv head, keys per prefix part, prefix parts
    int Po, kmin;              // own parts per row at most, keys per own part at least
    int prefix_groups;         // groups of 8 workgroups of prefix parts
    float sc;
};

// Own keys of sequence b and how they are cut: `parts` parts of `keys` keys, a multiple of 32.
struct OwnCut { int len, keys, parts; };
__device__ __forceinline__ OwnCut own_cut(const SharedArgs& a, int b) {
    OwnCut c{0, 32, 0};
    if (a.Po == 0) return c;   // no own keys in any sequence: no lengths either
    c.len = min(max(a.lens[b], 0), a.max_own);
    c.keys = max((c.len + a.Po - 1) / a.Po, a.kmin);
    c.keys = (c.keys + 31) & ~31;
    c.parts = (c.len + c.keys - 1) / c.keys;
    return c;
}

// Waves that stream own keys: each has a ring of two K and V stages (16 KiB at D = 64, 32 KiB at D = 128) in
// the LDS of the prefix parts' size at D = 128, 64 KiB, so that two workgroups fit a CU.
template <int D> constexpr int own_waves() { return D == 64 ? 4 : 2; }
template <int D> constexpr int shared_lds() { return 32768; }   // elements: 64 KiB

template <int D, bool kBf16>
__device__ __forceinline__ void prefix_part(const SharedArgs& a, int item, uint16_t* lds, int wave, int lane) {
    constexpr int QT = 2, ND = D / 32, NDT = D / 16;
    const int li = lane & 15, g = lane >> 4;
    // item = ((column / 8) * blocks + row block) * 8 + column % 8: the row blocks of a column (kv head and key
    // range) run on one XCD, which workgroups go to round-robin, and share the range in its L2
    const int col = (item >> 3) / a.blocks * 8 + (item & 7), blk = (item >> 3) % a.blocks;
    if (col >= a.nKVH * a.Pp) return;
    const int kvh = col % a.nKVH, part = col / a.nKVH;
    const int k0 = part * a.kpp, S = min(a.kpp, a.prefix - k0);
    const int rows = a.batch * a.G, r0 = blk * kBlockRows + wave * QT * 16;
    const uint16_t* Kh = a.Kp + kvh * a.p_hs + (long long)k0 * D;
    const uint16_t* Vh = a.Vp + kvh * a.p_hs + (long long)k0 * D;
    // row r of the kv head: sequence r / G, query head kvh G + r % G
    auto row_of = [&](int r) { return (size_t)(r / a.G) * a.nQH + (size_t)(kvh * a.G + r % a.G); };
    u32x4 qb[QT][ND];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const uint16_t* q = a.q + row_of(min(r0 + t * 16 + li, rows - 1)) * D;
#pragma unroll
        for (int c = 0; c < ND; ++c) qb[t][c] = *(const u32x4*)(q + c * 32 + g * 8);
    }
    const int ntiles = (S + pipe::kBc - 1) / pipe::kBc;
    const int t_main = min(S >= 96 ? (S - 96) / 64 + 1 : 0, min(ntiles, S / pipe::kBc) - 2);
    const block::Keys<false> kk{Kh, nullptr, D, 0, S, 1}, kv{Vh, nullptr, D, 0, S, 1};
    const block::Offsets own = block::own_offsets<D>(D, wave, lane);
    block::first_copies<D, false>(kk, kv, ntiles, own, lds, wave, lane);
    f32x4 o[QT][NDT], lacc[QT];
    float m[QT];
    block::attend<D, QT, kBf16, false, false>(kk, kv, block::Shape{S, ntiles, r0 < rows ? (S + 31) / 32 : 0, 0, t_main}, qb, o,
                                          lacc, m, own, lds, a.sc, wave, lane);
    const int PT = a.Pp + a.Po;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int r = r0 + t * 16 + li;
        if (r >= rows) continue;
        const size_t idx = row_of(r) * PT + part;
        float* dst = a.part_o + idx * D + g * 4;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *(f32x4*)(dst + dt * 16) = o[t][dt];
        if (g == 0) *(float2*)(a.part_ml + idx * 2) = make_float2(m[t], lacc[t][0]);
    }
}

template <int D, bool kBf16, bool kNT>
__device__ __forceinline__ void own_part(const SharedArgs& a, int item, uint16_t* lds, int wave, int lane) {
    constexpr int W = own_waves<D>(), ND = D / 32, NDT = D / 16;
    constexpr int kRing = stream::kDecStages * stream::kDecT * D;
    static_assert(2 * W * kRing <= shared_lds<D>(), "the rings fit the LDS");
    static_assert(W * 16 * (D + 2) * 4 <= shared_lds<D>() * 2, "the waves' results fit over the rings");
    const int li = lane & 15, g = lane >> 4;
    const int per_b = a.nKVH * a.HB;
    const int row = item % (a.batch * per_b), part = item / (a.batch * per_b);
    if (part >= a.Po) return;
    const int b = row / per_b, kvh = row % per_b / a.HB, sub = row % a.HB;
    const OwnCut cut = own_cut(a, b);
    if (part >= cut.parts) return;
    const int qh0 = kvh * a.G + sub * 16, nrows = min(16, a.G - sub * 16);
    const int s0 = part * cut.keys, s1 = min(cut.len, s0 + cut.keys);
    const int kpw = ((s1 - s0 + W - 1) / W + 31) & ~31;
    float* const po = (float*)lds;
    float* const pml = po + W * 16 * D;
    f32x4 o[1][NDT], lacc[1];
    float m[1];
    if (wave < W) {
        u32x4 qb[1][ND];
#pragma unroll
        for (int c = 0; c < ND; ++c) {
            qb[0][c] = u32x4{0u, 0u, 0u, 0u};
            if (li < nrows) qb[0][c] = *(const u32x4*)(a.q + ((size_t)b * a.nQH + qh0 + li) * D + c * 32 + g * 8);
        }
        const size_t head = ((size_t)b * a.nKVH + kvh) * (size_t)a.kv_hs;
        const int kbeg = min(s1, s0 + wave * kpw), kend = min(s1, kbeg + kpw);
        stream::stream_keys<D, kBf16, stream::kDecStages, kNT>(a.K + head, a.V + head, D, cut.len, kbeg, kend, 0, 0, a.sc, qb,
                                                               o, lacc, m, lds + wave * kRing, lds + (W + wave) * kRing, lane);
    }
    __syncthreads();   // every wave is done with its ring: reuse the LDS for the waves' results
    if (wave < W) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) *(f32x4*)(po + (wave * 16 + li) * D + dt * 16 + g * 4) = o[0][dt];
        if (g == 0) *(float2*)(pml + (wave * 16 + li) * 2) = make_float2(m[0], lacc[0][0]);
    }
    __syncthreads();
    const int PT = a.Pp + a.Po;
    for (int p = (int)threadIdx.x; p < nrows * (D / 4); p += 256) {
        const int h = p / (D / 4), d = 4 * (p % (D / 4));
        float M = kInitM, L = 0.f;
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, pml[(w * 16 + h) * 2]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 ml = *(const float2*)(pml + (w * 16 + h) * 2);
            const float wt = __builtin_amdgcn_exp2f(ml.x - M);
            L = fmaf(wt, ml.y, L);
            acc += *(const f32x4*)(po + (w * 16 + h) * D + d) * wt;
        }
        const size_t idx = ((size_t)b * a.nQH + qh0 + h) * PT + a.Pp + part;
        *(f32x4*)(a.part_o + idx * D + d) = acc;
        if (d == 0) *(float2*)(a.part_ml + idx * 2) = make_float2(M, L);
    }
}

// Workgroups of prefix parts first, in groups of 8, one per XCD: with own keys in the call they are one per CU
// (plan_shared), and the own parts that follow take the CUs' other places.
template <int D, bool kBf16, bool kNT>
__global__ __launch_bounds__(256, 2) void shared_parts(SharedArgs a) {
    __shared__ __attribute__((aligned(16))) uint16_t lds[shared_lds<D>()];
    const int lane = (int)(threadIdx.x & 63u);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int own = (int)blockIdx.x - a.prefix_groups * 8;
    if (own < 0) prefix_part<D, kBf16>(a, (int)blockIdx.x, lds, wave, lane);
    else own_part<D, kBf16, kNT>(a, own, lds, wave, lane);
}

// One wave per (batch, query head): its n parts joined (Pp of the prefix, then the own ones that exist).
template <int D, bool kBf16>
__global__ __launch_bounds__(256) void shared_join(SharedArgs a) {
    constexpr int EPL = D / 64;
    const int lane = (int)(threadIdx.x & 63u);
    const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (size_t)a.batch * a.nQH) return;
    const int PT = a.Pp + a.Po;
    const int n = a.Pp + own_cut(a, (int)(row / a.nQH)).parts;
    const float* ml = a.part_ml + row * PT * 2;
    const float* po = a.part_o + row * PT * D + lane * EPL;
    float M = kInitM;
    for (int i = lane; i < n; i += 64) M = fmaxf(M, ml[2 * i]);
    M = allreduce(M, Max{});
    float L = 0.f, acc[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int c = min(64, n - i0);
        float wl = 0.f;
        if (lane < c) {
            wl = __builtin_amdgcn_exp2f(ml[2 * (i0 + lane)] - M);
            L = fmaf(wl, ml[2 * (i0 + lane) + 1], L);
        }
        for (int j0 = 0; j0 < c; j0 += 16) {   // sixteen rows in flight; those past the count re-read the last, weighted 0
            float v[16][EPL];
#pragma unroll
            for (int jj = 0; jj < 16; ++jj)
#pragma unroll
                for (int e = 0; e < EPL; ++e) v[jj][e] = po[(size_t)(i0 + min(j0 + jj, c - 1)) * D + e];
#pragma unroll
            for (int jj = 0; jj < 16; ++jj) {
                const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wl), j0 + jj));
#pragma unroll
                for (int e = 0; e < EPL; ++e) acc[e] = fmaf(w, v[jj][e], acc[e]);
            }
        }
    }
    L = allreduce(L, Sum{});
    const float inv = L > 0.f ? 1.f / L : 1.f;   // a row that sees no key: O = 0
    uint16_t* o = a.o + row * D + lane * EPL;
    if constexpr (EPL == 2) *(uint32_t*)o = pack2<kBf16>(acc[0] * inv, acc[1] * inv);
    else o[0] = (uint16_t)pack2<kBf16>(acc[0] * inv, 0.f);
}

// ---- plan -----------------------------------------------------------------------------------------
struct SharedPlan {
    int G, HB, blocks, kpp, Pp, Po, kmin;
    long long prefix_groups, groups;
    size_t ws_bytes;
};

// A launch has fewer than 2^32 threads, and shared_join a wave per row (four to a workgroup).
constexpr long long kMaxRows = (1LL << 32) / 64 - 4;

bool plan_shared(const cdna4_shared_decode_cfg& c, SharedPlan& p) {
    if (c.D != 64 && c.D != 128) return false;
    if (c.nQHeads < 1 || c.nKVHeads < 1 || c.nQHeads % c.nKVHeads) return false;
    if (c.batch < 1 || c.prefix < 0 || c.max_own < 0) return false;
    if (c.prefix > 0x7fffffff - 1024 || c.max_own > 0x7fffffff - 1024) return false;
    if (c.stride_prefix != 0 && c.stride_prefix < c.prefix) return false;
    if (c.stride_kv != 0 && c.stride_kv < c.max_own) return false;
    const long long cus = device_cus(), slots = 2 * cus;
    p.G = c.nQHeads / c.nKVHeads;
    p.HB = (p.G + 15) / 16;
    const long long own_rows = (long long)c.batch * c.nKVHeads * p.HB;
    const long long rows = (long long)c.batch * p.G;
    if (rows > 0x7fffffff - kBlockRows || (long long)c.batch * c.nQHeads > kMaxRows) return false;
    p.blocks = (int)((rows + kBlockRows - 1) / kBlockRows);
    // prefix: parts of whole tiles
    p.Pp = 0;
    p.kpp = 64;
    if (c.prefix > 0) {
        const long long tiles = (c.prefix + 63) / 64, all = tiles * c.nKVHeads * p.blocks;
        // One part per CU (a CU with two runs each of them slower, and the parts' results are written and read
        // again: 64 sequences behind 8,192 keys, 32/8 heads D 128, 22.3 us with 256 parts, 27.5 with 128, 29.1
        // with 512), two where the parts stay long (256 behind 16,384: 73.8 against 81.4 us). With about as many
        // own keys, three quarters of that: their parts get the other CUs (64 behind 8,192 with 20-1,000 own
        // 29.6 against 32.2 us, 256 behind 16,384 with 64-2,048 142 against 151 us). Half the capacity is taken
        // for the own keys, whose number is on the device.
        const long long own = c.max_own / 2 / 64 * own_rows;
        const long long want = all >= 32 * slots && 8 * own < all ? slots : 2 * own >= all ? cus * 3 / 4 : cus;
        long long per = std::max(2LL, (all + want - 1) / want);
        per = std::min(per, tiles);
        p.kpp = (int)per * 64;
        p.Pp = (int)((tiles + per - 1) / per);
    }
    p.prefix_groups = ((long long)c.nKVHeads * p.Pp + 7) / 8 * p.blocks;
    // own keys
    p.Po = 0;
    p.kmin = 64;
    if (c.max_own > 0) {
        // Two rounds of parts at full lengths, of 64 to 1,024 keys, and up to 32 parts a row (more cost the join
        // more than they save: one sequence of 8,192 keys 10.7 us with 32, 17.5 with 128). 256 sequences of 64-2,048
        // keys: 108.8 us with 512 keys a part, 108.1 with 1,024, 113.7 with 2,048, 152 with 128.
        long long keys = (c.max_own * own_rows + 2 * slots - 1) / (2 * slots);
        keys = std::max({std::min(keys, 1024LL), 64LL, (c.max_own + 31LL) / 32});
        keys = (keys + 63) / 64 * 64;
        p.kmin = (int)keys;
        p.Po = (int)((c.max_own + keys - 1) / keys);
    }
    p.groups = p.prefix_groups + (own_rows * p.Po + 7) / 8;
    if (p.groups * 8 * 256 > 0xffffffffLL) return false;
    p.ws_bytes = (size_t)c.batch * c.nQHeads * (p.Pp + p.Po) * (size_t)(c.D + 2) * sizeof(float) + 256;
    return true;
}

template <int D, bool kBf16>
int launch_shared(const cdna4_shared_decode_cfg& c, const SharedPlan& p, const void* q, const void* Kp, const void* Vp,
                  const void* K, const void* V, const int* lens, void* o, void* ws, hipStream_t s) {
    SharedArgs a;
    a.q = (const uint16_t*)q; a.Kp = (const uint16_t*)Kp; a.Vp = (const uint16_t*)Vp; a.K = (const uint16_t*)K; a.V = (const uint16_t*)V;
    a.o = (uint16_t*)o;
    a.lens = lens;
    const size_t nml = (size_t)c.batch * c.nQHeads * (p.Pp + p.Po) * 2 * sizeof(float);
    a.part_ml = (float*)ws;
    a.part_o = (float*)((char*)ws + ((nml + 255) & ~(size_t)255));
    a.p_hs = (long long)(c.stride_prefix ? c.stride_prefix : c.prefix) * D;
    a.kv_hs = (long long)(c.stride_kv ? c.stride_kv : c.max_own) * D;
    a.nQH = c.nQHeads; a.nKVH = c.nKVHeads; a.G = p.G; a.HB = p.HB; a.batch = c.batch; a.prefix = c.prefix; a.max_own = c.max_own;
    a.blocks = p.blocks; a.kpp = p.kpp; a.Pp = p.Pp; a.Po = std::max(p.Po, 0); a.kmin = p.kmin;
    a.prefix_groups = (int)p.prefix_groups;
    a.sc = kLog2e / sqrtf((float)D);
    if (p.groups > 0) {
        const unsigned grid = (unsigned)(p.groups * 8);
        // own caches larger than the Infinity Cache are copied past it (stream::dma16)
        if (4.0 * c.batch * c.nKVHeads * c.max_own * D > 256.0 * 1024 * 1024) shared_parts<D, kBf16, true><<<grid, 256, 0, s>>>(a);
        else shared_parts<D, kBf16, false><<<grid, 256, 0, s>>>(a);
    }
    shared_join<D, kBf16><<<ceil_div((size_t)c.batch * c.nQHeads, 4), 256, 0, s>>>(a);
    return launch_status();
}

}  // namespace
}  // namespace cdna4

using namespace cdna4;

extern "C" size_t cdna4_attn_decode_shared_workspace_size(const cdna4_shared_decode_cfg* cfg) {
    SharedPlan p;
    if (!cfg || !plan_shared(*cfg, p)) return 0;
    return p.ws_bytes + 256;
}

extern "C" int cdna4_attn_decode_shared(const void* q, const void* K_prefix, const void* V_prefix, const void* K,
                                        const void* V, const int* lens, void* o, const cdna4_shared_decode_cfg* cfg,
                                        int dtype, void* workspace, size_t ws_bytes, cdna4_stream_t stream) {
    if (!cfg || (dtype != CDNA4_F16 && dtype != CDNA4_BF16)) return CDNA4_ERR_INVALID_VALUE;
    const cdna4_shared_decode_cfg& c = *cfg;
    if (c.batch == 0) return 0;
    SharedPlan p;
    if (!plan_shared(c, p)) return CDNA4_ERR_INVALID_VALUE;
    if (!q || !o || ((uintptr_t)q & 15u) || ((uintptr_t)o & 3u)) return CDNA4_ERR_INVALID_VALUE;
    if (c.prefix > 0 && (!K_prefix || !V_prefix || (((uintptr_t)K_prefix | (uintptr_t)V_prefix) & 15u))) return CDNA4_ERR_INVALID_VALUE;
    if (c.max_own > 0 && (!K || !V || (((uintptr_t)K | (uintptr_t)V) & 15u))) return CDNA4_ERR_INVALID_VALUE;
    if (c.max_own > 0 && (!lens || ((uintptr_t)lens & 3u))) return CDNA4_ERR_INVALID_VALUE;
    if (!workspace || ((uintptr_t)workspace & 15u) || ws_bytes < p.ws_bytes + 256) return CDNA4_ERR_INVALID_VALUE;
    if (int e = check_device()) return e;
    hipStream_t s = (hipStream_t)stream;
    const bool bf = dtype == CDNA4_BF16;
    if (c.D == 128)
        return bf ? launch_shared<128, true>(c, p, q, K_prefix, V_prefix, K, V, lens, o, workspace, s)
                  : launch_shared<128, false>(c, p, q, K_prefix, V_prefix, K, V, lens, o, workspace, s);
    return bf ? launch_shared<64, true>(c, p, q, K_prefix, V_prefix, K, V, lens, o, workspace, s)
              : launch_shared<64, false>(c, p, q, K_prefix, V_prefix, K, V, lens, o, workspace, s);
}

extern "C" int cdna4_attn_decode_shared_plan(const cdna4_shared_decode_cfg* cfg, int dtype, cdna3_plan_info* out) {
    SharedPlan p;
    if (!cfg || !out || (dtype != CDNA4_F16 && dtype != CDNA4_BF16) || !plan_shared(*cfg, p)) return CDNA4_ERR_INVALID_VALUE;
    out->kernel = CDNA4_KERNEL_DECODE_SHARED;
    out->waves = 4;
    out->rows = p.kpp;
    out->partials = p.Pp + p.Po;
    out->grid = p.groups * 8;
    out->workspace = p.ws_bytes + 256;
    return 0;
}
