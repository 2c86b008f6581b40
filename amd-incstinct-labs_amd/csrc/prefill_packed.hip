// Prompt attention over packed sequences for gfx950: prompts of different lengths one after another in
// token-major Q, K, V, causal within each, optionally behind a prefix of keys that all of them see.
//
// Token i of sequence s (rows cu[s] .. cu[s+1] - 1) sees the P prefix keys and its sequence's tokens 0 .. i:
//   O = sum_j 2^(c q.k_j - m) v_j / sum_j 2^(c q.k_j - m),  c = log2(e) / sqrt(D), m a running maximum.
// The kernels are the prompt kernels' tile machinery (attn_tile.hpp, attn_pipe.hpp) over one key axis per
// sequence, prefix keys 0 .. P - 1 and then the sequence's own, with no padding where they meet: key k lies
// in the prefix cache or in the packed rows, and the tile that holds both takes its addresses per lane.
//
// Lengths are read on the device (a captured call replays on other lengths): a workgroup finds its item,
// one block of queries of one sequence and head, from cu alone. Blocks are ordered by their index in the
// sequence, the last ones (the most keys) first, so that the hardware's in-order dispatch gives the chip a
// longest-first schedule whatever the lengths are.
#include <type_traits>
#include <algorithm>

#include "attn_tile.hpp"
#include "attn_stream.hpp"
#include "attn_block.hpp"

namespace cdna4 {
namespace {

using namespace tile;
using namespace pipe;
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
    int copy32;   // 1: a step's rows span < 4 GiB (32-bit copy offsets)
    float sc;     // log2(e) / sqrt(D)
};

// ---- work items ----------------------------------------------------------------------------------
// Blocks of sequence s with `rows` queries each; cu outside 0 .. total or decreasing is cut to it, so that
// no contents of cu lead outside the tensors.
__device__ __forceinline__ void seq_rows(const PackedArgs& a, int s, int& start, int& len) {
    start = min(max(a.cu[s], 0), a.total);
    len = min(max(a.cu[s + 1], start), a.total) - start;   // cut before the difference, which then cannot wrap
}

// Entry idx of the list of blocks, block index descending and sequences ascending within one index:
// f(d) = sum_s max(0, n_s - d) blocks have an index of d or more, so idx lies at the largest d with
// f(d) > idx, found by bisection; each lane holds the block counts of sequences lane, lane + 64, ..
// (kHeld in registers, the rest read again). Six wave sums at 64 blocks a sequence, ~0.3 us.
// False past the last block.
constexpr int kHeld = 4;
template <int kRows>
__device__ __forceinline__ bool packed_item(const PackedArgs& a, int idx, int lane, int& start, int& len, int& blk) {
    int n[kHeld];
    auto blocks = [&](int s) {
        int st, ln;
        if (s >= a.batch) return 0;
        seq_rows(a, s, st, ln);
        return (ln + kRows - 1) / kRows;
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
    // every lane holds a wave sum: readfirstlane keeps what follows from it scalar
    auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    if (idx >= scalar(allreduce(sum, Sum{}))) return false;
    auto above = [&](int d) {   // f(d)
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
    return blk * kRows < len;   // always, but for counts of overlapping sequences that pass 32 bits
}

// Head of workgroup i within one entry's nQH workgroups. Workgroups go to the XCDs round-robin: with nQH a
// multiple of 8 each XCD takes nQH / 8 neighbouring query heads, which share K and V heads in its L2.
__device__ __forceinline__ int item_head(int i, int nQH) {
    return (nQH & 7) ? i : (i & 7) * (nQH >> 3) + (i >> 3);
}

template <int D, bool kBf16>
__device__ __forceinline__ void store_rows(const f32x4 (&o)[D / 16], float l, uint16_t* dst) {
    const float inv = l > 0.f ? 1.f / l : 1.f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
        *(u32x2*)(dst + dt * 16) = u32x2{pack2<kBf16>(o[dt][0] * inv, o[dt][1] * inv), pack2<kBf16>(o[dt][2] * inv, o[dt][3] * inv)};
}

// ---- 128 queries per workgroup, two workgroups per CU ---------------------------------------------
// Four waves of 32 queries share 64-key K/V tiles in LDS, two slots each for K and V (64 KiB at D = 128), so
// that two workgroups fit a CU: while one fills its first tiles, masks its diagonal or stores, the other has
// the matrix cores. Tile t's regions (attn_pipe.hpp), with a barrier before each:
//   region 2t     S of chunk 2t + 1 (K t), P.V of chunk 2t (V t); copies V (t + 1) into the slot of V (t - 1)
//   region 2t + 1 S of chunk 2t + 2 (K t + 1), P.V of chunk 2t + 1; copies K (t + 2) into the slot of K t
// so each copy has the time of two regions to land.
template <int D, bool kBf16, bool kPrefix>
__global__ __launch_bounds__(256, 2) void fa_packed(PackedArgs a) {
    constexpr int QT = block::kQT, ND = D / 32, NDT = D / 16, BM = block::kRows;
    __shared__ __attribute__((aligned(16))) uint16_t lds[block::lds_elems<D>()];
    const int lane = (int)(threadIdx.x & 63u);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int li = lane & 15, g = lane >> 4;

    const int entry = (int)blockIdx.x / a.nQH;
    const int h = item_head((int)blockIdx.x - entry * a.nQH, a.nQH);
    int start, len, blk;
    if (!packed_item<BM>(a, entry, lane, start, len, blk)) return;
    const int P = kPrefix ? a.prefix : 0;
    const int q0 = blk * BM, qw0 = q0 + wave * QT * 16, S = P + len;
    const int kvh = h / a.G;
    const uint16_t* own_k = a.K + start * a.k_rs + kvh * a.k_hs;
    const uint16_t* own_v = a.V + start * a.k_rs + kvh * a.k_hs;
    const Keys<kPrefix> keys_k{own_k, a.Kp + kvh * a.p_hs, a.k_rs, P, S};
    const Keys<kPrefix> keys_v{own_v, a.Vp + kvh * a.p_hs, a.k_rs, P, S};
    u32x4 qb[QT][ND];
    {
        const uint16_t* Qh = a.Q + start * a.q_rs + h * a.q_hs;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int q = min(qw0 + t * 16 + li, len - 1);
#pragma unroll
            for (int c = 0; c < ND; ++c) qb[t][c] = *(const u32x4*)(Qh + q * a.q_rs + c * 32 + g * 8);
        }
    }
    const int ntiles = (P + min(q0 + BM, len) + kBc - 1) / kBc;
    const int wave_end = min(qw0 + QT * 16, len);                     // one past this wave's last query
    const int nch = wave_end > qw0 ? (P + wave_end + 31) / 32 : 0;     // the wave's chunks; 0: no queries
    // Main tiles: chunks 2t + 1 and 2t + 2 lie below the workgroup's first query, and the copies of
    // V (t + 1) and K (t + 2) are whole tiles that exist.
    int t_main = P + q0 >= 95 ? (P + q0 - 95) / 64 + 1 : 0;
    t_main = min(t_main, min(ntiles - 2, S / kBc - 2));
    if (!a.copy32) t_main = 0;

    f32x4 o[QT][NDT], lacc[QT];
    float m[QT];
    block::attend<D, kBf16, kPrefix, true>(keys_k, keys_v, block::Shape{S, ntiles, nch, P + qw0, t_main}, qb, o, lacc, m,
                                           lds, a.sc, wave, lane);

    uint16_t* Oh = a.O + start * a.o_rs + h * a.o_hs;
#pragma unroll
    for (int x = 0; x < QT; ++x) {
        const int q = qw0 + x * 16 + li;
        if (q < len) store_rows<D, kBf16>(o[x], lacc[x][0], Oh + q * a.o_rs + g * 4);
    }
}

}  // namespace

namespace {

int check_packed(const cdna4_packed_cfg* cfg, const cdna4_packed_strides* st, const void* Q, const void* K, const void* V,
                 const void* Kp, const void* Vp, const void* O, const int* cu, int dtype) {
    if (!cfg || !st) return CDNA4_ERR_INVALID_VALUE;
    const cdna4_packed_cfg& c = *cfg;
    if (c.D != 64 && c.D != 128) return CDNA4_ERR_INVALID_VALUE;
    if (dtype != CDNA4_F16 && dtype != CDNA4_BF16) return CDNA4_ERR_INVALID_VALUE;
    if (c.nQHeads < 1 || c.nKVHeads < 1 || c.nQHeads % c.nKVHeads) return CDNA4_ERR_INVALID_VALUE;
    if (c.batch < 0 || c.total < 0 || c.max_seq < 0 || c.max_seq > c.total || c.prefix < 0) return CDNA4_ERR_INVALID_VALUE;
    if (c.total > 0 && c.prefix > 0x7fffffff - 1024 - c.total) return CDNA4_ERR_INVALID_VALUE;   // keys are counted in 32 bits
    if (c.stride_prefix != 0 && c.stride_prefix < c.prefix) return CDNA4_ERR_INVALID_VALUE;
    const long long in[4] = {st->q_row, st->q_head, st->kv_row, st->kv_head};
    for (long long x : in)
        if (x < 0 || (x & 7)) return CDNA4_ERR_INVALID_VALUE;
    const long long out[2] = {st->o_row, st->o_head};
    for (long long x : out)
        if (x < 0 || (x & 3)) return CDNA4_ERR_INVALID_VALUE;
    if (st->q_row < c.D || st->kv_row < c.D || st->o_row < c.D) return CDNA4_ERR_INVALID_VALUE;
    if (c.batch == 0 || c.total == 0) return 0;
    if (!Q || !K || !V || !O || !cu || ((uintptr_t)cu & 3u)) return CDNA4_ERR_INVALID_VALUE;
    if ((((uintptr_t)Q | (uintptr_t)K | (uintptr_t)V) & 15u) || ((uintptr_t)O & 7u)) return CDNA4_ERR_INVALID_VALUE;
    if (c.prefix > 0 && (!Kp || !Vp || (((uintptr_t)Kp | (uintptr_t)Vp) & 15u))) return CDNA4_ERR_INVALID_VALUE;
    return 0;
}

struct PackedPlan { int kernel, waves, rows; long long grid; };

template <int D>
PackedPlan plan_packed(const cdna4_packed_cfg& c) {
    PackedPlan p{};
    p.kernel = CDNA4_KERNEL_PACKED_4W;
    p.waves = 4;
    p.rows = 128;
    // sum of ceil(len / rows) is at most total / rows + the sequences that are not empty
    p.grid = (long long)c.nQHeads * (c.total / p.rows + std::min(c.batch, c.total));
    return p;
}

template <int D, bool kBf16>
int launch_packed(const cdna4_packed_cfg& c, const cdna4_packed_strides& st, const void* Q, const void* K, const void* V,
                  const void* Kp, const void* Vp, void* O, const int* cu, hipStream_t s) {
    const PackedPlan p = plan_packed<D>(c);
    if (p.grid * 64 * p.waves > 0xffffffffLL) return CDNA4_ERR_INVALID_VALUE;
    PackedArgs a;
    a.Q = (const uint16_t*)Q; a.K = (const uint16_t*)K; a.V = (const uint16_t*)V; a.O = (uint16_t*)O;
    a.Kp = (const uint16_t*)Kp; a.Vp = (const uint16_t*)Vp;
    a.cu = cu;
    a.q_rs = st.q_row; a.q_hs = st.q_head; a.k_rs = st.kv_row; a.k_hs = st.kv_head; a.o_rs = st.o_row; a.o_hs = st.o_head;
    a.p_hs = (long long)(c.stride_prefix ? c.stride_prefix : c.prefix) * D;
    a.nQH = c.nQHeads; a.G = c.nQHeads / c.nKVHeads; a.batch = c.batch; a.total = c.total; a.prefix = c.prefix;
    a.copy32 = 256 * st.kv_row * 2 < (1LL << 32) ? 1 : 0;
    a.sc = kLog2e / sqrtf((float)D);
    const unsigned grid = (unsigned)p.grid;
    if (c.prefix) fa_packed<D, kBf16, true><<<grid, 256, 0, s>>>(a);
    else fa_packed<D, kBf16, false><<<grid, 256, 0, s>>>(a);
    return launch_status();
}

}  // namespace
}  // namespace cdna4

using namespace cdna4;

extern "C" int cdna4_attn_prefill_packed(const void* Q, const void* K, const void* V, const void* K_prefix,
                                         const void* V_prefix, void* O, const int* cu_seqlens, const cdna4_packed_cfg* cfg,
                                         const cdna4_packed_strides* strides, int dtype, cdna4_stream_t stream) {
    if (int e = check_packed(cfg, strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, dtype)) return e;
    if (cfg->batch == 0 || cfg->total == 0) return 0;
    if (int e = check_device()) return e;
    hipStream_t s = (hipStream_t)stream;
    const bool bf = dtype == CDNA4_BF16;
    if (cfg->D == 128)
        return bf ? launch_packed<128, true>(*cfg, *strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, s)
                  : launch_packed<128, false>(*cfg, *strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, s);
    return bf ? launch_packed<64, true>(*cfg, *strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, s)
              : launch_packed<64, false>(*cfg, *strides, Q, K, V, K_prefix, V_prefix, O, cu_seqlens, s);
}

extern "C" int cdna4_attn_prefill_packed_plan(const cdna4_packed_cfg* cfg, int dtype, cdna3_plan_info* out) {
    if (!cfg || !out) return CDNA4_ERR_INVALID_VALUE;
    const cdna4_packed_cfg& c = *cfg;
    if ((c.D != 64 && c.D != 128) || (dtype != CDNA4_F16 && dtype != CDNA4_BF16)) return CDNA4_ERR_INVALID_VALUE;
    if (c.nQHeads < 1 || c.nKVHeads < 1 || c.nQHeads % c.nKVHeads) return CDNA4_ERR_INVALID_VALUE;
    if (c.batch < 1 || c.total < 1 || c.max_seq < 0 || c.max_seq > c.total || c.prefix < 0) return CDNA4_ERR_INVALID_VALUE;
    const PackedPlan p = c.D == 128 ? plan_packed<128>(c) : plan_packed<64>(c);
    out->kernel = p.kernel;
    out->waves = p.waves;
    out->rows = p.rows;
    out->grid = p.grid;
    out->partials = 1;
    out->workspace = 0;
    return 0;
}
