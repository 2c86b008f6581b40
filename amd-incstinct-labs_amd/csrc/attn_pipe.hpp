// The software-pipelined region of the prompt-attention key loops (gfx950): S^T of one 32-key chunk on the
// matrix cores with the exponentials of the chunk before placed between its MFMAs, then the P.V product of
// that chunk, masks and the lazy rescale; and the asynchronous K/V tile copies around it. Shared by the
// kernels of prompts of one length (prefill.hip) and of packed prompts (prefill_packed.hip).
#pragma once
#include "attn_tile.hpp"
#include "attn_stream.hpp"

namespace cdna4 {
namespace pipe {

using namespace tile;

constexpr int kBc = 64;       // keys per K/V tile

// Masks chunk scores s whose first key is kb: key >= seqK or (causal) key > query -> -inf.
template <int QT>
__device__ __forceinline__ void mask_chunk(f32x4 (&s)[QT][2], int kb, int qw0, int seqK, int causal, int li, int g) {
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = kb + g * 8 + u * 4 + e;
                const int q = qw0 + t * 16 + li;
                if (key >= seqK || (causal && key > q)) s[t][u][e] = -INFINITY;
            }
}

// Causal mask of the chunk whose first key is the wave's first query (kb == qw0, both multiples of
// 32): key - query = 4u + e - (16t + li - 8g) for lane (li, g), so the pattern is the same for every
// such chunk, 2 VALU per score instead of mask_chunk's general form. Chunks below qw0 need no
// causal mask, and those above it lie past the wave's last query (never used).
template <int QT>
__device__ __forceinline__ void mask_diag(f32x4 (&s)[QT][2], int li, int g) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int dq = 16 * t + li - 8 * g;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * u + e > dq) s[t][u][e] = -INFINITY;
    }
}

// Per-lane raw maxima lm of a chunk and whether one exceeds its query's threshold thr = (m + kTau)
// / sc, i.e. whether a scaled score exceeds the reference maximum by more than kTau (the
// threshold is kept in raw score units so that the check per chunk needs no multiply).
template <int QT>
__device__ __forceinline__ bool check_raw(const f32x4 (&s)[QT][2], const float (&thr)[QT], float (&lm)[QT]) {
    bool need = false;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        float v = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) v = fmaxf(v, s[t][u][e]);
        lm[t] = v;
        need |= v > thr[t];
    }
    return need;
}

// rescale_rows, then the thresholds of the new reference maxima.
template <int D, int QT>
__device__ __forceinline__ void rescale_pipe(const float (&lm)[QT], float (&m)[QT], float (&thr)[QT],
                                             f32x4 (&o)[QT][D / 16], f32x4 (&lacc)[QT], float sc, float inv_sc) {
    rescale_rows<D, QT>(lm, m, o, lacc, sc);
#pragma unroll
    for (int t = 0; t < QT; ++t) thr[t] = (m[t] + kTau) * inv_sc;
}

// The copy of one full K/V tile a region issues between its MFMAs (kCopy): global bases of the
// tile's K and V rows, their LDS buffers, and the per-lane offsets of copy_offsets.
template <int NI>
struct TileCopy {
    static constexpr int kCount = 2 * NI;
    const uint16_t* kg; const uint16_t* vg;
    uint16_t* kd; uint16_t* vd;
    const uint32_t* koff; const uint32_t* voff;
    int wave, W;
    __device__ __forceinline__ void issue(int c) const {   // copy c of 2 NI: K parts, then V parts
        const int j = c % NI;
        if (c < NI) stream::dma16_s(kg, koff[j], kd + (j * W + wave) * 64 * 8);
        else stream::dma16_s(vg, voff[j], vd + (j * W + wave) * 64 * 8);
    }
};

// Region j (see above). Kn (K tile of chunk j + 1, half kcn) always points into the LDS ring;
// when chunk j + 1 does not exist for this wave (has_next false, tail only) the scores formed
// from it are ignored. Vc / kcc: V tile and half of chunk j. kTail: mask chunk j + 1. kTwo (bf16,
// tail tile 0 only): chunk j also enters with its weights' second bf16 term (see kLoKeys). CP: the copies
// the region issues (kCopy). kAnyDiag: the causal diagonal lies anywhere in a chunk (qw0 is the wave's
// first query plus the number of keys before the sequence, no multiple of 32).
template <int D, int QT, bool kBf16, bool kTail, bool kCopy, int NI, bool kTwo = false, class CP = TileCopy<NI>,
          bool kAnyDiag = false>
__device__ __forceinline__ void pipe_region(const char* Kn, int kcn, const char* Vc, int kcc, const LdsOffsets& off,
                                           const u32x4 (&qb)[QT][D / 32], f32x4 (&s)[QT][2], f32x4 (&o)[QT][D / 16],
                                           float (&m)[QT], float (&thr)[QT], f32x4 (&lacc)[QT], const u32x4& ones,
                                           bool has_next, int kbn, int qw0, int seqK, int causal, float sc,
                                           float inv_sc, int li, int g, const CP& cp) {
    constexpr int NK = (D / 32) * 2;   // K operand reads (ds_read_b128) of chunk j + 1, i = 2c + u
    constexpr int NV = D / 16;         // V^T operands of chunk j (two transpose reads each)
    constexpr int NP = QT * 8;         // P_j values per lane
    constexpr int SL = NP / NK;        // P values per interleave slot
    constexpr int kAhead = 2;          // LDS operand reads issued ahead of their MFMAs
    static_assert(NP % NK == 0, "the exponentials spread evenly over the slots");
    if constexpr (kTwo) {
        // Chunk j's keys lie below kLoKeys: first the P.V product of its weights' second bf16 term
        // (s holds chunk j's masked scores, m is the reference P_j is formed against; the sum into
        // O and l does not depend on the order), before chunk j + 1's scores are live.
        u32x4 pl[QT];
        softmax_lo_chunk<QT>(s, m, pl, sc);
        pv_chunk<D, QT, true>(Vc, off, pl, o, lacc, kcc);
        __builtin_amdgcn_sched_barrier(0);   // the region's reads stay after this block
    }
    float p[QT][8];
    u32x4 pb[QT];
    f32x4 sn[QT][2];
    u32x4 ka[NK];
    auto kread = [&](int i) {
        ka[i] = *(const u32x4*)(Kn + off.kc(i >> 1) + (kcn * 32 + (i & 1) * 4) * D * 2);
    };
    auto soft = [&](int v) {   // P value v (query tile v / 8, element v % 8)
        const int t = v >> 3, x = v & 7;
        p[t][x] = __builtin_amdgcn_exp2f(fmaf(s[t][x >> 2][x & 3], sc, -m[t]));
        if (x & 1) pb[t][x >> 1] = pack2<kBf16>(p[t][x - 1], p[t][x]);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kread(i);
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) sn[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
    // S^T of chunk j + 1, one K operand (QT MFMAs) per slot, SL values of P_j per slot. The
    // scheduling barriers keep the slots in this order.
    // Wave priority 2 here, 1 for the P.V part, 0 for the check and the copies between regions:
    // measured +1.7 to +2.7 % on the causal B4 H32 S8192 D128 prefill over equal priorities.
    __builtin_amdgcn_s_setprio(2);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < QT; ++t) sn[t][i & 1] = mfma<kBf16>(ka[i], qb[t][i >> 1], sn[t][i & 1]);
        if (i + kAhead < NK) kread(i + kAhead);
        // the region's copies spread over its NK slots (fa_pipe: one per odd slot): the waves'
        // copies then reach the texture unit spread over the region instead of all after the barrier
        if constexpr (kCopy) {
#pragma unroll
            for (int c = i * CP::kCount / NK; c < (i + 1) * CP::kCount / NK; ++c) cp.issue(c);
        }
#pragma unroll
        for (int v = 0; v < SL; ++v) soft(i * SL + v);
    }
    __builtin_amdgcn_sched_barrier(0);
    u32x4 va[NV];
    auto vread = [&](int dt) {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(Vc + off.vd(dt) + (kcc * 32) * D * 2));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4*)(Vc + off.vd(dt) + (kcc * 32 + 4) * D * 2));
        const u32x2 lo2 = __builtin_bit_cast(u32x2, lo), hi2 = __builtin_bit_cast(u32x2, hi);
        va[dt] = u32x4{lo2[0], lo2[1], hi2[0], hi2[1]};
    };
#pragma unroll
    for (int dt = 0; dt < kAhead; ++dt) vread(dt);
    __builtin_amdgcn_s_setprio(1);
    // l += row sums of exactly the rounded weights the product uses (all-ones A operand)
#pragma unroll
    for (int t = 0; t < QT; ++t) lacc[t] = mfma<kBf16>(ones, pb[t], lacc[t]);
#pragma unroll
    for (int dt = 0; dt < NV; ++dt) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < QT; ++t) o[t][dt] = mfma<kBf16>(va[dt], pb[t], o[t][dt]);
        if (dt + kAhead < NV) vread(dt + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if constexpr (kTail && kAnyDiag) {
        if (kbn + 31 > qw0) mask_chunk<QT>(sn, kbn, qw0, seqK, causal, li, g);
    } else if constexpr (kTail) {   // wave-uniform branches: most tail chunks need neither mask
        if (causal && kbn == qw0) mask_diag<QT>(sn, li, g);
        if (kbn + 32 > seqK) mask_chunk<QT>(sn, kbn, qw0, seqK, causal, li, g);
    }
    float lm[QT];
    bool need = check_raw<QT>(sn, thr, lm);
    if constexpr (kTail) need = need && has_next;
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[t][u] = sn[t][u];
    if (__builtin_amdgcn_ballot_w64(need)) rescale_pipe<D, QT>(lm, m, thr, o, lacc, sc, inv_sc);
}

// Asynchronous copy of keys [k0, k0 + kBc) of one head into an LDS tile (inline assembly, see
// stream::dma16), chunks placed by the K (kIsK) or the V swizzle.
template <int D, int W, bool kIsK>
__device__ __forceinline__ void copy_tile(const uint16_t* __restrict__ head, long long row_stride, int k0, int seqK,
                                          uint16_t* tile, int wave, int lane) {
    constexpr int CPR = D / 8;
    constexpr int NI = kBc * CPR / (64 * W);
    static_assert(NI >= 1 && NI * 64 * W == kBc * CPR, "tile copy must split evenly over the waves");
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int p0 = (j * W + wave) * 64;
        const int p = p0 + lane;
        const int r = p / CPR;
        const int lc = (p % CPR) ^ swz<D, kIsK>(r);
        const int key = min(k0 + r, seqK - 1);   // rows past the end re-read the last key (masked)
        stream::dma16(head + key * row_stride + lc * 8, tile + p0 * 8);
    }
}

// Per-lane byte offsets of the copy of a full tile (row r, swizzled 16-byte chunk lc), the same for
// every tile of a head, so formed once per work item: a full tile's copies then need only a
// wave-uniform base (stream::dma16_s).
template <int D, int W, bool kIsK>
__device__ __forceinline__ void copy_offsets(long long row_stride, int wave, int lane,
                                             uint32_t (&voff)[kBc * (D / 8) / (64 * W)]) {
    constexpr int CPR = D / 8;
    constexpr int NI = kBc * CPR / (64 * W);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int p = (j * W + wave) * 64 + lane;
        const int r = p / CPR;
        const int lc = (p % CPR) ^ swz<D, kIsK>(r);
        voff[j] = (uint32_t)(((long long)r * row_stride + lc * 8) * 2);
    }
}

// Copy of keys [k0, k0 + kBc), all inside the sequence, with the offsets above.
template <int D, int W>
__device__ __forceinline__ void copy_tile_full(const uint16_t* head, long long row_stride, int k0,
                                               const uint32_t (&voff)[kBc * (D / 8) / (64 * W)], uint16_t* tile,
                                               int wave) {
    constexpr int NI = kBc * (D / 8) / (64 * W);
    const uint16_t* base = head + (long long)k0 * row_stride;
#pragma unroll
    for (int j = 0; j < NI; ++j) stream::dma16_s(base, voff[j], tile + (j * W + wave) * 64 * 8);
}

}  // namespace pipe
}  // namespace cdna4
