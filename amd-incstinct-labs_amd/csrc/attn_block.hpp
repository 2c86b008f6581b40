// A block of 128 (or 64) queries against a key axis, the core of the packed prompt kernel (prefill_packed.hip) and of the
// shared prefix's part of a decode step (decode_shared.hip): four waves of 32 (16) queries over 64-key K/V tiles
// in LDS, the pipelined regions of attn_pipe.hpp, asynchronous copies two regions ahead.
#pragma once
#include <type_traits>

#include "attn_pipe.hpp"

namespace cdna4 {
namespace block {

using namespace tile;
using namespace pipe;

constexpr int kWaves = 4;
template <int QT> constexpr int rows_log2() { return QT == 2 ? 7 : 6; }   // queries per block: QT tiles of 16 per wave
template <int D> constexpr int lds_elems() { return 4 * kBc * D; }   // K slots 0, 1, V slots 0, 1
template <int D> constexpr int lds_v() { return 2 * kBc * D; }

// Keys of one sequence and kv head on the joint axis: k < P in the prefix, else own row k - P.
template <bool kPrefix>
struct Keys {
    const uint16_t *own, *pre;
    long long rs;
    int P, S;     // prefix keys, all keys
    int copy32;   // a tile's own rows span < 4 GiB: 32-bit offsets
    template <int D>
    __device__ __forceinline__ const uint16_t* row(int k) const {
        k = min(k, S - 1);   // rows past the end re-read the last key (masked)
        if constexpr (!kPrefix) return own + k * rs;
        else return k < P ? pre + (long long)k * D : own + (k - P) * rs;
    }
};

// Copy of `rows` keys from k0 on into an LDS slot by W waves, each lane's address formed by itself.
template <int D, int W, bool kIsK, bool kPrefix>
__device__ __forceinline__ void copy_any(const Keys<kPrefix>& k, int k0, int rows, uint16_t* dst, int wave, int lane) {
    constexpr int CPR = D / 8;
#pragma unroll
    for (int j = 0; j < rows * CPR / (64 * W); ++j) {
        const int p0 = (j * W + wave) * 64, p = p0 + lane, r = p / CPR;
        stream::dma16(k.template row<D>(k0 + r) + ((p % CPR) ^ swz<D, kIsK>(r)) * 8, dst + p0 * 8);
    }
}

// The copies of a whole step of K or of V, all in one source, that a region issues between its MFMAs: a
// wave-uniform base that moves on by whole rows per instruction, and per-lane offsets, of which two differ (a
// row's swizzle repeats every 32 rows, two instructions at D = 128).
template <int D, int W, int NI>
struct StepCopy {
    static constexpr int kCount = NI;
    static constexpr int kRows = 512 * W / D;   // rows of one instruction of all waves
    const uint16_t* base;
    uint16_t* dst;
    const uint32_t* off;   // [2]
    long long rs;
    int wave;
    __device__ __forceinline__ void issue(int c) const {
        stream::dma16_s(base + c * (kRows * rs), off[c & 1], dst + (c * W + wave) * 512);
    }
    template <bool kIsK>
    static __device__ __forceinline__ void offsets(long long rs, int wave, int lane, uint32_t (&off)[2]) {
        static_assert(kRows % 16 == 0, "rows 2 kRows apart have one swizzle");
        constexpr int CPR = D / 8;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int p = wave * 64 + lane, r = p / CPR, c = p % CPR;
            off[j] = (uint32_t)((r * rs + (c ^ swz<D, kIsK>(r + j * kRows)) * 8) * 2);
        }
    }
};

// The per-lane offsets of whole tiles' copies from own rows; those from a prefix (rows of D) are formed on use.
struct Offsets { uint32_t k[2], v[2]; };
template <int D>
__device__ __forceinline__ Offsets own_offsets(long long rs, int wave, int lane) {
    using CP = StepCopy<D, kWaves, kBc * (D / 8) / (64 * kWaves)>;
    Offsets o;
    CP::template offsets<true>(rs, wave, lane, o.k);
    CP::template offsets<false>(rs, wave, lane, o.v);
    return o;
}

// Copy of tile t into a slot: a whole tile of one source by a wave-uniform base and 32-bit offsets (a few scalar
// instructions), the others lane by lane.
template <int D, bool kIsK, bool kPrefix>
__device__ __forceinline__ void copy_tile(const Keys<kPrefix>& k, int t, const Offsets& own, uint16_t* dst, int wave, int lane) {
    constexpr int NI = kBc * (D / 8) / (64 * kWaves);
    using CP = StepCopy<D, kWaves, NI>;
    const int k0 = t * kBc;
    if (k.copy32 && k0 >= k.P && k0 + kBc <= k.S) {
        const CP c{k.own + (k0 - k.P) * k.rs, dst, kIsK ? own.k : own.v, k.rs, wave};
#pragma unroll
        for (int j = 0; j < NI; ++j) c.issue(j);
    } else if (kPrefix && k0 + kBc <= k.P) {
        uint32_t off[2];
        CP::template offsets<kIsK>(D, wave, lane, off);
        const CP c{k.pre + (long long)k0 * D, dst, off, D, wave};
#pragma unroll
        for (int j = 0; j < NI; ++j) c.issue(j);
    } else {
        copy_any<D, kWaves, kIsK>(k, k0, kBc, dst, wave, lane);
    }
}

// What the loop needs to know of a block: keys S on the joint axis, tiles ntiles, this wave's chunks nch (0:
// it has no queries), its first query on the key axis qv0 (causal), and main tiles t < t_main, whose chunks
// 2t + 1 and 2t + 2 every query sees and whose copies of V (t + 1) and K (t + 2) are whole tiles that exist.
struct Shape { int S, ntiles, nch, qv0, t_main; };

// The copies of K 0, V 0 and K 1, which attend waits for.
template <int D, bool kPrefix>
__device__ __forceinline__ void first_copies(const Keys<kPrefix>& keys_k, const Keys<kPrefix>& keys_v, int ntiles,
                                             const Offsets& own, uint16_t* lds, int wave, int lane) {
    copy_tile<D, true>(keys_k, 0, own, lds, wave, lane);
    copy_tile<D, false>(keys_v, 0, own, lds + lds_v<D>(), wave, lane);
    if (ntiles > 1) copy_tile<D, true>(keys_k, 1, own, lds + kBc * D, wave, lane);
}

// After first_copies: leaves the running base-2 maxima m, the sums lacc and O^T of the wave's queries (attn_tile.hpp's layout).
// Tile t's regions (attn_pipe.hpp), with a barrier before each:
//   region 2t     S of chunk 2t + 1 (K t), P.V of chunk 2t (V t); copies V (t + 1) into the slot of V (t - 1)
//   region 2t + 1 S of chunk 2t + 2 (K t + 1), P.V of chunk 2t + 1; copies K (t + 2) into the slot of K t
// so each copy has the time of two regions to land.
template <int D, int QT, bool kBf16, bool kPrefix, bool kCausal>
__device__ __forceinline__ void attend(const Keys<kPrefix>& keys_k, const Keys<kPrefix>& keys_v, const Shape& shape,
                                       const u32x4 (&qb)[QT][D / 32], f32x4 (&o)[QT][D / 16], f32x4 (&lacc)[QT],
                                       float (&m)[QT], const Offsets& own, uint16_t* lds, float sc, int wave,
                                       int lane) {
    constexpr int W = kWaves, NDT = D / 16;
    constexpr bool kAnyDiag = kPrefix || QT == 1;   // a wave's first query is no multiple of 32 on the key axis
    constexpr int kTile = kBc * D, NI = kBc * (D / 8) / (64 * W);
    const int li = lane & 15, g = lane >> 4;
    const int P = keys_k.P, S = shape.S, ntiles = shape.ntiles, nch = shape.nch, qv0 = shape.qv0, t_main = shape.t_main;
    uint16_t* const vlds = lds + lds_v<D>();
    auto copy_k = [&](int t) { copy_tile<D, true>(keys_k, t, own, lds + (t & 1) * kTile, wave, lane); };
    auto copy_v = [&](int t) { copy_tile<D, false>(keys_v, t, own, vlds + (t & 1) * kTile, wave, lane); };
    using CP = StepCopy<D, W, NI>;
    uint32_t koff[2] = {own.k[0], own.k[1]}, voff[2] = {own.v[0], own.v[1]};
    const float inv_sc = 1.f / sc;
    float thr[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        m[t] = kInitM;
        thr[t] = (kInitM + kTau) * inv_sc;
        lacc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < NDT; ++d) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const LdsOffsets off = lds_offsets<D>(li, g);
    u32x4 ones;
    {
        const uint32_t one2 = kBf16 ? 0x3F803F80u : 0x3C003C00u;
        ones = u32x4{one2, one2, one2, one2};
        asm volatile("" : "+v"(ones));
    }
    if (ntiles > 1) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * NI) : "memory");   // K 0 (V 0, K 1 newer)
    else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    __syncthreads();
    f32x4 s[QT][2];
    qk_chunk<D, QT, kBf16>((const char*)lds, off, qb, s, 0);
    {
        float lm[QT];
        if (32 > S || (kCausal && 31 > qv0)) mask_chunk<QT>(s, 0, qv0, S, kCausal, li, g);
        const bool need = check_raw<QT>(s, thr, lm) && nch > 0;
        if (__builtin_amdgcn_ballot_w64(need)) rescale_pipe<D, QT>(lm, m, thr, o, lacc, sc, inv_sc);
    }
    auto tile_iter = [&](int t, auto tail, auto two, int sl, const uint16_t* kb, const uint16_t* vb, long long rs) {
        constexpr bool kTail = decltype(tail)::value;
        constexpr bool kTwo = decltype(two)::value;
        const char* Kt = (const char*)(lds + sl * kTile);
        const char* Kn = (const char*)(lds + (sl ^ 1) * kTile);
        const char* Vt = (const char*)(vlds + sl * kTile);
        // V t landed (K t + 1 may be in flight); every wave is past region 2t - 1, the last reader of V t - 1
        if (kTail && t + 1 >= ntiles) asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" : : "n"(NI) : "memory");
        __syncthreads();
        if (kTail && t + 1 < ntiles) copy_v(t + 1);
        const int j0 = 2 * t;
        const CP cv{vb, vlds + (sl ^ 1) * kTile, voff, rs, wave};
        if (!kTail)
            pipe_region<D, QT, kBf16, false, true, NI, false, CP>(Kt, 1, Vt, 0, off, qb, s, o, m, thr, lacc, ones, true, (j0 + 1) * 32,
                                                                  qv0, S, kCausal, sc, inv_sc, li, g, cv);
        else if (j0 < nch)
            pipe_region<D, QT, kBf16, true, false, NI, kTwo, CP, kAnyDiag>(Kt, 1, Vt, 0, off, qb, s, o, m, thr, lacc, ones, j0 + 1 < nch,
                                                                 (j0 + 1) * 32, qv0, S, kCausal, sc, inv_sc, li, g, cv);
        // K t + 1 landed (V t + 1 may be in flight); every wave is past region 2t, the last reader of K t
        if (!kTail || t + 1 < ntiles) {
            asm volatile("s_waitcnt vmcnt(%0)" : : "n"(NI) : "memory");
            __syncthreads();
            if (kTail && t + 2 < ntiles) copy_k(t + 2);
        }
        const int j1 = 2 * t + 1;
        const CP ck{kb, lds + sl * kTile, koff, rs, wave};
        if (!kTail)
            pipe_region<D, QT, kBf16, false, true, NI, false, CP>(Kn, 0, Vt, 1, off, qb, s, o, m, thr, lacc, ones, true, (j1 + 1) * 32,
                                                                  qv0, S, kCausal, sc, inv_sc, li, g, ck);
        else if (j1 < nch)
            pipe_region<D, QT, kBf16, true, false, NI, kTwo, CP, kAnyDiag>(Kn, 0, Vt, 1, off, qb, s, o, m, thr, lacc, ones, j1 + 1 < nch,
                                                                 (j1 + 1) * 32, qv0, S, kCausal, sc, inv_sc, li, g, ck);
    };
    int t = 0;
    // bf16: keys 0..63 enter with their weights' second bf16 term where the queries see few keys
    if constexpr (kBf16) {
        if (t_main <= 0) {
            tile_iter(0, std::true_type{}, std::true_type{}, 0, nullptr, nullptr, 0);
            t = 1;
        }
    }
    // The joint axis in two passes: main tiles whose copies lie in the prefix, then (past the tiles whose
    // copies straddle its end, to an even tile) those whose copies lie in the sequence.
    bool pre = kPrefix;
    for (;;) {
        const long long rs = pre ? D : keys_k.rs;
        const uint16_t* kb = (pre ? keys_k.pre : keys_k.own - (long long)P * keys_k.rs) + 2LL * kBc * rs;
        const uint16_t* vb = (pre ? keys_v.pre : keys_v.own - (long long)P * keys_k.rs) + (long long)kBc * rs;
        const int t1 = pre ? min(t_main, P / kBc - 2) : t_main;   // main tiles of this source: t < t1
        if (pre) {
            CP::template offsets<true>(D, wave, lane, koff);
            CP::template offsets<false>(D, wave, lane, voff);
        }
#pragma unroll 1
        for (; t + 2 <= t1; t += 2) {
            tile_iter(t, std::false_type{}, std::false_type{}, 0, kb + (long long)t * kBc * rs, vb + (long long)t * kBc * rs, rs);
            tile_iter(t + 1, std::false_type{}, std::false_type{}, 1, kb + (long long)(t + 1) * kBc * rs, vb + (long long)(t + 1) * kBc * rs, rs);
        }
        // own main tiles begin where K (t + 2) and V (t + 1) lie past the prefix, at an even tile
        const int t2 = pre ? min(ntiles, ((P + kBc - 1) / kBc) & ~1) : ntiles;
#pragma unroll 1
        for (; t < t2; ++t) tile_iter(t, std::true_type{}, std::false_type{}, t & 1, nullptr, nullptr, 0);
        if (!pre) break;
        pre = false;
#pragma unroll
        for (int j = 0; j < 2; ++j) { koff[j] = own.k[j]; voff[j] = own.v[j]; }
    }
}

}  // namespace block
}  // namespace cdna4
