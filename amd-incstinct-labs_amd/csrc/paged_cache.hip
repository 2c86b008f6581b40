// The paged KV cache's writers (gfx950): tokens appended with norm and rotation on the way, and a batch of beams reordered.
//
// Append, for each head row x of a token: x' = x rsqrt(mean(x^2) + eps) w, then the pair (d, d + D/2) turned by the angle of its
// position, y_lo = c_lo x'_lo - s_lo x'_hi, y_hi = c_hi x'_hi + s_hi x'_lo; queries go to q_out, keys and values to row
// position % page of page tables[sequence][position / page]. Norm and rotation in fp32, or in fp64 for keys that become 4-bit codes: an
// fp32 rounding before the code's would take some values next to the middle of two codes to the wrong one.
// A wave holds the angles of one token for as many heads as leave the chip 16 waves per CU, four rounds of rows on their way at a
// time; no LDS. Bound by HBM: 24 prompts of 33-2,048 bf16 tokens, 32/8 heads, D 128, normed, with the keys written twice (348 MB) 70-74 us,
// 4.8 TB/s, what a copy reaches; chunks of 1,000-8,192 into MXFP4 (789 MB) 181-195 us, 4.2 TB/s, with the fp64 beside it. A step of four
// tokens: 3.4 us, the launch and two dependent loads.
//
// Reorder: the tables and lengths of the new rows, and the rows of their last pages that are not full, copied to pages of their own. 64 beams in
// eight layers (108 MB) 19-21 us, 5.3 TB/s; four beams in twelve layers 3.6 us.
#include <algorithm>

#include "paged.hpp"
#include "wave_primitives/detail/xlane.hpp"

namespace cdna4 {
namespace {

using namespace paged;
using wave::xlane::dpp_full;

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AppendArgs {
    cdna4_append_args p;
    int HK, page, lp, pages, max_pages, per_wave, chunks;   // per_wave: rounds of a wave over its heads
    long long table_stride;
};

// Sum, or maximum, over the D / 8 lanes that hold a row, or over the 8 lanes that hold a block of 32 values.
template <int kLanes, class T, class Op>
__device__ __forceinline__ T lanes_allreduce(T v, Op op) {
    v = op(v, dpp_full<wave::xlane::kQuadXor1>(v));
    v = op(v, dpp_full<wave::xlane::kQuadXor2>(v));
    v = op(v, dpp_full<wave::xlane::kRowHalfMirror>(v));
    if constexpr (kLanes == 16) v = op(v, dpp_full<wave::xlane::kRowMirror>(v));
    return v;
}

template <bool kBf16>
__device__ __forceinline__ float widen(uint32_t b) { return kBf16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b); }
template <bool kBf16>
__device__ __forceinline__ uint32_t narrow(float f) { return kBf16 ? f32_to_bf16_bits(f) : f32_to_f16_bits(f); }

template <bool kBf16>
__device__ __forceinline__ void widen4(uint2 u, float (&x)[4]) {
    x[0] = widen<kBf16>(u.x & 0xffffu);
    x[1] = widen<kBf16>(u.x >> 16);
    x[2] = widen<kBf16>(u.y & 0xffffu);
    x[3] = widen<kBf16>(u.y >> 16);
}
template <bool kBf16>
__device__ __forceinline__ uint2 narrow4(const float (&x)[4]) {
    return make_uint2(narrow<kBf16>(x[0]) | narrow<kBf16>(x[1]) << 16, narrow<kBf16>(x[2]) | narrow<kBf16>(x[3]) << 16);
}

// A row in D / 8 lanes: lane i holds elements 4 i .. 4 i + 3 of its lower half and the same of its upper one, so that
// the pairs of the rotation are in one lane and a block of 32 in 8 neighbouring ones.
constexpr int kAhead = 4;   // rounds whose loads a wave has in flight
struct Angles { f32x4 c_lo, s_lo, c_hi, s_hi; };

// Norm and rotation in F.
template <class F, int D>
__device__ __forceinline__ void norm_rope(F (&lo)[4], F (&hi)[4], bool norm, const float (&w_lo)[4], const float (&w_hi)[4], double eps, bool turn,
                                          const Angles& an) {
    if (norm) {
        F s = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fma(lo[e], lo[e], fma(hi[e], hi[e], s));
        s = lanes_allreduce<D / 8>(s, wave::xlane::Sum{});
        F r;
        if constexpr (sizeof(F) == 8) r = 1.0 / sqrt(s * (1.0 / D) + eps);
        else r = 1.f / sqrtf(s * (1.f / D) + (float)eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lo[e] = lo[e] * r * (F)w_lo[e];
            hi[e] = hi[e] * r * (F)w_hi[e];
        }
    }
    if (turn) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const F a = lo[e], b = hi[e];
            lo[e] = fma((F)an.c_lo[e], a, -(b * (F)an.s_lo[e]));
            hi[e] = fma((F)an.c_hi[e], b, a * (F)an.s_hi[e]);
        }
    }
}

// One wave per token and `per_wave` rounds of heads, a row for every D / 8 of its lanes: the angles are loaded once.
template <int D, bool kBf16, bool kFp4>
__global__ __launch_bounds__(256) void append_paged(AppendArgs a) {
    constexpr int kLanes = D / 8, kRows = 64 / kLanes;   // rows of a wave at a time
    const int lane = (int)(threadIdx.x & 63u), i = lane % kLanes;
    const long long item = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int t = (int)(item / a.chunks), chunk = (int)(item % a.chunks);
    if (t >= a.p.T) return;
    const int seq = a.p.seqs ? a.p.seqs[t] : t, pos = a.p.positions[t];
    const bool turn = a.p.cos_tab != nullptr;
    if (seq < 0 || seq >= a.p.batch || pos < 0 || (pos >> a.lp) >= a.max_pages || (turn && pos >= a.p.max_pos)) return;
    const int page = a.p.tables[seq * a.table_stride + (pos >> a.lp)], row = pos & (a.page - 1);
    const bool placed = page >= 0 && page < a.pages;
    const int slots = a.p.nQHeads + 2 * a.HK;
    Angles an;
    if (turn) {
        const float *c = a.p.cos_tab + (size_t)pos * D + 4 * i, *s = a.p.sin_tab + (size_t)pos * D + 4 * i;
        an.c_lo = *(const f32x4*)c;
        an.s_lo = *(const f32x4*)s;
        an.c_hi = *(const f32x4*)(c + D / 2);
        an.s_hi = *(const f32x4*)(s + D / 2);
    }
    float wq[2][4], wk[2][4];
    if (a.p.q_norm) {
        widen4<kBf16>(*(const uint2*)((const uint16_t*)a.p.q_norm + 4 * i), wq[0]);
        widen4<kBf16>(*(const uint2*)((const uint16_t*)a.p.q_norm + D / 2 + 4 * i), wq[1]);
    }
    if (a.p.k_norm) {
        widen4<kBf16>(*(const uint2*)((const uint16_t*)a.p.k_norm + 4 * i), wk[0]);
        widen4<kBf16>(*(const uint2*)((const uint16_t*)a.p.k_norm + D / 2 + 4 * i), wk[1]);
    }
    const size_t page_bytes = (size_t)a.page * row_bytes(D, kFp4);
    const size_t place = ((size_t)(placed ? page : 0) * a.HK) * page_bytes;
    const uint16_t *q = (const uint16_t*)a.p.q + t * a.p.q_row, *k = (const uint16_t*)a.p.k + t * a.p.k_row, *v = (const uint16_t*)a.p.v + t * a.p.v_row;
    const int slot0 = chunk * a.per_wave * kRows + lane / kLanes;
    for (int j0 = 0; j0 < a.per_wave; j0 += kAhead) {
        if (slot0 - lane / kLanes + j0 * kRows >= slots) break;
        uint2 in_lo[kAhead], in_hi[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {   // rows past the last re-read it
            const int slot = min(slot0 + (j0 + j) * kRows, slots - 1);
            const uint16_t* src = slot < a.p.nQHeads ? q + slot * D : slot < a.p.nQHeads + a.HK ? k + (slot - a.p.nQHeads) * D : v + (slot - a.p.nQHeads - a.HK) * D;
            in_lo[j] = *(const uint2*)(src + 4 * i);
            in_hi[j] = *(const uint2*)(src + D / 2 + 4 * i);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int slot = slot0 + (j0 + j) * kRows;
            if (slot >= slots || j0 + j >= a.per_wave) break;
            const bool is_q = slot < a.p.nQHeads, is_k = !is_q && slot < a.p.nQHeads + a.HK;
            const int h = is_q ? slot : is_k ? slot - a.p.nQHeads : slot - a.p.nQHeads - a.HK;
            const uint2 u_lo = in_lo[j], u_hi = in_hi[j];
            float lo[4], hi[4];
            widen4<kBf16>(u_lo, lo);
            widen4<kBf16>(u_hi, hi);
            uint16_t* out = nullptr;
            if (is_q) out = (uint16_t*)a.p.q_out + t * a.p.q_out_row + h * D + 4 * i;
            else if (is_k && a.p.k_out) out = (uint16_t*)a.p.k_out + t * a.p.k_out_row + h * D + 4 * i;
            else if (!is_k && a.p.v_out) out = (uint16_t*)a.p.v_out + t * a.p.v_out_row + h * D + 4 * i;
            char* pool = (char*)(is_k ? a.p.K_pages : a.p.V_pages) + place + h * page_bytes;
            if (kFp4 && !is_q) {
                if (is_k && (a.p.k_norm || turn)) {
                    double dlo[4], dhi[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) { dlo[e] = lo[e]; dhi[e] = hi[e]; }
                    norm_rope<double, D>(dlo, dhi, a.p.k_norm != nullptr, wk[0], wk[1], a.p.eps, turn, an);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { lo[e] = round_to_odd(dlo[e]); hi[e] = round_to_odd(dhi[e]); }
                }
                uint32_t m_lo = 0, m_hi = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    m_lo = max(m_lo, __builtin_bit_cast(uint32_t, lo[e]) & 0x7fffffffu);
                    m_hi = max(m_hi, __builtin_bit_cast(uint32_t, hi[e]) & 0x7fffffffu);
                }
                const uint32_t b_lo = scale_byte<kBf16>(lanes_allreduce<8>(m_lo, wave::xlane::Max{}));
                const uint32_t b_hi = scale_byte<kBf16>(lanes_allreduce<8>(m_hi, wave::xlane::Max{}));
                const uint32_t c_lo = encode4(lo, b_lo), c_hi = encode4(hi, b_hi);
                if (placed) {
                    uint8_t* code = (uint8_t*)pool + row * (D / 2) + 2 * i;
                    *(uint16_t*)code = (uint16_t)c_lo;
                    *(uint16_t*)(code + D / 4) = (uint16_t)c_hi;
                    if ((i & 7) == 0) {
                        uint8_t* scale = (uint8_t*)pool + a.page * (D / 2) + row * (D / 32) + (i >> 3);
                        scale[0] = (uint8_t)b_lo;
                        scale[D / 64] = (uint8_t)b_hi;
                    }
                }
                if (out) {
                    const float f_lo = f32_from_bits(b_lo << 23), f_hi = f32_from_bits(b_hi << 23);
                    *(uint2*)out = make_uint2(decode2<kBf16, 0>(c_lo, f_lo), decode2<kBf16, 1>(c_lo, f_lo));
                    *(uint2*)(out + D / 2) = make_uint2(decode2<kBf16, 0>(c_hi, f_hi), decode2<kBf16, 1>(c_hi, f_hi));
                }
            } else {
                uint2 r_lo = u_lo, r_hi = u_hi;
                if (is_q || is_k) {
                    const bool normed = is_q ? a.p.q_norm != nullptr : a.p.k_norm != nullptr;
                    if (!kBf16 && !normed && turn) {   // the bits of the other kernels that write a cache
                        const uint32_t x[4] = {u_lo.x & 0xffffu, u_lo.x >> 16, u_lo.y & 0xffffu, u_lo.y >> 16};
                        const uint32_t y[4] = {u_hi.x & 0xffffu, u_hi.x >> 16, u_hi.y & 0xffffu, u_hi.y >> 16};
                        uint32_t p[4], q[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) rope_pair(x[e], y[e], an.c_lo[e], an.s_lo[e], an.c_hi[e], an.s_hi[e], p[e], q[e]);
                        r_lo = make_uint2(p[0] | p[1] << 16, p[2] | p[3] << 16);
                        r_hi = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
                    } else if (normed || turn) {
                        float w_lo[4], w_hi[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            w_lo[e] = is_q ? wq[0][e] : wk[0][e];
                            w_hi[e] = is_q ? wq[1][e] : wk[1][e];
                        }
                        norm_rope<float, D>(lo, hi, normed, w_lo, w_hi, a.p.eps, turn, an);
                        r_lo = narrow4<kBf16>(lo);
                        r_hi = narrow4<kBf16>(hi);
                    }
                }
                if (!is_q && placed) {
                    uint16_t* dst = (uint16_t*)pool + row * D + 4 * i;
                    *(uint2*)dst = r_lo;
                    *(uint2*)(dst + D / 2) = r_hi;
                }
                if (out) {
                    *(uint2*)out = r_lo;
                    *(uint2*)(out + D / 2) = r_hi;
                }
            }
        }
    }
}

// A launch has fewer than 2^32 threads, and the largest calls take a wave per token.
constexpr int kMaxTokens = (1 << 26) - 8;

int check_append(const cdna4_append_args* p, const cdna4_paged_cache* c, int dtype) {
    if (!p || !c || !valid_cache(*c)) return CDNA4_ERR_INVALID_VALUE;
    if (dtype != CDNA4_F16 && dtype != CDNA4_BF16) return CDNA4_ERR_INVALID_VALUE;
    if (p->T < 0 || p->nQHeads < 0 || p->nQHeads > (1 << 20) || p->batch < 1 || p->max_pos < 0) return CDNA4_ERR_INVALID_VALUE;
    if (p->T > kMaxTokens) return CDNA4_ERR_INVALID_VALUE;
    if ((p->cos_tab == nullptr) != (p->sin_tab == nullptr)) return CDNA4_ERR_INVALID_VALUE;
    if (p->nQHeads > 0 && (p->q == nullptr) != (p->q_out == nullptr)) return CDNA4_ERR_INVALID_VALUE;
    if (!(p->eps >= 0.0)) return CDNA4_ERR_INVALID_VALUE;
    const long long qd = (long long)p->nQHeads * c->D, kd = (long long)c->nKVHeads * c->D;
    const long long rows[6] = {p->q_row, p->q_out_row, p->k_row, p->v_row, p->k_out_row, p->v_out_row};
    for (int i = 0; i < 6; ++i)
        if (rows[i] != 0 && (rows[i] < (i < 2 ? qd : kd) || (rows[i] & 3))) return CDNA4_ERR_INVALID_VALUE;
    if (p->T == 0) return 0;
    if (!p->k || !p->v || !p->K_pages || !p->V_pages || !p->tables || !p->positions) return CDNA4_ERR_INVALID_VALUE;
    if (p->nQHeads > 0 && !p->q) return CDNA4_ERR_INVALID_VALUE;
    const void* by8[] = {p->q, p->k, p->v, p->q_out, p->k_out, p->v_out, p->q_norm, p->k_norm};
    for (const void* x : by8)
        if ((uintptr_t)x & 7u) return CDNA4_ERR_INVALID_VALUE;
    const void* by16[] = {p->K_pages, p->V_pages, p->cos_tab, p->sin_tab};
    for (const void* x : by16)
        if ((uintptr_t)x & 15u) return CDNA4_ERR_INVALID_VALUE;
    const void* by4[] = {p->tables, p->seqs, p->positions};
    for (const void* x : by4)
        if ((uintptr_t)x & 3u) return CDNA4_ERR_INVALID_VALUE;
    // in place only row by row: waves write while others read
    auto same = [](const void* in, const void* out, long long in_row, long long out_row, long long packed) {
        return in && in == out && (in_row ? in_row : packed) != (out_row ? out_row : packed);
    };
    if (p->T > 1 && (same(p->q, p->q_out, p->q_row, p->q_out_row, qd) || same(p->k, p->k_out, p->k_row, p->k_out_row, kd) ||
                     same(p->v, p->v_out, p->v_row, p->v_out_row, kd))) return CDNA4_ERR_INVALID_VALUE;
    return 0;
}

template <int D>
int launch_append(const cdna4_append_args& p, const cdna4_paged_cache& c, int dtype, hipStream_t s) {
    constexpr int kRows = 64 / (D / 8);
    AppendArgs a;
    a.p = p;
    const long long qd = (long long)p.nQHeads * D, kd = (long long)c.nKVHeads * D;
    if (!p.q_row) a.p.q_row = qd;
    if (!p.q_out_row) a.p.q_out_row = qd;
    if (!p.k_row) a.p.k_row = kd;
    if (!p.v_row) a.p.v_row = kd;
    if (!p.k_out_row) a.p.k_out_row = kd;
    if (!p.v_out_row) a.p.v_out_row = kd;
    a.HK = c.nKVHeads; a.page = c.page; a.lp = log2_of(c.page); a.pages = c.pages; a.max_pages = c.max_pages;
    a.table_stride = table_stride(c);
    const int rounds = (p.nQHeads + 2 * c.nKVHeads + kRows - 1) / kRows;
    // a wave takes as many of its token's heads as leave the chip 16 waves per CU
    const long long waves = 16LL * device_cus();
    a.per_wave = (int)std::min<long long>(rounds, std::max<long long>(1, (long long)p.T * rounds / waves));
    a.chunks = (rounds + a.per_wave - 1) / a.per_wave;
    const unsigned grid = ceil_div((size_t)p.T * a.chunks, 4);
    const bool bf = dtype == CDNA4_BF16, fp4 = c.format == CDNA4_KV_MXFP4;
    if (bf && fp4) append_paged<D, true, true><<<grid, 256, 0, s>>>(a);
    else if (bf) append_paged<D, true, false><<<grid, 256, 0, s>>>(a);
    else if (fp4) append_paged<D, false, true><<<grid, 256, 0, s>>>(a);
    else append_paged<D, false, false><<<grid, 256, 0, s>>>(a);
    return launch_status();
}

// ---- reorder ----------------------------------------------------------------------------------------
struct ReorderArgs {
    const int *parents, *tables, *lens, *fresh;
    int *tables_out, *lens_out;
    char *K, *V;
    int HK, page, lp, pages, max_pages, rows_in, segs;   // segs: layers x 2 x heads
    int code, scale;                                      // bytes of a row; MXFP4: of its codes and of its scales
    long long table_stride, layer_stride;
};

// blockIdx.y: the row. Workgroup x copies heads x, x + gridDim.x, .. of the row's last page in K and V of all layers; the first
// one of a row also writes its table.
__global__ __launch_bounds__(256) void reorder_paged(ReorderArgs a) {
    const int i = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int p = a.parents[i];
    const bool used = p >= 0 && p < a.rows_in;
    const int n = used ? min(max(a.lens[p], 0), a.max_pages << a.lp) : 0;
    const int last = n >> a.lp, rest = n & (a.page - 1);
    const int* from = a.tables + (used ? p : 0) * a.table_stride;
    const int fresh = rest ? a.fresh[i] : 0, src = rest ? from[last] : 0;
    if (blockIdx.x == 0) {
        int* to = a.tables_out + i * a.table_stride;
        for (int j = tid; j < a.max_pages; j += 256) to[j] = !used ? -1 : rest && j == last ? fresh : from[j];
        if (tid == 0) a.lens_out[i] = n;
    }
    if (!rest || fresh == src || fresh < 0 || fresh >= a.pages || src < 0 || src >= a.pages) return;
    const size_t head = (size_t)a.page * (a.code + a.scale);
    for (int g = (int)blockIdx.x; g < a.segs; g += (int)gridDim.x) {
        const int h = g % a.HK, kv = g / a.HK & 1, layer = g / a.HK / 2;
        char* pool = (kv ? a.V : a.K) + layer * a.layer_stride + h * head;
        const char* x = pool + (size_t)src * a.HK * head;
        char* y = pool + (size_t)fresh * a.HK * head;
        for (int j = tid; j < rest * a.code / 16; j += 256) ((u32x4*)y)[j] = ((const u32x4*)x)[j];
        const size_t at = (size_t)a.page * a.code;
        for (int j = tid; j < rest * a.scale / 2; j += 256) ((uint16_t*)(y + at))[j] = ((const uint16_t*)(x + at))[j];
    }
}

}  // namespace
}  // namespace cdna4

using namespace cdna4;

extern "C" int cdna4_rope_append_paged(const cdna4_append_args* args, const cdna4_paged_cache* cache, int dtype, cdna4_stream_t stream) {
    if (int e = check_append(args, cache, dtype)) return e;
    if (args->T == 0) return 0;
    if (int e = check_device()) return e;
    return cache->D == 128 ? launch_append<128>(*args, *cache, dtype, (hipStream_t)stream)
                           : launch_append<64>(*args, *cache, dtype, (hipStream_t)stream);
}

extern "C" int cdna4_paged_reorder(const int* parents, const int* tables, const int* lens, const int* fresh, int* tables_out,
                                   int* lens_out, void* K_pages, void* V_pages, const cdna4_paged_cache* cache, int rows,
                                   int rows_in, int layers, long long layer_stride, cdna4_stream_t stream) {
    if (!cache || !paged::valid_cache(*cache)) return CDNA4_ERR_INVALID_VALUE;
    const cdna4_paged_cache& c = *cache;
    const bool fp4 = c.format == CDNA4_KV_MXFP4;
    const long long pool = (long long)c.pages * c.nKVHeads * c.page * paged::row_bytes(c.D, fp4);
    if (rows < 0 || rows > 65535 || rows_in < 1 || layers < 1 || layers > 1 << 12) return CDNA4_ERR_INVALID_VALUE;
    if (layer_stride != 0 && (layer_stride < pool || (layer_stride & 15))) return CDNA4_ERR_INVALID_VALUE;
    if (rows == 0) return 0;
    const void* words[6] = {parents, tables, lens, fresh, tables_out, lens_out};
    for (const void* w : words)
        if (!w || ((uintptr_t)w & 3u)) return CDNA4_ERR_INVALID_VALUE;
    if (tables_out == tables || lens_out == lens || lens_out == parents) return CDNA4_ERR_INVALID_VALUE;
    if (!K_pages || !V_pages || (((uintptr_t)K_pages | (uintptr_t)V_pages) & 15u)) return CDNA4_ERR_INVALID_VALUE;
    if (int e = check_device()) return e;
    ReorderArgs a;
    a.parents = parents; a.tables = tables; a.lens = lens; a.fresh = fresh;
    a.tables_out = tables_out; a.lens_out = lens_out;
    a.K = (char*)K_pages; a.V = (char*)V_pages;
    a.HK = c.nKVHeads; a.page = c.page; a.lp = paged::log2_of(c.page); a.pages = c.pages; a.max_pages = c.max_pages;
    a.rows_in = rows_in;
    a.segs = layers * 2 * c.nKVHeads;   // up to 2^12 x 2 x 2^16: 2^29
    a.code = fp4 ? c.D / 2 : 2 * c.D;
    a.scale = fp4 ? c.D / 32 : 0;
    a.table_stride = paged::table_stride(c);
    a.layer_stride = layer_stride ? layer_stride : pool;
    // a launch has fewer than 2^32 threads
    const int most = (int)((1LL << 24) / rows) - 1;
    reorder_paged<<<dim3((unsigned)(a.segs < most ? a.segs : most), (unsigned)rows), 256, 0, (hipStream_t)stream>>>(a);
    return launch_status();
}
