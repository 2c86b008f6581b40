// Logits of a batch made ready for the sampler (gfx950): penalties for repeated tokens, biases, grammar masks.
//
// Row m, token j, with c the number of times j was generated (history entries from prompt_len on) and s whether
// j is in the history at all (prompt or generated):
//   x = logit;  s: x = x > 0 ? x / repetition : x * repetition;  x -= c frequency + (c > 0) presence;
//   x += bias of j;  not allowed by the mask: x = -inf.
// All in fp32 whatever the logits' type, fp32 out.
//
// One launch: a workgroup serves one chunk of one row's vocabulary. It counts the history entries that fall
// into its chunk in LDS (integer atomics: the counts do not depend on their order), then streams the chunk, 16
// bytes per load, and applies everything in one pass. Bound by HBM: the logits read, the results written.
#include <algorithm>

#include "common.hpp"

namespace cdna4 {
namespace {

typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));   // rows of odd length start anywhere
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kSeen = 0x80000000u;   // in the prompt; lower bits: times generated

template <int kDtype>
__device__ __forceinline__ float widen(uint32_t b) {
    return kDtype == CDNA4_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

struct Penalty { float rep, freq, pres; };

__device__ __forceinline__ float penalise(float x, uint32_t word, const Penalty& p) {
    if (word) {
        x = x > 0.f ? x / p.rep : x * p.rep;
        const float c = (float)(word & ~kSeen);
        x = fmaf(-c, p.freq, x);
        if (c > 0.f) x -= p.pres;
    }
    return x;
}

template <int kDtype, int kThreads>
__global__ __launch_bounds__(kThreads) void process_logits_kernel(cdna4_logits_args a, int chunk) {
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];   // counts [chunk], then 1 + bias entry [chunk]
    const int tid = (int)threadIdx.x;
    const size_t m = blockIdx.y;
    const int c0 = (int)blockIdx.x * chunk, n = min(chunk, a.V - c0);
    Penalty p{a.repetition ? a.repetition[m] : 1.f, a.frequency ? a.frequency[m] : 0.f, a.presence ? a.presence[m] : 0.f};
    int hist = 0, made = 0;
    if (a.history && !(p.rep == 1.f && p.freq == 0.f && p.pres == 0.f)) {   // neutral penalties change nothing
        hist = a.history_len ? min(max(a.history_len[m], 0), a.history_max) : a.history_max;
        made = a.prompt_len ? min(max(a.prompt_len[m], 0), hist) : 0;
    }
    uint32_t* const bias_at = lds + (a.history ? chunk : 0);
    const bool penal = hist > 0;
    if (penal || a.n_bias) {
        const int words = (penal ? chunk : 0) + (a.n_bias ? chunk : 0);
        uint4* z = (uint4*)(penal ? lds : bias_at);
        for (int i = tid; i < words / 4; i += kThreads) z[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        const int* h = a.history + m * a.history_stride;
        for (int j = tid; j < hist; j += kThreads) {
            const uint32_t at = (uint32_t)h[j] - (uint32_t)c0;
            if (at < (uint32_t)n) {
                if (j < made) atomicOr(&lds[at], kSeen);
                else atomicAdd(&lds[at], 1u);
            }
        }
        const int* b = a.bias_ids + m * a.n_bias;
        for (int j = tid; j < a.n_bias; j += kThreads) {   // of several entries for one token the last counts
            const uint32_t at = (uint32_t)b[j] - (uint32_t)c0;
            if (at < (uint32_t)n) atomicMax(&bias_at[at], (uint32_t)j + 1u);
        }
        __syncthreads();
    }
    const float* bv = a.bias_values + m * a.n_bias;
    const uint32_t* mask = a.mask ? a.mask + m * a.mask_stride : nullptr;
    float* out = a.out + m * a.out_stride + c0;
    auto finish = [&](float x, int i) {   // token c0 + i
        if (penal) x = penalise(x, lds[i], p);
        if (a.n_bias) {
            const uint32_t e = bias_at[i];
            if (e) x += bv[e - 1];
        }
        return x;
    };
    constexpr int kVec = 8;
    const int nv = n / kVec;
    for (int v = tid; v < nv; v += kThreads) {
        const int i = v * kVec;
        float x[kVec];
        if constexpr (kDtype == CDNA4_F32) {
            const float* in = (const float*)a.logits + m * a.logits_stride + c0 + i;
            const f32x4_u lo = *(const f32x4_u*)in, hi = *(const f32x4_u*)(in + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[e] = lo[e]; x[4 + e] = hi[e]; }
        } else {
            const u32x4_u w = *(const u32x4_u*)((const uint16_t*)a.logits + m * a.logits_stride + c0 + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) { x[2 * e] = widen<kDtype>(w[e] & 0xffffu); x[2 * e + 1] = widen<kDtype>(w[e] >> 16); }
        }
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] = finish(x[e], i + e);
        if (mask) {   // c0 + i is a multiple of 8: the bits lie in one word
            const uint32_t bits = mask[(c0 + i) >> 5] >> ((c0 + i) & 31);
#pragma unroll
            for (int e = 0; e < kVec; ++e) if (!((bits >> e) & 1u)) x[e] = -INFINITY;
        }
        f32x4_u lo, hi;
#pragma unroll
        for (int e = 0; e < 4; ++e) { lo[e] = x[e]; hi[e] = x[4 + e]; }
        *(f32x4_u*)(out + i) = lo;
        *(f32x4_u*)(out + i + 4) = hi;
    }
    for (int i = nv * kVec + tid; i < n; i += kThreads) {   // the row's last V % 8 tokens
        float x;
        if constexpr (kDtype == CDNA4_F32) x = ((const float*)a.logits)[m * a.logits_stride + c0 + i];
        else x = widen<kDtype>(((const uint16_t*)a.logits)[m * a.logits_stride + c0 + i]);
        x = finish(x, i);
        if (mask && !((mask[(c0 + i) >> 5] >> ((c0 + i) & 31)) & 1u)) x = -INFINITY;
        out[i] = x;
    }
}

int check_logits(const cdna4_logits_args* a, int dtype) {
    if (!a) return CDNA4_ERR_INVALID_VALUE;
    if (dtype != CDNA4_F32 && dtype != CDNA4_F16 && dtype != CDNA4_BF16) return CDNA4_ERR_INVALID_VALUE;
    if (a->M < 0 || a->V < 1 || a->V > 0x7fffffff - 65536) return CDNA4_ERR_INVALID_VALUE;
    if (a->M > 65535) return CDNA4_ERR_INVALID_VALUE;   // rows are the grid's second axis
    if (a->logits_stride < a->V || a->out_stride < a->V) return CDNA4_ERR_INVALID_VALUE;
    if (a->history_max < 0 || a->history_max > (1 << 24) || a->n_bias < 0 || a->n_bias > (1 << 24)) return CDNA4_ERR_INVALID_VALUE;
    if (a->M == 0) return 0;
    const uintptr_t el = dtype == CDNA4_F32 ? 3u : 1u;
    if (!a->logits || !a->out || ((uintptr_t)a->logits & el) || ((uintptr_t)a->out & 3u)) return CDNA4_ERR_INVALID_VALUE;
    if (a->history && a->history_stride < a->history_max) return CDNA4_ERR_INVALID_VALUE;
    if (a->n_bias > 0 && (!a->bias_ids || !a->bias_values)) return CDNA4_ERR_INVALID_VALUE;
    if (a->mask && a->mask_stride < ((long long)a->V + 31) / 32) return CDNA4_ERR_INVALID_VALUE;
    const void* words[9] = {a->history, a->history_len, a->prompt_len, a->repetition, a->frequency, a->presence, a->bias_ids, a->bias_values, a->mask};
    for (const void* w : words)
        if ((uintptr_t)w & 3u) return CDNA4_ERR_INVALID_VALUE;
    return 0;
}

constexpr int kMaxChunk = 8192, kMinChunk = 1024;

int chunk_of(const cdna4_logits_args& a) {
    int chunk = kMaxChunk;
    while (chunk > kMinChunk && (long long)a.M * ((a.V + chunk - 1) / chunk) < 4LL * device_cus()) chunk >>= 1;
    return chunk;
}

template <int kDtype>
int launch_logits(const cdna4_logits_args& a, hipStream_t s) {
    const int chunk = chunk_of(a);
    const dim3 grid((unsigned)((a.V + chunk - 1) / chunk), (unsigned)a.M);
    const size_t lds = ((a.history ? (size_t)chunk : 0) + (a.n_bias ? (size_t)chunk : 0)) * 4;
    process_logits_kernel<kDtype, 256><<<grid, 256, lds, s>>>(a, chunk);
    return launch_status();
}

}  // namespace
}  // namespace cdna4

using namespace cdna4;

extern "C" int cdna4_process_logits(const cdna4_logits_args* args, int dtype, cdna4_stream_t stream) {
    if (int e = check_logits(args, dtype)) return e;
    if (args->M == 0) return 0;
    if (int e = check_device()) return e;
    cdna4_logits_args a = *args;
    if (a.history_max == 0) a.history = nullptr;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == CDNA4_F32) return launch_logits<CDNA4_F32>(a, s);
    return dtype == CDNA4_BF16 ? launch_logits<CDNA4_BF16>(a, s) : launch_logits<CDNA4_F16>(a, s);
}
