// Logits of a batch made ready for the sampler (gfx950): penalties for repeated tokens, biases, grammar masks.
//
// Row m, token j, with c the number of times j was generated (history entries from prompt_len on) and s whether
// j is in the history at all (prompt or generated):
//   x = logit;  s: x = x > 0 ? x / repetition : x * repetition;  x -= c frequency + (c > 0) presence;
//   x += bias of j;  not allowed by the mask: x = -inf.
// All in fp32 whatever the logits' type, fp32 out.
//
// One launch: a workgroup serves one chunk of one row's vocabulary. It reads the chunk's logits into registers, and
// while they are on their way counts the history entries that fall into the chunk in LDS (integer atomics: the
// counts do not depend on their order); then it applies penalties and mask and writes the chunk, 16 bytes per
// store. The few biases are added to what was written, behind a barrier. Bound by HBM, the logits read and the
// results written: 256 rows of 131,072 fp32 50 us called on inputs that change from call to call (5.4 TB/s), 44 in a graph on
// one set of inputs, which the caches hold in part; small calls by the chain of the row's scalars, its history and the
// counts (4 rows of 32,000 fp16 3.7 us in a graph).
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace cdna4 {
namespace {

typedef uint32_t u32x2_u __attribute__((ext_vector_type(2), aligned(2)));   // rows of odd length start anywhere
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4_u __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kSeen = 0x80000000u;   // in the prompt; lower bits: times generated
constexpr int kThreads = 256;
constexpr int kVec = 4;                   // tokens per load and store of a thread
constexpr int kBiasPerThread = 32;        // one bit each
constexpr int kMaxBias = kThreads * kBiasPerThread;

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

// NV vectors per thread: chunks of 1,024 NV tokens.
template <int kDtype, int NV>
__global__ __launch_bounds__(kThreads) void process_logits_kernel(cdna4_logits_args a) {
    constexpr int kChunk = kThreads * kVec * NV;
    constexpr int kFirst = 4;   // history vectors per thread that are loaded ahead of the logits
    extern __shared__ __attribute__((aligned(16))) uint32_t count[];   // [kChunk], with a history or biases
    const int tid = (int)threadIdx.x;
    const size_t m = blockIdx.y;
    const int c0 = (int)blockIdx.x * kChunk, n = min(kChunk, a.V - c0);
    Penalty p{a.repetition ? a.repetition[m] : 1.f, a.frequency ? a.frequency[m] : 0.f, a.presence ? a.presence[m] : 0.f};
    int hist = 0, made = 0;
    if (a.history && !(p.rep == 1.f && p.freq == 0.f && p.pres == 0.f)) {   // neutral penalties change nothing
        hist = a.history_len ? min(max(a.history_len[m], 0), a.history_max) : a.history_max;
        made = a.prompt_len ? min(max(a.prompt_len[m], 0), hist) : 0;
    }
    const bool penal = hist > 0;
    const int* h = a.history + m * a.history_stride;
    // Loads without a branch on the lane, so that all of them are in flight at once: lanes past the end read the
    // last vector again.
    i32x4_u first[kFirst];
    const bool vec_h = hist >= 4;
    if (vec_h) {
#pragma unroll
        for (int k = 0; k < kFirst; ++k) first[k] = *(const i32x4_u*)(h + min((k * kThreads + tid) * 4, hist - 4));
    }
    std::conditional_t<kDtype == CDNA4_F32, f32x4_u, u32x2_u> raw[NV];
    const uint32_t* mask = a.mask ? a.mask + m * a.mask_stride : nullptr;
    uint32_t bits[NV];
    if (n >= kVec) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int i = min((v * kThreads + tid) * kVec, n - kVec);
            if constexpr (kDtype == CDNA4_F32) raw[v] = *(const f32x4_u*)((const float*)a.logits + m * a.logits_stride + c0 + i);
            else raw[v] = *(const u32x2_u*)((const uint16_t*)a.logits + m * a.logits_stride + c0 + i);
        }
        if (mask) {
#pragma unroll
            for (int v = 0; v < NV; ++v) bits[v] = mask[(c0 + min((v * kThreads + tid) * kVec, n - 1)) >> 5];
        }
    }
    auto clear = [&]() {
        for (int i = tid; i < kChunk / 4; i += kThreads) ((uint4*)count)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    };
    // Of several biases for one token the last counts: the entries' places by a maximum in the array that the
    // counts take over afterwards. Bit k of `wins`: entry k kThreads + tid counts.
    const int* b = a.bias_ids + m * a.n_bias;
    uint32_t wins = 0;
    if (a.n_bias) {
        clear();
        for (int j = tid; j < a.n_bias; j += kThreads) {
            const uint32_t at = (uint32_t)b[j] - (uint32_t)c0;
            if (at < (uint32_t)n) atomicMax(&count[at], (uint32_t)j + 1u);
        }
        __syncthreads();
        for (int j = tid, k = 0; j < a.n_bias; j += kThreads, ++k) {
            const uint32_t at = (uint32_t)b[j] - (uint32_t)c0;
            if (at < (uint32_t)n && count[at] == (uint32_t)j + 1u) wins |= 1u << k;
        }
        __syncthreads();
    }
    if (penal) {
        clear();
        auto add = [&](int id, int j) {
            const uint32_t at = (uint32_t)id - (uint32_t)c0;
            if (at < (uint32_t)n) {
                if (j < made) atomicOr(&count[at], kSeen);
                else atomicAdd(&count[at], 1u);
            }
        };
        if (vec_h) {
#pragma unroll
            for (int k = 0; k < kFirst; ++k) {
                const int j = (k * kThreads + tid) * 4;
                if (j + 4 > hist) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) add(first[k][e], j + e);
            }
        }
        // what the vectors did not hold: entries past the first ones, or the last three at most
        for (int j = min(hist & ~3, kFirst * kThreads * 4) + tid; j < hist; j += kThreads) add(h[j], j);
        __syncthreads();
    }
    float* out = a.out + m * a.out_stride + c0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int i = (v * kThreads + tid) * kVec;
        if (i + kVec > n) continue;
        f32x4_u x;
        if constexpr (kDtype == CDNA4_F32) x = raw[v];
        else x = f32x4_u{widen<kDtype>(raw[v][0] & 0xffffu), widen<kDtype>(raw[v][0] >> 16), widen<kDtype>(raw[v][1] & 0xffffu), widen<kDtype>(raw[v][1] >> 16)};
        if (penal) {
            const uint4 w = *(const uint4*)(count + i);
            if (w.x | w.y | w.z | w.w) {
                x[0] = penalise(x[0], w.x, p);
                x[1] = penalise(x[1], w.y, p);
                x[2] = penalise(x[2], w.z, p);
                x[3] = penalise(x[3], w.w, p);
            }
        }
        if (mask) {   // c0 + i is a multiple of 4: the bits lie in one word
            const uint32_t w = bits[v] >> ((c0 + i) & 31);
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (!((w >> e) & 1u)) x[e] = -INFINITY;
        }
        *(f32x4_u*)(out + i) = x;
    }
    auto allowed = [&](int i) { return !mask || ((mask[(c0 + i) >> 5] >> ((c0 + i) & 31)) & 1u); };
    if (tid < (n & (kVec - 1))) {   // the row's last V % 4 tokens
        const int i = (n & ~(kVec - 1)) + tid;
        float x;
        if constexpr (kDtype == CDNA4_F32) x = ((const float*)a.logits)[m * a.logits_stride + c0 + i];
        else x = widen<kDtype>(((const uint16_t*)a.logits)[m * a.logits_stride + c0 + i]);
        if (penal) x = penalise(x, count[i], p);
        out[i] = allowed(i) ? x : -INFINITY;
    }
    if (a.n_bias) {
        __syncthreads();   // the workgroup's results are written
        const float* bv = a.bias_values + m * a.n_bias;
        for (int j = tid, k = 0; j < a.n_bias; j += kThreads, ++k) {
            const int at = b[j] - c0;
            if (((wins >> k) & 1u) && allowed(at)) out[at] += bv[j];
        }
    }
}

int check_logits(const cdna4_logits_args* a, int dtype) {
    if (!a) return CDNA4_ERR_INVALID_VALUE;
    if (dtype != CDNA4_F32 && dtype != CDNA4_F16 && dtype != CDNA4_BF16) return CDNA4_ERR_INVALID_VALUE;
    if (a->M < 0 || a->V < 1 || a->V > 0x7fffffff - 65536) return CDNA4_ERR_INVALID_VALUE;
    if (a->M > 65535) return CDNA4_ERR_INVALID_VALUE;   // rows are the grid's second axis
    if (a->logits_stride < a->V || a->out_stride < a->V) return CDNA4_ERR_INVALID_VALUE;
    if (a->history_max < 0 || a->history_max > (1 << 24) || a->n_bias < 0 || a->n_bias > kMaxBias) return CDNA4_ERR_INVALID_VALUE;
    if (a->M == 0) return 0;
    const uintptr_t el = dtype == CDNA4_F32 ? 3u : 1u;
    if (!a->logits || !a->out || ((uintptr_t)a->logits & el) || ((uintptr_t)a->out & 3u)) return CDNA4_ERR_INVALID_VALUE;
    // in place only element by element: workgroups of a row write while others read
    if (a->logits == a->out && (dtype != CDNA4_F32 || (a->M > 1 && a->logits_stride != a->out_stride))) return CDNA4_ERR_INVALID_VALUE;
    if (a->history && a->history_stride < a->history_max) return CDNA4_ERR_INVALID_VALUE;
    if (a->n_bias > 0 && (!a->bias_ids || !a->bias_values)) return CDNA4_ERR_INVALID_VALUE;
    if (a->mask && a->mask_stride < ((long long)a->V + 31) / 32) return CDNA4_ERR_INVALID_VALUE;
    const void* words[9] = {a->history, a->history_len, a->prompt_len, a->repetition, a->frequency, a->presence, a->bias_ids, a->bias_values, a->mask};
    for (const void* w : words)
        if ((uintptr_t)w & 3u) return CDNA4_ERR_INVALID_VALUE;
    return 0;
}

template <int kDtype>
int launch_logits(const cdna4_logits_args& a, hipStream_t s) {
    // chunks as large as leave the chip four workgroups per CU: the history is read once per chunk
    int nv = 8;
    while (nv > 1 && (long long)a.M * ((a.V + 1024 * nv - 1) / (1024 * nv)) < 4LL * device_cus()) nv >>= 1;
    const dim3 grid((unsigned)((a.V + 1024 * nv - 1) / (1024 * nv)), (unsigned)a.M);
    const size_t lds = a.history || a.n_bias ? (size_t)1024 * nv * 4 : 0;
    switch (nv) {
        case 8: process_logits_kernel<kDtype, 8><<<grid, kThreads, lds, s>>>(a); break;
        case 4: process_logits_kernel<kDtype, 4><<<grid, kThreads, lds, s>>>(a); break;
        case 2: process_logits_kernel<kDtype, 2><<<grid, kThreads, lds, s>>>(a); break;
        default: process_logits_kernel<kDtype, 1><<<grid, kThreads, lds, s>>>(a);
    }
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
