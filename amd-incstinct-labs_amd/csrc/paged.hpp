// The paged KV cache as its kernels see it (gfx950): places of rows in a pool, checks of the cache's description, and the 4-bit
// format's conversions.
#pragma once
#include "common.hpp"

namespace cdna4 {
namespace paged {

// Bytes of a page's rows of one head; MXFP4: codes, then scales.
__host__ __device__ __forceinline__ int row_bytes(int D, bool fp4) { return fp4 ? D / 2 + D / 32 : 2 * D; }

inline bool valid_cache(const cdna4_paged_cache& c) {
    if (c.D != 64 && c.D != 128) return false;
    if (c.page < 16 || c.page > 256 || (c.page & (c.page - 1))) return false;
    if (c.nKVHeads < 1 || c.pages < 1 || c.max_pages < 1) return false;
    if (c.nKVHeads > 1 << 16) return false;   // a page's bytes fit 32 bits: 2^16 heads x 256 rows x 256 bytes are 2^32
    if ((long long)c.max_pages * c.page >= 0x7fffffffLL - 1024) return false;
    if (c.format != CDNA4_KV_16 && c.format != CDNA4_KV_MXFP4) return false;
    if ((long long)c.nKVHeads * c.page * row_bytes(c.D, c.format == CDNA4_KV_MXFP4) > 0x7fffffffLL) return false;
    return c.table_stride == 0 || c.table_stride >= c.max_pages;
}

inline int log2_of(int page) { return __builtin_ctz((unsigned)page); }
inline long long table_stride(const cdna4_paged_cache& c) { return c.table_stride ? c.table_stride : c.max_pages; }

// ---- MXFP4 ------------------------------------------------------------------------------------------
// The scale byte of a block from the largest absolute value's fp32 bits: the smallest e with max < 7 2^e, so that the
// top code's 6 is as near to a value as any other grid value would be (the grid's next would be 8); 255 where a value
// is not finite (its bits are above every finite one's, which is why the maximum is taken of the bits).
template <bool kBf16>
__device__ __forceinline__ uint32_t scale_byte(uint32_t max_bits) {
    if (max_bits >= 0x7f800000u) return 255u;
    const int e = (int)(max_bits >> 23) - 129 + ((max_bits & 0x7fffffu) >= 0x600000u ? 1 : 0);
    return (uint32_t)(min(max(e, kBf16 ? -125 : -23), kBf16 ? 125 : 13) + 127);
}

// Four values as codes, 16 bits (v_cvt_scalef32_pk_fp4_f32: nearest, ties to the even code, up to 6 2^e).
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], uint32_t byte) {
    if (byte == 255u) return 0u;
    const float s = f32_from_bits(byte << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
    return c;
}

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// Two codes (byte kByte of c) as 16-bit values times the scale 2^(byte - 127), given as the fp32 number of those bits.
template <bool kBf16, int kByte>
__device__ __forceinline__ uint32_t decode2(uint32_t c, float scale) {
    if constexpr (kBf16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, kByte));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, kByte));
}

// fp64 -> fp32 rounded to odd: between two neighbours the one with an odd last bit, so that a further rounding to fewer
// bits gives what rounding the fp64 value itself would.
__device__ __forceinline__ float round_to_odd(double d) {
    const float f = (float)d;
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    const double back = (double)f;
    if (back == d || (b & 1u) || (b & 0x7f800000u) == 0x7f800000u) {
        // exact, odd already, or infinite: a finite value past the largest fp32 is that value, whose last bit is odd
        return __builtin_isinf(f) && !__builtin_isinf(d) ? f32_from_bits(b - 1u) : f;
    }
    return f32_from_bits(__builtin_fabs(d) > __builtin_fabs(back) ? b + 1u : b - 1u);
}

}  // namespace paged
}  // namespace cdna4
