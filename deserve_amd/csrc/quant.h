// Pages of 8-bit K/V.  A page of a layer is a record of bytes: the codes of K, then of V, by head and token - (2, Hkv, P, D) in
// e4m3 (OCP: 3 bits behind the point, largest value 448, no infinity) -, then one fp32 scale for each half and head,
// (2, Hkv), and padding to a multiple of 128, so that rows of 128 dims are whole cache lines.  A value is code * scale of its block, the
// tokens of one page and head.  By head, since a workgroup of the attention reads one head: a block is then contiguous.  The scales
// lie in the record, so that pages are swapped, gathered and scattered as they are.
//
// Scales are powers of two: e4m3 has an exponent of its own, so that a finer scale would gain at most half a bit of
// the few codes under 2^-6, while with powers of two code * scale is exact in bf16 and a block whose scale grows is rounded anew only
// where its codes fall under 2^-6.
#pragma once

#include "mfma.h"

namespace dskv {

struct QuantShape {
    int num_pages, page_size, n_kv_heads, head_dim;
    long head_bytes, half_bytes, page_bytes;      // of a page: a head's block, K, all
};
static inline int64_t quant_page_bytes(int64_t page_size, int64_t n_kv_heads, int64_t head_dim)
{
    return (2 * page_size * n_kv_heads * head_dim + 8 * n_kv_heads + 127) / 128 * 128;
}
static inline QuantShape quant_shape(int num_pages, int page_size, int n_kv_heads, int head_dim)
{
    const long head = (long)page_size * head_dim;
    return {num_pages, page_size, n_kv_heads, head_dim, head, n_kv_heads * head, quant_page_bytes(page_size, n_kv_heads, head_dim)};
}

constexpr uint32_t kLeastScale = 0x00800000u;      // 2^-126
constexpr uint8_t kNoNumberCode = 0x7F;

// The least power of two, as bits, that takes `most` (finite, not negative) to 448 = 0.875 * 2^9 or less.
__device__ __forceinline__ uint32_t needed_scale(float most)
{
    const uint32_t bits = __builtin_bit_cast(uint32_t, most);
    const uint32_t exponent = (bits >> 23) + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);     // most <= 1.75 * 2^(exponent - 127)
    return (max(exponent, 9u) - 8u) << 23;
}
// A stored scale: bits of a power of two, or what a page holds that nothing was ever written to (0 then).
__device__ __forceinline__ uint32_t stored_scale(uint32_t bits)
{
    return (bits & 0x807FFFFFu) == 0 && bits >= kLeastScale && bits < 0x7F800000u ? bits : 0u;
}
// 1 / 2^e for 2^-126 <= 2^e <= 2^126
__device__ __forceinline__ float reciprocal_of(uint32_t scale) { return __builtin_bit_cast(float, 0x7F000000u - scale); }

typedef float f32x2_t __attribute__((ext_vector_type(2)));
// 8 codes <-> 8 floats
__device__ __forceinline__ void decode8(u32x2 codes, float *f)
{
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[w], true);
        f[4 * w] = lo.x;
        f[4 * w + 1] = lo.y;
        f[4 * w + 2] = hi.x;
        f[4 * w + 3] = hi.y;
    }
}
// Rounded to nearest, ties to even: by at most 2^-4 of the value, or 2^-10 under 2^-6.
__device__ __forceinline__ u32x2 encode8(const float *f)
{
    u32x2 codes;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * w], f[4 * w + 1], 0, false);
        codes[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * w + 2], f[4 * w + 3], word, true);
    }
    return codes;
}

}  // namespace dskv
