// The paged cache in 8 bits (include/gdn_attention_hip.h): where things lie in it, its checks, and its arithmetic.
//
// A scale is a power of two, so a code's value and the step to a page's next scale are exact but for the code's own rounding: e4m3 keeps its
// four significant bits under a larger scale until it runs into its smallest exponent, and a page that grows token by token loses nothing
// to the rescaling of what it holds (integers would be rounded again with each).
#pragma once

#include "gdn_attention_hip.h"
#include "gdn_common.h"

namespace gdn {

constexpr int CACHE_LOWEST = -100;  // a page of (nearly) zeros: 2^-100 448 is far below what bf16 activations hold

typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

// the smallest e with top <= 448 2^e: 448 = 1.75 2^8, so one more where the significand passes 1.75
__device__ __forceinline__ int cache_exponent(float top) {
    return max((int)((__builtin_bit_cast(unsigned, top) + 0x1fffffu) >> 23) - 127 - 8, CACHE_LOWEST);
}

__device__ __forceinline__ int cache_scale(const uint8_t* scales, int64_t at) { return min(max((int)scales[at], CACHE_LOWEST + 127), 247) - 127; }

// 2^e, e from -126 to 127
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, (unsigned)(e + 127) << 23); }

// four values to four codes; what is not finite becomes NaN
__device__ __forceinline__ unsigned cache_codes(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// The page that holds position `index` * P and on of sequence n, or -1.
__device__ __forceinline__ int cache_page(const gdn_paged_cache& c, int n, int64_t index) {
    if (index < 0 || index >= c.table_pages) return -1;
    const int page = c.table[n * c.table_stride + index];
    return page >= 0 && page < c.pages ? page : -1;
}

inline bool cache_aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline int check_cache(const gdn_paged_cache& c) {
    if (c.pages <= 0 || c.P <= 0 || c.HK <= 0 || c.D <= 0 || c.N <= 0 || c.table_pages <= 0 || c.table_stride < 0) return GDN_ERR_SHAPE;
    if (c.P % 16 != 0 || c.P > 256 || c.D % 16 != 0 || c.D > 256 || c.HK > 65535) return GDN_ERR_UNSUPPORTED;
    if ((int64_t)c.table_pages * c.P > INT32_MAX) return GDN_ERR_UNSUPPORTED;  // positions in 32 bits
    return GDN_OK;
}

inline int check_cache_pointers(const gdn_paged_cache& c) {
    if (c.k_codes == nullptr || c.v_codes == nullptr || c.k_scales == nullptr || c.v_scales == nullptr || c.table == nullptr) return GDN_ERR_NULL;
    return cache_aligned(c.k_codes, 16) && cache_aligned(c.v_codes, 16) && cache_aligned(c.table, 4) ? GDN_OK : GDN_ERR_ALIGN;
}

}  // namespace gdn
