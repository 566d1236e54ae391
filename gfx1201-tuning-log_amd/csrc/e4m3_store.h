// Conversions of the kernels that write e4m3 caches (cache_write.hip, rope_append.hip).
#pragma once
#include "fp8kv_common.h"

namespace fp8kv {

// e4m3fn codes of two fp32 values, finite or not: NaN -> 0x7F with the sign bit; everything else is
// clamped to +-448 (exact) and converted with round to nearest even.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b)
{
    const float ca = __builtin_fminf(__builtin_fmaxf(a, -448.f), 448.f);
    const float cb = __builtin_fminf(__builtin_fmaxf(b, -448.f), 448.f);
    uint32_t r = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(ca, cb, 0, false) & 0xFFFFu;
    if (a != a) r = (r & 0xFF00u) | 0x7Fu | ((__float_as_uint(a) >> 24) & 0x80u);
    if (b != b) r = (r & 0x00FFu) | 0x7F00u | ((__float_as_uint(b) >> 16) & 0x8000u);
    return r;
}

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t bits) { return __uint_as_float(bits << 16); }

}  // namespace fp8kv
