// e4m3 bytes on gfx950: conversions of the paged cache's kernels.
#pragma once
#include "pgn_common.h"

// exponent of the smallest scale of a page
#define PGN_CACHE_SCALE_FLOOR (-100)

// Four fp32 -> four e4m3 bytes, nearest even.  The values are at most 448 in magnitude (the page's scale sees to that).
__device__ __forceinline__ unsigned pgn_fp8_pack4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// The same where values may be infinite or NaN: an infinity has no e4m3 form and becomes NaN, so that an overflow
// upstream stays visible.
__device__ __forceinline__ unsigned pgn_fp8_pack4_any(float a, float b, float c, float d) {
    unsigned u = pgn_fp8_pack4(a, b, c, d);
    if (!(fabsf(a) < INFINITY)) u |= 0x7fu;
    if (!(fabsf(b) < INFINITY)) u |= 0x7f00u;
    if (!(fabsf(c) < INFINITY)) u |= 0x7f0000u;
    if (!(fabsf(d) < INFINITY)) u |= 0x7f000000u;
    return u;
}

// Four e4m3 bytes times f (a power of two, at most 1) -> e4m3.
__device__ __forceinline__ unsigned pgn_fp8_rescale4(unsigned w, float f) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return pgn_fp8_pack4_any(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}
