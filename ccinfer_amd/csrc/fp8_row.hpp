// Quantisation of one row of an fp8 (OCP E4M3) cache, for the kernels that write one
// (kv_fp8.hip states the layout and the reasons).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.hpp"

namespace ccinfer::hipk {

// The row scale: the smallest power of two P >= 2^-126 with amax <= 448 P (448 = 0.875 *
// 2^9), 0 for an all-zero row, and 2^126 for a row holding an infinity (its infinities
// store as +-448 and dequantise to +-inf again; its finite elements store as zeros).
__device__ __forceinline__ float fp8_row_scale(float amax) {
    if (!(amax > 0.f)) return 0.f;
    if (__builtin_isinf(amax)) return 0x1p126f;
    int e;
    const float f = frexpf(amax, &e);  // amax = f * 2^e, f in [0.5, 1)
    int p = e - 9 + (f > 0.875f ? 1 : 0);
    p = p < -126 ? -126 : p;
    return ldexpf(1.0f, p);
}

// What a row of this scale is multiplied by (exact: a power of two); 0 for scale 0.
__device__ __forceinline__ float fp8_row_inverse(float scale) {
    return scale > 0.f ? 1.0f / scale : 0.f;
}

// Two elements over the row's scale -> E4M3 bytes, nearest even, past +-448 to +-448, a NaN to
// the NaN code (in sources compiled with NaNs honoured).
__device__ __forceinline__ uint32_t fp8_pair(float a, float b) {
    a = a != a ? a : fminf(fmaxf(a, -448.0f), 448.0f);
    b = b != b ? b : fminf(fmaxf(b, -448.0f), 448.0f);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false)) & 0xffffu;
}

__device__ __forceinline__ int64_t fp8_scale_index(int64_t slot, int h, int heads) {
    return (slot / kFp8Block * heads + h) * kFp8Block + slot % kFp8Block;
}

}  // namespace ccinfer::hipk
