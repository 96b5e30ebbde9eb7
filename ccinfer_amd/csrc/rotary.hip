// Rotary positions for q and k rows, with or without the RMSNorm of each head and the write of
// K and V into the paged cache in the same pass.
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + offset)      (norm; else y = x)
//   pair (a, b) of y -> (a cos - b sin, b cos + a sin) with (cos, sin) = table[position][pair]
//
// Pairs: element p with p + R/2 (half layout) or 2p with 2p + 1 (interleaved), p < R/2, where R
// is the table's width; elements from R on are not rotated. The inverse turns by -sin: it is
// the gradient, and takes a rotated row back. Everything between the bf16 row read and the row
// written is float32 and rounded once, unlike ccinfer_qkv_prologue, which follows the
// reference's kernels and their bf16 values in between (src/kernel/norm/rms_norm.cu:22-88,
// src/kernel/pos/rope.cu:14-43).
//
// A row is one head of one token; it is read once and written once, which bounds the kernels
// by memory (or, for a few tokens, by latency).
#include <hip/hip_runtime.h>

#include <cstdint>

#include "attn_common.hpp"
#include "fp8_row.hpp"
#include "kernels.hpp"

namespace ccinfer::hipk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}

// One wavefront per row; lane l takes the pairs l, l + 64, ... A row's elements are read and
// written by the same lane, so a call may write where it reads. Any even head_dim up to 1024,
// any 2-byte alignment and stride.
template <bool kInterleaved, bool kFp8>
__global__ __launch_bounds__(kThreads) void rotary_rows_kernel(RotaryArgs a) {
    constexpr int kSteps = kRotaryMaxHeadDim / 2 / kWave;
    const int lane = threadIdx.x & 63;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
    const int heads = a.sec[0].heads + a.sec[1].heads + a.sec[2].heads;
    if (row >= static_cast<int64_t>(a.tokens) * heads) return;
    const int t = static_cast<int>(row / heads);
    int h = static_cast<int>(row - static_cast<int64_t>(t) * heads);
    int s = 0;
    while (h >= a.sec[s].heads) h -= a.sec[s++].heads;
    const RotarySection& c = a.sec[s];
    int64_t out_row = t;
    if (c.to_cache) {
        out_row = a.slot_mapping[t];
        if (out_row < 0 || out_row >= a.max_slots) return;
    }
    const int half = a.rotary_dim / 2, pairs = a.head_dim / 2;
    const int pos = a.positions[t];
    const bool rotate = c.rotate && pos >= 0 && pos < a.rope_max;
    const float2* table = a.rope_cache + static_cast<int64_t>(rotate ? pos : 0) * half;
    const __bf16* src = c.src + t * c.src_t + h * c.src_h;

    float x0[kSteps], x1[kSteps];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int p = lane + i * kWave;
        const bool halves = !kInterleaved && p < half;
        x0[i] = p < pairs ? static_cast<float>(src[halves ? p : 2 * p]) : 0.f;
        x1[i] = p < pairs ? static_cast<float>(src[halves ? p + half : 2 * p + 1]) : 0.f;
        sum += x0[i] * x0[i] + x1[i] * x1[i];
    }
    float inv = 1.f;
    if (c.norm) inv = rsqrtf(wave_sum(sum) / static_cast<float>(a.head_dim) + a.eps);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int p = lane + i * kWave;
        if (p < pairs) {
            const bool halves = !kInterleaved && p < half;
            if (c.norm) {
                const __bf16* w = c.weight + h * c.weight_h;
                x0[i] *= inv * (static_cast<float>(w[halves ? p : 2 * p]) + a.weight_offset);
                x1[i] *= inv * (static_cast<float>(w[halves ? p + half : 2 * p + 1]) +
                                a.weight_offset);
            }
            if (rotate && p < half) {
                const float2 cs = table[p];
                const float sn = cs.y * a.sin_sign;
                const float u = x0[i] * cs.x - x1[i] * sn;
                x1[i] = x1[i] * cs.x + x0[i] * sn;
                x0[i] = u;
            }
            amax = fmaxf(amax, fmaxf(fabsf(x0[i]), fabsf(x1[i])));
        }
    }
    if (kFp8 && c.to_cache) {
        const float scale = fp8_row_scale(wave_max(amax));
        const float by = fp8_row_inverse(scale);
        uint8_t* dst = static_cast<uint8_t*>(c.dst) + out_row * c.dst_t + h * c.dst_h;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int p = lane + i * kWave;
            if (p >= pairs) continue;
            const bool halves = !kInterleaved && p < half;
            const uint32_t q = fp8_pair(x0[i] * by, x1[i] * by);
            dst[halves ? p : 2 * p] = static_cast<uint8_t>(q);
            dst[halves ? p + half : 2 * p + 1] = static_cast<uint8_t>(q >> 8);
        }
        if (lane == 0) c.scale[fp8_scale_index(out_row, h, c.heads)] = scale;
        return;
    }
    __bf16* dst = static_cast<__bf16*>(c.dst) + out_row * c.dst_t + h * c.dst_h;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int p = lane + i * kWave;
        if (p >= pairs) continue;
        const bool halves = !kInterleaved && p < half;
        dst[halves ? p : 2 * p] = static_cast<__bf16>(x0[i]);
        dst[halves ? p + half : 2 * p + 1] = static_cast<__bf16>(x1[i]);
    }
}

}  // namespace

hipError_t rotary_rows(const RotaryArgs& a, bool interleaved, bool fp8, hipStream_t stream) {
    const int64_t rows =
        static_cast<int64_t>(a.tokens) * (a.sec[0].heads + a.sec[1].heads + a.sec[2].heads);
    const unsigned grid = static_cast<unsigned>((rows + kWaves - 1) / kWaves);
    if (interleaved) {
        if (fp8)
            rotary_rows_kernel<true, true><<<grid, kThreads, 0, stream>>>(a);
        else
            rotary_rows_kernel<true, false><<<grid, kThreads, 0, stream>>>(a);
    } else {
        if (fp8)
            rotary_rows_kernel<false, true><<<grid, kThreads, 0, stream>>>(a);
        else
            rotary_rows_kernel<false, false><<<grid, kThreads, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace ccinfer::hipk
