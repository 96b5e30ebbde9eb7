// The (cos, sin) table of rotary positions, with the frequencies scaled for long contexts.
//
//   table[i][p] = m * (cos, sin)((first + i) * f_p),   f_p = theta^(-2p / R) before scaling
//
// The reference builds its table on the host in float32 (src/model/rope/rope_cache.cpp),
// unscaled. Angles of far positions need more than 32 bits: at position 10^6 a float32 angle is
// off by up to 0.03. Here it is held in quarter turns as a double: with g = 4 f / (2 pi),
//   q = rint(n g)      (by adding 1.5 * 2^52, whose low bits are then q itself)
//   r = n g - q        (one fused product and sum: rounded once, at most 1/2)
// so r is off by the 2^-53 of g (3e-11 quarter turns at 10^6 positions) and goes to float32 with
// 2^-24 of itself, into the Taylor series of sine and cosine on [-pi/4, pi/4], cut where the
// next term is under 2e-9 ((pi/4)^11 / 11!).
//
// The table is only written, so the rate of plain stores bounds it: 2^20 positions x 32 pairs
// (268 MB) take 42.9 us, 6.3 TB/s, where a fill of 2 GiB reaches 6.9. Two pairs (16 bytes) a
// store, streamed; the two-double-operation reduction keeps the arithmetic (about 27 operations
// an entry) under the stores' time.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace ccinfer::hipk {
namespace {

constexpr int kThreads = 256;
constexpr int kSteps = 2;  // positions of a lane

// Frequencies in quarter turns a position, by value: the call needs no upload and can be
// captured.
struct Quarters {
    double per_position[kRopeMaxPairs];
};

// m * (cos, sin) of n g quarter turns.
__device__ __forceinline__ float2 cos_sin_quarters(double n, double g, float m) {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
    const double shifted = __builtin_fma(n, g, kRound);
    const uint32_t k = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, shifted));
    const float y =
        static_cast<float>(__builtin_fma(n, g, kRound - shifted)) * 1.57079632679489662f;
    const float z = y * y;
    const float s =
        y + y * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
    const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 +
                                                                  z * (-1.f / 3628800)))));
    // quarter 1: (-s, c), 2: (-c, -s), 3: (s, -c)
    const float cs = (k & 1) ? s : c, sn = (k & 1) ? c : s;
    const uint32_t flip_c = ((k + 1) & 2) << 30, flip_s = (k & 2) << 30;
    return make_float2(__uint_as_float(__float_as_uint(cs) ^ flip_c) * m,
                       __uint_as_float(__float_as_uint(sn) ^ flip_s) * m);
}

typedef f32x4 f32x4_a8 __attribute__((aligned(8)));

// A workgroup takes kSteps times `rows` positions; lane (row, column) the kPer pairs of its
// column. Two steps share the frequencies' load; with one, 40960 x 64 pairs take 5.9 us instead
// of 5.2, with eight 2^20 x 32 pairs 48.5 us instead of 42.9 (too few workgroups write at once).
template <int kPer>
__global__ __launch_bounds__(kThreads) void rope_table_kernel(Quarters quarters, int pairs,
                                                              int rows, int count, int first,
                                                              float m, float2* __restrict__ out) {
    const int columns = pairs / kPer;
    const int row = threadIdx.x / columns;
    if (row >= rows) return;
    const int p = (threadIdx.x - row * columns) * kPer;
    double g[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) g[k] = quarters.per_position[p + k];
    const int64_t step = static_cast<int64_t>(gridDim.x) * kSteps * rows;
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * kSteps * rows + row; i0 < count;
         i0 += step) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int64_t i = i0 + k * rows;
            if (i >= count) break;
            const double n = static_cast<double>(first + i);
            float2* to = out + i * pairs + p;
            if constexpr (kPer == 2) {
                const float2 a = cos_sin_quarters(n, g[0], m), b = cos_sin_quarters(n, g[1], m);
                __builtin_nontemporal_store(f32x4{a.x, a.y, b.x, b.y},
                                            reinterpret_cast<f32x4_a8*>(to));
            } else {
                *to = cos_sin_quarters(n, g[0], m);
            }
        }
    }
}

}  // namespace

// Frequencies (radians a position) of the pairs of `rotary_dim` elements, and the factor m of
// cos and sin. False for parameters outside their ranges.
bool rope_frequencies(int rotary_dim, double theta, int scaling, const double* prm, double* freq,
                      double* magnitude) {
    const int pairs = rotary_dim / 2;
    if (rotary_dim < 2 || rotary_dim % 2 != 0 || pairs > kRopeMaxPairs) return false;
    if (!std::isfinite(theta) || !(theta > 1.0)) return false;
    *magnitude = 1.0;
    if (scaling != kRopeNone) {
        if (prm == nullptr) return false;
        for (int i = 0; i < kRopeParams; ++i)
            if (!std::isfinite(prm[i])) return false;
        if (scaling != kRopeFactors && !(prm[kRopeFactor] >= 1.0)) return false;
    }
    const double by = scaling != kRopeNone ? prm[kRopeFactor] : 1.0;
    const double length = scaling != kRopeNone ? prm[kRopeOriginalMax] : 0.0;
    const double fast = scaling != kRopeNone ? prm[kRopeFast] : 0.0;
    const double slow = scaling != kRopeNone ? prm[kRopeSlow] : 0.0;
    const double given = scaling != kRopeNone ? prm[kRopeMagnitude] : 0.0;
    if (given < 0.0) return false;
    double base = theta;
    if (scaling == kRopeNtk) {
        // the base grows so that the slowest pair is stretched by the whole factor
        if (rotary_dim <= 2) return false;
        base = theta * std::pow(by, static_cast<double>(rotary_dim) / (rotary_dim - 2));
        if (!std::isfinite(base)) return false;
    }
    double lo = 0.0, hi = 0.0;
    if (scaling == kRopeYarn || scaling == kRopeBands) {
        if (!(length >= 1.0) || !(fast > slow) || !(slow > 0.0)) return false;
    }
    if (scaling == kRopeYarn) {
        // the pair that makes `turns` turns over the original length
        auto pair_at = [&](double turns) {
            return rotary_dim * std::log(length / (2.0 * M_PI * turns)) / (2.0 * std::log(theta));
        };
        lo = std::fmax(std::floor(pair_at(fast)), 0.0);
        hi = std::fmin(std::ceil(pair_at(slow)), rotary_dim - 1.0);
        *magnitude = by > 1.0 ? 0.1 * std::log(by) + 1.0 : 1.0;
    }
    if (scaling != kRopeNone && given > 0.0) *magnitude = given;
    for (int p = 0; p < pairs; ++p) {
        const double f = std::pow(base, -2.0 * p / rotary_dim);
        switch (scaling) {
            case kRopeNone:
            case kRopeNtk:
                freq[p] = f;
                break;
            case kRopeLinear:
                freq[p] = f / by;
                break;
            case kRopeYarn: {
                const double r = std::fmin(std::fmax((p - lo) / std::fmax(hi - lo, 0.001), 0.0), 1.0);
                freq[p] = f / by * r + f * (1.0 - r);
                break;
            }
            case kRopeBands: {
                // `fast` turns or more over the original length: unscaled; `slow` or fewer:
                // stretched; between them blended
                const double turns = length * f / (2.0 * M_PI);
                const double r = std::fmin(std::fmax((turns - slow) / (fast - slow), 0.0), 1.0);
                freq[p] = (1.0 - r) * f / by + r * f;
                break;
            }
            case kRopeFactors: {
                const double d = prm[kRopeParams + p];
                if (!std::isfinite(d) || !(d > 0.0)) return false;
                freq[p] = f / d;
                break;
            }
            default:
                return false;
        }
        if (!std::isfinite(freq[p])) return false;
    }
    return true;
}

hipError_t build_rope_cache(const double* freq, int pairs, double magnitude, int first, int count,
                            void* out, hipStream_t stream) {
    Quarters quarters{};
    for (int p = 0; p < pairs; ++p) quarters.per_position[p] = freq[p] * (2.0 / M_PI);
    const int rows = kThreads / (pairs % 2 == 0 ? pairs / 2 : pairs);
    const int each = rows * kSteps;
    const unsigned grid = static_cast<unsigned>(
        std::min<int64_t>(1 << 22, (static_cast<int64_t>(count) + each - 1) / each));
    auto* to = static_cast<float2*>(out);
    const float m = static_cast<float>(magnitude);
    if (pairs % 2 == 0)
        rope_table_kernel<2><<<grid, kThreads, 0, stream>>>(quarters, pairs, rows, count, first, m,
                                                            to);
    else
        rope_table_kernel<1><<<grid, kThreads, 0, stream>>>(quarters, pairs, rows, count, first, m,
                                                            to);
    return hipGetLastError();
}

}  // namespace ccinfer::hipk
