// The (cos, sin) table of rotary positions, with the frequencies scaled for long contexts.
//
//   table[i][p] = m * (cos, sin)((first + i) * f_p),   f_p = theta^(-2p / R) before scaling
//
// The reference builds its table on the host in float32 (src/model/rope/rope_cache.cpp),
// unscaled. Angles of far positions need more than 32 bits: at position 10^6 a float32 angle is
// off by up to 0.03. Here the angle is held in turns (of 2 pi) as a double: x = position *
// f_p / (2 pi) is off by 2^-53 of itself (2e-11 turns at 10^6), its whole turns and quarter
// turns come off exactly, and what is left, at most an eighth of a turn, goes to float32 with
// 2^-24 of itself and into the Taylor series of sine and cosine, cut where the next term is
// under 2e-9 (pi/4 to the eleventh over 11!).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "kernels.hpp"

namespace ccinfer::hipk {
namespace {

constexpr int kThreads = 256;

// Frequencies in turns a position, by value: the call needs no upload and can be captured.
struct Turns {
    double per_position[kRopeMaxPairs];
};

// m * (cos, sin) of `turns` turns.
__device__ __forceinline__ float2 cos_sin_turns(double turns, float m) {
    const double t = turns - __builtin_rint(turns);  // [-1/2, 1/2], exact
    const double q = __builtin_rint(4.0 * t);        // quarter turns, -2..2
    const float y = static_cast<float>((t - 0.25 * q) * 6.283185307179586476925);
    const float z = y * y;
    const float s =
        y + y * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
    const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 +
                                                                  z * (-1.f / 3628800)))));
    const int k = static_cast<int>(q) & 3;
    float cs = (k & 1) ? s : c, sn = (k & 1) ? c : s;
    cs = (k == 1 || k == 2) ? -cs : cs;
    sn = (k & 2) ? -sn : sn;
    return make_float2(cs * m, sn * m);
}

__global__ __launch_bounds__(kThreads) void rope_table_kernel(Turns turns, int pairs,
                                                              int64_t entries, int first, float m,
                                                              float2* __restrict__ out) {
    const int64_t e = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (e >= entries) return;
    const int64_t i = e / pairs;
    const int p = static_cast<int>(e - i * pairs);
    out[e] = cos_sin_turns((static_cast<double>(first) + static_cast<double>(i)) *
                               turns.per_position[p],
                           m);
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
    Turns turns{};
    for (int p = 0; p < pairs; ++p) turns.per_position[p] = freq[p] / (2.0 * M_PI);
    const int64_t entries = static_cast<int64_t>(count) * pairs;
    const unsigned grid = static_cast<unsigned>((entries + kThreads - 1) / kThreads);
    rope_table_kernel<<<grid, kThreads, 0, stream>>>(turns, pairs, entries, first,
                                                     static_cast<float>(magnitude),
                                                     static_cast<float2*>(out));
    return hipGetLastError();
}

}  // namespace ccinfer::hipk
