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
// next term is under 2e-9 ((pi/4)^11 / 11!). The series run in float32, and pi/2 and m are
// rounded to it: an entry is off by 2.8e-8 of m in the mean (its nearest float32 by 2.0e-8), and
// where m is no float32 itself by up to 2^-24 more, for all entries alike. With both constants in
// two parts and m inside the series that was 2.6e-8 to 3.2e-8, and 42.8 to 44.3 us where this
// takes 40.9 to 41.6: not kept.
//
// The table is only written, so the rate of plain stores bounds it: 2^20 positions x 32 pairs
// (268 MB) take 40 to 45 us on different machines, 6.0 to 6.7 TB/s, where a fill of 2 GiB reaches
// 6.9. Two entries (16 bytes) a
// store, streamed; the reduction in three double operations keeps the arithmetic (about 27
// operations an entry) under the stores' time.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace ccinfer::hipk {
namespace {

constexpr int kThreads = 256;
constexpr int kSteps = 2;

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

constexpr int kGroupEntries = 2 * kThreads;  // entries that a workgroup stores at a time, 4 KiB
constexpr int kMagicBits = 20;

// The table as one run of entries: a workgroup takes kSteps times 4 KiB of it, a lane two
// entries side by side, whatever the number of pairs. (By positions, a workgroup's share is no
// multiple of a line at most widths, and its edges are written in two parts: 4.5 to 4.8 TB/s
// instead of 6.3.) One step takes 44.6 us instead of 41.4 for 2^20 x 32 pairs, four 45.3.
// `magic` is 2^20 / pairs rounded up: x * magic >> 20 is x / pairs for x < pairs + 512. The
// workgroup's own division is on the scalar unit, in 32 bits where the table allows it (in 64
// 42.4 us instead of 40.8).
__global__ __launch_bounds__(kThreads) void rope_table_kernel(Quarters quarters, int pairs,
                                                              uint32_t magic,
                                                              int64_t entries, int first, float m,
                                                              float2* __restrict__ out) {
    __shared__ double g[kRopeMaxPairs];
    for (int p = threadIdx.x; p < pairs; p += kThreads) g[p] = quarters.per_position[p];
    __syncthreads();
    const int64_t step = static_cast<int64_t>(gridDim.x) * kSteps * kGroupEntries;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kSteps * kGroupEntries; base < entries;
         base += step) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int64_t from = base + k * kGroupEntries;  // of the workgroup
            const int row =
                entries <= INT_MAX
                    ? static_cast<int>(static_cast<uint32_t>(from) / static_cast<uint32_t>(pairs))
                    : static_cast<int>(from / pairs);
            const uint32_t x =
                static_cast<uint32_t>(from - static_cast<int64_t>(row) * pairs) + 2 * threadIdx.x;
            const int64_t e = from + 2 * threadIdx.x;
            if (e >= entries) return;
            const uint32_t q = x * magic >> kMagicBits;
            const int p0 = static_cast<int>(x - q * pairs);
            const bool wraps = p0 + 1 == pairs;
            const int p1 = wraps ? 0 : p0 + 1;
            const int n0 = first + row + static_cast<int>(q), n1 = n0 + (wraps ? 1 : 0);
            const float2 a = cos_sin_quarters(static_cast<double>(n0), g[p0], m);
            if (e + 1 < entries) {
                const float2 b = cos_sin_quarters(static_cast<double>(n1), g[p1], m);
                __builtin_nontemporal_store(f32x4{a.x, a.y, b.x, b.y},
                                            reinterpret_cast<f32x4_a8*>(out + e));
            } else {
                out[e] = a;
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
    const int64_t entries = static_cast<int64_t>(count) * pairs;
    constexpr int64_t kEach = kSteps * kGroupEntries;
    const unsigned grid =
        static_cast<unsigned>(std::min<int64_t>(1 << 22, (entries + kEach - 1) / kEach));
    const uint32_t magic = ((1u << kMagicBits) + pairs - 1) / pairs;
    rope_table_kernel<<<grid, kThreads, 0, stream>>>(quarters, pairs, magic, entries, first,
                                                     static_cast<float>(magnitude),
                                                     static_cast<float2*>(out));
    return hipGetLastError();
}

}  // namespace ccinfer::hipk
