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

#include <algorithm>
#include <cstdint>
#include <type_traits>

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

// The heads that the kernel below leaves: under sixteen elements, and those of about a thousand
// whose rotated part and rest do not fit its 64 lanes. One wavefront per row; lane l takes the
// pairs l, l + 64, ... A row's elements are read and written by the same lane, so a call may
// write where it reads.
template <bool kInterleaved, bool kFp8, int kSteps>
__device__ __forceinline__ void rotary_row(const RotaryArgs& a, int64_t row) {
    const int lane = threadIdx.x & 63;
    const int heads = a.sec[0].heads + a.sec[1].heads + a.sec[2].heads;
    const int t = static_cast<int>(row / heads);
    int h = static_cast<int>(row - static_cast<int64_t>(t) * heads);
    RotarySection c = a.sec[0];
    if (h >= c.heads) {
        h -= c.heads;
        c = a.sec[1];
        if (h >= c.heads) {
            h -= c.heads;
            c = a.sec[2];
        }
    }
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
    if (c.norm) inv = rsqrtf(wave_sum(sum) * a.per_elem + a.eps);
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

template <bool kInterleaved, bool kFp8, int kSteps>
__global__ __launch_bounds__(kThreads) void rotary_rows_kernel(RotaryArgs a) {
    const int64_t rows = static_cast<int64_t>(a.tokens) *
                         (a.sec[0].heads + a.sec[1].heads + a.sec[2].heads);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + wave; row < rows;
         row += static_cast<int64_t>(gridDim.x) * kWaves)
        rotary_row<kInterleaved, kFp8, kSteps>(a, row);
}

// The kernel for heads of sixteen elements or more. A row is held by G lanes,
// one chunk a lane, two segments of eight elements:
//   split chunk       pairs p .. p + 7 of the half layout: elements p .. and R/2 + p ..
//   tail chunk        two segments of the elements from R on (half layout)
//   other rows        two segments of the row: interleaved ones, with their pairs inside, and v
// so both elements of every pair are in one lane in either layout, and the lanes' first (and
// second) segments lie side by side: a load or store takes whole lines. A wavefront holds 64 / G
// rows of one section of one token, and all its loads are on their way before the first is
// needed; no row is split between wavefronts, so a call may write where it reads. Where a length
// is no multiple of its segment, the last one is moved back to end with it: its first elements
// are another lane's too, which counts them in the sum of squares and writes the same values.
// Only where fewer than eight pairs are rotated, or fewer than eight elements are not, does a
// segment reach into elements that are treated otherwise; they are left out, and the rest is
// stored element by element. kWhole: the head is a multiple of sixteen and R of sixteen
// (interleaved: eight), so there is nothing of this. Segments start at any even byte; the loads
// and stores claim 2-byte alignment, which the hardware takes at full width.
//
// Bound by memory: 12288 tokens of 16 q and 2 x 8 kv heads of 128 (208 MB) take 38.9 us with the
// norm and the cache write, 5.3 TB/s, where a copy of as many bytes takes 40.2 and
// ccinfer_qkv_prologue on the same rows, slots and positions 41.5 (three sets of inputs in turn;
// one set again and again, which the last-level cache holds in part: 34.7, 29.3 and 34.7). Into
// an fp8 cache 40.7, at the copy's rate 34.8; 8191 tokens x 40 heads half rotated 30.7. What that
// took: eight wavefronts a SIMD (63 registers; at five, with two
// rows a lane sharing (cos, sin) and weights, 46.8 us), stores with the streaming hint (41.5
// without; a prefill that reads the rows afterwards takes the same time either way), and whole
// lines a store (a lane's two segments side by side instead: 28 % more bytes written where they
// are streamed).
//
// What is left. Half-layout widths that are no multiple of 16: segments that reach into one
// another are stored twice in part and need a select an element in the sums. A row rotated in 50
// or 120 of 128 elements also takes nine lanes, so a wavefront holds seven rows instead of eight:
// 40 us instead of 32 (one wavefront a row: 124). With the norm, 12288 tokens of 16 q and 8 kv
// heads: 120 of 128 65.0 us (128 of 128 38.9), all of 120 48.0. Few kv heads: a wavefront holds
// rows of one section of one token, so with one kv head of 128 seven eighths of the K and V ones
// are idle: 8 q and 1 kv heads run at 3.5 TB/s, 14 and 2 or 28 and 4 at 4.5.
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
typedef f32x4 f32x4_a8 __attribute__((aligned(8)));

constexpr int kSegment = 8;
constexpr int kChunkElems = 2 * kSegment;

template <int Ctrl>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), Ctrl, 0xf, 0xf, true));
}

// op over the `lanes` lanes that hold a row, the same ones' order in each, so that every lane gets
// the same bits: pairs of lanes where they are a power of two, else one after the other.
template <typename Op>
__device__ __forceinline__ float row_reduce(float v, int lanes, bool power, int first, Op op) {
    if (power) {
        if (lanes > 1) v = op(v, dpp<0xB1>(v));   // quad_perm 1,0,3,2
        if (lanes > 2) v = op(v, dpp<0x4E>(v));   // quad_perm 2,3,0,1
        if (lanes > 4) v = op(v, dpp<0x141>(v));  // row_half_mirror: the other quad of eight
        if (lanes > 8) v = op(v, dpp<0x140>(v));  // row_mirror: the other eight of sixteen
        if (lanes > 16) v = op(v, __shfl_xor(v, 16, 64));
        if (lanes > 32) v = op(v, __shfl_xor(v, 32, 64));
        return v;
    }
    float all = __shfl(v, first, 64);
    for (int i = 1; i < lanes; ++i) all = op(all, __shfl(v, first + i, 64));
    return all;
}

__device__ __forceinline__ float elem(const u32x4& w, int i) {
    return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
}

__device__ __forceinline__ u32x4 load_segment(const __bf16* p) {
    return *reinterpret_cast<const u32x4_a2*>(p);
}

struct VecPlan {
    int lanes;        // G
    bool power;       // G is a power of two
    int split;        // split chunks of a rotated row (half layout), 0 for interleaved
    int chunks;       // chunks of a q or k row
    int plain;        // chunks of a v row
    int units[3];     // wavefronts of a section and token
    bool whole;       // no segment was moved back, and none crosses R
};

template <bool kInterleaved, bool kFp8, bool kWhole>
__global__ __launch_bounds__(kThreads, 8) void rotary_vec_kernel(RotaryArgs a, VecPlan plan) {
    const int lane = threadIdx.x & 63;
    const int in_slab = lane / plan.lanes;
    const int sub = lane - in_slab * plan.lanes;
    const int per_slab = kWave / plan.lanes;
    const uint32_t units = plan.units[0] + plan.units[1] + plan.units[2];
    const uint32_t total = static_cast<uint32_t>(a.tokens) * units;
    const int half = a.rotary_dim / 2;
    for (uint32_t id = blockIdx.x * kWaves +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
         id < total; id += gridDim.x * kWaves) {
        const int t = static_cast<int>(id / units);
        // asked for first: the table's row waits for the position, the rows for nothing
        const int pos = a.positions[t];
        const int slot = a.slot_mapping != nullptr ? a.slot_mapping[t] : -1;
        int u = static_cast<int>(id - static_cast<uint32_t>(t) * units);
        int s = 0;
        while (u >= plan.units[s]) u -= plan.units[s++];
        const RotarySection& c = a.sec[s];
        const int chunks = s == 2 ? plan.plain : plan.chunks;
        const bool live = sub < chunks && in_slab < per_slab;
        const int chunk = min(sub, chunks - 1);
        const bool split = s < 2 && chunk < plan.split;
        // where its segments start, and which of their elements are this lane's: [lo, hi)
        int seg_a, seg_b, lo_a = 0, lo_b = 0, hi = kSegment;
        bool others = false;  // the elements that are not may not be written
        if (split) {
            seg_a = max(0, min(chunk * kSegment, half - kSegment));
            seg_b = half + seg_a;
            lo_a = lo_b = chunk * kSegment - seg_a;
            hi = min(kSegment, half);
            others = half < kSegment;
        } else {
            const bool tail = s < 2 && plan.split > 0;
            const int n = tail ? chunks - plan.split : chunks;
            const int ua = tail ? a.rotary_dim + (chunk - plan.split) * kSegment
                                : chunk * kSegment;
            const int ub = ua + n * kSegment;
            const bool two = ub < a.head_dim;
            seg_a = min(ua, a.head_dim - kSegment);
            seg_b = two ? min(ub, a.head_dim - kSegment) : seg_a;
            lo_a = ua - seg_a;
            lo_b = two ? ub - seg_b : kSegment;
            others = tail && a.head_dim - a.rotary_dim < kSegment;
        }
        auto mine = [&](int i) {
            return i < kSegment ? i >= lo_a && i < hi
                                : i - kSegment >= lo_b && i - kSegment < hi;
        };
        const int h = u * per_slab + in_slab;
        const bool store = live && h < c.heads;
        const int h_in = min(h, c.heads - 1);
        const __bf16* row = c.src + t * c.src_t + h_in * c.src_h;
        const u32x4 xa = load_segment(row + seg_a), xb = load_segment(row + seg_b);
        int64_t out_row = t;
        if (c.to_cache) {
            if (slot < 0 || slot >= a.max_slots) continue;
            out_row = slot;
        }
        // (cos, sin) of the chunk's eight pairs; `turn` bit i: pair i is rotated (kWhole: any)
        float cs[kSegment], sn[kSegment];
        uint32_t turn = 0;
        if (c.rotate) {
            if (pos >= 0 && pos < a.rope_max) {
                const float2* table = a.rope_cache + static_cast<int64_t>(pos) * half;
                auto load_pairs = [&](int i0, int n, int first) {  // n pairs from `first` on
#pragma unroll
                    for (int i = 0; i < kSegment / 2; ++i) {
                        if (2 * i < i0 || 2 * i >= i0 + n) continue;
                        const f32x4 v =
                            *reinterpret_cast<const f32x4_a8*>(table + first + 2 * i - i0);
                        cs[2 * i] = v[0], sn[2 * i] = v[1];
                        cs[2 * i + 1] = v[2], sn[2 * i + 1] = v[3];
                    }
                };
                if (!kInterleaved && (kWhole || half >= kSegment)) {
                    // all of a chunk's pairs are rotated, or none
                    turn = split ? 0xffu : 0u;
                    load_pairs(0, kSegment, split ? seg_a : 0);
                } else if (kWhole) {
                    // all of a segment's four pairs, or none
                    const int pa = seg_a / 2, pb = seg_b / 2;
                    turn = (pa < half ? 0x0fu : 0u) | (pb < half ? 0xf0u : 0u);
                    load_pairs(0, kSegment / 2, pa < half ? pa : 0);
                    load_pairs(kSegment / 2, kSegment / 2, pb < half ? pb : 0);
                } else if (split || kInterleaved) {
#pragma unroll
                    for (int i = 0; i < kSegment; ++i) {
                        const int p = split            ? i
                                      : i < kSegment / 2 ? seg_a / 2 + i
                                                         : seg_b / 2 + i - kSegment / 2;
                        const float2 v = table[min(p, half - 1)];
                        cs[i] = v.x, sn[i] = v.y;
                        turn |= p < half ? 1u << i : 0u;
                    }
                }
            }
        }
        u32x4 wa{}, wb{};
        if (c.norm) {
            const __bf16* from = c.weight + h_in * c.weight_h;
            wa = load_segment(from + seg_a);
            wb = load_segment(from + seg_b);
        }
        if (a.sin_sign < 0.f) {
#pragma unroll
            for (int i = 0; i < kSegment; ++i) sn[i] = -sn[i];
        }
        float x[kChunkElems];
#pragma unroll
        for (int i = 0; i < kSegment; ++i) {
            x[i] = elem(xa, i);
            x[kSegment + i] = elem(xb, i);
        }
        if (c.norm) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kChunkElems; ++i) {
                if constexpr (kWhole)
                    sum += x[i] * x[i];
                else
                    sum += mine(i) ? x[i] * x[i] : 0.f;
            }
            sum = row_reduce(live ? sum : 0.f, plan.lanes, plan.power, lane - sub,
                             [](float p, float q) { return p + q; });
            const float inv = rsqrtf(sum * a.per_elem + a.eps);
#pragma unroll
            for (int i = 0; i < kSegment; ++i) {
                x[i] *= inv * (elem(wa, i) + a.weight_offset);
                x[kSegment + i] *= inv * (elem(wb, i) + a.weight_offset);
            }
        }
        // under a branch or a select, so that nothing of a pair that is not rotated meets
        // another one's infinity
#pragma unroll
        for (int g = 0; g < 2; ++g) {  // four pairs at a time
            if ((turn >> (4 * g) & 0xfu) == 0) continue;
#pragma unroll
            for (int i = 4 * g; i < 4 * g + 4; ++i) {
                const int p = kInterleaved ? 2 * i : i;
                const int q = kInterleaved ? 2 * i + 1 : kSegment + i;
                const float u0 = x[p] * cs[i] - x[q] * sn[i];
                const float u1 = x[q] * cs[i] + x[p] * sn[i];
                const bool r = kWhole || !kInterleaved || ((turn >> i) & 1);
                x[p] = r ? u0 : x[p];
                x[q] = r ? u1 : x[q];
            }
        }
        if (kFp8 && c.to_cache) {
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < kChunkElems; ++i)
                amax = kWhole || mine(i) ? fmaxf(amax, fabsf(x[i])) : amax;
            amax = row_reduce(amax, plan.lanes, plan.power, lane - sub,
                              [](float p, float q) { return fmaxf(p, q); });
            const float scale = fp8_row_scale(amax);
            const float by = fp8_row_inverse(scale);
            if (!store) continue;
            uint8_t* dst = static_cast<uint8_t*>(c.dst) + out_row * c.dst_t + h * c.dst_h;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint32_t q[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    q[i] = fp8_pair(x[g * kSegment + 2 * i] * by,
                                    x[g * kSegment + 2 * i + 1] * by);
                uint8_t* to = dst + (g == 0 ? seg_a : seg_b);
                if (kWhole || !others) {
                    *reinterpret_cast<u32x2_a1*>(to) = u32x2{q[0] | q[1] << 16, q[2] | q[3] << 16};
                } else {
#pragma unroll
                    for (int i = 0; i < kSegment; ++i)
                        if (mine(g * kSegment + i))
                            to[i] = static_cast<uint8_t>(q[i / 2] >> (8 * (i & 1)));
                }
            }
            if (sub == 0) c.scale[fp8_scale_index(out_row, h, c.heads)] = scale;
            continue;
        }
        if (!store) continue;
        __bf16* dst = static_cast<__bf16*>(c.dst) + out_row * c.dst_t + h * c.dst_h;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = pack_bf16x2(x[g * kSegment + 2 * i], x[g * kSegment + 2 * i + 1]);
            __bf16* to = dst + (g == 0 ? seg_a : seg_b);
            if (kWhole || !others) {
                __builtin_nontemporal_store(w, reinterpret_cast<u32x4_a2*>(to));
            } else {
#pragma unroll
                for (int i = 0; i < kSegment; ++i)
                    if (mine(g * kSegment + i)) to[i] = static_cast<__bf16>(x[g * kSegment + i]);
            }
        }
    }
}

// Whether the chunks above cover a row of this shape, and how.
bool vec_plan(const RotaryArgs& a, bool interleaved, VecPlan& plan) {
    const int d = a.head_dim, r = a.rotary_dim;
    if (d < kChunkElems) return false;
    auto up = [](int n, int m) { return (n + m - 1) / m; };
    plan.split = interleaved ? 0 : up(r / 2, kSegment);
    plan.plain = up(d, kChunkElems);
    plan.chunks = interleaved ? plan.plain : plan.split + up(d - r, kChunkElems);
    const int most = std::max(plan.chunks, plan.plain);
    if (most > kWave) return false;
    int power = 1;
    while (power < most) power *= 2;
    // A power of two of lanes has the shorter reduction; as many lanes as chunks hold more rows a
    // wavefront. At nine chunks (7 rows or 4) the rotation of 8191 tokens x 40 heads takes 40 us
    // or 48, with norm and fp8 write 68 or 81; at five (12 or 8) a head of 64 rotated in 30 with
    // the norm 31 or 33; at six (10 or 8) the rotation 23.7 or 22.9, with the norm 28.1 or 25.9.
    // At 17 to 21 (3 or 2) 4096 tokens x 40 heads of 272 to 336 take 38 to 42 or 44 to 47, with
    // norm and write 54 to 59 or 66 to 69.
    plan.lanes = kWave / most * 2 >= kWave / power * 3 ? most : power;
    plan.power = plan.lanes == power;
    plan.whole = r % (interleaved ? kSegment : kChunkElems) == 0 && d % kChunkElems == 0;
    for (int s = 0; s < 3; ++s) plan.units[s] = up(a.sec[s].heads, kWave / plan.lanes);
    return true;
}

}  // namespace

hipError_t rotary_rows(const RotaryArgs& a, bool interleaved, bool fp8, hipStream_t stream) {
    constexpr int64_t kMostGroups = 1 << 20;  // the kernels go on from there
    auto with = [&](auto inter, auto to_fp8) {
        constexpr bool kInter = decltype(inter)::value, kFp8 = decltype(to_fp8)::value;
        auto groups = [&](int64_t waves) {
            return static_cast<unsigned>(std::min(kMostGroups, (waves + kWaves - 1) / kWaves));
        };
        const int64_t rows = static_cast<int64_t>(a.tokens) *
                             (a.sec[0].heads + a.sec[1].heads + a.sec[2].heads);
        VecPlan plan;
        if (!vec_plan(a, kInter, plan)) {
            if (a.head_dim <= 2 * kWave)
                rotary_rows_kernel<kInter, kFp8, 1><<<groups(rows), kThreads, 0, stream>>>(a);
            else
                rotary_rows_kernel<kInter, kFp8, kRotaryMaxHeadDim / 2 / kWave>
                    <<<groups(rows), kThreads, 0, stream>>>(a);
            return;
        }
        const int64_t waves = static_cast<int64_t>(a.tokens) *
                              (plan.units[0] + plan.units[1] + plan.units[2]);
        if (plan.whole)
            rotary_vec_kernel<kInter, kFp8, true><<<groups(waves), kThreads, 0, stream>>>(a, plan);
        else
            rotary_vec_kernel<kInter, kFp8, false><<<groups(waves), kThreads, 0, stream>>>(a, plan);
    };
    using std::false_type;
    using std::true_type;
    if (interleaved)
        fp8 ? with(true_type{}, true_type{}) : with(true_type{}, false_type{});
    else
        fp8 ? with(false_type{}, true_type{}) : with(false_type{}, false_type{});
    return hipGetLastError();
}

}  // namespace ccinfer::hipk
