// Attention of NT tiles of 16 query rows over 32-token chunks of the paged cache, one wavefront:
// the device code that the attention of drafted trees (tree_attn.hip) and the decode over
// selected blocks (sparse_attn.hip) share.
//
// Layout of the products (as in decode_core.hpp): S^T = K . Q^T and O^T = V^T . P^T, so that the
// probabilities leave the first product in the lanes that the second one takes them from. Lane
// (j = lane & 15, g = lane >> 4) holds row j of a tile; its eight scores of a chunk are those of
// tokens T(g, e) = 16 (e / 4) + 4 g + e % 4, and acc[t][n][r] is O[16 t + j][NV (4 g + r) + n].
//
// K and V of a chunk have one set of registers each: K of the next chunk is asked for when the
// scores are done, V when the second product is, so a chunk and a half is in flight on the
// average while the register file holds one, and two tiles of rows fit beside it at two
// wavefronts a SIMD.
#pragma once

#include <type_traits>

#include "attn_common.hpp"

namespace ccinfer::hipk::rows {

constexpr int kBlock = 16;
constexpr int kChunk = 32;
constexpr int kWaves = 4;  // wavefronts of a workgroup

template <int D>
struct Shape {
    static constexpr int kSteps = D / 32;   // first product: steps of 32 dims
    static constexpr int kNV = D / 16;      // dims of V a lane holds of a token
    static constexpr int kVWords = D / 32;  // the same in 32-bit words of bf16
};

// A pointer to what no kernel writes while this one runs: wave-uniform loads through it go to the
// scalar unit, whose waits do not wait for the vector loads in flight.
__device__ __forceinline__ const __attribute__((address_space(4))) int32_t* unwritten(
    const int32_t* p) {
    return (const __attribute__((address_space(4))) int32_t*)(reinterpret_cast<uintptr_t>(p));
}

// One layer's cache of rows of D dims, or, padded, of dr < D, a multiple of 8 (the rest of D counts
// as zeros).
template <int D, bool F8, bool Pad>
struct Cache {
    static constexpr bool kF8 = F8;
    const std::conditional_t<F8, uint8_t, __bf16>* k;
    const std::conditional_t<F8, uint8_t, __bf16>* v;
    const float* ks;
    const float* vs;
    int hkv;
    int dr;
    __device__ __forceinline__ int dims() const { return Pad ? dr : D; }
};

// One chunk: two blocks, wave-uniform. Tokens [0, lim) of a block that is `on` are there; what
// is not is read from a token that is (never from a slot that holds nothing, whose bits may be
// anything: a probability of 0 does not take a NaN away), so lim >= 1 and pb names a block of
// the row unless the whole chunk is off.
struct Pair {
    int pb[2];
    int lim[2];
    bool on[2];
    __device__ __forceinline__ bool any() const { return on[0] || on[1]; }
    __device__ __forceinline__ bool whole() const {
        return on[0] && on[1] && lim[0] == kBlock && lim[1] == kBlock;
    }
};

// pb < 0 or lim <= 0: the block is not there.
__device__ __forceinline__ Pair make_pair(int pb0, int lim0, int pb1, int lim1) {
    Pair p;
    p.on[0] = pb0 >= 0 && lim0 > 0;
    p.on[1] = pb1 >= 0 && lim1 > 0;
    const int l0 = min(lim0, kBlock), l1 = min(lim1, kBlock);
    p.pb[0] = p.on[0] ? pb0 : (p.on[1] ? pb1 : 0);
    p.lim[0] = p.on[0] ? l0 : (p.on[1] ? l1 : 1);
    p.pb[1] = p.on[1] ? pb1 : p.pb[0];
    p.lim[1] = p.on[1] ? l1 : p.lim[0];
    return p;
}

template <int D, bool F8>
struct KRegs {
    // fp8: 16 bytes of a row hold two steps' dims 64 s + 16 g .. + 16 (q_dim says the same)
    u32x4 k[2][F8 ? Shape<D>::kSteps / 2 : Shape<D>::kSteps];
    u32x4 s[F8 ? 2 : 1];
};

template <int D, bool F8>
struct VRegs {
    uint32_t v[8][F8 ? (Shape<D>::kNV + 3) / 4 : Shape<D>::kVWords];
    u32x4 s[F8 ? 2 : 1];
};

// First of the eight dims that lane group g holds in step kk.
template <bool F8>
__device__ __forceinline__ int q_dim(int kk, int g) {
    return F8 ? 64 * (kk >> 1) + 16 * g + 8 * (kk & 1) : (kk * 4 + g) * 8;
}

// A block's first row of head h, wave-uniform: loads take it from scalar registers and a 32-bit
// offset a lane (a block has at most 2^30 bytes).
template <class Elem, class C>
__device__ __forceinline__ const Elem* block_rows(const Elem* base, const C& c, int pb, int h) {
    return base + (static_cast<int64_t>(pb) * kBlock * c.hkv + h) * c.dims();
}

template <class C>
__device__ __forceinline__ u32x4 load_scales(const float* base, const C& c, int pb, int h, int g) {
    return load16(base + (static_cast<int64_t>(pb) * c.hkv + h) * kBlock +
                  static_cast<uint32_t>(4 * g));
}

template <int D, bool F8, bool Pad>
__device__ __forceinline__ void load_k(KRegs<D, F8>& r, const Cache<D, F8, Pad>& c, const Pair& p,
                                       int h, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const uint32_t stride = static_cast<uint32_t>(c.hkv) * c.dims();
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const auto* blk = block_rows(c.k, c, p.pb[b], h);
        const uint32_t row = static_cast<uint32_t>(min(i, p.lim[b] - 1)) * stride;
        if constexpr (F8) {
#pragma unroll
            for (int s = 0; s < Shape<D>::kSteps / 2; ++s)
                r.k[b][s] = load16(blk + (row + 64 * s + 16 * g));
            r.s[b] = load_scales(c.ks, c, p.pb[b], h, g);
        } else {
#pragma unroll
            for (int kk = 0; kk < Shape<D>::kSteps; ++kk) {
                const int dim = q_dim<false>(kk, g);
                const bool ok = !Pad || dim < c.dr;
                r.k[b][kk] = load16(blk + (row + (ok ? dim : 0)));
                // a dim past the row meets q's zero, but 0 x inf is none
                if (!ok) r.k[b][kk] = u32x4{0u, 0u, 0u, 0u};
            }
        }
    }
}

template <int D, bool F8, bool Pad>
__device__ __forceinline__ void load_v(VRegs<D, F8>& r, const Cache<D, F8, Pad>& c, const Pair& p,
                                       int h, int lane) {
    constexpr int NV = Shape<D>::kNV;
    const int i = lane & 15, g = lane >> 4;
    const uint32_t stride = static_cast<uint32_t>(c.hkv) * c.dims();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int b = e >> 2;
        const auto* blk = block_rows(c.v, c, p.pb[b], h);
        const uint32_t row = static_cast<uint32_t>(min(4 * g + (e & 3), p.lim[b] - 1)) * stride;
        if constexpr (F8) {
            if constexpr (NV == 8) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(blk + (row + i * NV));
                r.v[e][0] = w[0];
                r.v[e][1] = w[1];
            } else {
                r.v[e][0] = *reinterpret_cast<const uint32_t*>(blk + (row + i * NV));
            }
        } else if constexpr (NV == 4) {
            const u32x2 w =
                *reinterpret_cast<const u32x2*>(blk + (row + (!Pad || i * NV < c.dr ? i * NV : 0)));
            r.v[e][0] = w[0];
            r.v[e][1] = w[1];
        } else {
            // dims past the row read its start: columns of O that are not stored
#pragma unroll
            for (int x = 0; x < NV / 8; ++x) {
                const int dim = i * NV + 8 * x;
                const u32x4 w = load16(blk + (row + (!Pad || dim < c.dr ? dim : 0)));
#pragma unroll
                for (int y = 0; y < 4; ++y) r.v[e][4 * x + y] = w[y];
            }
        }
    }
    if constexpr (F8) {
#pragma unroll
        for (int b = 0; b < 2; ++b) r.s[b] = load_scales(c.vs, c, p.pb[b], h, g);
    }
}

template <int D, int NT>
struct State {
    f32x4 acc[NT][Shape<D>::kNV];
    float m[NT];  // running maximum, base 2, the same in a row's four lanes
    float l[NT];  // this lane's part of the sum
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int n = 0; n < Shape<D>::kNV; ++n) acc[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
            m[t] = kNegInf;
            l[t] = 0.f;
        }
    }
};

// Word w of the bf16 pairs of token T(g, e).
template <int D, bool F8>
__device__ __forceinline__ uint32_t v_word(const VRegs<D, F8>& r, int e, int w) {
    if constexpr (F8) {
        return (w & 1) ? e4m3x2_to_bf16x2<true>(r.v[e][w >> 1])
                       : e4m3x2_to_bf16x2<false>(r.v[e][w >> 1]);
    } else {
        return r.v[e][w];
    }
}

// Zeros in place of the infinities and NaN of this lane's V; whether there were any. (An exponent
// of all ones plus one, or an fp8 NaN's seven ones plus one, carries into the sign's place.)
template <int D, bool F8>
__device__ __forceinline__ bool clear_unbounded(VRegs<D, F8>& r) {
    constexpr uint32_t kExp = F8 ? 0x7f7f7f7fu : 0x7f807f80u;
    constexpr uint32_t kOne = F8 ? 0x01010101u : 0x00800080u;
    constexpr uint32_t kSign = F8 ? 0x80808080u : 0x80008000u;
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (auto& w : r.v[e]) any |= ((w & kExp) + kOne) & kSign;
    const bool found = __builtin_amdgcn_ballot_w64(any != 0) != 0;
    if (found) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (auto& w : r.v[e]) {
                const uint32_t bad = ((w & kExp) + kOne) & kSign;
                w &= ~((bad >> (F8 ? 7 : 15)) * (F8 ? 0xffu : 0xffffu));
            }
    }
    return found;
}

// Chunks first, first + stride, ... below last of the rows. chunk(c): the Pair of chunk c (asked
// for two chunks ahead: the ids' way to the scalar registers is hidden behind a chunk's work).
// seen(c, t, bits): false where every row of tile t sees all that is there of the chunk, else
// bits has a bit for each of its 32 tokens that this lane's row sees. In such chunks the matrix
// product leaves out infinities and NaN of V, which would reach rows that do not see their token
// (0 x inf); true if there were any: add_unbounded then brings them to the rows that do.
template <int D, bool F8, bool Pad, int NT, class Chunks, class Seen>
__device__ __forceinline__ bool attend(State<D, NT>& st, const bf16x8 (&q)[NT][Shape<D>::kSteps],
                                       const Cache<D, F8, Pad>& cache, int h, int first, int last,
                                       int stride, float scale_log2, int lane, Chunks chunk,
                                       Seen seen) {
    constexpr int S = Shape<D>::kSteps;
    constexpr int NV = Shape<D>::kNV;
    if (first >= last) return false;
    bool left_out = false;
    const int g = lane >> 4;
    KRegs<D, F8> k;
    VRegs<D, F8> v;
    Pair cur = chunk(first);
    Pair next = chunk(min(first + stride, last - 1));
    load_k(k, cache, cur, h, lane);
    load_v(v, cache, cur, h, lane);
    for (int c = first;; c += stride) {
        const bool more = c + stride < last;
        const Pair after = chunk(min(c + 2 * stride, last - 1));
        float sc[NT][8];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            f32x4 s4[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) s4[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < S; ++kk) {
                u32x4 w;
                if constexpr (F8) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t bytes = k.k[b][kk >> 1][2 * (kk & 1) + x];
                        w[2 * x] = e4m3x2_to_bf16x2<false>(bytes);
                        w[2 * x + 1] = e4m3x2_to_bf16x2<true>(bytes);
                    }
                } else {
                    w = k.k[b][kk];
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    s4[t] = mfma16x16x32(__builtin_bit_cast(bf16x8, w), q[t][kk], s4[t]);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f =
                        F8 ? scale_log2 * __uint_as_float(k.s[F8 ? b : 0][r]) : scale_log2;
                    sc[t][4 * b + r] = s4[t][r] * f;
                }
        }
        if (more) load_k(k, cache, next, h, lane);
        if (cur.any()) {
            bool hidden = false;  // wave-uniform: some score is masked
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                uint32_t bits = 0xffffffffu;
                const bool some = seen(c, t, bits);
                if (some || !cur.whole()) {
                    hidden |= some;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int b = e >> 2, key = 4 * g + (e & 3);
                        const bool ok = cur.on[b] && key < cur.lim[b] &&
                                        ((bits >> (16 * b + key)) & 1u) != 0;
                        sc[t][e] = ok ? sc[t][e] : kNegInf;
                    }
                }
            }
            float p[NT][8];
            bf16x8 pop[NT];
            float alpha[NT];
            bool grew = false;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float top = fmaxf(fmaxf(fmaxf(sc[t][0], sc[t][1]), fmaxf(sc[t][2], sc[t][3])),
                                  fmaxf(fmaxf(sc[t][4], sc[t][5]), fmaxf(sc[t][6], sc[t][7])));
                top = fmaxf(st.m[t], wave_max_xor16_32(top));
                const float use = top == kNegInf ? 0.f : top;  // nothing seen yet: exp2(-inf)
                alpha[t] = __builtin_amdgcn_exp2f(st.m[t] - use);
                grew |= top != st.m[t];
                st.m[t] = top;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[t][e] = __builtin_amdgcn_exp2f(sc[t][e] - use);
                    sum += p[t][e];
                }
                st.l[t] = st.l[t] * alpha[t] + sum;
                if constexpr (F8) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        // a masked token's scale may be anything; a NaN stays one
                        p[t][e] = __float_as_uint(p[t][e]) != 0u
                                      ? p[t][e] * __uint_as_float(v.s[F8 ? e >> 2 : 0][e & 3])
                                      : 0.f;
                }
                u32x4 pw;
                // probabilities in bf16 (2^-8 of each, and the matrix unit takes no wider ones); the
                // sum is of the unrounded ones
#pragma unroll
                for (int x = 0; x < 4; ++x) pw[x] = pack_bf16x2(p[t][2 * x], p[t][2 * x + 1]);
                pop[t] = __builtin_bit_cast(bf16x8, pw);
            }
            if (__builtin_amdgcn_ballot_w64(grew) != 0) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int n = 0; n < NV; ++n) st.acc[t][n] = st.acc[t][n] * alpha[t];
            }
            if (hidden) left_out |= clear_unbounded<D, F8>(v);
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                u32x4 vw;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    vw[x] = pick_halves(v_word<D, F8>(v, 2 * x, n >> 1),
                                        v_word<D, F8>(v, 2 * x + 1, n >> 1), n & 1);
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    st.acc[t][n] =
                        mfma16x16x32(__builtin_bit_cast(bf16x8, vw), pop[t], st.acc[t][n]);
            }
        }
        if (!more) break;
        load_v(v, cache, next, h, lane);
        cur = next;
        next = after;
    }
    return left_out;
}

// The infinities and NaN of V that attend left out, added to the rows that see their tokens (a
// sum with one in it is one, whatever its weight). Rare, and written for few registers: element
// by element.
template <int D, bool F8, bool Pad, int NT, class Chunks, class Seen>
__device__ __forceinline__ void add_unbounded(State<D, NT>& st, const Cache<D, F8, Pad>& cache,
                                              int h, int first, int last, int stride, int lane,
                                              Chunks chunk, Seen seen) {
    constexpr int NV = Shape<D>::kNV;
    for (int c = first; c < last; c += stride) {
        uint32_t bits[NT];
        bool some = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            bits[t] = 0;
            some |= seen(c, t, bits[t]);
        }
        if (!some) continue;
        const Pair p = chunk(c);
#pragma unroll 1
        for (int key = 0; key < kChunk; ++key) {
            const int b = key >> 4;
            if (!p.on[b] || (key & 15) >= p.lim[b]) continue;
            const int64_t slot = static_cast<int64_t>(p.pb[b]) * kBlock + (key & 15);
            const auto* row = cache.v + (slot * cache.hkv + h) * cache.dims();
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    const int dim = NV * (4 * (lane >> 4) + r) + n;
                    uint32_t f = 0;
                    if (!Pad || dim < cache.dr) {
                        if constexpr (F8)
                            f = (row[dim] & 0x7f) == 0x7f ? 0x7fc00000u : 0u;
                        else
                            f = static_cast<uint32_t>(
                                    reinterpret_cast<const uint16_t*>(row)[dim]) << 16;
                    }
                    const bool bad = (f & 0x7f800000u) == 0x7f800000u;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        if (bad && ((bits[t] >> key) & 1u) != 0)
                            st.acc[t][n][r] += __uint_as_float(f);
                }
        }
    }
}

// The q operand of a tile: lane (j, g) holds the dims q_dim(kk, g) .. + 8 of its row, zeros for
// a row that is not there and dims past the row's end.
template <int D, bool F8, bool Pad>
__device__ __forceinline__ void load_q(bf16x8 (&q)[Shape<D>::kSteps], const __bf16* row, bool live,
                                       int dr, int lane) {
#pragma unroll
    for (int kk = 0; kk < Shape<D>::kSteps; ++kk) {
        const int dim = q_dim<F8>(kk, lane >> 4);
        // (a row that is not there points at one that is)
        const bool ok = live && (!Pad || dim < dr);
        u32x4 w = load16(row + (!Pad || dim < dr ? dim : 0));
        if (!ok) w = u32x4{0u, 0u, 0u, 0u};
        q[kk] = __builtin_bit_cast(bf16x8, w);
    }
}

// A row's columns of this lane in the merges: D / 64 next to one another.
template <int D>
__device__ __forceinline__ void store_bf16_row(__bf16* out, const float (&x)[D / 64], float inv,
                                               int dr, int lane) {
    constexpr int P = D / 64;
    if (lane * P >= dr) return;
    if constexpr (P == 1) {
        out[lane] = static_cast<__bf16>(x[0] * inv);
    } else {
        uint32_t* o = reinterpret_cast<uint32_t*>(out + lane * P);
#pragma unroll
        for (int y = 0; y < P / 2; ++y)
            o[y] = pack_bf16x2(x[2 * y] * inv, x[2 * y + 1] * inv);
    }
}

// What a row's sums are multiplied by: 0 where it saw nothing. (By its bits: sources that do not
// honour NaNs would take a NaN sum for none.)
__device__ __forceinline__ float inverse_sum(float l) {
    return __float_as_uint(l) != 0u ? 1.f / l : 0.f;
}

// LDS of a workgroup's partial rows: rows are 4 floats longer than D, so that the 16 rows that
// lanes write at once lie in different banks.
template <int D, int NT>
struct Parts {
    static constexpr int kRows = 16 * NT;
    static constexpr int kStride = D + 4;
    float acc[kWaves][kRows][kStride];
    float m[kWaves][kRows];
    float l[kWaves][kRows];
};

// A wavefront's rows into LDS.
template <int D, int NT>
__device__ __forceinline__ void put_part(Parts<D, NT>& parts, const State<D, NT>& st, int wave,
                                         int lane) {
    constexpr int NV = Shape<D>::kNV;
    const int j = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float l = wave_sum_xor16_32(st.l[t]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < NV; n += 4) {
                const f32x4 w = {st.acc[t][n][r], st.acc[t][n + 1][r], st.acc[t][n + 2][r],
                                 st.acc[t][n + 3][r]};
                *reinterpret_cast<f32x4*>(&parts.acc[wave][16 * t + j][NV * (4 * g + r) + n]) = w;
            }
        if (g == 0) {
            parts.m[wave][16 * t + j] = st.m[t];
            parts.l[wave][16 * t + j] = l;
        }
    }
}

// Row `row` of the parts of wavefronts from, from + step, ... (`count` of them): this lane's
// columns of the sum over them, with the row's maximum and sum.
template <int D, int NT>
__device__ __forceinline__ void sum_parts(const Parts<D, NT>& parts, int row, int from, int step,
                                          int count, int lane, float (&x)[D / 64], float& m,
                                          float& l) {
    constexpr int P = D / 64;
    m = kNegInf;
    for (int w = 0; w < count; ++w) m = fmaxf(m, parts.m[from + w * step][row]);
    l = 0.f;
#pragma unroll
    for (int y = 0; y < P; ++y) x[y] = 0.f;
    // a part that saw nothing, or only NaN, has maximum -inf, and zeros or NaN
    const float use = m == kNegInf ? 0.f : m;
    for (int w = 0; w < count; ++w) {
        const int at = from + w * step;
        const float f = __builtin_amdgcn_exp2f(parts.m[at][row] - use);
        l += parts.l[at][row] * f;
#pragma unroll
        for (int y = 0; y < P; ++y) x[y] += parts.acc[at][row][lane * P + y] * f;
    }
}

}  // namespace ccinfer::hipk::rows
