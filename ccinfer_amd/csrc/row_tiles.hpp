// Attention of NT tiles of 16 query rows over 32-token chunks of the paged cache, one wavefront:
// the device code that the attention of drafted trees (tree_attn.hip) and the decode over
// selected blocks (sparse_attn.hip) share.
//
// Layout of the products (as in decode_core.hpp): S^T = K . Q^T and O^T = V^T . P^T, so that the
// probabilities leave the first product in the lanes that the second one takes them from. Lane
// (j = lane & 15, g = lane >> 4) holds row j of a tile; its eight scores of a chunk are those of
// tokens T(g, e) = 16 (e / 4) + 4 g + e % 4, and acc[t][n][r] is O[16 t + j][NV (4 g + r) + n],
// or [16 n + 4 g + r] where V comes out of LDS transposed (Tr).
//
// Two ways of the chunks. One wavefront by itself (attend) loads K and V into registers, one set
// each: K of the next chunk is asked for when the scores are done, V when the second product is, so
// a chunk and a half is in flight on the average. Wavefronts with different rows and the same
// chunks (attend_shared) copy each chunk once into a ring in LDS: the first product wants 16 rows
// of K in 16 neighbouring lanes, in memory a read of 16 lines at once, of which the address unit
// takes one a cycle, and every wavefront by itself would ask for them again (48 trees of 8 to 64
// nodes, 735 MB, the kernel under a tracer: 383 us, the address unit busy for all of it; through the
// ring 255, and 238 with V out of LDS transposed, which saves 32 of 170 vector instructions a chunk).
#pragma once

#include <type_traits>

#include "attn_common.hpp"

namespace ccinfer::hipk::rows {

constexpr int kBlock = 16;
constexpr int kChunk = 32;

template <int D>
struct Shape {
    static constexpr int kSteps = D / 32;   // first product: steps of 32 dims
    static constexpr int kNV = D / 16;      // dims of V a lane holds of a token
    static constexpr int kVWords = D / 32;  // the same in 32-bit words of bf16
};

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
    uint32_t on;  // a bit a block
    __device__ __forceinline__ bool is_on(int b) const { return ((on >> b) & 1u) != 0; }
    __device__ __forceinline__ bool whole() const {
        return on == 3u && lim[0] + lim[1] == 2 * kBlock;
    }
};

// pb < 0 or lim <= 0: the block is not there.
__device__ __forceinline__ Pair make_pair(int pb0, int lim0, int pb1, int lim1) {
    if ((pb0 | pb1) >= 0 && min(lim0, lim1) >= kBlock)  // nearly always
        return Pair{{pb0, pb1}, {kBlock, kBlock}, 3u};
    Pair p;
    const bool on0 = pb0 >= 0 && lim0 > 0, on1 = pb1 >= 0 && lim1 > 0;
    const int l0 = min(lim0, kBlock), l1 = min(lim1, kBlock);
    p.on = (on0 ? 1u : 0u) | (on1 ? 2u : 0u);
    p.pb[0] = on0 ? pb0 : (on1 ? pb1 : 0);
    p.lim[0] = on0 ? l0 : (on1 ? l1 : 1);
    p.pb[1] = on1 ? pb1 : p.pb[0];
    p.lim[1] = on1 ? l1 : p.lim[0];
    return p;
}

// A chunk's K and V in registers. K: lane (i, g) has of token i of each block the dims q_dim(kk, g)
// .. + 8 of every step (fp8: 16 bytes hold two steps'). V: dims NV i .. of tokens T(g, e), or (Tr)
// dim 16 n + i of tokens T(g, 0..7), the operands as they are. The scales of an fp8 chunk: of
// tokens 4 g .. of each block.
template <int D, bool F8>
struct KRegs {
    u32x4 k[2][F8 ? Shape<D>::kSteps / 2 : Shape<D>::kSteps];
    u32x4 s[F8 ? 2 : 1];
};
template <int D, bool F8, bool Tr = false>
struct VRegs {
    static_assert(!Tr || !F8);
    static constexpr int kRows = Tr ? Shape<D>::kNV : 8;
    static constexpr int kWords = Tr ? 4 : (F8 ? (Shape<D>::kNV + 3) / 4 : Shape<D>::kVWords);
    uint32_t v[kRows][kWords];
    u32x4 s[F8 ? 2 : 1];
};

// A chunk's K and V in LDS: 32 rows of kPieces 16-byte pieces each. Piece x of row r lies at place
// x ^ swizzle(r) of its row: the 16 rows that lanes read at once then lie in different banks.
template <bool F8>
struct TileScales {};
template <>
struct TileScales<true> {
    float scales[2][kChunk];  // of K, of V
};
template <int D, bool F8>
struct Tile : TileScales<F8> {
    static constexpr int kPieces = D * (F8 ? 1 : 2) / 16;
    static constexpr int kBytes = kChunk * kPieces * 16;
    static constexpr int kLoads = kBytes / (64 * 16);  // of K, and of V: a wavefront moves 1 KB
    static __device__ __forceinline__ int swizzle(int row) {
        constexpr int kRowsPerLine = kPieces >= 16 ? 1 : 16 / kPieces;  // a line of 256 bytes
        return (row / kRowsPerLine) & ((kPieces < 16 ? kPieces : 16) - 1);
    }
    static constexpr int kRowBytes = 16 * kPieces;
    static constexpr uint32_t kKvAt = F8 ? sizeof(TileScales<true>) : 0;
    alignas(256) char kv[2][kBytes];
};
static_assert(sizeof(TileScales<true>) == 256 && sizeof(Tile<64, true>) == 256 + 2 * 2048 &&
              sizeof(Tile<64, false>) == 2 * 4096);

// First of the eight dims that lane group g holds in step kk.
template <bool F8>
__device__ __forceinline__ int q_dim(int kk, int g) {
    return F8 ? 64 * (kk >> 1) + 16 * g + 8 * (kk & 1) : (kk * 4 + g) * 8;
}

// A block's first row of head h, wave-uniform: loads take it from scalar registers and an offset
// in bytes a lane (rows are less than 2^24 bytes apart: the entries see to it).
template <class Elem, class C>
__device__ __forceinline__ const char* block_rows(const Elem* base, const C& c, int pb, int h) {
    return reinterpret_cast<const char*>(
        base + (static_cast<int64_t>(pb) * kBlock * c.hkv + h) * c.dims());
}

template <class C>
__device__ __forceinline__ u32x4 load_scales(const float* base, const C& c, int pb, int h, int g) {
    return load16(reinterpret_cast<const char*>(
                      base + (static_cast<int64_t>(pb) * c.hkv + h) * kBlock) +
                  static_cast<uint32_t>(16 * g));
}

template <int D, bool F8, bool Pad>
__device__ __forceinline__ void load_k(KRegs<D, F8>& r, const Cache<D, F8, Pad>& c, const Pair& p,
                                       int h, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const uint32_t stride = static_cast<uint32_t>(c.hkv) * c.dims() * (F8 ? 1 : 2);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const char* blk = block_rows(c.k, c, p.pb[b], h);
        const uint32_t row = __umul24(min(i, p.lim[b] - 1), stride);
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
                r.k[b][kk] = load16(blk + (row + (ok ? 2 * dim : 0)));
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
    const uint32_t stride = static_cast<uint32_t>(c.hkv) * c.dims() * (F8 ? 1 : 2);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int b = e >> 2;
        const char* blk = block_rows(c.v, c, p.pb[b], h);
        const uint32_t row = __umul24(min(4 * g + (e & 3), p.lim[b] - 1), stride);
        if constexpr (F8) {
            if constexpr (NV == 8) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(blk + (row + i * NV));
                r.v[e][0] = w[0];
                r.v[e][1] = w[1];
            } else {
                r.v[e][0] = *reinterpret_cast<const uint32_t*>(blk + (row + i * NV));
            }
        } else if constexpr (NV == 4) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(
                blk + (row + (!Pad || i * NV < c.dr ? 2 * i * NV : 0)));
            r.v[e][0] = w[0];
            r.v[e][1] = w[1];
        } else {
            // dims past the row read its start: columns of O that are not stored
#pragma unroll
            for (int x = 0; x < NV / 8; ++x) {
                const int dim = i * NV + 8 * x;
                const u32x4 w = load16(blk + (row + (!Pad || dim < c.dr ? 2 * dim : 0)));
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

__device__ const uint32_t kZeros[4] = {0u, 0u, 0u, 0u};

// Where copies go: `ring` by the name of another variable. Taken as writes to the ring, each would
// make the compiler wait for all of them before the next read of any tile; the loop's own waits
// and meetings order them.
struct LdsCopy {
    using Byte = __attribute__((address_space(3))) char;
    Byte* name;
    uint32_t ring;  // bytes from there
    __device__ __forceinline__ LdsCopy(void* other, const void* ring_)
        : name((Byte*)other),
          ring(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((Byte*)const_cast<void*>(ring_))) -
               static_cast<uint32_t>(reinterpret_cast<uintptr_t>((Byte*)other))) {}
    __device__ __forceinline__ __attribute__((address_space(3))) void* at(uint32_t off) const {
        uint32_t o = ring + off;
        asm("" : "+s"(o));
        return (__attribute__((address_space(3))) void*)(name + o);
    }
};

// Copies chunks into tiles. Instruction z of K, or of V, moves the 64 pieces from row z kRows on;
// of all of them wavefront r of Of asks for its part (the same number for each: where there are
// fewer than wavefronts, some ask for the same again). The part of one of several lies in K or in
// V, that of one of four or more in one of the blocks.
template <int Of, int D, bool F8, bool Pad>
struct Copier {
    using T = Tile<D, F8>;
    static constexpr int kRows = 64 / T::kPieces;
    static constexpr int kEach = 2 * T::kLoads >= Of ? 2 * T::kLoads / Of : 1;
    static constexpr int kAsked = kEach + (F8 ? 1 : 0);
    static_assert(Of <= 2 || Of % 4 == 0);
    static_assert(2 * T::kLoads % Of == 0 || Of % (2 * T::kLoads) == 0);
    const Cache<D, F8, Pad>& cache;
    int h, lane, x0;
    uint32_t stride;  // bytes of a token's heads
    LdsCopy to;
    __device__ __forceinline__ Copier(const Cache<D, F8, Pad>& c, int h_, int r, int lane_,
                                      const LdsCopy& to_)
        : cache(c), h(h_), lane(lane_), to(to_) {
        x0 = Of == 1 ? 0 : r % (2 * T::kLoads / kEach) * kEach;
        stride = static_cast<uint32_t>(c.hkv) * c.dims() * (F8 ? 1 : 2);
    }
    // Head h of a block's first token, of K or V.
    __device__ __forceinline__ const char* block(bool of_v, int pb) const {
        return reinterpret_cast<const char*>((of_v ? cache.v : cache.k) +
                                             static_cast<int64_t>(h) * cache.dims()) +
               static_cast<uint64_t>(static_cast<uint32_t>(pb)) * (stride * kBlock);
    }
    // Instruction z of K (of_v false) or V, of a tile at byte `tile` of the ring.
    __device__ __forceinline__ void one(uint32_t tile, const char* blk, int lim, bool of_v,
                                        int z) const {
        const int row0 = z * kRows & (kBlock - 1);  // wave-uniform
        const int row = lane / T::kPieces;
        // swizzle(row0 + row): the bits of the two do not meet
        const int piece = lane % T::kPieces ^ T::swizzle(row) ^ T::swizzle(row0);
        const bool past = Pad && 8 * piece >= cache.dr;
        // rows past the last are copies of it
        const char* src = blk + (__umul24(min(row0 + row, lim - 1), stride) +
                                 static_cast<uint32_t>(past ? 0 : 16 * piece));
        // a dim of K past the row meets q's zero, but 0 x inf is none; one of V goes to columns
        // that are not stored
        if (past && !of_v) src = reinterpret_cast<const char*>(kZeros);
        __builtin_amdgcn_global_load_lds(
            src, to.at(tile + T::kKvAt + ((of_v ? T::kLoads : 0) + z) * 64 * 16), 16, 0, 0);
    }
    // The scales of K, of V, or of both.
    __device__ __forceinline__ void scales(uint32_t tile, const Pair& p, bool of_k,
                                           bool of_v) const {
        const float* scale = lane < kChunk ? cache.ks : cache.vs;
        const int pb = (lane & kBlock) != 0 ? p.pb[1] : p.pb[0];
        const float* src = scale + (static_cast<int64_t>(pb) * cache.hkv + h) * kBlock +
                           (lane & (kBlock - 1));
        // (scales come first in a tile)
        if (lane < kChunk ? of_k : of_v)
            __builtin_amdgcn_global_load_lds(src, to.at(tile), 4, 0, 0);
    }
    // This wavefront's part of a chunk, into tile `slot` of the ring.
    __device__ __forceinline__ void ask(int slot, const Pair& p) const {
        const uint32_t tile = static_cast<uint32_t>(slot) * sizeof(T);
        const bool of_v = x0 >= T::kLoads;
        const int z0 = x0 % T::kLoads;
        if constexpr (Of >= 4) {
            const bool second = z0 >= T::kLoads / 2;
            const int lim = second ? p.lim[1] : p.lim[0];
            const char* blk = block(of_v, second ? p.pb[1] : p.pb[0]);
#pragma unroll
            for (int y = 0; y < kEach; ++y) one(tile, blk, lim, of_v, z0 + y);
        } else {
            half(tile, p, of_v);
        }
        if constexpr (F8) scales(tile, p, true, true);
    }
    // All of a chunk's K, or V.
    __device__ __forceinline__ void half(uint32_t tile, const Pair& p, bool of_v) const {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const char* blk = block(of_v, p.pb[b]);
#pragma unroll
            for (int y = 0; y < T::kLoads / 2; ++y)
                one(tile, blk, p.lim[b], of_v, b * (T::kLoads / 2) + y);
        }
    }
    // The same of a wavefront by itself (Of = 1), with the scales.
    __device__ __forceinline__ void ask_half(const Pair& p, bool of_v) const {
        half(0, p, of_v);
        if constexpr (F8) scales(0, p, !of_v, of_v);
    }
};

template <int D, bool F8>
__device__ __forceinline__ void read_k(KRegs<D, F8>& r, const Tile<D, F8>& tile, int lane) {
    using T = Tile<D, F8>;
    constexpr int kEach = sizeof(r.k[0]) / 16;
    const int i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const int row = 16 * b + i;
            r.k[b][x] = *reinterpret_cast<const u32x4*>(
                tile.kv[0] + (row * T::kPieces + ((4 * x + g) ^ T::swizzle(row))) * 16);
        }
        if constexpr (F8) r.s[b] = *reinterpret_cast<const u32x4*>(&tile.scales[0][16 * b + 4 * g]);
    }
}

// fp8: the lane's dims of each token.
template <int D>
__device__ __forceinline__ void read_v(VRegs<D, true>& r, const Tile<D, true>& tile, int lane) {
    using T = Tile<D, true>;
    constexpr int kWords = VRegs<D, true>::kWords;
    const int i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int row = 16 * (e >> 2) + 4 * g + (e & 3);
        const int byte = i * kWords * 4;
        const char* from = tile.kv[1] + row * T::kRowBytes +
                           ((byte / 16 ^ T::swizzle(row)) * 16 + byte % 16);
        if constexpr (kWords == 1) {
            r.v[e][0] = *reinterpret_cast<const uint32_t*>(from);
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(from);
            r.v[e][0] = w[0];
            r.v[e][1] = w[1];
        }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
        r.s[b] = *reinterpret_cast<const u32x4*>(&tile.scales[1][16 * b + 4 * g]);
}

// bf16: LDS hands each 16 lanes four tokens' 16 dims transposed, a lane's being one dim of them;
// lane s gives the place of four dims, 4 (s % 4) .., of token s / 4.
template <int D>
__device__ __forceinline__ void read_v(VRegs<D, false, true>& r, const Tile<D, false>& tile,
                                       int lane) {
    using T = Tile<D, false>;
    using Four = short __attribute__((ext_vector_type(4)));
    using InLds = __attribute__((address_space(3))) Four*;
    const int row = lane >> 2;
    // of dims 4 (s % 4) ..; those of 16 n + .. lie at `at` ^ 32 n
    int at = row * T::kRowBytes + (((lane & 3) / 2 ^ T::swizzle(row)) * 16 + (lane & 1) * 8);
    asm("" : "+v"(at));  // one register, not one for each n through the loop
#pragma unroll
    for (int n = 0; n < Shape<D>::kNV; ++n) {
        const char* from = tile.kv[1] + (at ^ 32 * n);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const u32x2 w = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (InLds)const_cast<char*>(from + b * kBlock * T::kRowBytes)));
            r.v[n][2 * b] = w[0];
            r.v[n][2 * b + 1] = w[1];
        }
    }
}

// Until all but the newest n loads of this wavefront have landed, and all its LDS reads.
template <int n>
__device__ __forceinline__ void wait_loads_but() {
    static_assert(n < 64);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | ((n >> 4) << 14));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Until this wavefront's LDS reads have arrived: what they read may be written again. (The copies
// that write it are hidden from the compiler, see LdsCopy: a read stays before them by the clobber.)
__device__ __forceinline__ void wait_reads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The workgroup's wavefronts meet; what they copied into LDS before may be read after.
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

template <int D, int NT, bool Tr = false>
struct State {
    static constexpr bool kTr = Tr;
    f32x4 acc[NT][Shape<D>::kNV];
    float m[NT];  // what the exponents are taken from, base 2, the same in a row's four lanes
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
    // The dim of acc[.][n][r] in lane group g.
    static __device__ __forceinline__ int dim(int n, int r, int g) {
        return Tr ? 16 * n + 4 * g + r : Shape<D>::kNV * (4 * g + r) + n;
    }
    // Four neighbouring dims of a row, set x of kNV, from dim four_dim(x, g) on.
    __device__ __forceinline__ f32x4 four(int t, int x) const {
        if constexpr (Tr) {
            return acc[t][x];
        } else {
            const int r = x % 4, n = x / 4 * 4;
            return f32x4{acc[t][n][r], acc[t][n + 1][r], acc[t][n + 2][r], acc[t][n + 3][r]};
        }
    }
    static __device__ __forceinline__ int four_dim(int x, int g) {
        return Tr ? dim(x, 0, g) : dim(x / 4 * 4, x % 4, g);
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
template <int D, bool F8, bool Tr>
__device__ __forceinline__ bool clear_unbounded(VRegs<D, F8, Tr>& r) {
    constexpr uint32_t kExp = F8 ? 0x7f7f7f7fu : 0x7f807f80u;
    constexpr uint32_t kOne = F8 ? 0x01010101u : 0x00800080u;
    constexpr uint32_t kSign = F8 ? 0x80808080u : 0x80008000u;
    uint32_t any = 0;
#pragma unroll
    for (auto& row : r.v)
#pragma unroll
        for (auto& w : row) any |= ((w & kExp) + kOne) & kSign;
    const bool found = __builtin_amdgcn_ballot_w64(any != 0) != 0;
    if (found) {
#pragma unroll
        for (auto& row : r.v)
#pragma unroll
            for (auto& w : row) {
                const uint32_t bad = ((w & kExp) + kOne) & kSign;
                w &= ~((bad >> (F8 ? 7 : 15)) * (F8 ? 0xffu : 0xffffu));
            }
    }
    return found;
}

// Zeros in place of what this lane's V holds of tokens that are not there: copies of ones that are,
// of whose infinities a probability of 0 would make NaN.
template <int D, bool F8>
__device__ __forceinline__ void clear_absent(VRegs<D, F8>& r, const Pair& p, int lane) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // token T(g, e)
        const bool there = p.is_on(e >> 2) && 4 * (lane >> 4) + (e & 3) < p.lim[e >> 2];
#pragma unroll
        for (auto& w : r.v[e]) w = there ? w : 0u;
    }
}

// Products of q with K: sc[t][e] of row j and token T(g, e), times the token's scale in an fp8
// cache; the logits' factor follows in the exponent.
template <int D, bool F8, int NT>
__device__ __forceinline__ void first_product(float (&sc)[NT][8],
                                              const bf16x8 (&q)[NT][Shape<D>::kSteps],
                                              const KRegs<D, F8>& k) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        f32x4 s4[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) s4[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < Shape<D>::kSteps; ++kk) {
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
            for (int r = 0; r < 4; ++r)
                sc[t][4 * b + r] =
                    F8 ? s4[t][r] * __uint_as_float(k.s[F8 ? b : 0][r]) : s4[t][r];
    }
}

// Masks the scores of a chunk that some row does not see whole. seen(c, t, bits): false where
// every row of tile t sees all that is there of the chunk, else bits has a bit for each of its 32
// tokens that this lane's row sees. Returns whether it masked any (wave-uniform).
template <int NT, class Seen>
__device__ __forceinline__ bool mask_scores(float (&sc)[NT][8], const Pair& p, int c, int lane,
                                            Seen seen) {
    uint32_t bits[NT];
    bool hidden = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        bits[t] = 0xffffffffu;
        hidden |= seen(c, t, bits[t]);
    }
    const bool part = hidden || !p.whole();
    if (part) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int b = e >> 2, key = 4 * (lane >> 4) + (e & 3);
                const bool ok =
                    p.is_on(b) && key < p.lim[b] && ((bits[t] >> (16 * b + key)) & 1u) != 0;
                sc[t][e] = ok ? sc[t][e] : kNegInf;
            }
    }
    return part;
}

// The reference that the exponents are taken from follows the maximum only when a score passes it
// by 2^8: probabilities up to 256 are as good in floating point, and without a new one nothing is
// compared across lanes and no sum is scaled.
template <int D, int NT, bool Tr>
__device__ __forceinline__ void follow_maximum(State<D, NT, Tr>& st, const float (&sc)[NT][8],
                                               float scale_log2) {
    float top[NT];
    bool passed = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        top[t] = fmaxf(fmaxf(fmaxf(sc[t][0], sc[t][1]), fmaxf(sc[t][2], sc[t][3])),
                       fmaxf(fmaxf(sc[t][4], sc[t][5]), fmaxf(sc[t][6], sc[t][7]))) *
                 scale_log2;
        passed |= top[t] > st.m[t] + 8.f;
    }
    if (__builtin_amdgcn_ballot_w64(passed) != 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float m = fmaxf(st.m[t], wave_max_xor16_32(top[t]));
            // (nothing seen yet: sums of zeros)
            const float f = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(st.m[t] - m);
            st.m[t] = m;
            st.l[t] *= f;
#pragma unroll
            for (int n = 0; n < Shape<D>::kNV; ++n) st.acc[t][n] = st.acc[t][n] * f;
        }
    }
}

// Probabilities and the second product. `clear`: V's infinities and NaN are left out (see
// add_unbounded); returns whether there were any.
template <int D, bool F8, int NT, bool Tr>
__device__ __forceinline__ bool second_product(State<D, NT, Tr>& st, const float (&sc)[NT][8],
                                               VRegs<D, F8, Tr>& v, float scale_log2,
                                               bool clear) {
    const bool found = clear && clear_unbounded(v);
    bf16x8 pop[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float from = st.m[t] == kNegInf ? 0.f : st.m[t];
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e], scale_log2, -from));
            st.l[t] += p[e];
        }
        if constexpr (F8) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                // a masked token's scale may be anything; a NaN stays one
                p[e] = __float_as_uint(p[e]) != 0u
                           ? p[e] * __uint_as_float(v.s[F8 ? e >> 2 : 0][e & 3])
                           : 0.f;
        }
        u32x4 pw;
        // probabilities in bf16 (2^-8 of each, and the matrix unit takes no wider ones); the sum
        // is of the unrounded ones
#pragma unroll
        for (int x = 0; x < 4; ++x) pw[x] = pack_bf16x2(p[2 * x], p[2 * x + 1]);
        pop[t] = __builtin_bit_cast(bf16x8, pw);
    }
#pragma unroll
    for (int n = 0; n < Shape<D>::kNV; ++n) {
        u32x4 vw;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if constexpr (Tr)
                vw[x] = v.v[n][x];
            else
                vw[x] = pick_halves(v_word<D, F8>(v, 2 * x, n >> 1),
                                    v_word<D, F8>(v, 2 * x + 1, n >> 1), n & 1);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
            st.acc[t][n] = mfma16x16x32(__builtin_bit_cast(bf16x8, vw), pop[t], st.acc[t][n]);
    }
    return found;
}

// Chunks first, first + stride, ... below last of the rows of one wavefront. next(): their Pairs,
// one after the other (the last one again behind it), from ids that lie in the wavefront's lanes:
// a scalar load a chunk would make every wait for LDS wait for it too. Every row sees all tokens
// that are there.
template <int D, bool F8, bool Pad, int NT, class Next>
__device__ __forceinline__ void attend(State<D, NT>& st, const bf16x8 (&q)[NT][Shape<D>::kSteps],
                                       const Cache<D, F8, Pad>& cache, int h, int first, int last,
                                       int stride, float scale_log2, int lane, Next& next) {
    if (first >= last) return;
    KRegs<D, F8> k;
    VRegs<D, F8> v;
    Pair cur = next();
    load_k(k, cache, cur, h, lane);
    // K before V here as in the loop: the waits count loads in their order
    __builtin_amdgcn_sched_barrier(0);
    load_v(v, cache, cur, h, lane);
    __builtin_amdgcn_sched_barrier(0);
    int c = first;
    // One chunk; with More, K and V of the next one are asked for on the way.
    auto step = [&](auto more) {
        constexpr bool More = decltype(more)::value;
        Pair after = cur;
        if constexpr (More) after = next();
        float sc[NT][8];
        first_product<D, F8, NT>(sc, q, k);
        if constexpr (More) load_k(k, cache, after, h, lane);
        const bool part =
            mask_scores<NT>(sc, cur, c, lane, [](int, int, uint32_t&) { return false; });
        follow_maximum(st, sc, scale_log2);
        if (part) clear_absent(v, cur, lane);
        second_product(st, sc, v, scale_log2, false);
        if constexpr (More) {
            load_v(v, cache, after, h, lane);
            cur = after;
            c += stride;
        }
    };
    while (c + stride < last) step(std::true_type{});
    step(std::false_type{});
}

// The same through a tile in LDS of the wavefront's own, with few registers: K and V of the next
// chunk are asked for as soon as this one's have been read from their place. Rows see what `seen`
// says (mask_scores). Chunks of which some row does not see all, or of which not all is there, are
// multiplied without the infinities and NaN of V, which would reach rows that do not see their token
// (0 x inf); true if there were any: add_unbounded then brings them to the rows that do.
template <int D, bool F8, bool Pad, int NT, class Next, class Seen>
__device__ __forceinline__ bool attend_alone(State<D, NT, !F8>& st,
                                             const bf16x8 (&q)[NT][Shape<D>::kSteps],
                                             const Cache<D, F8, Pad>& cache,
                                             const Tile<D, F8>& tile, const LdsCopy& copies,
                                             int h, int first, int last, int stride,
                                             float scale_log2, int lane, Next& next, Seen seen) {
    if (first >= last) return false;
    constexpr int kHalf = Tile<D, F8>::kLoads + (F8 ? 1 : 0);
    const Copier<1, D, F8, Pad> copier(cache, h, 0, lane, copies);
    bool left_out = false;
    Pair cur = next();
    copier.ask_half(cur, false);
    copier.ask_half(cur, true);
    for (int c = first; c < last; c += stride) {
        const bool more = c + stride < last;
        Pair after = cur;
        if (more) after = next();
        wait_loads_but<kHalf>();  // K is there
        float sc[NT][8];
        {
            KRegs<D, F8> k;
            read_k<D, F8>(k, tile, lane);
            if (more) {
                wait_reads();
                copier.ask_half(after, false);
            }
            first_product<D, F8, NT>(sc, q, k);
        }
        const bool part = mask_scores<NT>(sc, cur, c, lane, seen);
        follow_maximum(st, sc, scale_log2);
        if (more)
            wait_loads_but<kHalf>();  // V is there
        else
            wait_loads_but<0>();
        VRegs<D, F8, !F8> v;
        read_v(v, tile, lane);
        if (more) {
            wait_reads();
            copier.ask_half(after, true);
        }
        left_out |= second_product(st, sc, v, scale_log2, part);
        cur = after;
    }
    return left_out;
}

// The same for Of wavefronts of a workgroup that take the chunks first, first + stride, ... below
// last together, each with rows of its own; all wavefronts of the workgroup call it with the same
// number of steps, those whose chunks end earlier with nothing to do in the last one. ring: the
// Depth tiles of these wavefronts (copies: the same place for the copies). They meet every Group
// steps; a tile is asked for Depth - Group steps before it is read, when all have left the steps
// that read its place, one a step: requests are under way all the time. (Meetings every three or
// four steps, or all of a group's tiles asked for at once: the same time.)
template <int Of, int Depth, int D, bool F8, bool Pad, int NT, class Next, class Seen>
__device__ __forceinline__ bool attend_shared(State<D, NT, !F8>& st,
                                              const bf16x8 (&q)[NT][Shape<D>::kSteps],
                                              const Cache<D, F8, Pad>& cache,
                                              const Tile<D, F8>* ring, const LdsCopy& copies,
                                              int r, int h, int first, int last, int stride,
                                              int steps, bool busy, float scale_log2, int lane,
                                              Next& next, Seen seen) {
    constexpr int Group = Depth >= 8 ? 2 : 1;
    constexpr int kAhead = Depth - Group;
    const Copier<Of, D, F8, Pad> copier(cache, h, r, lane, copies);
    constexpr int kAsked = Copier<Of, D, F8, Pad>::kAsked;
    bool left_out = false;
    uint32_t on = 0;  // two bits a tile that was asked for and is to be read: its blocks are there
    int asked = 0;    // how many those are
    auto ask = [&](int s) {
        const Pair p = next();
        on |= p.on << (2 * asked);
        ++asked;
        copier.ask(s % Depth, p);
    };
    for (int x = 0; x < min(kAhead, steps); ++x) ask(x);
    for (int s = 0; s < steps; s += Group) {
        // this wavefront's part of the next Group tiles; newer ones may be under way
        if (s + kAhead <= steps)
            wait_loads_but<(kAhead - Group) * kAsked>();
        else
            wait_loads_but<0>();
        meet();
#pragma unroll
        for (int x = 0; x < Group; ++x) {
            if (s + kAhead + x < steps) ask(s + kAhead + x);
            const int c = first + (s + x) * stride;
            const Pair pair = next.read(c, on & 3u);
            on >>= 2;
            --asked;
            if (!busy || s + x >= steps || c >= last) continue;
            const Tile<D, F8>& tile = ring[(s + x) % Depth];
            float sc[NT][8];
            {
                KRegs<D, F8> k;
                read_k<D, F8>(k, tile, lane);
                first_product<D, F8, NT>(sc, q, k);
            }
            VRegs<D, F8, !F8> v;
            read_v(v, tile, lane);
            const bool part = mask_scores<NT>(sc, pair, c, lane, seen);
            follow_maximum(st, sc, scale_log2);
            left_out |= second_product(st, sc, v, scale_log2, part);
        }
    }
    return left_out;
}

// The infinities and NaN of V that attend left out, added to the rows that see their tokens (a
// sum with one in it is one, whatever its weight). Rare, and written for few registers: element
// by element.
template <int D, bool F8, bool Pad, int NT, bool Tr, class Chunks, class Seen>
__device__ __forceinline__ void add_unbounded(State<D, NT, Tr>& st, const Cache<D, F8, Pad>& cache,
                                              int h, int first, int last, int stride, int lane,
                                              Chunks chunk, Seen seen) {
    constexpr int NV = Shape<D>::kNV;
    for (int c = first; c < last; c += stride) {
        uint32_t bits[NT];
        bool some = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            bits[t] = 0xffffffffu;
            some |= seen(c, t, bits[t]);
        }
        const Pair p = chunk(c);
        if (!some && p.whole()) continue;
#pragma unroll 1
        for (int key = 0; key < kChunk; ++key) {
            const int b = key >> 4;
            if (!p.is_on(b) || (key & 15) >= p.lim[b]) continue;
            const int64_t slot = static_cast<int64_t>(p.pb[b]) * kBlock + (key & 15);
            const auto* row = cache.v + (slot * cache.hkv + h) * cache.dims();
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    const int dim = st.dim(n, r, lane >> 4);
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

// What a row's sums are multiplied by: 0 where it saw nothing. (By its bits: sources that do not
// honour NaNs would take a NaN sum for none.)
__device__ __forceinline__ float inverse_sum(float l) {
    return __float_as_uint(l) != 0u ? 1.f / l : 0.f;
}

// Place for half a workgroup's sums, lane by lane.
template <int D, int NT, int Waves>
struct Exchange {
    f32x4 acc[Waves / 2][NT * Shape<D>::kNV][64];
    float m[Waves / 2][NT][64];
    float l[Waves / 2][NT][64];
};

// Adds up the sums of the `parts` (a power of two) wavefronts that took different chunks of the
// same rows into those of part 0: in each round the upper half hands its own over. A workgroup's
// wavefronts are `part * groups + group`; all of them call it.
template <int D, int NT, bool Tr, int Waves>
__device__ __forceinline__ void add_parts(Exchange<D, NT, Waves>& x, State<D, NT, Tr>& st, int part,
                                          int parts, int group, int groups, int lane) {
    constexpr int NV = Shape<D>::kNV;
    for (int half = parts / 2; half >= 1; half /= 2) {
        if (part >= half && part < 2 * half) {
            const int at = (part - half) * groups + group;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int n = 0; n < NV; ++n) x.acc[at][t * NV + n][lane] = st.acc[t][n];
                x.m[at][t][lane] = st.m[t];
                x.l[at][t][lane] = st.l[t];
            }
        }
        __syncthreads();
        if (part < half) {
            const int at = part * groups + group;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float mo = x.m[at][t][lane];
                const float m = fmaxf(st.m[t], mo);
                // a part that saw nothing, or only NaN, has -inf, and zeros or NaN
                const float use = m == kNegInf ? 0.f : m;
                const float f = __builtin_amdgcn_exp2f(st.m[t] - use);
                const float fo = __builtin_amdgcn_exp2f(mo - use);
                st.m[t] = m;
                st.l[t] = st.l[t] * f + x.l[at][t][lane] * fo;
#pragma unroll
                for (int n = 0; n < NV; ++n)
                    st.acc[t][n] = st.acc[t][n] * f + x.acc[at][t * NV + n][lane] * fo;
            }
        }
        if (half > 1) __syncthreads();
    }
}

// Row j of tile t, finished, to `row` (bf16, dr elements).
template <int D, bool Pad, int NT, bool Tr>
__device__ __forceinline__ void store_row(const State<D, NT, Tr>& st, int t, float l, __bf16* row,
                                          int dr, int lane) {
    const float inv = inverse_sum(l);
#pragma unroll
    for (int x = 0; x < Shape<D>::kNV; ++x) {
        const int dim = st.four_dim(x, lane >> 4);
        const f32x4 f = st.four(t, x) * inv;
        const u32x2 w = {pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])};
        if (!Pad || dim < dr) *reinterpret_cast<u32x2*>(row + dim) = w;
    }
}

// The same as it is, to D floats.
template <int D, int NT, bool Tr>
__device__ __forceinline__ void store_part(const State<D, NT, Tr>& st, int t, float* row,
                                           int lane) {
#pragma unroll
    for (int x = 0; x < Shape<D>::kNV; ++x)
        *reinterpret_cast<f32x4*>(row + st.four_dim(x, lane >> 4)) = st.four(t, x);
}

// Pieces 0 .. n - 1 of a row, piece s in row at(s) of the parts, added up: a lane has D / 64
// columns next to one another in x; returns the sum. Eight pieces are under way at once while there
// are that many (one after the other waits for memory at each: 32 pieces of 8 x 128 rows of 128 dims
// take 33.3 us, so 30.5, and 16.4 with twice the wavefronts).
template <int D, class At>
__device__ __forceinline__ float merge_row(float (&x)[D / 64], int n, const float* part_acc,
                                           const float2* part_ml, int lane, At at) {
    constexpr int P = D / 64;
    float m = kNegInf, l = 0.f;
#pragma unroll
    for (int y = 0; y < P; ++y) x[y] = 0.f;
    auto add = [&](int s0, auto count) {
        constexpr int N = decltype(count)::value;
        float2 ml[N];
        float a[N][P];
        float top = m;
#pragma unroll
        for (int z = 0; z < N; ++z) {
            const int64_t row = at(s0 + z);
            ml[z] = part_ml[row];
#pragma unroll
            for (int y = 0; y < P; ++y) a[z][y] = part_acc[row * D + lane * P + y];
        }
#pragma unroll
        for (int z = 0; z < N; ++z) top = fmaxf(top, ml[z].x);
        const float use = top == kNegInf ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - use);
        l *= f;
#pragma unroll
        for (int y = 0; y < P; ++y) x[y] *= f;
#pragma unroll
        for (int z = 0; z < N; ++z) {
            const float w = __builtin_amdgcn_exp2f(ml[z].x - use);
            l += ml[z].y * w;
#pragma unroll
            for (int y = 0; y < P; ++y) x[y] += a[z][y] * w;
        }
        m = top;
    };
    int s = 0;
    for (; s + 8 <= n; s += 8) add(s, std::integral_constant<int, 8>{});
    for (; s + 2 <= n; s += 2) add(s, std::integral_constant<int, 2>{});
    if (s < n) add(s, std::integral_constant<int, 1>{});
    return l;
}

// A merge's lane has D / 64 columns of a row next to one another.
template <int D>
__device__ __forceinline__ void store_columns(__bf16* out, const float (&x)[D / 64], float inv,
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

// A workgroup's LDS: chunks, and, when all wavefronts are done with them, their sums.
template <int D, bool F8, int NT, int Waves, int Tiles>
union Shared {
    Exchange<D, NT, Waves> sums;
    Tile<D, F8> tiles[Tiles];
};

}  // namespace ccinfer::hipk::rows
