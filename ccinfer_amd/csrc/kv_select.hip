// Which blocks of a long context a decode step looks at: bounds of each block's keys, kept beside
// the cache, the most that a query can make of a block by them, and the best blocks by that.
//
// bounds: bf16 [blocks][kv heads][2][head_dim], the smallest and the largest of the block's keys
// element by element: 1/16 of the bytes of the block's K and V in a bf16 cache, about 1/8 in an fp8
// one. A score by them costs an eighth of reading K (fp8: a quarter). It is never below the block's
// largest logit but for float32's rounding and, over an fp8 cache with scales that are no powers of two,
// that of the bounds to the nearest bf16.
#include <algorithm>
#include <cmath>

#include "attn_common.hpp"
#include "kernels.hpp"
#include "row_tiles.hpp"

namespace ccinfer::hipk {
namespace {

constexpr int kBlock = 16;
constexpr int kThreads = 256;
constexpr float kInf = __builtin_inff();

// ---- bounds ----------------------------------------------------------------------

// Inclusive sums of one int a thread over the workgroup; all = the total. Every thread calls it.
template <int Threads>
__device__ __forceinline__ int group_inclusive(int v, int& all, int* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(v, off);
        if (lane >= off) v += y;
    }
    __syncthreads();  // lds may hold an earlier call's sums
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < Threads / 64; ++w) {
        v += w < wave ? lds[w] : 0;
        all += lds[w];
    }
    return v;
}

// Blocks of row b that its new tokens touch: [first, last).
struct Touched {
    int first, last, ctx;
};

__device__ __forceinline__ Touched touched(const int32_t* ctx, const int32_t* qsl, int b,
                                           int mbpr) {
    const int c = ctx[b];
    const int n = qsl != nullptr ? qsl[b + 1] - qsl[b] : 1;
    Touched t{0, 0, c};
    if (c <= 0 || n <= 0) return t;
    t.first = max(c - n, 0) / kBlock;
    t.last = min((c - 1) / kBlock + 1, mbpr);
    t.last = max(t.last, t.first);
    return t;
}

// A thread takes eight dims of one block: 16 loads of 16 (fp8: 8) bytes in flight, whole rows of
// all heads across the lanes. Tokens that the block does not hold are read as its last one. Rows
// that share a block which one of them does not fill (query tokens of one request) all take the
// tokens of the longest of them, so that it does not matter whose bounds are written last.
// Bound by the reads: 11 operations an element leave room at HBM's rate (16 prompts, 287 MB: 64 us,
// 4.5 TB/s; 48 rows' newest blocks: 4.2 us).
template <bool F8>
__global__ __launch_bounds__(kThreads) void key_bounds_kernel(
    const void* __restrict__ k_cache, const float* __restrict__ k_scale,
    __bf16* __restrict__ bounds, const int32_t* __restrict__ table,
    const int32_t* __restrict__ ctx, const int32_t* __restrict__ qsl, int batch, int mbpr, int hkv,
    int head_dim) {
    __shared__ int starts[kBoundsMaxRequests + 1];
    __shared__ int sums[kThreads / 64];
    constexpr int kPer = kBoundsMaxRequests / kThreads;
    const int per_head = head_dim / 8;
    const int pieces = hkv * per_head;
    int items = batch;
    if (qsl != nullptr) {
        const int per = (batch + kThreads - 1) / kThreads;
        int n[kPer], sum = 0;
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            const int b = static_cast<int>(threadIdx.x) * per + x;
            n[x] = 0;
            if (x < per && b < batch) {
                const Touched t = touched(ctx, qsl, b, mbpr);
                n[x] = t.last - t.first;
            }
            sum += n[x];
        }
        int at = group_inclusive<kThreads>(sum, items, sums) - sum;
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            const int b = static_cast<int>(threadIdx.x) * per + x;
            if (x < per && b < batch) {
                starts[b] = at;
                at += n[x];
            }
        }
        __syncthreads();
    }
    const int64_t work = static_cast<int64_t>(items) * pieces;
    const int lane = threadIdx.x & 63;
    // whole wavefronts, the threads behind the last piece with it once more
    for (int64_t x0 = static_cast<int64_t>(blockIdx.x) * kThreads; x0 < work;
         x0 += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int64_t x = min(x0 + threadIdx.x, work - 1);
        const int item = static_cast<int>(x / pieces);
        const int piece = static_cast<int>(x - static_cast<int64_t>(item) * pieces);
        int b = item;
        if (qsl != nullptr) {  // the last row that starts at or before the item
            int lo = 0, hi = batch - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (starts[mid] <= item) lo = mid; else hi = mid - 1;
            }
            b = lo;
        }
        const Touched t = touched(ctx, qsl, b, mbpr);
        const int blk = t.first + (qsl != nullptr ? item - starts[b] : 0);
        const int pb = blk < t.last ? table[static_cast<int64_t>(b) * mbpr + blk] : -1;
        int held = min(t.ctx - blk * kBlock, kBlock);
        // the lanes' unfinished blocks, one after the other: every lane looks at other rows (48
        // rows 3.6 -> 4.2 us, 1024 5.4 -> 9.0, 2048 9.6 -> 20.8: a line of the table for each pair
        // of rows; only of longer contexts, asked for once those are there: 4.3, 10.0 and 22.5)
        uint64_t open = __builtin_amdgcn_ballot_w64(pb >= 0 && held < kBlock);
        while (open != 0) {
            const int of = __builtin_ctzll(open);
            const int pb0 = __builtin_amdgcn_readlane(pb, of);
            const int blk0 = __builtin_amdgcn_readlane(blk, of);
            int longest = 0;
            for (int r = lane; r < batch; r += 64) {
                const int c = ctx[r];
                if (table[static_cast<int64_t>(r) * mbpr + blk0] == pb0) longest = max(longest, c);
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) longest = max(longest, __shfl_xor(longest, off));
            const bool same = pb == pb0 && blk == blk0;
            if (same) held = min(longest - blk * kBlock, kBlock);
            open &= ~__builtin_amdgcn_ballot_w64(same);
        }
        if (pb < 0) continue;
        const int h = piece / per_head;
        const int dim = (piece - h * per_head) * 8;
        const int64_t row = static_cast<int64_t>(hkv) * head_dim;
        const int64_t base = static_cast<int64_t>(pb) * kBlock * row + static_cast<int64_t>(piece) * 8;
        float lo[8], hi[8];
        uint32_t top[8];  // of the magnitudes: past infinity's for a NaN
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            lo[d] = kInf;
            hi[d] = -kInf;
            top[d] = 0;
        }
        auto take = [&](int d, float v) {
            lo[d] = fminf(lo[d], v);
            hi[d] = fmaxf(hi[d], v);
            top[d] = max(top[d], __float_as_uint(v) & 0x7fffffffu);
        };
        if constexpr (F8) {
            const uint8_t* k = static_cast<const uint8_t*>(k_cache) + base;
            const float* s = k_scale + (static_cast<int64_t>(pb) * hkv + h) * kBlock;
            u32x2 w[kBlock];
            float sc[kBlock];
#pragma unroll
            for (int i = 0; i < kBlock; ++i) {
                const int at = min(i, held - 1);
                w[i] = *reinterpret_cast<const u32x2*>(k + at * row);
                sc[i] = s[at];
            }
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint32_t p0 = e4m3x2_to_bf16x2<false>(w[i][y]);
                    const uint32_t p1 = e4m3x2_to_bf16x2<true>(w[i][y]);
                    take(4 * y, __uint_as_float(p0 << 16) * sc[i]);
                    take(4 * y + 1, __uint_as_float(p0 & 0xffff0000u) * sc[i]);
                    take(4 * y + 2, __uint_as_float(p1 << 16) * sc[i]);
                    take(4 * y + 3, __uint_as_float(p1 & 0xffff0000u) * sc[i]);
                }
        } else {
            const __bf16* k = static_cast<const __bf16*>(k_cache) + base;
            u32x4 w[kBlock];
#pragma unroll
            for (int i = 0; i < kBlock; ++i) w[i] = load16(k + min(i, held - 1) * row);
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    take(2 * y, __uint_as_float(w[i][y] << 16));
                    take(2 * y + 1, __uint_as_float(w[i][y] & 0xffff0000u));
                }
        }
        // Both bounds of an element with a NaN are NaN. The values are bf16 already (an fp8 value
        // times a power of two is one; times another scale it is rounded to the nearest).
        u32x4 out[2];
#pragma unroll
        for (int d = 0; d < 8; ++d)
            if (top[d] > 0x7f800000u) lo[d] = hi[d] = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            out[0][y] = pack_bf16x2(lo[2 * y], lo[2 * y + 1]);
            out[1][y] = pack_bf16x2(hi[2 * y], hi[2 * y + 1]);
        }
        __bf16* o = bounds + (static_cast<int64_t>(pb) * hkv + h) * 2 * head_dim + dim;
        *reinterpret_cast<u32x4*>(o) = out[0];
        *reinterpret_cast<u32x4*>(o + head_dim) = out[1];
    }
}

// ---- scores ------------------------------------------------------------------------

__device__ __forceinline__ float nan_max(float a, float b) {
    return a > b || a != a ? a : b;
}

// The halves of two bf16 with a clear sign, and those with a set one; the others become zeros.
__device__ __forceinline__ uint32_t of_sign(uint32_t w, bool negative) {
    const uint32_t lo = ((w & 0x8000u) != 0) == negative ? w & 0xffffu : 0u;
    const uint32_t hi = ((w & 0x80000000u) != 0) == negative ? w & 0xffff0000u : 0u;
    return lo | hi;
}

// sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo with q's positive and negative parts: two
// matrix products over the rows of bounds. A wavefront takes `tiles` times 16 blocks of one (row,
// kv head); rows of the product are the group's query heads (a missing one repeats the first: the
// maximum does not mind), columns the blocks. Bound by the reads of bounds. The product wants 16
// rows of bounds in 16 neighbouring lanes, in memory a read of 16 lines at once (the 48 rows
// below read like that: 143 us); so the rows are copied as they lie, two tiles under
// way, and leave LDS in the product's order (48 rows, 325 MB: 71.7 us, 4.5 TB/s).
// D: dims that the product counts, rows of fewer filled with zeros.
template <int D>
__global__ __launch_bounds__(kThreads) void score_kernel(
    const __bf16* __restrict__ q, const __bf16* __restrict__ bounds,
    const int32_t* __restrict__ table, const int32_t* __restrict__ ctx, float* __restrict__ scores,
    int mbpr, int hq, int hkv, int head_dim, float scale, int spans, int tiles) {
    constexpr int S = D / 32;                      // steps of the products
    constexpr int kPieces = D / 4;                 // of 16 bytes in a row: D of lo, then D of hi
    constexpr int kRows = 64 / kPieces;            // that one instruction copies
    constexpr int kAsked = 16 / kRows;             // instructions a tile
    constexpr int kTileBytes = 16 * 16 * kPieces;  // 16 blocks
    __shared__ __align__(16) char lds[kThreads / 64][2][kTileBytes];
    __shared__ __align__(16) uint32_t lds_copy[4];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // heads first: those of a block lie side by side in memory (spans first: 101.6 us)
    const int h = blockIdx.x % hkv, bs = blockIdx.x / hkv;
    const int span = bs % spans, b = bs / spans;
    const int j0 = (span * (kThreads / 64) + wave) * 16 * tiles;
    if (j0 >= mbpr) return;
    const int G = hq / hkv;
    const int i = lane & 15, g = lane >> 4;
    const int c = ctx[b];
    const int64_t blocks64 = c > 0 ? (static_cast<int64_t>(c) + kBlock - 1) / kBlock : 0;
    const int blocks = blocks64 > mbpr ? 0 : static_cast<int>(blocks64);
    const int there = min(tiles, (blocks - j0 + 15) / 16);
    const bool mine = lane < 16 * tiles && j0 + lane < mbpr;
    float* out = scores + (static_cast<int64_t>(b) * hkv + h) * mbpr + j0;
    int id = -1;
    if (mine && j0 + lane < blocks) id = table[static_cast<int64_t>(b) * mbpr + j0 + lane];
    float best = -kInf;  // of block j0 + lane
    // Place x of row r holds piece x ^ r: lanes read 16 rows at once, from different banks.
    const uint32_t stride = static_cast<uint32_t>(hkv) * 2 * head_dim * 2;  // bytes of a block's rows
    const char* base = reinterpret_cast<const char*>(bounds + static_cast<int64_t>(h) * 2 * head_dim);
    const rows::LdsCopy to(lds_copy, lds[wave]);
    auto ask = [&](int t) {
#pragma unroll
        for (int z = 0; z < kAsked; ++z) {
            const int row = z * kRows + lane / kPieces;
            const int piece = (lane % kPieces) ^ row;
            const int dim = 8 * (piece % (D / 8));
            // a block that is not there is read as block 0, and its score replaced
            const uint32_t pb = static_cast<uint32_t>(max(__shfl(id, 16 * t + row), 0));
            const char* src = base + static_cast<uint64_t>(pb) * stride +
                              2 * (dim + (piece < D / 8 ? 0 : head_dim));
            if (dim >= head_dim) src = reinterpret_cast<const char*>(rows::kZeros);
            __builtin_amdgcn_global_load_lds(
                src, to.at(static_cast<uint32_t>((t & 1) * kTileBytes + z * 64 * 16)), 16, 0, 0);
        }
    };
    for (int g0 = 0; g0 < G && there > 0; g0 += 16) {
        const int head = h * G + (g0 + i < G ? g0 + i : g0);
        const __bf16* qrow = q + (static_cast<int64_t>(b) * hq + head) * head_dim;
        u32x4 w[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int dim = (s * 4 + g) * 8;
            w[s] = load16(qrow + (dim < head_dim ? dim : 0));
            if (dim >= head_dim) w[s] = u32x4{0u, 0u, 0u, 0u};
        }
        // the waits below count the copies as the newest loads
        __builtin_amdgcn_sched_barrier(0);
        ask(0);
        if (there > 1) ask(1);
        bf16x8 qp[S], qn[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            u32x4 p, n;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                p[y] = of_sign(w[s][y], false);
                n[y] = of_sign(w[s][y], true);
            }
            qp[s] = __builtin_bit_cast(bf16x8, p);
            qn[s] = __builtin_bit_cast(bf16x8, n);
        }
        for (int t = 0; t < there; ++t) {
            if (t + 1 < there)
                rows::wait_loads_but<kAsked>();
            else
                rows::wait_loads_but<0>();
            const char* row = lds[wave][t & 1] + i * 16 * kPieces;
            u32x4 lo[S], hi[S];
#pragma unroll
            for (int s = 0; s < S; ++s) {
                lo[s] = *reinterpret_cast<const u32x4*>(row + ((4 * s + g) ^ i) * 16);
                hi[s] = *reinterpret_cast<const u32x4*>(row + ((D / 8 + 4 * s + g) ^ i) * 16);
            }
            if (t + 2 < there) {
                rows::wait_reads();
                ask(t + 2);
            }
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; ++s) {
                sum = mfma16x16x32(qp[s], __builtin_bit_cast(bf16x8, hi[s]), sum);
                sum = mfma16x16x32(qn[s], __builtin_bit_cast(bf16x8, lo[s]), sum);
            }
            float m = nan_max(nan_max(sum[0], sum[1]), nan_max(sum[2], sum[3]));
            m = nan_max(m, __shfl_xor(m, 16));
            m = nan_max(m, __shfl_xor(m, 32));
            if (g == t) best = nan_max(best, m * scale);
        }
        // the next heads' copies: behind these reads
        rows::wait_reads();
    }
    if (mine) out[lane] = id >= 0 ? best : -kInf;
}

// ---- selection -----------------------------------------------------------------------

// Order of the scores as whole numbers; a NaN before everything.
__device__ __forceinline__ uint32_t order_of(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if ((u & 0x7fffffffu) == 0u) return 0x80000000u;  // -0 and +0 tie
    return (u >> 31) != 0 ? ~u : u | 0x80000000u;
}

constexpr int kBins = 256;

// The blocks of one (row, kv head): the first and the last ones, and of the others the best by
// score. The value that the last chosen one has is found by counting: the range from the lowest
// to the highest key is cut into 256 bins, the bin in which the count from above reaches what is
// wanted becomes the next range, until a bin fits exactly or holds one value; of that value the
// lowest blocks are taken. Scores lie close together, so cutting the range that they fill takes
// two or three rounds and spreads the counters, where their leading bits would meet in a few.
// A thread holds `Per` blocks that lie next to one another: ranks come from one scan. A chain of
// meetings: 9.0 us for one row of 1251 blocks, 11 for 48 rows of up to 2000 (256 threads of eight
// blocks: 9.4 and 9.7, a loss for one row and a gain for many; 1024 bins: 11.1 and 11.5; scores asked
// for before the context is there: 8.7 and 10.8, but for registers that the longest rows do not have:
// with 64 blocks a thread 40 of them are spilled as it is).
template <int Threads, int Per>
__global__ __launch_bounds__(Threads) void select_kernel(const float* __restrict__ scores,
                                                         const int32_t* __restrict__ ctx,
                                                         int32_t* __restrict__ selected, int mbpr,
                                                         int hkv, int take, int first, int last) {
    __shared__ int bins[kBins];
    __shared__ int sums[Threads / 64];
    __shared__ uint32_t edge_lo[Threads / 64], edge_hi[Threads / 64];
    __shared__ int found_bin, found_above, found_count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.x / hkv;
    const float* row = scores + static_cast<int64_t>(blockIdx.x) * mbpr;
    int32_t* out = selected + static_cast<int64_t>(blockIdx.x) * take;
    const int c = ctx[b];
    const int64_t blocks64 = c > 0 ? (static_cast<int64_t>(c) + kBlock - 1) / kBlock : 0;
    const int n = blocks64 > mbpr ? 0 : static_cast<int>(blocks64);
    if (n <= take) {
        for (int x = tid; x < take; x += Threads) out[x] = x < n ? x : -1;
        return;
    }
    // n > take >= first + last: the two ends are apart
    const int tail = n - last;
    int want = take - first - last;
    uint32_t key[Per];
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int x = 0; x < Per; ++x) {
        const int j = tid * Per + x;
        key[x] = 0;
        if (j >= first && j < tail) {
            key[x] = order_of(row[j]);
            lo = min(lo, key[x]);
            hi = max(hi, key[x]);
        }
    }
    auto candidate = [&](int x) {
        const int j = tid * Per + x;
        return j >= first && j < tail;
    };
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        lo = min(lo, static_cast<uint32_t>(__shfl_xor(static_cast<int>(lo), off)));
        hi = max(hi, static_cast<uint32_t>(__shfl_xor(static_cast<int>(hi), off)));
    }
    if (lane == 0) {
        edge_lo[wave] = lo;
        edge_hi[wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Threads / 64; ++w) {
        lo = min(lo, edge_lo[w]);
        hi = max(hi, edge_hi[w]);
    }
    // Keys above `from` are taken (at and above, where `whole`), and `want` of those equal to it.
    uint32_t from = hi;
    bool whole = false;
    if (want > 0) {
        while (true) {
            const uint32_t range = hi - lo;
            const int bits = range == 0 ? 0 : 32 - __builtin_clz(range);
            const int shift = max(bits - 8, 0);
            for (int x = tid; x < kBins; x += Threads) bins[x] = 0;
            __syncthreads();
#pragma unroll
            for (int x = 0; x < Per; ++x)
                if (candidate(x) && key[x] >= lo && key[x] <= hi)
                    atomicAdd(&bins[(key[x] - lo) >> shift], 1);
            __syncthreads();
            if (wave == 0) {
                // lane 0 holds the four highest bins
                int each[4], sum = 0;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    each[y] = bins[kBins - 1 - (4 * lane + y)];
                    sum += each[y];
                }
                int incl = sum;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const int y = __shfl_up(incl, off);
                    if (lane >= off) incl += y;
                }
                int above = incl - sum;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    if (above < want && want <= above + each[y]) {
                        found_bin = kBins - 1 - (4 * lane + y);
                        found_above = above;
                        found_count = each[y];
                    }
                    above += each[y];
                }
            }
            __syncthreads();
            want -= found_above;
            lo += static_cast<uint32_t>(found_bin) << shift;
            hi = lo + min(hi - lo, (1u << shift) - 1u);  // lo + 2^shift may pass 32 bits
            if (found_count == want || lo == hi) {
                from = lo;
                whole = found_count == want;
                break;
            }
        }
    }
    // Ties by index, then places.
    int before = 0, all;
    if (!whole && want > 0) {
        int same = 0;
#pragma unroll
        for (int x = 0; x < Per; ++x) same += candidate(x) && key[x] == from;
        before = group_inclusive<Threads>(same, all, sums) - same;
    }
    const bool any = take > first + last;
    int mine = 0;
    uint64_t chosen = 0;
#pragma unroll
    for (int x = 0; x < Per; ++x) {
        const int j = tid * Per + x;
        bool yes = j < first || (j >= tail && j < n);
        if (any && candidate(x)) {
            if (key[x] > from || (whole && key[x] == from)) {
                yes = true;
            } else if (key[x] == from) {
                yes = before < want;
                ++before;
            }
        }
        chosen |= static_cast<uint64_t>(yes) << x;
        mine += yes;
    }
    int at = group_inclusive<Threads>(mine, all, sums) - mine;
#pragma unroll
    for (int x = 0; x < Per; ++x)
        if ((chosen >> x) & 1) out[at++] = tid * Per + x;
}

template <int Threads, int Per>
hipError_t launch_select(const float* scores, const int32_t* ctx, int32_t* selected, int batch,
                         int mbpr, int hkv, int take, int first, int last, hipStream_t stream) {
    hipLaunchKernelGGL((select_kernel<Threads, Per>), dim3(static_cast<unsigned>(batch) * hkv),
                       dim3(Threads), 0, stream, scores, ctx, selected, mbpr, hkv, take, first,
                       last);
    return hipGetLastError();
}

}  // namespace

hipError_t update_key_bounds(const void* k, const float* k_scale, void* bounds,
                             const int32_t* table, const int32_t* ctx, const int32_t* qsl,
                             int batch, int mbpr, int hkv, int head_dim, hipStream_t stream) {
    // At most eight workgroups a CU, which stride over the blocks that turn out to be touched.
    const int64_t pieces = static_cast<int64_t>(hkv) * (head_dim / 8);
    const int64_t most = pieces * batch * (qsl != nullptr ? mbpr : 1);
    const unsigned grid = static_cast<unsigned>(
        std::min<int64_t>((most + kThreads - 1) / kThreads, 2048));
    auto* kernel = k_scale != nullptr ? key_bounds_kernel<true> : key_bounds_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, stream, k, k_scale,
                       static_cast<__bf16*>(bounds), table, ctx, qsl, batch, mbpr, hkv, head_dim);
    return hipGetLastError();
}

hipError_t score_kv_blocks(const void* q, const void* bounds, const int32_t* table,
                           const int32_t* ctx, float* scores, int batch, int mbpr, int hq, int hkv,
                           int head_dim, hipStream_t stream) {
    // 64 blocks a wavefront, or 16 where that keeps fewer than two of them a SIMD busy (one row of
    // 1251 blocks: 6.4 us and 4.2)
    const int64_t waves = (static_cast<int64_t>(mbpr) + 63) / 64 * batch * hkv;
    const int tiles = waves < 2048 ? 1 : 4;
    const int each = kThreads / 4 * tiles;  // blocks of a workgroup
    const int spans = (mbpr + each - 1) / each;
    const float scale = 1.0f / sqrtf(static_cast<float>(head_dim));
    auto* kernel = head_dim <= 64    ? score_kernel<64>
                   : head_dim <= 128 ? score_kernel<128>
                                     : score_kernel<256>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(spans) * batch * hkv), dim3(kThreads), 0,
                       stream, static_cast<const __bf16*>(q), static_cast<const __bf16*>(bounds),
                       table, ctx, scores, mbpr, hq, hkv, head_dim, scale, spans, tiles);
    return hipGetLastError();
}

hipError_t select_kv_blocks(const float* scores, const int32_t* ctx, int32_t* selected, int batch,
                            int mbpr, int hkv, int take, int first, int last, hipStream_t stream) {
    // the fewest blocks a thread that cover the table row, whatever the number of rows (the figures of
    // eight a thread stand at the kernel)
    if (mbpr <= 256 * 4)
        return launch_select<256, 4>(scores, ctx, selected, batch, mbpr, hkv, take, first, last,
                                     stream);
    if (mbpr <= 1024 * 4)
        return launch_select<1024, 4>(scores, ctx, selected, batch, mbpr, hkv, take, first, last,
                                      stream);
    if (mbpr <= 1024 * 16)
        return launch_select<1024, 16>(scores, ctx, selected, batch, mbpr, hkv, take, first, last,
                                       stream);
    return launch_select<1024, 64>(scores, ctx, selected, batch, mbpr, hkv, take, first, last,
                                   stream);
}

}  // namespace ccinfer::hipk
