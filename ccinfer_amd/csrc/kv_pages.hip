// Pages of the paged KV cache: blocks copied over all layers, block tables of requests changed
// on the device with counted references, and the pool compacted.
//
// The reference keeps its allocator on the host (src/cache/kv_cache_manager.cpp): a request that
// is forked, cut back or finished costs a walk over host lists and an upload of its table row.
// Here the pool is one array of reference counts on the device (0 = free; a count below 0, from
// owners that were not counted, is neither free nor held); what a call hands out
// is always the lowest-numbered free blocks, in item order, so its results do not depend on the
// order in which workgroups run. The only atomics are integer additions to the counts.
//
// Every call reads the tables and counts as they were before it: a first launch takes a bitmap
// of the free blocks (kChunk blocks a workgroup, one ballot per 64) and, for update, copies the
// source rows; the launches after it select from the bitmap (a prefix over the chunks' counts,
// then over a chunk's words) and never from counts that others are changing.
//
// The copies of cache data are bounded by memory: 16 bytes a lane, a block of one layer's K or V
// by one workgroup.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace ccinfer::hipk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kChunk = 1024;                // blocks whose bitmap one workgroup takes
constexpr int kChunkWords = kChunk / kWave;
constexpr int kWaveWords = kChunkWords / kWaves;
static_assert(kWaveWords * kWaves == kChunkWords && kChunkWords <= kWave);

constexpr int kOk = 0;
constexpr int kInvalidArgument = 6;    // ErrorCode::InvalidArgument
constexpr int kExhausted = 12;         // ErrorCode::KVBlockExhausted
constexpr int kInvalidTable = 14;      // ErrorCode::KVInvalidBlockTable

constexpr size_t kAlign = 256;
size_t align_up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }

int chunks_of(int blocks) { return (blocks + kChunk - 1) / kChunk; }

// ---- data --------------------------------------------------------------------

// Bytes from src to dst by the whole workgroup as units of T, kAhead of them a lane at a time:
// all loads of a round are on their way before its first store. The first round's loads may be
// asked for before it is known where they go. Stored with the streaming hint (900 blocks x 24
// layers: 482 us against 500 without it; with streaming loads as well 552).
template <typename T>
struct Copy {
    static constexpr int kAhead = 8;
    static constexpr int kRound = kThreads * kAhead;
    const T* src = nullptr;
    int n = 0;  // units; a block's bytes fit 31 bits
    T v[kAhead];

    __device__ __forceinline__ void load(int first) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = first + k * kThreads + static_cast<int>(threadIdx.x);
            if (i < n) v[k] = src[i];
        }
    }
    __device__ __forceinline__ void start(const char* from, int64_t bytes) {
        src = reinterpret_cast<const T*>(from);
        n = static_cast<int>(bytes / static_cast<int64_t>(sizeof(T)));
        load(0);
    }
    __device__ __forceinline__ void finish(char* to) {
        T* dst = reinterpret_cast<T*>(to);
        for (int first = 0; first < n; first += kRound) {
            if (first > 0) load(first);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = first + k * kThreads + static_cast<int>(threadIdx.x);
                if (i < n) __builtin_nontemporal_store(v[k], dst + i);
            }
        }
    }
};

// Part `part` (layer, then K or V) of the caches: its first `tokens` tokens of block `from`, to
// block `to`.
template <typename T>
struct PartCopy {
    Copy<T> data;
    char* cache;
    float* scale;
    float first_scale;
    int64_t block_bytes;

    __device__ __forceinline__ void start(const KvLayers& kv, int part, int from, int tokens) {
        const int layer = part >> 1;
        const bool is_v = part & 1;
        block_bytes = kv.token_bytes * kv.block_size;
        cache = (is_v ? kv.v : kv.k) + layer * kv.layer_stride;
        scale = is_v ? kv.v_scale : kv.k_scale;
        data.start(cache + from * block_bytes, kv.token_bytes * tokens);
        if (scale == nullptr) return;
        scale += layer * kv.scale_layer_stride;
        const int n = kv.heads * kFp8Block;  // [head][16]
        if (static_cast<int>(threadIdx.x) < n)
            first_scale = scale[static_cast<int64_t>(from) * n + threadIdx.x];
    }
    __device__ __forceinline__ void finish(const KvLayers& kv, int from, int to, int tokens) {
        data.finish(cache + to * block_bytes);
        if (scale == nullptr) return;
        const int n = kv.heads * kFp8Block;
        for (int i = threadIdx.x; i < n; i += kThreads)
            if (i % kFp8Block < tokens)
                scale[static_cast<int64_t>(to) * n + i] =
                    i < kThreads ? first_scale : scale[static_cast<int64_t>(from) * n + i];
    }
};

template <typename T>
__device__ __forceinline__ void copy_part(const KvLayers& kv, int part, int from, int to,
                                          int tokens) {
    PartCopy<T> c;
    c.start(kv, part, from, tokens);
    c.finish(kv, from, to, tokens);
}

// The unit that every copy of these caches can move in: 16 bytes where every token starts at a
// multiple of 16 (an update's copies end behind a token), else an element.
int copy_unit(const KvLayers& kv) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(kv.k) | reinterpret_cast<uintptr_t>(kv.v) |
                          static_cast<uintptr_t>(kv.layer_stride) |
                          static_cast<uintptr_t>(kv.token_bytes);
    return all % 16 == 0 ? 16 : (kv.k_scale == nullptr ? 2 : 1);
}

template <typename F>
hipError_t with_unit(const KvLayers& kv, F&& launch) {
    switch (copy_unit(kv)) {
        case 16: launch(u32x4{}); break;
        case 2: launch(uint16_t{}); break;
        default: launch(uint8_t{}); break;
    }
    return hipGetLastError();
}

// ---- copy --------------------------------------------------------------------

// Workgroup (x, y): pair x, parts y, y + gridDim.y, ... Pairs outside the pool and of a block
// with itself are nothing to do. A pair conflicts where another one writes its blocks, or reads
// the block that it writes (the same pair twice does not); it is left out, and told.
template <typename T>
__global__ __launch_bounds__(kThreads) void copy_blocks_kernel(KvLayers kv,
                                                               const int32_t* __restrict__ src,
                                                               const int32_t* __restrict__ dst,
                                                               int pairs, int32_t* status) {
    const int i = blockIdx.x;
    const int from = src[i], to = dst[i];
    auto in_pool = [&](int b) { return b >= 0 && b < kv.blocks; };
    if (!in_pool(from) || !in_pool(to) || from == to) return;
    bool conflict = false;
    for (int j = threadIdx.x; j < pairs; j += kThreads) {
        const int s = src[j], d = dst[j];
        if (!in_pool(s) || !in_pool(d) || s == d || (s == from && d == to)) continue;
        conflict |= d == to || d == from || s == to;
    }
    if (__syncthreads_or(conflict)) {
        if (status != nullptr && threadIdx.x == 0 && blockIdx.y == 0) *status = kInvalidArgument;
        return;
    }
    for (int part = blockIdx.y; part < 2 * kv.layers; part += gridDim.y)
        copy_part<T>(kv, part, from, to, kv.block_size);
}

// ---- bitmap of the free blocks -------------------------------------------------

// Chunk c: one bit per block, set where it is free, and how many are.
__device__ __forceinline__ void free_bitmap(const int32_t* __restrict__ refs, int blocks, int c,
                                            uint64_t* __restrict__ bitmap,
                                            int32_t* __restrict__ counts) {
    __shared__ int wave_count[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int word = wave * kWaveWords;
    int ref[kWaveWords];
#pragma unroll
    for (int k = 0; k < kWaveWords; ++k)
        ref[k] = refs[min(c * kChunk + (word + k) * kWave + lane, blocks - 1)];
    int count = 0;
#pragma unroll
    for (int k = 0; k < kWaveWords; ++k) {
        const int b = c * kChunk + (word + k) * kWave + lane;
        const uint64_t bits = __ballot(b < blocks && ref[k] == 0);
        if (lane == 0) bitmap[static_cast<int64_t>(c) * kChunkWords + word + k] = bits;
        count += __popcll(bits);
    }
    if (lane == 0) wave_count[wave] = count;
    __syncthreads();
    if (threadIdx.x == 0) {
        int n = 0;
        for (int w = 0; w < kWaves; ++w) n += wave_count[w];
        counts[c] = n;
    }
}

template <int Ctrl, int Rows>
__device__ __forceinline__ int dpp_or_0(int v) {
    return __builtin_amdgcn_update_dpp(0, v, Ctrl, Rows, 0xf, true);
}

// Sum of the lanes up to this one: row_shr 1, 2, 4, 8 inside rows of sixteen, then the last lane
// of each row and of each half to those behind it.
__device__ __forceinline__ int wave_inclusive(int v) {
    v += dpp_or_0<0x111, 0xf>(v);
    v += dpp_or_0<0x112, 0xf>(v);
    v += dpp_or_0<0x114, 0xf>(v);
    v += dpp_or_0<0x118, 0xf>(v);
    v += dpp_or_0<0x142, 0xa>(v);
    v += dpp_or_0<0x143, 0xc>(v);
    return v;
}

// For each of N values: its sum over the workgroup (total), and over the threads before this
// one (returned in place of the value).
template <int N>
__device__ __forceinline__ void group_exclusive(int (&v)[N], int (&total)[N]) {
    __shared__ int sums[N][kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) inc[k] = wave_inclusive(v[k]);
    __syncthreads();  // the last call's reads of sums
    if (lane == 63) {
#pragma unroll
        for (int k = 0; k < N; ++k) sums[k][wave] = inc[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        int before = 0;
        total[k] = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            before += w < wave ? sums[k][w] : 0;
            total[k] += sums[k][w];
        }
        v[k] = before + inc[k] - v[k];
    }
}

__device__ __forceinline__ int group_exclusive(int v, int& total) {
    int in[1] = {v}, all[1];
    group_exclusive(in, all);
    total = all[0];
    return in[0];
}

// The free blocks among `bits` (those of 64 blocks from `block` on, the first of rank `rank`) of
// ranks [lo, hi) to put(rank, block).
template <typename F>
__device__ __forceinline__ void put_word(uint64_t bits, int block, int rank, int lo, int hi,
                                         F&& put) {
    for (; bits != 0 && rank < hi; bits &= bits - 1, ++rank)
        if (rank >= lo) put(rank, block + __builtin_ctzll(bits));
}

// The free blocks of ranks [lo, hi), lowest first, to put(rank, block); by the whole workgroup.
// A chunk that holds some of them is found by the prefix over the chunks' counts, a word by the
// prefix over the chunk's.
template <typename F>
__device__ __forceinline__ void select_free(const uint64_t* __restrict__ bitmap,
                                            const int32_t* __restrict__ counts, int chunks, int lo,
                                            int hi, F&& put) {
    __shared__ int list_chunk[kThreads], list_rank[kThreads];
    __shared__ int list_n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0;
    for (int c0 = 0; c0 < chunks && base < hi; c0 += kThreads) {
        const int c = c0 + static_cast<int>(threadIdx.x);
        const int n = c < chunks ? counts[c] : 0;
        int total;
        const int first = base + group_exclusive(n, total);
        if (threadIdx.x == 0) list_n = 0;
        __syncthreads();
        if (n > 0 && first < hi && first + n > lo) {
            const int at = atomicAdd(&list_n, 1);  // any order: ranks go with their chunk
            list_chunk[at] = c;
            list_rank[at] = first;
        }
        __syncthreads();
        for (int k = wave; k < list_n; k += kWaves) {
            uint64_t bits = 0;
            if (lane < kChunkWords)
                bits = bitmap[static_cast<int64_t>(list_chunk[k]) * kChunkWords + lane];
            const int here = __popcll(bits);
            put_word(bits, list_chunk[k] * kChunk + lane * kWave,
                     list_rank[k] + wave_inclusive(here) - here, lo, hi, put);
        }
        __syncthreads();
        base += total;
    }
}

// ---- update ------------------------------------------------------------------

// What the first launch says of an item that can be done.
struct ItemPlan {
    int32_t need;    // blocks from the pool
    int32_t shared;  // leading blocks that are the source row's
    int32_t total;   // blocks of the new row
    int32_t length;
    int32_t from;    // block whose first `part` tokens the first of its new blocks gets, or -1
    int32_t part;
    int32_t held;    // blocks of the old row
};

struct UpdateWorkspace {
    uint64_t* bitmap;
    int32_t* counts;
    int32_t* needs;  // blocks that an item needs, or the status that it fails with, negated
    ItemPlan* plans;
    int32_t* staged;  // [items][width]: the blocks that the new row takes from the source row
};

size_t update_layout(int items, int width, int blocks, char* ws, UpdateWorkspace* out) {
    const int chunks = chunks_of(blocks);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes);
        return ws + here;
    };
    char* bitmap = take(static_cast<size_t>(chunks) * kChunkWords * sizeof(uint64_t));
    char* counts = take(static_cast<size_t>(chunks) * sizeof(int32_t));
    char* needs = take(static_cast<size_t>(items) * sizeof(int32_t));
    char* plans = take(static_cast<size_t>(items) * sizeof(ItemPlan));
    char* staged = take(static_cast<size_t>(items) * width * sizeof(int32_t));
    if (out != nullptr)
        *out = {reinterpret_cast<uint64_t*>(bitmap), reinterpret_cast<int32_t*>(counts),
                reinterpret_cast<int32_t*>(needs), reinterpret_cast<ItemPlan*>(plans),
                reinterpret_cast<int32_t*>(staged)};
    return at;
}

// Workgroups [0, chunks): the bitmap. Then one per item: its arguments and the blocks of the two
// rows are checked, its plan made, the source row's blocks copied. Three dependent reads: the
// item, its rows and contexts, the counts of their blocks (3.3 us).
__global__ __launch_bounds__(kThreads) void update_plan_kernel(TableUpdate u, KvLayers kv,
                                                               int blocks, int chunks,
                                                               UpdateWorkspace ws) {
    if (static_cast<int>(blockIdx.x) < chunks) {
        free_bitmap(u.refs, blocks, blockIdx.x, ws.bitmap, ws.counts);
        return;
    }
    const int i = blockIdx.x - chunks;
    const int bs = kv.block_size;
    const int d = u.dst[i], s = u.src != nullptr ? u.src[i] : d;
    const int asked = u.lengths != nullptr ? u.lengths[i] : -1;
    const int most = u.width * bs;
    bool bad = d < 0 || d >= u.rows || s < -1 || s >= u.rows || asked < -1 || asked > most;
    // the first entries of both rows are asked for with the contexts, not after them
    const int32_t* src_row = u.table + static_cast<int64_t>(min(max(s, 0), u.rows - 1)) * u.width;
    const int32_t* dst_row = u.table + static_cast<int64_t>(min(max(d, 0), u.rows - 1)) * u.width;
    const int entry = min(static_cast<int>(threadIdx.x), u.width - 1);
    const int src_entry = src_row[entry], dst_entry = dst_row[entry];
    const int src_ctx = u.ctx[min(max(s, 0), u.rows - 1)], old = u.ctx[min(max(d, 0), u.rows - 1)];
    for (int j = threadIdx.x; j < u.items; j += kThreads) bad |= j != i && u.dst[j] == d;
    ItemPlan p{};
    p.from = -1;
    auto tell = [&](int status) {
        if (threadIdx.x == 0) {
            ws.needs[i] = status == kOk ? p.need : -status;
            ws.plans[i] = p;
        }
    };
    if (__syncthreads_or(bad)) return tell(kInvalidArgument);
    const int have = s < 0 ? 0 : src_ctx;
    if (have < 0 || have > most || old < 0 || old > most) return tell(kInvalidTable);
    p.length = asked < 0 ? have : asked;
    const int kept = min(p.length, have);
    const int known = (kept + bs - 1) / bs;
    p.part = kept % bs;
    p.total = (p.length + bs - 1) / bs;
    p.held = (old + bs - 1) / bs;
    auto good = [&](int b) { return b >= 0 && b < blocks && u.refs[b] > 0; };
    bad = false;
    for (int j = threadIdx.x; j < known; j += kThreads) {
        const int b = j < kThreads ? src_entry : src_row[j];
        bad |= !good(b);
        ws.staged[static_cast<int64_t>(i) * u.width + j] = b;
    }
    for (int j = threadIdx.x; j < p.held; j += kThreads)
        bad |= !good(j < kThreads ? dst_entry : dst_row[j]);
    if (__syncthreads_or(bad)) return tell(kInvalidTable);
    const int last = known > 0 ? src_row[known - 1] : -1;
    // A block that is filled in part goes on being written: it may have one owner only. A row
    // that is cut back into a block of its own leaves it to rows that take it over as a whole
    // block in the same call.
    bool taken = false;
    if (p.part > 0 && s == d && u.src != nullptr && old >= known * bs) {
        for (int j = threadIdx.x; j < u.items; j += kThreads) {
            const int n = u.lengths != nullptr ? u.lengths[j] : -1;
            taken |= u.src[j] == d && j != i && (n < 0 || n >= known * bs);
        }
        taken = __syncthreads_or(taken);
    }
    const bool copied = p.part > 0 && (s != d || u.refs[last] > 1 || taken);
    p.shared = known - (copied ? 1 : 0);
    p.need = p.total - p.shared;
    p.from = copied ? last : -1;
    tell(copied && kv.layers == 0 && u.copy_src == nullptr ? kInvalidArgument : kOk);
}

// Workgroup (i, y): y = 0 changes the table row and the counts of item i; every y copies its
// parts of the block that was filled in part. All read the plans of all items first: one that
// cannot be done keeps the call from changing anything. What is copied is asked for as soon as
// the item's plan is there, before it is known where it goes. kSmall: the pool has at most
// kThreads words, a word a lane, asked for at the start.
// Bound by its chain of reads (plans and bitmap, source block, store): 48 beams of 8 layers 7.4
// us, of which 25 MB of copies take 4.8, and 4 items 3.8; with the plan 11.3 and 7.3 in all. It
// was 16.6 and 11.1 with a reduction for each sum and the copies' loads after the selection. Rows
// that grow by a token and copy nothing: 64 take 7.0 with the plan, 256 7.7, 1024 12.2, for under
// 0.4 us of bytes.
template <typename T, bool kSmall>
__global__ __launch_bounds__(kThreads) void update_apply_kernel(TableUpdate u, KvLayers kv,
                                                                int chunks, UpdateWorkspace ws) {
    const int i = blockIdx.x;
    const int tid = threadIdx.x;
    ItemPlan p{};
    p.from = -1;
    if (i < u.items) p = ws.plans[i];
    if (blockIdx.y > 0 && p.from < 0) return;
    uint64_t word = 0;
    if (kSmall && tid < chunks * kChunkWords) word = ws.bitmap[tid];
    // sums over the items and the pool: blocks asked for, those of the items before this one,
    // free ones, items of each failure
    int v[5] = {}, all[5];
    for (int j = tid; j < u.items; j += kThreads) {
        const int need = ws.needs[j];
        v[0] += max(need, 0);
        v[1] += j < i ? max(need, 0) : 0;
        v[3] += need == -kInvalidArgument;
        v[4] += need == -kInvalidTable;
    }
    if constexpr (kSmall) {
        v[2] = __popcll(word);
    } else {
        for (int c = tid; c < chunks; c += kThreads) v[2] += ws.counts[c];
    }
    PartCopy<T> ahead;
    const int parts = 2 * kv.layers;
    const bool copies = p.from >= 0 && kv.layers > 0;  // parts: at least as many as workgroups
    if (copies) ahead.start(kv, blockIdx.y, p.from, p.part);
    group_exclusive(v, all);
    const int status = all[3] > 0   ? kInvalidArgument
                       : all[4] > 0 ? kInvalidTable
                       : all[0] > all[2] ? kExhausted
                                         : kOk;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *u.status = status;
    const bool tells = u.copy_src != nullptr && blockIdx.y == 0 && i < u.items;
    if (status != kOk && tells && tid == 0) u.copy_src[i] = u.copy_dst[i] = -1;
    if (status != kOk || i >= u.items) return;

    const int lo = all[1];
    auto select = [&](int hi, auto&& put) {
        if constexpr (kSmall)
            put_word(word, tid * kWave, v[2], lo, hi, put);
        else
            select_free(ws.bitmap, ws.counts, chunks, lo, hi, put);
    };
    __shared__ int to;
    if (blockIdx.y == 0) {
        const int d = u.dst[i], s = u.src != nullptr ? u.src[i] : d;
        int32_t* row = u.table + static_cast<int64_t>(d) * u.width;
        const int32_t* staged = ws.staged + static_cast<int64_t>(i) * u.width;
        // a row that goes on from itself keeps its references to what it keeps
        const int same = s == d ? p.shared : 0;
        for (int j = tid; j < p.held; j += kThreads)
            if (j >= same) atomicAdd(&u.refs[row[j]], -1);
        __syncthreads();
        for (int j = tid; j < u.width; j += kThreads) {
            if (j < p.shared) {
                const int b = staged[j];
                row[j] = b;
                if (j >= same) atomicAdd(&u.refs[b], 1);
            } else if (j >= p.total) {
                row[j] = -1;
            }
        }
        select(lo + p.need, [&](int rank, int b) {
            row[p.shared + rank - lo] = b;
            atomicAdd(&u.refs[b], 1);
            if (rank == lo) to = b;
        });
        if (tid == 0) u.ctx[d] = p.length;
    } else if (copies) {
        select(lo + 1, [&](int, int b) { to = b; });
    }
    if (!copies && !tells) return;
    __syncthreads();
    if (tells && tid == 0) {
        u.copy_src[i] = p.from;
        u.copy_dst[i] = p.from >= 0 ? to : -1;
    }
    if (!copies) return;
    ahead.finish(kv, p.from, to, p.part);
    for (int part = blockIdx.y + gridDim.y; part < parts; part += gridDim.y)
        copy_part<T>(kv, part, p.from, to, p.part);
}

// ---- compact -----------------------------------------------------------------

struct CompactWorkspace {
    uint64_t* bitmap;
    int32_t* counts;
    int32_t* moves;   // [0]: how many blocks move
    int32_t* movers;  // rank -> block that moves, its count, its place
    int32_t* counts_of;
    int32_t* holes;
    int32_t* rank_of;  // block that moves -> rank
};

size_t compact_layout(int blocks, char* ws, CompactWorkspace* out) {
    const int chunks = chunks_of(blocks);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes);
        return ws + here;
    };
    const size_t half = (static_cast<size_t>(blocks) / 2 + 1) * sizeof(int32_t);
    char* bitmap = take(static_cast<size_t>(chunks) * kChunkWords * sizeof(uint64_t));
    char* counts = take(static_cast<size_t>(chunks) * sizeof(int32_t));
    char* moves = take(sizeof(int32_t));
    char* movers = take(half);
    char* counts_of = take(half);
    char* holes = take(half);
    char* rank_of = take(static_cast<size_t>(blocks) * sizeof(int32_t));
    if (out != nullptr) {
        auto i32 = [](char* p) { return reinterpret_cast<int32_t*>(p); };
        *out = {reinterpret_cast<uint64_t*>(bitmap), i32(counts), i32(moves), i32(movers),
                i32(counts_of), i32(holes), i32(rank_of)};
    }
    return at;
}

__global__ __launch_bounds__(kThreads) void free_bitmap_kernel(const int32_t* refs, int blocks,
                                                               uint64_t* bitmap,
                                                               int32_t* counts) {
    free_bitmap(refs, blocks, blockIdx.x, bitmap, counts);
}

// The live blocks (all that are not free) from n_live on (the movers) and the free ones below
// n_live (the holes) are equally many, at most half of the pool; the j-th lowest mover goes to
// the j-th lowest hole.
// Workgroup c lists those of its chunk and writes its blocks' counts and new numbers, the
// movers' own (known once all holes are) aside.
__global__ __launch_bounds__(kThreads) void compact_plan_kernel(const int32_t* refs, int blocks,
                                                                int chunks, CompactWorkspace ws,
                                                                int32_t* refs_out,
                                                                int32_t* __restrict__ remap,
                                                                int32_t* __restrict__ num_live) {
    __shared__ int word_free[kChunkWords];  // free blocks of the chunk before a word
    const int c = blockIdx.x;
    const int lane = threadIdx.x & 63;
    constexpr int kEach = kChunk / kThreads;
    int counts[kEach];  // of this lane's blocks, asked for first
#pragma unroll
    for (int k = 0; k < kEach; ++k)
        counts[k] = refs[min(c * kChunk + k * kThreads + static_cast<int>(threadIdx.x), blocks - 1)];
    int free_sum[2] = {}, free_all[2];  // free blocks of all chunks, of those before this one
    for (int j = threadIdx.x; j < chunks; j += kThreads) {
        const int n = ws.counts[j];
        free_sum[0] += n;
        free_sum[1] += j < c ? n : 0;
    }
    group_exclusive(free_sum, free_all);
    const int n_live = blocks - free_all[0], free_before = free_all[1];
    // holes: free blocks below n_live, whole chunks and the words of the chunk it lies in
    const int cut = n_live / kChunk;
    int below = 0, holes;
    for (int j = threadIdx.x; j < cut; j += kThreads) below += ws.counts[j];
    if (cut < chunks && threadIdx.x < kChunkWords) {
        const int at = n_live - cut * kChunk - static_cast<int>(threadIdx.x) * kWave;
        const uint64_t bits =
            ws.bitmap[static_cast<int64_t>(cut) * kChunkWords + threadIdx.x];
        const uint64_t mask = at <= 0 ? 0 : (at >= 64 ? ~0ull : (1ull << at) - 1);
        below += __popcll(bits & mask);
    }
    group_exclusive(below, holes);
    if (threadIdx.x < kWave) {
        int n = 0;
        if (lane < kChunkWords)
            n = __popcll(ws.bitmap[static_cast<int64_t>(c) * kChunkWords + lane]);
        const int before_word = wave_inclusive(n) - n;
        if (lane < kChunkWords) word_free[lane] = before_word;
    }
    __syncthreads();
    if (c == 0 && threadIdx.x == 0) {
        *num_live = n_live;
        ws.moves[0] = holes;
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int k = e * kThreads + threadIdx.x;
        const int b = c * kChunk + k;
        if (b >= blocks) break;
        const int word = k / kWave;
        const uint64_t bits = ws.bitmap[static_cast<int64_t>(c) * kChunkWords + word];
        const uint64_t low = (1ull << (k % kWave)) - 1;
        const bool is_free = (bits >> (k % kWave)) & 1;
        const int free_rank = free_before + word_free[word] + __popcll(bits & low);
        const int count = counts[e];
        int out = 0, to = -1;
        if (is_free) {
            if (b < n_live) ws.holes[free_rank] = b;
        } else if (b < n_live) {
            out = count;
            to = b;
        } else {
            const int rank = b - free_rank - (n_live - holes);
            ws.movers[rank] = b;
            ws.counts_of[rank] = count;
            ws.rank_of[b] = rank;
        }
        refs_out[b] = out;
        remap[b] = to;
    }
}

// Workgroups [0, table_groups): the table's entries. The others: the moves, each with its counts
// and its new number, part by part; how many there are only the device knows.
template <typename T>
__global__ __launch_bounds__(kThreads) void compact_move_kernel(const int32_t* table,
                                                                int64_t entries, KvLayers kv,
                                                                int table_groups,
                                                                CompactWorkspace ws,
                                                                const int32_t* num_live,
                                                                int32_t* table_out,
                                                                int32_t* refs_out,
                                                                int32_t* remap) {
    if (static_cast<int>(blockIdx.x) < table_groups) {
        const int n_live = *num_live;
        for (int64_t e = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; e < entries;
             e += static_cast<int64_t>(table_groups) * kThreads) {
            const int b = table[e];
            int to = b;
            if (b >= kv.blocks)
                to = -1;
            else if (b >= 0) {
                const uint64_t bits = ws.bitmap[b / kWave];
                if ((bits >> (b % kWave)) & 1)
                    to = -1;
                else if (b >= n_live)
                    to = ws.holes[ws.rank_of[b]];
            }
            table_out[e] = to;
        }
        return;
    }
    const int parts = max(1, 2 * kv.layers);
    const int moves = ws.moves[0];
    const int64_t units = static_cast<int64_t>(moves) * parts;
    const int groups = gridDim.x - table_groups;
    for (int64_t q = blockIdx.x - table_groups; q < units; q += groups) {
        const int part = static_cast<int>(q / moves);
        const int j = static_cast<int>(q - static_cast<int64_t>(part) * moves);
        const int from = ws.movers[j], to = ws.holes[j];
        if (part == 0 && threadIdx.x == 0) {
            refs_out[to] = ws.counts_of[j];
            remap[from] = to;
        }
        if (kv.layers > 0) copy_part<T>(kv, part, from, to, kv.block_size);
    }
}

}  // namespace

hipError_t copy_kv_blocks(const KvLayers& kv, const int32_t* src, const int32_t* dst, int pairs,
                          int32_t* status, hipStream_t stream) {
    // Enough workgroups to keep the chip full to the end, and no more lists checked than that
    // takes: with 16384, 900 blocks x 24 layers take 466 us (5.8 TB/s of counted traffic), with
    // 4096 482, with 1024 540.
    const int parts = 2 * kv.layers;
    const int split = std::min(parts, std::max(1, (16384 + pairs - 1) / pairs));
    const dim3 grid(static_cast<unsigned>(pairs), static_cast<unsigned>(split));
    return with_unit(kv, [&](auto unit) {
        copy_blocks_kernel<decltype(unit)><<<grid, kThreads, 0, stream>>>(kv, src, dst, pairs,
                                                                          status);
    });
}

size_t update_tables_workspace_bytes(int items, int width, int blocks) {
    return update_layout(items, width, blocks, nullptr, nullptr);
}

hipError_t update_block_tables(const TableUpdate& u, const KvLayers& kv, void* workspace,
                               hipStream_t stream) {
    const int chunks = chunks_of(kv.blocks);
    UpdateWorkspace ws;
    update_layout(u.items, u.width, kv.blocks, static_cast<char*>(workspace), &ws);
    update_plan_kernel<<<static_cast<unsigned>(chunks + u.items), kThreads, 0, stream>>>(
        u, kv, kv.blocks, chunks, ws);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    // Workgroups of an item share its parts: as many as there are parts where the items are few,
    // and one where they are so many that they fill the chip themselves.
    const int items = std::max(1, u.items);
    const int split = std::max(1, std::min(2 * kv.layers, (4096 + items - 1) / items));
    const dim3 grid(static_cast<unsigned>(items), static_cast<unsigned>(split));
    return with_unit(kv, [&](auto unit) {
        using T = decltype(unit);
        if (chunks * kChunkWords <= kThreads)
            update_apply_kernel<T, true><<<grid, kThreads, 0, stream>>>(u, kv, chunks, ws);
        else
            update_apply_kernel<T, false><<<grid, kThreads, 0, stream>>>(u, kv, chunks, ws);
    });
}

size_t compact_workspace_bytes(int blocks) { return compact_layout(blocks, nullptr, nullptr); }

hipError_t compact_kv_blocks(const int32_t* table, const int32_t* refs, int64_t entries,
                             const KvLayers& kv, int32_t* table_out, int32_t* refs_out,
                             int32_t* remap, int32_t* num_live, void* workspace,
                             hipStream_t stream) {
    const int chunks = chunks_of(kv.blocks);
    CompactWorkspace ws;
    compact_layout(kv.blocks, static_cast<char*>(workspace), &ws);
    free_bitmap_kernel<<<static_cast<unsigned>(chunks), kThreads, 0, stream>>>(
        refs, kv.blocks, ws.bitmap, ws.counts);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    compact_plan_kernel<<<static_cast<unsigned>(chunks), kThreads, 0, stream>>>(
        refs, kv.blocks, chunks, ws, refs_out, remap, num_live);
    err = hipGetLastError();
    if (err != hipSuccess) return err;
    const int table_groups =
        static_cast<int>(std::min<int64_t>(256, (entries + kThreads - 1) / kThreads));
    // 8192 workgroups over the moves: 994 blocks x 12 layers (1.56 GB) take 298-304 us, the rate
    // of a copy (5.2 TB/s); 122 fp8 blocks x 24 layers 33-35. With 2048 323 in all instead of 311,
    // and 44 instead of 40.
    const int64_t most = static_cast<int64_t>(kv.blocks / 2 + 1) * std::max(1, 2 * kv.layers);
    const int move_groups = static_cast<int>(std::min<int64_t>(8192, most));
    return with_unit(kv, [&](auto unit) {
        compact_move_kernel<decltype(unit)>
            <<<static_cast<unsigned>(table_groups + move_groups), kThreads, 0, stream>>>(
                table, entries, kv, table_groups, ws, num_live, table_out, refs_out, remap);
    });
}

}  // namespace ccinfer::hipk
