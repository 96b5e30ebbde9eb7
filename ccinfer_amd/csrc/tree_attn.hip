// Attention of drafted tokens over the paged cache: several new tokens a request, each of which
// sees the committed context and those of the request's new tokens that its mask names (its
// ancestors in a tree of drafts, itself among them).
//
//   request b: n = query_start_loc[b + 1] - query_start_loc[b] nodes in rows query_start_loc[b]
//   + i of q; context_lens[b] tokens with them, node j at position context_lens[b] - n + j.
//   Row i sees position p if p < context_lens[b] - n, or if bit p - (context_lens[b] - n) of its
//   mask is set. o = sum softmax(q k / sqrt d) v; zeros for a row that sees nothing.
//
// The G query heads of a kv head and the nodes make one matrix of n G rows, so a tree of 64 nodes
// at G = 4 fills the 256 rows of a workgroup, and K and V are read once for all of them. Rows are
// worked in blocks of up to eight wavefronts' (32 each, 16 at head dims over 128). In a block of
// few rows, wavefronts share the chunks instead: up to a wavefront's rows each of the eight takes
// chunks of its own, up to two wavefronts' four pairs do, and so on; what they found is added up
// in LDS.
//
// Work is cut without knowing the lengths on the host: the (request, row block) items of a kv
// head, laid end to end in units of their cost, are cut into `slots` equal ranges, one for each
// workgroup, which finds its own by a scan over the requests. An item that lies in one slot goes
// straight to the output; the pieces of one that is cut go to the workspace, and the workgroups
// of a second launch, one set for each slot in which a cut item begins, add them up.
//
// What bounds it: with few rows an item's start and end, in which nothing else is under way (8
// requests of 2048 tokens and 8 nodes, 32 / 8 heads of 128: 36.5 us, 1.9 TB/s; 248 of 64 tokens and 8 of
// 8192: 153 us, 2.4 TB/s); with all 256 rows of a block (256 operations a byte) the two wavefronts
// of each SIMD, which meet and then do the same phase at once: 140 vector and 95 scalar instructions a
// chunk, LDS reads and the waits between the products leave the matrix unit busy for 22 % of the
// time. 48 trees of 8 to 64 nodes over 735 MB of K and V: 238 us a call, the merge with it (3.1 TB/s,
// 0.44 PFLOP/s); over an fp8 cache (394 MB) 329, whose conversions come on top. One tree of 26 nodes
// over 1187 tokens, 16 / 8 heads: 22 us a call; under a tracer 17.5, of which the scan of the requests
// takes 2, the start 5 and the chunks 7, and 3.9 for the merge. Head dims of 72 to 120 spill 27
// registers (120: 259 us, 689 MB), those over 128 have half the wavefronts and a quarter of the rows a
// block (256: 1129 us, 1470 MB).
#include <algorithm>

#include "kernels.hpp"
#include "row_tiles.hpp"

namespace ccinfer::hipk {
namespace {

using namespace rows;

constexpr int kMaxRequests = kTreeMaxBatch;
constexpr int kMergeWaves = 4;
// Workgroups of the merge a slot, 8 of at most 256 rows each (16: 32 pieces of 128 rows 30.5 us
// in place of 16.4; 64: no faster, and 48 trees 16.9 in place of 14.8).
constexpr int kMergeSplit = 32;

// Wavefronts of a workgroup, and tiles of 16 rows of each. One workgroup a CU: the ring fills its
// LDS. At head dims over 128 a wavefront needs the registers of two.
template <int D>
constexpr int kWaves = D <= 128 ? 8 : 4;
template <int D>
constexpr int kTiles = D <= 128 ? 2 : 1;
template <int D>
constexpr int kBlockRows = kWaves<D> * 16 * kTiles<D>;

// The cut item that begins in a slot: its rows, and the last slot that holds a piece of it
// (rows 0: none).
struct SlotDesc {
    int first_token;  // row of q of its request's node 0
    int first_row;    // of its request's n G rows
    int rows;
    int last_slot;
};

template <int D, bool F8, bool Pad>
struct TreeArgs {
    const __bf16* q;
    Cache<D, F8, Pad> cache;
    const int32_t* table;
    const int32_t* qsl;
    const int32_t* ctx;
    const uint32_t* mask;
    __bf16* out;
    int batch, total, mbpr, hq, words;
    float scale_log2;
    uint32_t by_group;  // 2^32 / (hq / hkv), rounded up: quotients by it are its high products
    int slots;      // of each kv head
    int min_units;  // of a slot
    int row_cap;    // rows of a workspace piece
    float* part_acc;
    float2* part_ml;
    SlotDesc* desc;
};

// A request as the kernels see it (prefill's rules: rows past `total` and requests whose context
// is shorter than their nodes are left out).
struct Request {
    int first;   // row of q
    int nodes;   // rows that are there
    int n;       // nodes that the context counts
    int before;  // committed tokens
    int end;     // tokens that the table row holds
};

__device__ __forceinline__ Request request_of(int from, int to, int c, int total, int mbpr) {
    Request r;
    r.first = from;
    r.n = to - r.first;
    r.before = c - r.n;
    r.nodes = min(to, total) - r.first;
    r.end = min(c, mbpr * kBlock);
    // (the inputs, not their differences, which broken ones may have taken past 32 bits)
    if (from < 0 || to <= from || c < r.n || r.nodes < 0) r.nodes = 0;
    return r;
}

// Units of all requests together stay below this (the host refuses other shapes).
constexpr int kMaxUnits = 1 << 30;

// Wavefronts of a block of this many rows that have rows of their own.
template <int R>
__device__ __forceinline__ int row_groups(int rows) {
    return rows <= R ? 1 : (rows <= 2 * R ? 2 : (rows <= 4 * R ? 4 : 8));
}

// Cost of a chunk, whatever the rows of its block (4 units in place of 5 for up to half the rows:
// the same to 1 % slower). Several units, so that the ranges are nearly equal: with one, 8 requests
// of 2048 tokens take 41 us in place of 36.6.
constexpr int kChunkUnits = 4;
// Cost of an item's start and end: rows of q, the first chunks' way, sums joined and stored, 20 to
// 30 thousand cycles (left out, a slot may get many short requests: 248 of 64 tokens with 8 of
// 8192 take 286 us in place of 154).
constexpr int kStartUnits = 32;

// Units of a request's row blocks.
template <int D>
__device__ __forceinline__ int request_units(const Request& r, int G) {
    if (r.nodes <= 0) return 0;
    const int rows = r.nodes * G;
    const int blocks = (rows - 1) / kBlockRows<D> + 1;
    const int chunks = (r.end + kChunk - 1) / kChunk;
    return blocks * (kStartUnits + chunks * kChunkUnits);
}

// The blocks of chunks first, first + stride, ... below last of a table row, one chunk after the
// other (the last one again behind them), 64 chunks at a time in the wavefront's lanes: lane 2 k
// + x of `ids[w]` holds block x of chunk 32 w + k.
struct BlockIds {
    const int32_t* table;
    int end, stride, last, lane;
    int c;  // of the next Pair
    int k;  // its place
    int ids[2];
    __device__ __forceinline__ BlockIds(const int32_t* t, int first, int last_, int stride_,
                                        int end_, int lane_)
        : table(t), end(end_), stride(stride_), last(last_), lane(lane_), c(first), k(0) {
        load();
    }
    __device__ __forceinline__ void load() {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int chunk = c + (32 * w + (lane >> 1)) * stride;
            const int block = 2 * chunk + (lane & 1);
            ids[w] = chunk < last && block * kBlock < end ? table[block] : -1;
        }
        // here, where it is rare: a load that may be under way at a use makes the compiler wait
        // for the copies into LDS there too
        __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    __device__ __forceinline__ Pair operator()() {
        const int w = k >= 64 ? ids[1] : ids[0];
        const int left = end - c * kChunk;
        const Pair p = make_pair(__builtin_amdgcn_readlane(w, k & 63), left,
                                 __builtin_amdgcn_readlane(w, (k & 63) + 1), left - kBlock);
        if (c + stride < last) {
            c += stride;
            k += 2;
            if (k == 128) {
                k = 0;
                load();
            }
        }
        return p;
    }
    // Of chunk c, whose blocks `on` are there: what its scores are masked by.
    __device__ __forceinline__ Pair read(int c_, uint32_t on) const {
        const int left = end - c_ * kChunk;
        return Pair{{0, 0}, {min(left, kBlock), min(left - kBlock, kBlock)}, on};
    }
};

template <int D, bool F8, bool Pad>
__global__ __launch_bounds__(kWaves<D> * 64, kWaves<D> / 4) void tree_attention_kernel(
    TreeArgs<D, F8, Pad> a) {
    constexpr int NT = kTiles<D>;
    constexpr int R = 16 * NT;
    constexpr int W = kWaves<D>;
    constexpr int kThreads = W * 64;
    constexpr int kPerThread = kMaxRequests / kThreads;  // requests of a thread
    __shared__ __align__(16) Shared<D, F8, NT, W, W> shared;
    __shared__ __align__(16) uint32_t lds_copy[4];
    __shared__ int starts[kMaxRequests + 1];
    __shared__ int froms[kMaxRequests], tos[kMaxRequests], ctxs[kMaxRequests];
    __shared__ int64_t wave_sum[W];
    __shared__ int first_request;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hkv = a.cache.hkv;
    const int G = a.hq / hkv, dr = a.cache.dims();
    const int h = blockIdx.x % hkv, slot = blockIdx.x / hkv;
    SlotDesc* desc = a.desc + static_cast<int64_t>(h) * a.slots + slot;

    // Where each request's units start.
    const int per = (a.batch + kThreads - 1) / kThreads;
    int units[kPerThread];
    int64_t sum = 0;  // requests that overlap (a broken query_start_loc) may pass 32 bits
#pragma unroll
    for (int x = 0; x < kPerThread; ++x) {
        const int b = tid * per + x;
        units[x] = 0;
        if (x < per && b < a.batch) {
            const int from = a.qsl[b], to = a.qsl[b + 1], c = a.ctx[b];
            froms[b] = from;
            tos[b] = to;
            ctxs[b] = c;
            units[x] = request_units<D>(request_of(from, to, c, a.total, a.mbpr), G);
        }
        sum += units[x];
    }
    int64_t incl = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t y = __shfl_up(incl, off);
        if (lane >= off) incl += y;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    int64_t before = incl - sum, total_units = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        before += w < wave ? wave_sum[w] : 0;
        total_units += wave_sum[w];
    }
    // past the host's bound: no request is worked on
    const int all = total_units < kMaxUnits ? static_cast<int>(total_units) : 0;
    int at = static_cast<int>(before);
    const int quota = max((all + a.slots - 1) / a.slots, a.min_units);
    const int u0 = slot * quota;
    const int u1 = min(all, u0 + quota);
#pragma unroll
    for (int x = 0; x < kPerThread; ++x) {
        const int b = tid * per + x;
        if (x < per && b < a.batch) {
            starts[b] = at;
            if (at <= u0 && u0 < at + units[x]) first_request = b;
            at += units[x];
        }
    }
    if (tid == 0) starts[a.batch] = all;
    __syncthreads();
    if (u0 >= u1) {
        if (tid == 0) *desc = SlotDesc{0, 0, 0, 0};
        return;
    }
    // (2^32 / 1 has no place in 32 bits)
    auto node_of = [&](int r) {
        return G == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), a.by_group));
    };
    SlotDesc own{0, 0, 0, 0};
    int b = first_request;
    for (int u = __builtin_amdgcn_readfirstlane(u0); u < u1;) {
        while (starts[b + 1] <= u) ++b;
        b = __builtin_amdgcn_readfirstlane(b);
        const Request req = request_of(__builtin_amdgcn_readfirstlane(froms[b]),
                                       __builtin_amdgcn_readfirstlane(tos[b]),
                                       __builtin_amdgcn_readfirstlane(ctxs[b]), a.total, a.mbpr);
        const int all_rows = req.nodes * G;
        const int chunks = (req.end + kChunk - 1) / kChunk;
        const int item = kStartUnits + chunks * kChunkUnits;
        const int local = u - __builtin_amdgcn_readfirstlane(starts[b]);
        const int rb = local / item;
        const int row0 = rb * kBlockRows<D>;
        const int block_rows = min(all_rows - row0, kBlockRows<D>);
        const int from = local - rb * item;
        const int to = min(item, from + (u1 - u));
        // a chunk belongs to the slot that its first unit lies in
        const int c0 = (max(from - kStartUnits, 0) + kChunkUnits - 1) / kChunkUnits;
        const int c1 = (max(to - kStartUnits, 0) + kChunkUnits - 1) / kChunkUnits;
        const bool whole = from == 0 && to == item;
        const int which = from == 0 ? 1 : 0;  // piece of the slot: begins in it, or before it
        if (from == 0 && to < item)
            own = SlotDesc{req.first, row0, block_rows, (u - from + item - 1) / quota};

        // Wavefronts by rows, and those of the same rows by chunks.
        const int groups = row_groups<R>(block_rows);
        const int share = W / groups;
        const int group = wave % groups, part = wave / groups;
        State<D, NT, !F8> st;
        st.clear();
        const bool busy = group * R < block_rows;
        bf16x8 q[NT][Shape<D>::kSteps];
        const uint32_t* mask_row[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int row = group * R + 16 * t + (lane & 15);
            const bool live = row < block_rows;
            const int r = row0 + (live ? row : 0);
            const int node = node_of(r);
            const int64_t token = req.first + node;
            load_q<D, F8, Pad>(q[t], a.q + (token * a.hq + h * G + (r - node * G)) * dr, live, dr,
                               lane);
            mask_row[t] = a.mask + token * a.words;
        }
        const int32_t* table = a.table + static_cast<int64_t>(b) * a.mbpr;
        BlockIds ids(table, c0 + part, c1, share, req.end, lane);
        auto chunk = [&](int c) {
            const int cb = c * kChunk;
            return make_pair(table[2 * c], req.end - cb,
                             cb + kBlock < req.end ? table[2 * c + 1] : -1, req.end - cb - kBlock);
        };
        auto seen = [&](int c, int t, uint32_t& bits) {
            const int o = c * kChunk - req.before;  // tree node of the chunk's first token
            if (o <= -kChunk) return false;
            const uint32_t* m = mask_row[t];
            if (o < 0) {
                bits = (m[0] << -o) | ((1u << -o) - 1u);
            } else {
                const int w = o >> 5;
                const uint32_t lo = w < a.words ? m[w] : 0u;
                const uint32_t hi = w + 1 < a.words ? m[w + 1] : 0u;
                bits = static_cast<uint32_t>(((static_cast<uint64_t>(hi) << 32) | lo) >> (o & 31));
            }
            return true;
        };
        const int steps = (c1 - c0 + share - 1) / share;
        bool left_out;
        if (c0 >= c1)
            left_out = false;
        else if (groups == 1)
            left_out = attend_alone(st, q, a.cache, shared.tiles[wave],
                                    LdsCopy(lds_copy, shared.tiles + wave), h, c0 + part, c1,
                                    share, a.scale_log2, lane, ids, seen);
        else if (groups == 2)
            left_out = attend_shared<2, 2>(
                st, q, a.cache, shared.tiles + 2 * part,
                LdsCopy(lds_copy, shared.tiles + 2 * part), group, h, c0 + part, c1, share, steps,
                busy, a.scale_log2, lane, ids, seen);
        else if (groups == 4)
            left_out = attend_shared<4, 4>(
                st, q, a.cache, shared.tiles + 4 * part,
                LdsCopy(lds_copy, shared.tiles + 4 * part), group, h, c0 + part, c1, share, steps,
                busy, a.scale_log2, lane, ids, seen);
        else if constexpr (W == 8)
            left_out = attend_shared<8, 8>(st, q, a.cache, shared.tiles,
                                           LdsCopy(lds_copy, shared.tiles), group, h, c0, c1, 1,
                                           steps, busy, a.scale_log2, lane, ids, seen);
        else
            left_out = false;
        if (left_out)
            add_unbounded(st, a.cache, h, c0 + part, c1, share, lane, chunk, seen);

        __syncthreads();  // the tiles' place is the sums' now
        add_parts(shared.sums, st, part, share, group, groups, lane);
        if (part == 0) {
            const int64_t piece = (static_cast<int64_t>(h) * a.slots + slot) * 2 + which;
            float* pa = a.part_acc + piece * a.row_cap * D;
            float2* pm = a.part_ml + piece * a.row_cap;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int row = group * R + 16 * t + (lane & 15);
                const float l = wave_sum_xor16_32(st.l[t]);
                if (row >= block_rows) continue;
                if (whole) {
                    const int r = row0 + row;
                    const int node = node_of(r);
                    const int64_t token = req.first + node;
                    store_row<D, Pad>(
                        st, t, l, a.out + (token * a.hq + h * G + (r - node * G)) * dr, dr, lane);
                } else {
                    store_part(st, t, pa + static_cast<int64_t>(row) * D, lane);
                    if (lane < 16) pm[row] = float2{st.m[t], l};
                }
            }
        }
        __syncthreads();
        u += to - from;
    }
    if (tid == 0) *desc = own;
}

// Rows of the cut items, a wavefront each in turn: the pieces of slots [slot, last_slot], the
// first of them the slot's item that begins in it, the others those that begin before them.
template <int D>
__global__ __launch_bounds__(kMergeWaves * 64) void tree_merge_kernel(
    const SlotDesc* desc, const float* part_acc, const float2* part_ml, __bf16* out, int slots,
    int row_cap, int hq, int hkv, int dr) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % hkv, slot = blockIdx.x / hkv;
    const int G = hq / hkv;
    const SlotDesc d = desc[static_cast<int64_t>(h) * slots + slot];
    const int64_t base = (static_cast<int64_t>(h) * slots + slot) * 2;
    for (int row = blockIdx.y * kMergeWaves + wave; row < d.rows;
         row += kMergeSplit * kMergeWaves) {
        float x[D / 64];
        const int pieces = d.last_slot - slot + 1;
        const float l = merge_row<D>(x, pieces, part_acc, part_ml, lane, [&](int s) {
            return (base + 2 * s + (s == 0 ? 1 : 0)) * row_cap + row;
        });
        const int r = d.first_row + row;
        const int node = r / G;
        store_columns<D>(
            out + ((static_cast<int64_t>(d.first_token) + node) * hq + h * G + (r - node * G)) * dr,
            x, inverse_sum(l), dr, lane);
    }
}

// Workgroups that the chip holds at once: one for each of 256 CUs.
constexpr int kResident = 256;
// Units of a slot at least: a start and eight chunks, one for each wavefront of a block of few rows
// (twice as many: 8 requests of 2048 tokens 38.5 us in place of 36.6; half: one of 1000 21.3 in
// place of 20.4).
constexpr int kMinUnits = kStartUnits + 8 * kChunkUnits;

int slots_of(int hkv) { return std::max(1, kResident / hkv); }

int mfma_dim(int head_dim) { return head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256); }

int row_cap_of(int total, int hq, int hkv, int D) {
    const int64_t rows = static_cast<int64_t>(total) * (hq / hkv);
    return static_cast<int>(std::min<int64_t>(rows, D <= 128 ? kBlockRows<128> : kBlockRows<256>));
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

struct TreeWorkspace {
    size_t desc = 0, ml = 0, acc = 0, bytes = 0;
};

TreeWorkspace workspace_of(int total, int hq, int hkv, int D) {
    TreeWorkspace w;
    const size_t slots = static_cast<size_t>(slots_of(hkv)) * hkv;
    const size_t cap = row_cap_of(total, hq, hkv, D);
    w.ml = align256(slots * sizeof(SlotDesc));
    w.acc = w.ml + align256(slots * 2 * cap * sizeof(float2));
    w.bytes = w.acc + slots * 2 * cap * D * sizeof(float);
    return w;
}

template <int D, bool F8, bool Pad>
hipError_t launch(const TreeAttention& t, void* workspace, hipStream_t stream) {
    const TreeWorkspace w = workspace_of(t.total, t.hq, t.hkv, D);
    char* ws = static_cast<char*>(workspace);
    TreeArgs<D, F8, Pad> a;
    a.q = static_cast<const __bf16*>(t.q);
    using Elem = std::conditional_t<F8, uint8_t, __bf16>;
    a.cache = {static_cast<const Elem*>(t.k), static_cast<const Elem*>(t.v), t.k_scale, t.v_scale,
               t.hkv, t.head_dim};
    a.table = t.table;
    a.qsl = t.qsl;
    a.ctx = t.ctx;
    a.mask = reinterpret_cast<const uint32_t*>(t.mask);
    a.out = static_cast<__bf16*>(t.out);
    a.batch = t.batch;
    a.total = t.total;
    a.mbpr = t.mbpr;
    a.hq = t.hq;
    a.words = t.words;
    a.scale_log2 = kLog2e / sqrtf(static_cast<float>(t.head_dim));
    const uint64_t group = static_cast<uint64_t>(t.hq / t.hkv);
    a.by_group = static_cast<uint32_t>(((uint64_t{1} << 32) + group - 1) / group);
    a.slots = slots_of(t.hkv);
    a.min_units = kMinUnits;
    a.row_cap = row_cap_of(t.total, t.hq, t.hkv, D);
    a.desc = reinterpret_cast<SlotDesc*>(ws + w.desc);
    a.part_ml = reinterpret_cast<float2*>(ws + w.ml);
    a.part_acc = reinterpret_cast<float*>(ws + w.acc);
    const unsigned grid = static_cast<unsigned>(a.slots) * t.hkv;
    hipLaunchKernelGGL((tree_attention_kernel<D, F8, Pad>), dim3(grid), dim3(kWaves<D> * 64), 0, stream, a);
    if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    hipLaunchKernelGGL((tree_merge_kernel<D>), dim3(grid, kMergeSplit), dim3(kMergeWaves * 64), 0,
                       stream,
                       a.desc, a.part_acc, a.part_ml, a.out, a.slots, a.row_cap, t.hq, t.hkv,
                       t.head_dim);
    return hipGetLastError();
}

}  // namespace

bool tree_attention_supported(int batch, int total, int mbpr, int hq, int hkv, int head_dim,
                              bool fp8) {
    if (batch > kTreeMaxBatch || head_dim > 256 || head_dim % 8 != 0) return false;
    if (fp8 && head_dim != 64 && head_dim != 128) return false;
    // units: the chunks of a row block, and its start
    const int64_t block = head_dim <= 128 ? kBlockRows<128> : kBlockRows<256>;
    const int64_t blocks = static_cast<int64_t>(total) * (hq / hkv) / block + batch;
    const int64_t units = kStartUnits + kChunkUnits * (static_cast<int64_t>(mbpr) / 2 + 1);
    // by_group gives the quotients of rows whose product with the group is below 2^32
    const int64_t group = hq / hkv;
    if (static_cast<int64_t>(total) * group >= (int64_t{1} << 32) / group) return false;
    // below 2^28 row blocks the product keeps 64 bits; a request's and all requests' units, and
    // the ends of the slots, keep 32
    return blocks < (int64_t{1} << 28) && units * blocks < kMaxUnits &&
           slots_of(hkv) <= kMaxUnits / kMinUnits;
}

size_t tree_attention_workspace_bytes(int total, int hq, int hkv, int head_dim) {
    return workspace_of(total, hq, hkv, mfma_dim(head_dim)).bytes;
}

hipError_t tree_attention(const TreeAttention& t, void* workspace, hipStream_t stream) {
    const bool fp8 = t.k_scale != nullptr;
    const int d = t.head_dim;
    switch (mfma_dim(d)) {
        case 64:
            return fp8 ? launch<64, true, false>(t, workspace, stream)
                   : d == 64 ? launch<64, false, false>(t, workspace, stream)
                             : launch<64, false, true>(t, workspace, stream);
        case 128:
            return fp8 ? launch<128, true, false>(t, workspace, stream)
                   : d == 128 ? launch<128, false, false>(t, workspace, stream)
                              : launch<128, false, true>(t, workspace, stream);
        default:
            return d == 256 ? launch<256, false, false>(t, workspace, stream)
                            : launch<256, false, true>(t, workspace, stream);
    }
}

}  // namespace ccinfer::hipk
