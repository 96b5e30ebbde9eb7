// Attention of drafted tokens over the paged cache: several new tokens a request, each of which
// sees the committed context and those of the request's new tokens that its mask names (its
// ancestors in a tree of drafts, itself among them).
//
//   request b: n = query_start_loc[b + 1] - query_start_loc[b] nodes in rows query_start_loc[b]
//   + i of q; context_lens[b] tokens with them, node j at position context_lens[b] - n + j.
//   Row i sees position p if p < context_lens[b] - n, or if bit p - (context_lens[b] - n) of its
//   mask is set. o = sum softmax(q k / sqrt d) v; zeros for a row that sees nothing.
//
// The G query heads of a kv head and the nodes make one matrix of n G rows, so a tree of 16
// nodes at G = 4 fills 64 rows and K and V are read once for all of them. Rows are worked in
// blocks of up to four wavefronts' tiles (kRows each). Up to kRows rows all four wavefronts take
// different chunks of the same rows, up to 2 kRows two by two, beyond that every wavefront has
// rows of its own and the same chunks as the others, at about the same time: what one asks of
// HBM the others find in L1 or L2.
//
// Work is cut without knowing the lengths on the host: the (request, row block) items of a kv
// head, laid end to end in units of their cost, are cut into `slots` equal ranges, one for each
// workgroup, which finds its own by a scan over the requests. An item that lies in one slot goes
// straight to the output; the pieces of one that is cut go to the workspace, and the workgroups
// of a second launch, one set for each slot in which a cut item begins, add them up.
#include <algorithm>

#include "kernels.hpp"
#include "row_tiles.hpp"

namespace ccinfer::hipk {
namespace {

using namespace rows;

constexpr int kThreads = kWaves * 64;
constexpr int kMaxRequests = kTreeMaxRequests;
constexpr int kPerThread = kMaxRequests / kThreads;
constexpr int kMergeSplit = 8;  // workgroups of the merge a slot: 16 of at most 128 rows each

// Two tiles of 16 rows a wavefront, one at head dims over 128 (two would need 320 registers).
template <int D>
constexpr int kTiles = D <= 128 ? 2 : 1;

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

template <class Ptr>
__device__ __forceinline__ Request request_of(Ptr qsl, Ptr ctx, int b, int total, int mbpr) {
    Request r;
    r.first = qsl[b];
    const int to = qsl[b + 1];
    const int c = ctx[b];
    r.n = to - r.first;
    r.before = c - r.n;
    r.nodes = min(to, total) - r.first;
    r.end = min(c, mbpr * kBlock);
    if (r.first < 0 || r.n <= 0 || r.before < 0 || r.nodes < 0) r.nodes = 0;
    return r;
}

// Units of all requests together stay below this (the host refuses other shapes).
constexpr int kMaxUnits = 1 << 30;

// Cost of a chunk for a block of this many rows. A block of one wavefront's rows reads as many
// bytes as one of four and computes a quarter.
template <int R>
__device__ __forceinline__ int chunk_units(int rows) {
    return rows <= R ? 2 : (rows <= 2 * R ? 3 : 4);
}

// Units of a request's row blocks.
template <int R>
__device__ __forceinline__ int request_units(const Request& r, int G) {
    if (r.nodes <= 0) return 0;
    const int rows = r.nodes * G;
    const int full = (rows - 1) / (4 * R);
    const int chunks = (r.end + kChunk - 1) / kChunk;
    return chunks * (4 * full + chunk_units<R>(rows - full * 4 * R));
}

template <int D, bool F8, bool Pad>
__global__ __launch_bounds__(kThreads, 2) void tree_attention_kernel(TreeArgs<D, F8, Pad> a) {
    constexpr int NT = kTiles<D>;
    constexpr int R = 16 * NT;
    __shared__ Parts<D, NT> parts;
    __shared__ int starts[kMaxRequests + 1];
    __shared__ int64_t wave_sum[kWaves];
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
        units[x] = x < per && b < a.batch
                       ? request_units<R>(request_of(a.qsl, a.ctx, b, a.total, a.mbpr), G)
                       : 0;
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
    for (int w = 0; w < kWaves; ++w) {
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
    SlotDesc own{0, 0, 0, 0};
    int b = first_request;
    for (int u = __builtin_amdgcn_readfirstlane(u0); u < u1;) {
        while (starts[b + 1] <= u) ++b;
        b = __builtin_amdgcn_readfirstlane(b);
        const Request req = request_of(unwritten(a.qsl), unwritten(a.ctx), b, a.total, a.mbpr);
        const int all_rows = req.nodes * G;
        const int chunks = (req.end + kChunk - 1) / kChunk;
        const int full = (all_rows - 1) / (4 * R);
        const int local = u - __builtin_amdgcn_readfirstlane(starts[b]);
        const int rb = min(local / (4 * chunks), full);
        const int row0 = rb * 4 * R;
        const int block_rows = min(all_rows - row0, 4 * R);
        const int weight = chunk_units<R>(block_rows);
        const int item = chunks * weight;
        const int from = local - rb * 4 * chunks;
        const int to = min(item, from + (u1 - u));
        // a chunk belongs to the slot that its first unit lies in
        const int c0 = (from + weight - 1) / weight, c1 = (to + weight - 1) / weight;
        const bool whole = from == 0 && to == item;
        const int which = from == 0 ? 1 : 0;  // piece of the slot: begins in it, or before it
        if (from == 0 && to < item)
            own = SlotDesc{req.first, row0, block_rows, (u - from + item - 1) / quota};

        // Wavefronts by rows, and those of the same rows by chunks.
        const int groups = block_rows <= R ? 1 : (block_rows <= 2 * R ? 2 : 4);
        const int share = kWaves / groups;
        const int group = wave % groups, part = wave / groups;
        State<D, NT> st;
        st.clear();
        const bool busy = group * R < block_rows;
        if (busy) {
            bf16x8 q[NT][Shape<D>::kSteps];
            const uint32_t* mask_row[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int row = group * R + 16 * t + (lane & 15);
                const bool live = row < block_rows;
                const int r = row0 + (live ? row : 0);
                const int node = r / G;
                const int64_t token = req.first + node;
                load_q<D, F8, Pad>(q[t], a.q + (token * a.hq + h * G + (r - node * G)) * dr, live,
                                   dr, lane);
                mask_row[t] = a.mask + token * a.words;
            }
            const auto table = unwritten(a.table) + static_cast<int64_t>(b) * a.mbpr;
            auto chunk = [&](int c) {
                const int cb = c * kChunk;
                const int pb0 = table[2 * c];
                const int pb1 = cb + kBlock < req.end ? table[2 * c + 1] : -1;
                return make_pair(pb0, req.end - cb, pb1, req.end - cb - kBlock);
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
                    bits = static_cast<uint32_t>(((static_cast<uint64_t>(hi) << 32) | lo) >>
                                                 (o & 31));
                }
                return true;
            };
            if (attend(st, q, a.cache, h, c0 + part, c1, share, a.scale_log2, lane,
                                  chunk, seen))
                add_unbounded(st, a.cache, h, c0 + part, c1, share, lane, chunk, seen);
        }

        const int64_t piece = (static_cast<int64_t>(h) * a.slots + slot) * 2 + which;
        float* pa = a.part_acc + piece * a.row_cap * D;
        float2* pm = a.part_ml + piece * a.row_cap;
        put_part<D, NT>(parts, st, wave, lane);
        __syncthreads();
        for (int row = wave; row < block_rows; row += kWaves) {
            float x[D / 64], m, l;
            sum_parts<D, NT>(parts, row % R, row / R, groups, share, lane, x, m, l);
            if (whole) {
                const int r = row0 + row;
                const int node = r / G;
                const int64_t token = req.first + node;
                store_bf16_row<D>(a.out + (token * a.hq + h * G + (r - node * G)) * dr, x,
                                  inverse_sum(l), dr, lane);
            } else {
#pragma unroll
                for (int y = 0; y < D / 64; ++y)
                    pa[static_cast<int64_t>(row) * D + lane * (D / 64) + y] = x[y];
                if (lane == 0) pm[row] = float2{m, l};
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
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(
    const SlotDesc* desc, const float* part_acc, const float2* part_ml, __bf16* out, int slots,
    int row_cap, int hq, int hkv, int dr) {
    constexpr int P = D / 64;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % hkv, slot = blockIdx.x / hkv;
    const int G = hq / hkv;
    const SlotDesc d = desc[static_cast<int64_t>(h) * slots + slot];
    const int64_t base = (static_cast<int64_t>(h) * slots + slot) * 2;
    for (int row = blockIdx.y * kWaves + wave; row < d.rows; row += kMergeSplit * kWaves) {
        float m = kNegInf, l = 0.f, x[P];
#pragma unroll
        for (int y = 0; y < P; ++y) x[y] = 0.f;
        for (int s = slot; s <= d.last_slot; ++s) {
            const int64_t at = (base + 2 * (s - slot) + (s == slot ? 1 : 0)) * row_cap + row;
            const float2 ml = part_ml[at];
            const float top = fmaxf(m, ml.x);
            const float use = top == kNegInf ? 0.f : top;
            const float f = __builtin_amdgcn_exp2f(m - use);
            const float fs = __builtin_amdgcn_exp2f(ml.x - use);
            l = l * f + ml.y * fs;
#pragma unroll
            for (int y = 0; y < P; ++y)
                x[y] = x[y] * f + part_acc[at * D + lane * P + y] * fs;
            m = top;
        }
        const int r = d.first_row + row;
        const int node = r / G;
        store_bf16_row<D>(
            out + ((static_cast<int64_t>(d.first_token) + node) * hq + h * G + (r - node * G)) * dr,
            x, inverse_sum(l), dr, lane);
    }
}

// Workgroups that the chip holds at once, two for each of 256 CUs.
constexpr int kResident = 512;
// Units of a slot at least: four chunks for a wavefront of a small block.
constexpr int kMinUnits = 32;

int slots_of(int hkv) { return std::max(1, kResident / hkv); }

int mfma_dim(int head_dim) { return head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256); }

int row_cap_of(int total, int hq, int hkv, int D) {
    const int wave_rows = D <= 128 ? 32 : 16;
    const int64_t rows = static_cast<int64_t>(total) * (hq / hkv);
    return static_cast<int>(std::min<int64_t>(rows, 4 * wave_rows));
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
    a.slots = slots_of(t.hkv);
    a.min_units = kMinUnits;
    a.row_cap = row_cap_of(t.total, t.hq, t.hkv, D);
    a.desc = reinterpret_cast<SlotDesc*>(ws + w.desc);
    a.part_ml = reinterpret_cast<float2*>(ws + w.ml);
    a.part_acc = reinterpret_cast<float*>(ws + w.acc);
    const unsigned grid = static_cast<unsigned>(a.slots) * t.hkv;
    hipLaunchKernelGGL((tree_attention_kernel<D, F8, Pad>), dim3(grid), dim3(kThreads), 0, stream, a);
    if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    hipLaunchKernelGGL((tree_merge_kernel<D>), dim3(grid, kMergeSplit), dim3(kThreads), 0, stream,
                       a.desc, a.part_acc, a.part_ml, a.out, a.slots, a.row_cap, t.hq, t.hkv,
                       t.head_dim);
    return hipGetLastError();
}

}  // namespace

bool tree_attention_supported(int batch, int total, int mbpr, int hq, int hkv, int head_dim,
                              bool fp8) {
    if (batch > kTreeMaxRequests || head_dim > 256 || head_dim % 8 != 0) return false;
    if (fp8 && head_dim != 64 && head_dim != 128) return false;
    // units: 4 a chunk and row block
    const int D = mfma_dim(head_dim);
    const int64_t block = D <= 128 ? 128 : 64;
    const int64_t blocks = static_cast<int64_t>(total) * (hq / hkv) / block + batch;
    const int64_t units = 4 * (static_cast<int64_t>(mbpr) / 2 + 1);
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
