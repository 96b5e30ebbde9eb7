// What a step of drafted tokens needs around its attention (tree_attn.hip): the trees' masks,
// positions and cache slots before it, and the confirmed path with its K and V after it.
//
// Both are chains of dependent reads over a few integers: latency. A workgroup stages its
// request's arrays in LDS once, so that every step of a walk is an LDS read. Plan of 26 nodes 2.4 us,
// of 192 requests of 4 to 64 nodes 4.2; acceptance of one request over 24 layers 4.9 (under a tracer,
// which adds to each). 96 requests with 34 MB of K and V to move: 16.8 us a call, 2.0 TB/s. Each of the
// 1152 workgroups walks before it moves, and their LDS (41 KB, for 2048 nodes) lets three run on a CU
// at once: they come in two rounds.
#include <algorithm>
#include <cstdint>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace ccinfer::hipk {
namespace {

constexpr int kThreads = 256;
constexpr int kInvalid = 6;  // the status of build_batch_metadata

// Mask of node i: the bits of its ancestors and its own; a thread walks up from its node and
// writes each word as it leaves it (parents come before their children, so words come in
// descending order). Position: committed tokens + depth. Slot: where position committed + i
// lies, since two nodes of one depth need a slot each.
__global__ __launch_bounds__(kThreads) void draft_tree_kernel(
    const int32_t* __restrict__ parents, const int32_t* __restrict__ qsl,
    const int32_t* __restrict__ ctx, const int32_t* __restrict__ table, int total, int mbpr,
    int words, int max_nodes, uint32_t* __restrict__ mask, int32_t* __restrict__ positions,
    int32_t* __restrict__ slots, int32_t* __restrict__ status) {
    __shared__ int16_t up[kTreeMaxNodes];
    const int b = blockIdx.x;
    const int first = qsl[b], n = qsl[b + 1] - first, c = ctx[b];
    const int before = c - n;
    const bool range_ok = first >= 0 && n >= 0 && first <= total - n;
    const bool ok = range_ok && c >= n && n <= max_nodes;  // (before may have passed 32 bits)
    // Rows [from, to) that are there get no mask, position or slot.
    auto leave_out = [&](int from, int to) {
        for (int64_t t = max(from, 0) + threadIdx.x; t < min(to, total); t += kThreads) {
            for (int w = 0; w < words; ++w) mask[t * words + w] = 0u;
            positions[t] = -1;
            slots[t] = -1;
        }
    };
    // Those of no request too: left as they were, a captured step's cache write would go to the
    // slots of an earlier replay with more nodes.
    if (range_ok && b == 0) leave_out(0, first);
    if (range_ok && b == static_cast<int>(gridDim.x) - 1) leave_out(first + n, total);
    if (!ok) {
        leave_out(first, qsl[b + 1]);  // (n may have passed 32 bits)
        if (threadIdx.x == 0) status[b] = kInvalid;
        return;
    }
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int p = parents[first + i];
        const bool good = p >= -1 && p < i;
        bad |= !good;
        up[i] = static_cast<int16_t>(good ? p : -1);
    }
    __syncthreads();
    const int32_t* row = table + static_cast<int64_t>(b) * mbpr;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int pos = before + i;
        int blk = pos / 16 < mbpr ? row[pos / 16] : -1;
        if (blk > INT32_MAX / 16) blk = -1;  // a slot past 32 bits would be another block's
        bad |= blk < 0;
        uint32_t* m = mask + static_cast<int64_t>(first + i) * words;
        int at = words - 1;
        uint32_t bits = 0;
        int depth = -1;
        for (int p = i; p >= 0; p = up[p]) {
            for (; at > (p >> 5); --at) {
                m[at] = bits;
                bits = 0;
            }
            bits |= 1u << (p & 31);
            ++depth;
        }
        for (; at >= 0; --at) {
            m[at] = bits;
            bits = 0;
        }
        positions[first + i] = before + depth;
        slots[first + i] = blk < 0 ? -1 : blk * 16 + pos % 16;
    }
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) status[b] = bad ? kInvalid : 0;
}

// A request's accepted path, found by every workgroup of the request for itself (a walk of a few
// LDS reads costs less than a second launch): from node 0, the lowest child whose drafted token
// is what the model says after the node. Then the workgroup's columns of all layers: node p_k's
// row goes to the slot of position committed + k. p_k >= k and p grows, so a destination is never
// a later node's source, and the rows of eight nodes are read before they are written: memory
// that two nodes share needs no other order.
template <typename T>
__global__ __launch_bounds__(kThreads) void accept_kernel(AcceptDrafts a, KvLayers kv, int parts) {
    __shared__ int16_t up[kTreeMaxNodes];
    __shared__ int32_t draft[kTreeMaxNodes];
    __shared__ int32_t target[kTreeMaxNodes];
    __shared__ int16_t path[kTreeMaxNodes];
    __shared__ int32_t moves_src[kTreeMaxNodes];
    __shared__ int32_t moves_dst[kTreeMaxNodes];
    __shared__ int count, moves;
    const int b = blockIdx.x / parts, part = blockIdx.x % parts;
    const int lane = threadIdx.x & 63;
    const int first = a.qsl[b], n = a.qsl[b + 1] - first, c = a.ctx[b];
    const int before = c - n;
    const bool range_ok = first >= 0 && n >= 0 && first <= a.total - n;
    // What the plan refused was not written to the cache, or not all of it: nothing of it is taken.
    const bool planned = a.status == nullptr || a.status[b] == 0;
    if (!planned || !range_ok || c < n || n <= 0 || n > kTreeMaxNodes) {
        if (part == 0) {
            const int from = max(first, 0);
            const int to = min(a.total, a.qsl[b + 1]);  // (n may have passed 32 bits)
            for (int t = from + static_cast<int>(threadIdx.x); t < to; t += kThreads) {
                a.nodes[t] = -1;
                a.tokens[t] = -1;
            }
            if (threadIdx.x == 0) {
                a.accepted[b] = 0;
                a.lengths[b] = !planned && range_ok && c >= n ? before : c;
            }
        }
        return;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int p = a.parents[first + i];
        up[i] = static_cast<int16_t>(p >= -1 && p < i ? p : -1);
        draft[i] = a.draft[first + i];
        target[i] = a.target[first + i];
    }
    __syncthreads();
    if (threadIdx.x < kWave) {
        int now = 0, k = 0;
        while (true) {
            if (lane == 0) path[k] = static_cast<int16_t>(now);
            ++k;
            const int said = target[now];
            int child = -1;
            for (int i0 = now + 1; i0 < n && child < 0; i0 += kWave) {
                const int i = i0 + lane;
                const bool good = i < n && up[i] == now && draft[i] == said;
                const uint64_t hit = __builtin_amdgcn_ballot_w64(good);
                if (hit != 0) child = i0 + __builtin_ctzll(hit);
            }
            if (child < 0) break;
            now = child;
        }
        if (lane == 0) count = k;
    }
    __syncthreads();
    const int taken = count;
    if (part == 0) {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int node = i < taken ? path[i] : -1;
            a.nodes[first + i] = node;
            a.tokens[first + i] = node >= 0 ? target[node] : -1;
        }
        if (threadIdx.x == 0) {
            a.accepted[b] = taken;
            a.lengths[b] = before + taken;
        }
    }
    if (kv.layers == 0) return;

    // The rows that move, in the order of the path.
    const int bs = kv.block_size;
    const int32_t* row = a.table + static_cast<int64_t>(b) * a.mbpr;
    auto slot_of = [&](int pos) {
        const int blk = pos / bs < a.mbpr ? row[pos / bs] : -1;
        return blk >= 0 && blk < kv.blocks ? blk * bs + pos % bs : -1;
    };
    if (threadIdx.x < kWave) {
        int at = 0;
        for (int k0 = 0; k0 < taken; k0 += kWave) {
            const int k = k0 + lane;
            int src = -1, dst = -1;
            if (k < taken && path[k] != k) {
                src = slot_of(before + path[k]);
                dst = slot_of(before + k);
            }
            const bool go = src >= 0 && dst >= 0;
            const uint64_t all = __builtin_amdgcn_ballot_w64(go);
            if (go) {
                const int x = at + __popcll(all & ((1ull << lane) - 1));
                moves_src[x] = src;
                moves_dst[x] = dst;
            }
            at += __popcll(all);
        }
        if (lane == 0) moves = at;
    }
    __syncthreads();
    const int n_moves = moves;
    if (n_moves == 0) return;
    const int pieces = static_cast<int>(kv.token_bytes / static_cast<int64_t>(sizeof(T)));
    const int64_t columns = static_cast<int64_t>(kv.layers) * 2 * pieces;
    for (int64_t x = static_cast<int64_t>(part) * kThreads + threadIdx.x; x < columns;
         x += static_cast<int64_t>(parts) * kThreads) {
        const int64_t of = x / pieces;
        char* base = (of & 1 ? kv.v : kv.k) + (of >> 1) * kv.layer_stride +
                     (x - of * pieces) * static_cast<int64_t>(sizeof(T));
        for (int k0 = 0; k0 < n_moves; k0 += 8) {
            T r[8];
#pragma unroll
            for (int y = 0; y < 8; ++y)
                r[y] = *reinterpret_cast<const T*>(
                    base + moves_src[min(k0 + y, n_moves - 1)] * kv.token_bytes);
#pragma unroll
            for (int y = 0; y < 8; ++y)
                if (k0 + y < n_moves)
                    *reinterpret_cast<T*>(base + moves_dst[k0 + y] * kv.token_bytes) = r[y];
        }
    }
    if (kv.k_scale == nullptr) return;
    const int64_t scale_columns = static_cast<int64_t>(kv.layers) * 2 * kv.heads;
    for (int64_t x = static_cast<int64_t>(part) * kThreads + threadIdx.x; x < scale_columns;
         x += static_cast<int64_t>(parts) * kThreads) {
        const int64_t of = x / kv.heads;
        const int64_t h = x - of * kv.heads;
        float* base = (of & 1 ? kv.v_scale : kv.k_scale) + (of >> 1) * kv.scale_layer_stride;
        auto at = [&](int slot) {
            return (static_cast<int64_t>(slot / kFp8Block) * kv.heads + h) * kFp8Block +
                   slot % kFp8Block;
        };
        for (int k0 = 0; k0 < n_moves; k0 += 8) {
            float r[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) r[y] = base[at(moves_src[min(k0 + y, n_moves - 1)])];
#pragma unroll
            for (int y = 0; y < 8; ++y)
                if (k0 + y < n_moves) base[at(moves_dst[k0 + y])] = r[y];
        }
    }
}

}  // namespace

hipError_t build_draft_tree(const int32_t* parents, const int32_t* qsl, const int32_t* ctx,
                            const int32_t* table, int batch, int total, int mbpr, int words,
                            int max_nodes, int32_t* mask, int32_t* positions, int32_t* slots,
                            int32_t* status, hipStream_t stream) {
    hipLaunchKernelGGL(draft_tree_kernel, dim3(batch), dim3(kThreads), 0, stream, parents, qsl, ctx,
                       table, total, mbpr, words, max_nodes, reinterpret_cast<uint32_t*>(mask),
                       positions, slots, status);
    return hipGetLastError();
}

hipError_t accept_draft_tokens(const AcceptDrafts& a, const KvLayers& kv, hipStream_t stream) {
    const bool wide = kv.token_bytes % 16 == 0 && kv.layer_stride % 16 == 0 &&
                      (reinterpret_cast<uintptr_t>(kv.k) | reinterpret_cast<uintptr_t>(kv.v)) % 16 == 0;
    const int64_t columns = kv.layers * 2 * (kv.token_bytes / (wide ? 16 : 1));
    // a column a thread, up to 2048 workgroups in all (three run on a CU at once, by their LDS)
    const int64_t most = std::max<int64_t>(1, 2048 / a.batch);
    const int parts = static_cast<int>(
        std::clamp<int64_t>((columns + kThreads - 1) / kThreads, 1, most));
    const dim3 grid(static_cast<unsigned>(a.batch) * parts);
    if (wide)
        hipLaunchKernelGGL(accept_kernel<u32x4>, grid, dim3(kThreads), 0, stream, a, kv, parts);
    else
        hipLaunchKernelGGL(accept_kernel<uint8_t>, grid, dim3(kThreads), 0, stream, a, kv, parts);
    return hipGetLastError();
}

}  // namespace ccinfer::hipk
