// Decode attention over selected blocks of the context: each (request, kv head) has a list of
// blocks of its own (kv_select.hip makes one), and the request's newest token attends to the
// positions below its context length that lie in them.
//
// A workgroup takes a (request, kv head) and 16 of its query heads, or a part of its list: the
// wavefronts take chunks of two blocks in turn and are added up in LDS; parts go to the workspace
// and a second launch adds them. Lists have a length that the host knows, so the parts are cut
// there. The ids of a wavefront's blocks lie in its lanes, one each, found by one read of the list
// and one of the table before the first chunk. Bound by the reads: 48 rows of 128 blocks, fp8, 32
// / 8 heads of 128 (203 MB) 45.4 us, 4.5 TB/s, and 4.7 for the merge; one row of 160 blocks, bf16,
// 16 / 8 heads 6.6 and 2.8: start, two dependent reads of ids, one or two chunks a wavefront.
#include <algorithm>
#include <cmath>

#include "kernels.hpp"
#include "row_tiles.hpp"

namespace ccinfer::hipk {
namespace {

using namespace rows;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTile = 16;  // query heads of a workgroup

template <int D, bool F8, bool Pad>
struct SparseArgs {
    const __bf16* q;
    Cache<D, F8, Pad> cache;
    const int32_t* table;
    const int32_t* ctx;
    const int32_t* selected;
    __bf16* out;
    int mbpr, hq, take, splits, tiles;
    float scale_log2;
    float* part_acc;  // [batch][kv heads][tiles][splits][16][D]
    float2* part_ml;
};

// The context of a decode row, 0 where the table row is too short for it (decode's rule).
__device__ __forceinline__ int decode_ctx(int c, int mbpr) {
    return c > 0 && (static_cast<int64_t>(c) + kBlock - 1) / kBlock <= mbpr ? c : 0;
}

template <int D, bool F8, bool Pad>
__global__ __launch_bounds__(kThreads, D <= 128 ? 3 : 1) void sparse_decode_kernel(SparseArgs<D, F8, Pad> a) {
    __shared__ Exchange<D, 1, kWaves> sums;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hkv = a.cache.hkv, dr = a.cache.dims();
    const int G = a.hq / hkv;
    const int split = blockIdx.x % a.splits;
    const int item = blockIdx.x / a.splits;  // ((b * hkv) + h) * tiles + tile
    const int tile = item % a.tiles;
    const int bh = item / a.tiles;
    const int h = bh % hkv, b = bh / hkv;
    const int heads = min(G - tile * kTile, kTile);
    const int head0 = h * G + tile * kTile;
    const int ctx = decode_ctx(a.ctx[b], a.mbpr);

    // Chunks of this wavefront: first, first + stride, ...; lane 2 k + x has block x of the k-th.
    const int chunks = (a.take + 1) / 2;
    const int first = split * kWaves + wave, stride = a.splits * kWaves;
    const int entry = 2 * (first + (lane >> 1) * stride) + (lane & 1);
    int block = -1, lim = 0;
    if (entry < a.take) {
        const int j = a.selected[static_cast<int64_t>(bh) * a.take + entry];
        if (j >= 0 && static_cast<int64_t>(j) * kBlock < ctx) {
            block = a.table[static_cast<int64_t>(b) * a.mbpr + j];
            lim = ctx - j * kBlock;
        }
    }
    State<D, 1> st;
    st.clear();
    bf16x8 q[1][Shape<D>::kSteps];
    const int row = lane & 15;
    load_q<D, F8, Pad>(q[0],
                       a.q + (static_cast<int64_t>(b) * a.hq + head0 + min(row, heads - 1)) * dr,
                       row < heads, dr, lane);
    int k = 0;
    const int last_k = 2 * ((chunks - 1 - first) / stride);
    auto next = [&] {
        const Pair p = make_pair(__builtin_amdgcn_readlane(block, k), __builtin_amdgcn_readlane(lim, k),
                                 __builtin_amdgcn_readlane(block, k + 1),
                                 __builtin_amdgcn_readlane(lim, k + 1));
        k = min(k + 2, last_k);
        return p;
    };
    attend(st, q, a.cache, h, first, chunks, stride, a.scale_log2, lane, next);
    add_parts(sums, st, wave, kWaves, 0, 1, lane);
    if (wave != 0) return;
    const float l = wave_sum_xor16_32(st.l[0]);
    if (row >= heads) return;
    if (a.splits == 1) {
        store_row<D, Pad>(st, 0, l, a.out + (static_cast<int64_t>(b) * a.hq + head0 + row) * dr,
                             dr, lane);
    } else {
        const int64_t at = static_cast<int64_t>(blockIdx.x) * kTile + row;
        store_part(st, 0, a.part_acc + at * D, lane);
        if (lane < 16) a.part_ml[at] = float2{st.m[0], l};
    }
}

// A wavefront a row of the output.
template <int D>
__global__ __launch_bounds__(kThreads) void sparse_merge_kernel(const float* part_acc,
                                                                const float2* part_ml, __bf16* out,
                                                                int64_t rows, int hq, int hkv,
                                                                int splits, int tiles, int dr) {
    const int lane = threadIdx.x & 63;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves +
                        __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= rows) return;
    const int64_t b = row / hq;
    const int head = static_cast<int>(row - b * hq);
    const int G = hq / hkv;
    const int h = head / G, g = head - h * G;
    const int64_t item = (b * hkv + h) * tiles + g / kTile;
    float x[D / 64];
    const float l = merge_row<D>(x, splits, part_acc, part_ml, lane, [&](int s) {
        return (item * splits + s) * kTile + g % kTile;
    });
    store_columns<D>(out + row * dr, x, inverse_sum(l), dr, lane);
}

// Workgroups that keep the chip busy, and chunks a wavefront at least where a list is cut (a part
// costs a merge's launch and its rows through memory).
constexpr int kBusy = 512;
constexpr int kMinChunks = 2;
constexpr int kMaxChunks = 32;  // of a wavefront: their blocks lie in its lanes

int splits_of(int batch, int hq, int hkv, int take) {
    const int64_t tiles = (hq / hkv + kTile - 1) / kTile;
    const int64_t items = static_cast<int64_t>(batch) * hkv * tiles;
    const int64_t chunks = (static_cast<int64_t>(take) + 1) / 2;
    const int64_t least = (chunks + kWaves * kMaxChunks - 1) / (kWaves * kMaxChunks);
    const int64_t most = std::max<int64_t>(1, chunks / (kWaves * kMinChunks));
    return static_cast<int>(std::max(least, std::min(most, (kBusy + items - 1) / items)));
}

int mfma_dim(int head_dim) { return head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256); }

int64_t part_rows(int batch, int hq, int hkv, int take) {
    const int64_t tiles = (hq / hkv + kTile - 1) / kTile;
    return static_cast<int64_t>(batch) * hkv * tiles * splits_of(batch, hq, hkv, take) * kTile;
}

template <int D, bool F8, bool Pad>
hipError_t launch(const SparseDecode& s, void* workspace, hipStream_t stream) {
    SparseArgs<D, F8, Pad> a;
    a.q = static_cast<const __bf16*>(s.q);
    using Elem = std::conditional_t<F8, uint8_t, __bf16>;
    a.cache = {static_cast<const Elem*>(s.k), static_cast<const Elem*>(s.v), s.k_scale, s.v_scale,
               s.hkv, s.head_dim};
    a.table = s.table;
    a.ctx = s.ctx;
    a.selected = s.selected;
    a.out = static_cast<__bf16*>(s.out);
    a.mbpr = s.mbpr;
    a.hq = s.hq;
    a.take = s.take;
    a.splits = splits_of(s.batch, s.hq, s.hkv, s.take);
    a.tiles = (s.hq / s.hkv + kTile - 1) / kTile;
    a.scale_log2 = kLog2e / sqrtf(static_cast<float>(s.head_dim));
    a.part_ml = nullptr;
    a.part_acc = nullptr;
    if (a.splits > 1) {
        const int64_t rows = part_rows(s.batch, s.hq, s.hkv, s.take);
        a.part_acc = static_cast<float*>(workspace);
        a.part_ml = reinterpret_cast<float2*>(a.part_acc + rows * D);
    }
    const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(s.batch) * s.hkv * a.tiles *
                                                a.splits);
    hipLaunchKernelGGL((sparse_decode_kernel<D, F8, Pad>), dim3(grid), dim3(kThreads), 0, stream, a);
    if (const hipError_t err = hipGetLastError(); err != hipSuccess || a.splits == 1) return err;
    const int64_t rows = static_cast<int64_t>(s.batch) * s.hq;
    hipLaunchKernelGGL((sparse_merge_kernel<D>),
                       dim3(static_cast<unsigned>((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0,
                       stream, a.part_acc, a.part_ml, a.out, rows, s.hq, s.hkv, a.splits, a.tiles,
                       s.head_dim);
    return hipGetLastError();
}

}  // namespace

size_t sparse_decode_workspace_bytes(int batch, int hq, int hkv, int head_dim, int take) {
    if (splits_of(batch, hq, hkv, take) == 1) return 0;
    return static_cast<size_t>(part_rows(batch, hq, hkv, take)) *
           (mfma_dim(head_dim) * sizeof(float) + sizeof(float2));
}

hipError_t sparse_decode(const SparseDecode& s, void* workspace, hipStream_t stream) {
    const bool fp8 = s.k_scale != nullptr;
    const int d = s.head_dim;
    switch (mfma_dim(d)) {
        case 64:
            return fp8 ? launch<64, true, false>(s, workspace, stream)
                   : d == 64 ? launch<64, false, false>(s, workspace, stream)
                             : launch<64, false, true>(s, workspace, stream);
        case 128:
            return fp8 ? launch<128, true, false>(s, workspace, stream)
                   : d == 128 ? launch<128, false, false>(s, workspace, stream)
                              : launch<128, false, true>(s, workspace, stream);
        default:
            return d == 256 ? launch<256, false, false>(s, workspace, stream)
                            : launch<256, false, true>(s, workspace, stream);
    }
}

}  // namespace ccinfer::hipk
