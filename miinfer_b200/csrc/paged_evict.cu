// Eviction from a paged cache by accumulated attention weight: which positions of a sequence stay, and their rows moved together.
//
// Of L > keep positions the first `sinks` and the last `recent` stay, and of the middle the k = keep - sinks - recent with the largest weights; each kv
// head chooses for itself.  Two kernels:
//
//  * paged_choose_kernel, a cluster of CTAs for a (sequence, kv head).  The k-th largest weight of the middle is found digit by digit (radix
//    selection): a weight becomes a 32-bit key that orders as the weights do, and four passes count the keys under the digits found so far by their next
//    eight bits, in shared memory, every CTA over its own stretch of positions, all counts together through distributed shared memory.  What is left is
//    the key T of the k-th largest and how many of the positions that share it stay, the lowest ones; a position's place among those that stay is
//    then a count over the ones before it (a scan over warps, CTAs, and the lanes' ballots).
//  * paged_move_kernel copies the rows.  With a table of its own for the target nothing can collide, and rows are spread over the device.  In place, row r
//    comes from a position >= r, so a cluster takes a (sequence, kv head, side) and moves the rows in rounds of what its threads hold in registers: all
//    of a round is read before any of it is written (a cluster barrier), and what a round writes no later round reads.
//
// The choice is bound by its chain of passes (the weights come from HBM once and from L2 or L1 after that), the copy by HBM.
#include "paged_common.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace b200kv {

namespace cg = cooperative_groups;

namespace {

constexpr int kChooseThreads = 512, kChooseWarps = kChooseThreads / 32;
constexpr uint32_t kMaxCluster = 8;

struct EvictParams {
    Paged pool;
    const int32_t* target_table;
    uint32_t target_max_pages;
    const float* weights;
    uint32_t weights_stride, keep, sinks, recent;
    int32_t* kept;
    float* new_weights;
    int32_t* new_lengths;
};

// Keys order as the weights do; a NaN is the least, and the two zeros are one.
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t u = __float_as_uint(w), magnitude = u & 0x7fffffffu;   // on the bits: arithmetic of this build flushes subnormal numbers
    if (magnitude > 0x7f800000u) return 0;
    return magnitude == 0 || u == magnitude ? magnitude | 0x80000000u : ~u;   // minus infinity: 0x007fffff
}

__global__ void __launch_bounds__(kChooseThreads) paged_choose_kernel(const __grid_constant__ EvictParams p) {
    __shared__ uint32_t counts[2][256];      // of a pass, two in turn: a CTA may still be read while its next pass counts
    __shared__ uint32_t sums[256];
    __shared__ uint32_t warp_above[kChooseWarps], warp_equal[kChooseWarps];
    __shared__ uint32_t totals[2];           // of this CTA's stretch: positions above the threshold, and at it
    __shared__ uint32_t found[2];            // a pass's digit, and how many of the chosen lie at or below it
    pdl_launch_dependents();
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks();
    const uint32_t s = blockIdx.y, head = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Span span = span_of(p.pool, s);
    const uint32_t H = p.pool.view.kv_heads, L = span.length, keep = p.keep;
    const float* weights = p.weights + (static_cast<size_t>(s) * H + head) * p.weights_stride;
    int32_t* kept = p.kept + (static_cast<size_t>(s) * H + head) * keep;
    float* new_weights = p.new_weights == nullptr ? nullptr : p.new_weights + (static_cast<size_t>(s) * H + head) * keep;
    if (head == 0 && rank == 0 && tid == 0) p.new_lengths[s] = static_cast<int32_t>(min(L, keep));
    const uint32_t step = ctas * kChooseThreads, me = rank * kChooseThreads + tid;
    if (L <= keep) {   // the whole cluster
        for (uint32_t r = me; r < keep; r += step) {
            kept[r] = r < L ? static_cast<int32_t>(r) : -1;
            if (new_weights != nullptr) new_weights[r] = r < L ? weights[r] : 0.0f;
        }
        return;
    }
    const uint32_t mid0 = p.sinks, mid1 = L - p.recent;
    uint32_t wanted = keep - p.sinks - p.recent;
    for (uint32_t r = me; r < p.sinks + p.recent; r += step) {   // what stays in any case
        const uint32_t j = r < p.sinks ? r : L - p.recent + (r - p.sinks), to = r < p.sinks ? r : keep - p.recent + (r - p.sinks);
        kept[to] = static_cast<int32_t>(j);
        if (new_weights != nullptr) new_weights[to] = weights[j];
    }
    if (wanted == 0) return;
    // this CTA's stretch of the middle, in whole warps
    const uint32_t share = ((mid1 - mid0 + ctas - 1) / ctas + 31) / 32 * 32;
    const uint32_t a = min(mid0 + rank * share, mid1), b = min(a + share, mid1);

    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        uint32_t* mine = counts[pass & 1];
        if (tid < 256) mine[tid] = 0;
        __syncthreads();
        for (uint32_t j = a + tid; j < b; j += kChooseThreads) {
            const uint32_t key = key_of(weights[j]);
            if (pass == 0 || (key >> (shift + 8)) == prefix) atomicAdd(&mine[(key >> shift) & 255u], 1u);
        }
        cluster.sync();
        if (tid < 256) {
            uint32_t n = 0;
            for (uint32_t c = 0; c < ctas; ++c) n += cluster.map_shared_rank(mine, c)[tid];
            sums[tid] = n;
        }
        __syncthreads();
        if (warp == 0) {   // lane l: digits 8l .. 8l + 7; the digit at which the count from the top reaches `wanted`
            uint32_t own = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) own += sums[8 * lane + i];
            uint32_t above = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_down_sync(0xffffffffu, above, o);
                if (lane + o < 32) above += v;
            }
            above -= own;      // keys in higher lanes' digits
            if (above < wanted && above + own >= wanted) {
                for (int i = 7; i >= 0; --i) {
                    const uint32_t n = sums[8 * lane + i];
                    if (above + n >= wanted) { found[0] = 8 * lane + i; found[1] = wanted - above; break; }
                    above += n;
                }
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | found[0];
        wanted = found[1];
    }
    // `prefix` is the key of the last that stays, `wanted` how many positions with that key do.

    // Places: a warp's positions lie in one piece, 32 at a time in order.
    const uint32_t piece = ((b - a + kChooseWarps - 1) / kChooseWarps + 31) / 32 * 32;
    const uint32_t w0 = min(a + warp * piece, b), w1 = min(w0 + piece, b);
    uint32_t above = 0, equal = 0;
    for (uint32_t j0 = w0; j0 < w1; j0 += 32) {
        const uint32_t key = j0 + lane < w1 ? key_of(weights[j0 + lane]) : 0;
        above += __popc(__ballot_sync(0xffffffffu, j0 + lane < w1 && key > prefix));
        equal += __popc(__ballot_sync(0xffffffffu, j0 + lane < w1 && key == prefix));
    }
    if (lane == 0) { warp_above[warp] = above; warp_equal[warp] = equal; }
    __syncthreads();
    if (tid == 0) {
        uint32_t ta = 0, te = 0;
        for (int w = 0; w < kChooseWarps; ++w) { ta += warp_above[w]; te += warp_equal[w]; }
        totals[0] = ta; totals[1] = te;
    }
    cluster.sync();
    uint32_t before_above = 0, before_equal = 0;
    for (uint32_t c = 0; c < rank; ++c) {
        const uint32_t* t = cluster.map_shared_rank(totals, c);
        before_above += t[0];
        before_equal += t[1];
    }
    for (uint32_t w = 0; w < warp; ++w) { before_above += warp_above[w]; before_equal += warp_equal[w]; }
    const uint32_t lower = (1u << lane) - 1;
    for (uint32_t j0 = w0; j0 < w1; j0 += 32) {
        const bool in = j0 + lane < w1;
        const float w = in ? weights[j0 + lane] : 0.0f;
        const uint32_t key = key_of(w);
        const uint32_t is_above = __ballot_sync(0xffffffffu, in && key > prefix), is_equal = __ballot_sync(0xffffffffu, in && key == prefix);
        const uint32_t rank_above = before_above + __popc(is_above & lower), rank_equal = before_equal + __popc(is_equal & lower);
        if (in && (key > prefix || (key == prefix && rank_equal < wanted))) {
            const uint32_t to = p.sinks + rank_above + min(rank_equal, wanted);
            kept[to] = static_cast<int32_t>(j0 + lane);
            if (new_weights != nullptr) new_weights[to] = w;
        }
        before_above += __popc(is_above);
        before_equal += __popc(is_equal);
    }
    cluster.sync();   // no CTA leaves while another may read its counts
}

// ---- the rows -----------------------------------------------------------------------------------------------------------

constexpr int kMoveThreads = 256;
constexpr int kHeld = 8;   // 16-byte pieces a thread has in flight

// One side's rows: pieces of 16 bytes of data, and the row's scales as one piece of 2, 8 or 16 bytes.
struct Side {
    uint8_t* data;
    uint8_t* scales;             // null for fp16
    uint32_t pieces;             // 16-byte pieces of a row
    uint32_t scale_bytes;
};
__device__ __forceinline__ Side side_of(const b200kv_paged_view& v, uint32_t side) {
    const bool q8 = side == 0 ? is_k_q8(v.quant_mode) : is_v_q8(v.quant_mode);
    Side x;
    x.data = q8 ? reinterpret_cast<uint8_t*>(side == 0 ? v.key_q8 : v.value_q8) : static_cast<uint8_t*>(side == 0 ? v.key_f16 : v.value_f16);
    x.scales = q8 ? static_cast<uint8_t*>(side == 0 ? v.key_scales : v.value_scales) : nullptr;
    x.pieces = v.head_dim * (q8 ? 1 : 2) / 16;
    x.scale_bytes = q8 ? v.head_dim / v.qblock * 2 : 0;
    return x;
}
__device__ __forceinline__ uint4 load_scales(const uint8_t* at, uint32_t bytes) {
    if (bytes == 16) return *reinterpret_cast<const uint4*>(at);
    if (bytes == 8) { const uint2 v = *reinterpret_cast<const uint2*>(at); return make_uint4(v.x, v.y, 0, 0); }
    return make_uint4(*reinterpret_cast<const uint16_t*>(at), 0, 0, 0);
}
__device__ __forceinline__ void store_scales(uint8_t* at, uint32_t bytes, const uint4& v) {
    if (bytes == 16) *reinterpret_cast<uint4*>(at) = v;
    else if (bytes == 8) *reinterpret_cast<uint2*>(at) = make_uint2(v.x, v.y);
    else *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(v.x);
}

// IN_PLACE: blockIdx.x is a CTA of the cluster of this (sequence, kv head, side).  Otherwise it takes its share of the rows alone.
template <bool IN_PLACE>
__global__ void __launch_bounds__(kMoveThreads) paged_move_kernel(const __grid_constant__ EvictParams p) {
    pdl_wait();   // the choice comes from the kernel just before
    pdl_launch_dependents();   // behind the wait: this kernel writes cache rows
    const uint32_t s = blockIdx.y, H = p.pool.view.kv_heads, head = blockIdx.z >> 1, side = blockIdx.z & 1;
    const Span span = span_of(p.pool, s);
    const uint32_t rows = min(span.length, p.keep);
    if (IN_PLACE && span.length <= p.keep) return;   // the whole cluster: every row is where it goes
    const Side x = side_of(p.pool.view, side);
    const int32_t* kept = p.kept + (static_cast<size_t>(s) * H + head) * p.keep;
    const int32_t* target = p.target_table + static_cast<size_t>(s) * p.target_max_pages;
    const uint32_t slot_mask = (1u << p.pool.page_shift) - 1;
    const uint32_t per_row = x.pieces + (x.scales != nullptr ? 1 : 0);   // the last piece of a row: its scales
    const uint32_t row_bytes = x.pieces * 16;
    // a thread's piece number n: row n / per_row, piece n % per_row
    uint4 v[kHeld];
    uint32_t to[kHeld], piece[kHeld];     // target row of the sequence; 0xffffffff where there is nothing to move
    auto fetch = [&](uint32_t first, uint32_t stride, uint32_t end) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint32_t n = first + i * stride;
            to[i] = 0xffffffffu;
            if (n >= end) continue;
            const uint32_t r = n / per_row;
            const int j = kept[r];
            if (j < 0 || static_cast<uint32_t>(j) >= span.length || (IN_PLACE && static_cast<uint32_t>(j) == r)) continue;
            const long long row = row_of(p.pool, s, head, static_cast<uint32_t>(j));
            to[i] = r;
            piece[i] = n % per_row;
            v[i] = make_uint4(0, 0, 0, 0);
            if (row < 0) continue;        // a page outside the pool reads as zeros
            if (piece[i] < x.pieces) v[i] = *reinterpret_cast<const uint4*>(x.data + static_cast<size_t>(row) * row_bytes + piece[i] * 16);
            else v[i] = load_scales(x.scales + static_cast<size_t>(row) * x.scale_bytes, x.scale_bytes);
        }
    };
    auto store = [&] {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            if (to[i] == 0xffffffffu) continue;
            const long long page = page_row(p.pool, target[to[i] >> p.pool.page_shift], head);
            if (page < 0) continue;
            const size_t row = static_cast<size_t>(page) + (to[i] & slot_mask);
            if (piece[i] < x.pieces) *reinterpret_cast<uint4*>(x.data + row * row_bytes + piece[i] * 16) = v[i];
            else store_scales(x.scales + row * x.scale_bytes, x.scale_bytes, v[i]);
        }
    };
    const uint64_t all = static_cast<uint64_t>(rows) * per_row;
    const uint64_t round = static_cast<uint64_t>(gridDim.x) * kMoveThreads * kHeld;
    if constexpr (IN_PLACE) {
        // Whole rows a round: a row that a later round still reads must not be written in this one.
        cg::cluster_group cluster = cg::this_cluster();
        const uint32_t rows_a_round = static_cast<uint32_t>(round / per_row);
        for (uint32_t r0 = 0; r0 < rows; r0 += rows_a_round) {
            const uint32_t end = min(r0 + rows_a_round, rows) * per_row;
            fetch(r0 * per_row + blockIdx.x * kMoveThreads + threadIdx.x, gridDim.x * kMoveThreads, end);
            cluster.sync();
            store();
        }
    } else {
        for (uint64_t n0 = static_cast<uint64_t>(blockIdx.x) * kMoveThreads * kHeld; n0 < all; n0 += round) {
            fetch(static_cast<uint32_t>(n0) + threadIdx.x, kMoveThreads, static_cast<uint32_t>(min(all, n0 + kMoveThreads * kHeld)));
            store();
        }
    }
}

cudaError_t launch_cluster(void (*kernel)(EvictParams), dim3 grid, uint32_t threads, uint32_t cluster, bool behind, cudaStream_t stream, const EvictParams& p) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = behind || launch_overlap_tail() > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_paged_evict(const b200kv_paged_view* view, const b200kv_paged_batch* batch, const int32_t* target_table, uint32_t target_max_pages,
                                  const float* weights, uint32_t weights_stride, uint32_t keep, uint32_t sinks, uint32_t recent, int32_t* kept,
                                  float* new_weights, int32_t* new_lengths, void* stream) {
    int rc = validate_paged(view, batch);
    if (rc != B200KV_OK) return rc;
    if (batch->sequences == 0) return B200KV_OK;
    const auto word = [](const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
    if (!word(target_table) || !word(weights) || !word(kept) || !word(new_lengths) || (new_weights != nullptr && !word(new_weights))) return B200KV_ERR_INVALID;
    if (keep == 0 || static_cast<uint64_t>(sinks) + recent > keep || new_lengths == batch->lengths) return B200KV_ERR_INVALID;
    if (weights_stride < batch->max_length) return B200KV_ERR_INVALID;
    if (keep > 0x7fffffffu / 40 || static_cast<uint64_t>(target_max_pages) * view->page_size < std::min(keep, batch->max_length)) return B200KV_ERR_RANGE;   // 33 pieces of a row at most
    if (view->kv_heads > 32767u) return B200KV_ERR_UNSUPPORTED;                                                                 // two grid rows a head
    const uint64_t heads = static_cast<uint64_t>(batch->sequences) * view->kv_heads;
    const uintptr_t w0 = reinterpret_cast<uintptr_t>(weights), w1 = w0 + heads * weights_stride * 4, n0 = reinterpret_cast<uintptr_t>(new_weights);
    if (new_weights != nullptr && n0 < w1 && w0 < n0 + heads * keep * 4) return B200KV_ERR_INVALID;
    if (target_table == batch->page_table && target_max_pages != batch->max_pages) return B200KV_ERR_INVALID;
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    const EvictParams p{paged_of(*view, *batch), target_table, target_max_pages, weights, weights_stride, keep, sinks, recent, kept, new_weights, new_lengths};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint32_t cluster = 1;
    while (cluster < kMaxCluster && static_cast<uint64_t>(batch->max_length) > static_cast<uint64_t>(cluster) * 4 * kChooseThreads) cluster *= 2;
    B200KV_CUDA_TRY(launch_cluster(paged_choose_kernel, dim3(cluster, batch->sequences, view->kv_heads), kChooseThreads, cluster, false, s, p));
    const uint64_t pieces = static_cast<uint64_t>(std::min(keep, batch->max_length)) * (view->head_dim / 8 + 1);
    const uint64_t blocks = std::max<uint64_t>(1, (pieces + kMoveThreads * kHeld - 1) / (kMoveThreads * kHeld));
    if (target_table == batch->page_table) {
        uint32_t wide = 1;
        while (wide < kMaxCluster && wide < blocks) wide *= 2;
        B200KV_CUDA_TRY(launch_cluster(paged_move_kernel<true>, dim3(wide, batch->sequences, 2 * view->kv_heads), kMoveThreads, wide, true, s, p));
    } else {
        const uint64_t most = std::max<uint64_t>(1, 16ull * device_sms() / (2 * heads));
        B200KV_CUDA_TRY(launch_behind(paged_move_kernel<false>, dim3(static_cast<uint32_t>(std::min(blocks, most)), batch->sequences, 2 * view->kv_heads),
                                      dim3(kMoveThreads), 0, s, p));
    }
    return B200KV_OK;
}
