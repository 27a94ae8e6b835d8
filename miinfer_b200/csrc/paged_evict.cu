// Eviction from a paged cache by accumulated attention weight: which positions of a sequence stay, and their rows moved together.
//
// Of L > keep positions the first `sinks` and the last `recent` stay, and of the middle the k = keep - sinks - recent with the largest weights; each kv
// head chooses for itself.  Two kernels:
//
//  * paged_choose_kernel, a CTA for a (sequence, kv head) of up to 16384 positions, a cluster of up to eight for more; a thread keeps its keys in registers
//    (beyond 131072 positions it makes them again).  The k-th largest weight of the middle is found digit by digit (radix selection): a weight becomes a 32-bit
//    key that orders as the weights do, and three passes count the keys under the digits found so far by their next eleven bits, in shared memory, every CTA
//    over its own stretch of positions, a cluster's counts together through distributed shared memory.  (Four passes of eight bits: weights share sign and
//    exponent, so a first digit without any of the mantissa has most of them wait for a handful of words; 8000 weights 12 us, 70000 21.)  What is left is the key T of the k-th largest and how many
//    of the positions that share it stay, the lowest ones; a position's place among those that stay is then a count over the ones before it (a
//    scan over warps, CTAs, and the lanes' ballots).
//  * paged_move_kernel copies the rows, a warp a few at a time: its lanes look up a row each, source and target, then all of the rows' pieces are under way
//    together.  With a table of its own for the target nothing can collide, and rows are spread over the device.  In place, row r comes from a
//    position >= r, so a cluster takes a (sequence, kv head, side) and moves the rows in rounds: all of a round is read before any of it is written (a
//    cluster barrier), and what a round writes no later round reads.
//
// The choice is bound by its chain of passes, the copy by HBM and the chain of its lookups.
#include "paged_common.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace b200kv {

namespace cg = cooperative_groups;

namespace {

constexpr int kChooseThreads = 1024, kChooseWarps = kChooseThreads / 32;
constexpr uint32_t kMaxCluster = 8;
constexpr int kKept = 16;            // keys of a thread in registers
constexpr uint32_t kDigits = 2048;   // of a pass

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

// CACHED: a thread has no more than kKept keys.
template <bool CACHED>
__global__ void __launch_bounds__(kChooseThreads) paged_choose_kernel(const __grid_constant__ EvictParams p) {
    __shared__ uint32_t counts[2][kDigits];  // of a pass, two in turn: a CTA may still be read while its next pass counts
    __shared__ uint32_t warp_sums[kChooseWarps];
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
    // this CTA's stretch of the middle, and this warp's piece of it, 32 positions at a time
    const uint32_t share = ((mid1 - mid0 + ctas - 1) / ctas + 31) / 32 * 32;
    const uint32_t a = min(mid0 + rank * share, mid1), b = min(a + share, mid1);
    const uint32_t piece = ((b - a + kChooseWarps - 1) / kChooseWarps + 31) / 32 * 32;
    const uint32_t w0 = min(a + warp * piece, b), w1 = min(w0 + piece, b);
    uint32_t mine[CACHED ? kKept : 1];
    if constexpr (CACHED) {
        float w[kKept];
#pragma unroll
        for (int i = 0; i < kKept; ++i) w[i] = w0 + 32 * i + lane < w1 ? weights[w0 + 32 * i + lane] : 0.0f;
#pragma unroll
        for (int i = 0; i < kKept; ++i) mine[i] = key_of(w[i]);
    }
    // f(position, key, whether there is one) for this lane's positions, in order; the whole warp
    auto each = [&](auto f) {
        if constexpr (CACHED) {
#pragma unroll
            for (int i = 0; i < kKept; ++i) {
                const uint32_t j = w0 + 32 * i;
                if (j < w1) f(j + lane, mine[i], j + lane < w1);
            }
        } else {
#pragma unroll 4
            for (uint32_t j = w0; j < w1; j += 32) f(j + lane, j + lane < w1 ? key_of(weights[j + lane]) : 0u, j + lane < w1);
        }
    };
    for (uint32_t r = me; r < p.sinks + p.recent; r += step) {   // what stays in any case
        const uint32_t j = r < p.sinks ? r : L - p.recent + (r - p.sinks), to = r < p.sinks ? r : keep - p.recent + (r - p.sinks);
        kept[to] = static_cast<int32_t>(j);
        if (new_weights != nullptr) new_weights[to] = weights[j];
    }
    if (wanted == 0) return;

    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, above_bits = pass == 0 ? 0 : pass == 1 ? 21 : 10;   // 11, 11 and 10 bits
        uint32_t* own = counts[pass & 1];
        for (uint32_t i = tid; i < kDigits / 4; i += kChooseThreads) reinterpret_cast<uint4*>(own)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const uint32_t mask = pass == 2 ? 1023u : 2047u;
        if (pass == 0) {
            each([&](uint32_t, uint32_t key, bool there) {
                if (there) atomicAdd(&own[key >> 21], 1u);
            });
        } else {
            each([&](uint32_t, uint32_t key, bool there) {
                if (there && (key >> above_bits) == prefix) atomicAdd(&own[(key >> shift) & mask], 1u);
            });
        }
        if (ctas > 1) cluster.sync();
        else __syncthreads();
        // a thread's two digits, from the top: how many keys have them, and how many a higher one
        const uint32_t top = kDigits - 2 - 2 * tid;
        uint2 n = make_uint2(0, 0);
        if (ctas > 1) {
#pragma unroll
            for (uint32_t c = 0; c < kMaxCluster; ++c) {
                if (c >= ctas) break;
                const uint2 v = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(own, c) + top);
                n.x += v.x;
                n.y += v.y;
            }
        } else {
            n = *reinterpret_cast<const uint2*>(own + top);
        }
        uint32_t inc = n.x + n.y;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) warp_sums[warp] = inc;
        __syncthreads();
        const uint32_t higher = __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0u) + inc - n.x - n.y;
        if (higher < wanted && higher + n.x + n.y >= wanted) {
            const bool upper = higher + n.y >= wanted;
            found[0] = top + (upper ? 1 : 0);
            found[1] = wanted - higher - (upper ? 0 : n.y);
        }
        __syncthreads();
        prefix = pass == 0 ? found[0] : pass == 1 ? prefix << 11 | found[0] : prefix << 10 | found[0];
        wanted = found[1];
    }
    // `prefix` is the key of the last that stays, `wanted` how many positions with that key do.

    uint32_t above = 0, equal = 0;
    each([&](uint32_t, uint32_t key, bool there) {
        above += __popc(__ballot_sync(0xffffffffu, there && key > prefix));
        equal += __popc(__ballot_sync(0xffffffffu, there && key == prefix));
    });
    if (lane == 0) { warp_above[warp] = above; warp_equal[warp] = equal; }
    __syncthreads();
    // what lies before this warp's piece: in the CTA's other pieces, and in the stretches of the CTAs before
    uint32_t x = warp_above[lane], y = warp_equal[lane];
    static_assert(kChooseWarps == 32);
    if (ctas > 1 && warp == 0) {
        const uint32_t tx = __reduce_add_sync(0xffffffffu, x), ty = __reduce_add_sync(0xffffffffu, y);
        if (lane == 0) { totals[0] = tx; totals[1] = ty; }
    }
    uint32_t before_above = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0), before_equal = __reduce_add_sync(0xffffffffu, lane < warp ? y : 0);
    if (ctas > 1) {
        cluster.sync();
        for (uint32_t c = 0; c < rank; ++c) {
            const uint32_t* t = cluster.map_shared_rank(totals, c);
            before_above += t[0];
            before_equal += t[1];
        }
    }
    const uint32_t lower = (1u << lane) - 1;
    each([&](uint32_t j, uint32_t key, bool there) {
        const uint32_t is_above = __ballot_sync(0xffffffffu, there && key > prefix), is_equal = __ballot_sync(0xffffffffu, there && key == prefix);
        const uint32_t rank_above = before_above + __popc(is_above & lower), rank_equal = before_equal + __popc(is_equal & lower);
        if (there && (key > prefix || (key == prefix && rank_equal < wanted))) {
            const uint32_t to = p.sinks + rank_above + min(rank_equal, wanted);
            kept[to] = static_cast<int32_t>(j);
            if (new_weights != nullptr) new_weights[to] = weights[j];
        }
        before_above += __popc(is_above);
        before_equal += __popc(is_equal);
    });
    if (ctas > 1) cluster.sync();   // no CTA leaves while another may read its counts
}

// ---- the rows -----------------------------------------------------------------------------------------------------------

constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32;
constexpr int kHeld = 8;   // 16-byte pieces a thread has in flight

// One side's rows: 16-byte pieces of data, and the row's scales of 2, 8 or 16 bytes.
struct Side {
    uint8_t* data;
    uint8_t* scales;             // null for fp16
    uint32_t pieces;             // 16-byte pieces of a row: 8, 16 or 32
    uint32_t scale_bytes;
};
__host__ __device__ inline uint32_t pieces_of_side(const b200kv_paged_view& v, uint32_t side) { return v.head_dim * ((side == 0 ? is_k_q8(v.quant_mode) : is_v_q8(v.quant_mode)) ? 1 : 2) / 16; }
__device__ __forceinline__ Side side_of(const b200kv_paged_view& v, uint32_t side) {
    const bool q8 = side == 0 ? is_k_q8(v.quant_mode) : is_v_q8(v.quant_mode);
    Side x;
    x.data = q8 ? reinterpret_cast<uint8_t*>(side == 0 ? v.key_q8 : v.value_q8) : static_cast<uint8_t*>(side == 0 ? v.key_f16 : v.value_f16);
    x.scales = q8 ? static_cast<uint8_t*>(side == 0 ? v.key_scales : v.value_scales) : nullptr;
    x.pieces = pieces_of_side(v, side);
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
    const uint32_t s = blockIdx.y, H = p.pool.view.kv_heads, head = blockIdx.z >> 1, side = blockIdx.z & 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Span span = span_of(p.pool, s);
    const uint32_t rows = min(span.length, p.keep);
    if (IN_PLACE && span.length <= p.keep) return;   // the whole cluster: every row is where it goes
    const Side x = side_of(p.pool.view, side);
    const int32_t* kept = p.kept + (static_cast<size_t>(s) * H + head) * p.keep;
    const int32_t* source = pages_of(p.pool, s);
    const int32_t* target = p.target_table + static_cast<size_t>(s) * p.target_max_pages;
    const uint32_t slot_mask = (1u << p.pool.page_shift) - 1, row_bytes = x.pieces * 16;
    const uint32_t batch = 32 * kHeld / x.pieces, per_step = 32 / x.pieces == 0 ? 1 : 32 / x.pieces;   // rows of a warp at a time; of one of its steps
    const uint32_t sub = lane / x.pieces, piece = lane % x.pieces;
    // lane l < batch: row r0 + l, where it comes from (-1: of no page, zeros) and where it goes (-1: nowhere)
    long long from = -1, to = -1;
    uint4 v[kHeld], sc = make_uint4(0, 0, 0, 0);
    auto fetch = [&](uint32_t r0) {
        from = to = -1;
        const uint32_t r = r0 + lane;
        if (lane < batch && r < rows) {
            const int j = kept[r];
            const int there = target[r >> p.pool.page_shift];
            if (j >= 0 && static_cast<uint32_t>(j) < span.length && !(IN_PLACE && static_cast<uint32_t>(j) == r)) {
                from = page_row(p.pool, source[static_cast<uint32_t>(j) >> p.pool.page_shift], head);
                if (from >= 0) from += static_cast<uint32_t>(j) & slot_mask;
                to = page_row(p.pool, there, head);
                if (to >= 0) to += r & slot_mask;
            }
        }
        sc = make_uint4(0, 0, 0, 0);
        if (x.scales != nullptr && from >= 0) sc = load_scales(x.scales + static_cast<size_t>(from) * x.scale_bytes, x.scale_bytes);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const long long row = __shfl_sync(0xffffffffu, from, i * per_step + sub);
            v[i] = make_uint4(0, 0, 0, 0);
            if (row >= 0) v[i] = *reinterpret_cast<const uint4*>(x.data + static_cast<size_t>(row) * row_bytes + piece * 16);
        }
    };
    auto store = [&] {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const long long row = __shfl_sync(0xffffffffu, to, i * per_step + sub);
            if (row >= 0) *reinterpret_cast<uint4*>(x.data + static_cast<size_t>(row) * row_bytes + piece * 16) = v[i];
        }
        if (x.scales != nullptr && to >= 0) store_scales(x.scales + static_cast<size_t>(to) * x.scale_bytes, x.scale_bytes, sc);
    };
    const uint32_t round = gridDim.x * kMoveWarps * batch, first = (blockIdx.x * kMoveWarps + warp) * batch;
    for (uint64_t r0 = 0; r0 < rows; r0 += round) {
        const uint64_t mine = r0 + first;
        fetch(static_cast<uint32_t>(min(mine, static_cast<uint64_t>(rows))));
        if constexpr (IN_PLACE) cg::this_cluster().sync();   // a row that this round still reads must not be written yet
        store();
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
    if (keep == 0 || static_cast<uint64_t>(sinks) + recent > keep) return B200KV_ERR_INVALID;
    if (weights_stride < batch->max_length) return B200KV_ERR_INVALID;
    if (keep > 0x7fffffffu / 40 || static_cast<uint64_t>(target_max_pages) * view->page_size < std::min(keep, batch->max_length)) return B200KV_ERR_RANGE;
    if (view->kv_heads > 32767u) return B200KV_ERR_UNSUPPORTED;                                                                 // two grid rows a head
    const uint64_t heads = static_cast<uint64_t>(batch->sequences) * view->kv_heads;
    if (new_weights != nullptr && share(new_weights, heads * keep * 4, weights, heads * weights_stride * 4)) return B200KV_ERR_INVALID;
    const uint64_t S = batch->sequences;   // what one CTA writes of these, another may not have read yet
    const auto over_the_batch = [&](const void* out, uint64_t bytes) {
        return share(out, bytes, batch->lengths, S * 4) || share(out, bytes, batch->query_starts, (S + 1) * 4) || share(out, bytes, batch->page_table, S * batch->max_pages * 4) ||
               share(out, bytes, target_table, S * target_max_pages * 4);
    };
    if (over_the_batch(kept, heads * keep * 4) || over_the_batch(new_lengths, S * 4) || (new_weights != nullptr && over_the_batch(new_weights, heads * keep * 4))) return B200KV_ERR_INVALID;
    if (target_table == batch->page_table && target_max_pages != batch->max_pages) return B200KV_ERR_INVALID;
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    const EvictParams p{paged_of(*view, *batch), target_table, target_max_pages, weights, weights_stride, keep, sinks, recent, kept, new_weights, new_lengths};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint32_t cluster = 1;
    constexpr uint64_t kOfCta = static_cast<uint64_t>(kChooseThreads) * kKept;
    while (cluster < kMaxCluster && batch->max_length > cluster * kOfCta) cluster *= 2;
    // (a stretch is rounded up to whole warps, so a little less than all registers hold)
    const bool cached = batch->max_length <= cluster * (kOfCta - kChooseThreads);
    B200KV_CUDA_TRY(launch_cluster(cached ? paged_choose_kernel<true> : paged_choose_kernel<false>, dim3(cluster, batch->sequences, view->kv_heads), kChooseThreads, cluster, false, s, p));
    const uint32_t rows = std::min(keep, batch->max_length), batch_rows = 32 * kHeld / std::max(pieces_of_side(*view, 0), pieces_of_side(*view, 1));
    const uint32_t blocks = std::max<uint32_t>(1, (rows + kMoveWarps * batch_rows - 1) / (kMoveWarps * batch_rows));
    if (target_table == batch->page_table) {
        uint32_t wide = 1;
        while (wide < kMaxCluster && wide < blocks) wide *= 2;
        B200KV_CUDA_TRY(launch_cluster(paged_move_kernel<true>, dim3(wide, batch->sequences, 2 * view->kv_heads), kMoveThreads, wide, true, s, p));
    } else {
        const uint64_t most = std::max<uint64_t>(1, 16ull * device_sms() / (2 * heads));
        B200KV_CUDA_TRY(launch_behind(paged_move_kernel<false>, dim3(static_cast<uint32_t>(std::min<uint64_t>(blocks, most)), batch->sequences, 2 * view->kv_heads),
                                      dim3(kMoveThreads), 0, s, p));
    }
    return B200KV_OK;
}
