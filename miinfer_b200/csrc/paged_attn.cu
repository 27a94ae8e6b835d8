// Attention of a ragged batch of new tokens over a paged cache: what a call launches, and the kernels around the chunk kernel (prefill_tc5.cu).
//
//   o_i = sum_j exp(s_ij - lse_i) v_j,  s_ij = scale q_i.k_j,  lse_i = log sum_j exp s_ij,  j over what token i sees: j <= i, and under a window of w positions
//   only j > i - w and the first sinks.
//
// Sequences of a few query rows take the streaming kernel (paged_decode.cu), the others the chunk kernel; a call launches what its bounds allow, and the
// kernels find their sequences.
//
// The host knows bounds, the device the lengths, so a call over chunks begins with paged_prepare_kernel: one block lays out the work (which rows and tiles each
// CTA of the chunk kernel takes, how many of them share a row tile) while the others gather the visible rows into an fp16 copy, tile by tile
// as the chunk kernel's TMA reads them (int8 rows dequantised, rows that nobody sees zero).  (As a kernel of its own ahead of the gather the layout was 12 us of
// a call: a chain of latencies.)  The chunk kernel follows, and the merge of what its CTAs left for shared row tiles, each launched while the one before
// still runs.
//
// Measured, us, prepare / chunk kernel / merge: 512 new tokens over 8192, 24 / 4 heads of 256, q8_0: 131 to 135 in all (9 / 115 / 6); two chunks of 333 over up to 5000 beside
// 14 single tokens, 32 / 8 heads of 128, q8_0: 132 (10 / 77 / 6, the tokens' kernel 35); 2048 over 6001 under a window of 1024, fp16: 82 (a CTA has 18 tiles of
// 0.5 and 7 of set-up, Q and output).
#include "decode_common.cuh"
#include "dequant.cuh"
#include "paged_decode.cuh"
#include "paged_plan.cuh"

#include <algorithm>
#include <cmath>
#include <utility>

namespace b200kv {

namespace {

constexpr uint32_t kCandidates = 31;       // sizes of a piece that the layout chooses from: the smallest an eleventh of a row tile
constexpr int kPrepareThreads = 256;

// Estimated costs of the chunk kernel, us, as the single-sequence launch's (pick_kv_splits): a tile, a CTA's set-up and output, a merge, a partial.
// Of the plain instances; scored ones, whose tiles take up to a third longer (past a cap, twice as long), are split by the same.
struct ChunkCosts { float tile, cta, last_wave, merge, part; };   // last_wave: of a wave, where it is not full

struct PrepareParams {
    Paged pool;
    ChunkPlan* plan;
    ChunkItem* items;
    uint32_t* groups;           // first item of each shared row tile
    uint32_t max_items, max_parts, scratch_tiles;
    uint32_t group, window, sinks, sms;
    uint32_t few_rows;          // sequences of at most so many query rows are the other kernel's
    ChunkCosts costs;
    __half* out[2];             // the copy, K and V: [kv_head][scratch_tiles * kChunkTile][D]
    // tokens with ranges of their own: of every row tile (chunk_slot) its walk {tiles, skip}, of every sequence of the chunk kernel's {lowest position seen, the sinks aside, one
    // behind the last}
    const int32_t* ranges;
    uint2* tile_bounds;
    uint2* bounds;
    uint2* walks;               // the same as tile_bounds, in the list's order
    uint32_t max_walks;         // room of each of the two
    __device__ __forceinline__ bool mine(const Span& span) const { return span.tokens > 0 && static_cast<uint64_t>(span.tokens) * group > few_rows; }
    __device__ __forceinline__ uint32_t row_tiles(const Span& span) const { return (span.tokens * group + kChunkRows - 1) / kChunkRows; }
};

// Where a sequence's tiles lie.
template <bool RANGED>
__device__ __forceinline__ ChunkTiles tiles_of(const PrepareParams& p, const Span& span, uint32_t s) {
    if constexpr (RANGED) {
        const uint2 b = p.bounds[s];
        return chunk_tiles_between(b.x, b.y, p.sinks);
    } else {
        return chunk_tiles(span.base(), span.length, p.window, p.sinks);
    }
}

struct Sums { uint32_t a, b, c; };
__device__ __forceinline__ Sums add(const Sums& x, const Sums& y) { return {x.a + y.a, x.b + y.b, x.c + y.c}; }
// Exclusive sums over the block's threads in order, and the total.
__device__ __forceinline__ Sums scan(Sums v, Sums* total, Sums* scratch) {
    constexpr int kWarps = kPrepareThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Sums inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Sums u{__shfl_up_sync(0xffffffffu, inc.a, o), __shfl_up_sync(0xffffffffu, inc.b, o), __shfl_up_sync(0xffffffffu, inc.c, o)};
        if (lane >= o) inc = add(inc, u);
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    Sums before{0, 0, 0}, all{0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before = add(before, scratch[w]);
        all = add(all, scratch[w]);
    }
    *total = all;
    return {before.a + inc.a - v.a, before.b + inc.b - v.b, before.c + inc.c - v.c};
}
// The last s < sequences with starts[s] <= x.
__device__ __forceinline__ uint32_t last_from(const uint32_t* starts, uint32_t sequences, uint32_t x) {
    uint32_t lo = 0, hi = sequences;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (starts[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The tiles that row tile `r` of a sequence walks, and how many behind the sinks' it skips.
struct Walk { uint32_t tiles, skip; };
__device__ __forceinline__ Walk walk_of(const PrepareParams& p, const Span& span, const ChunkTiles& t, uint32_t r) {
    const uint32_t t_first = r * kChunkRows / p.group, t_last = min((r + 1) * kChunkRows - 1, span.tokens * p.group - 1) / p.group;
    const int last = span.base() + static_cast<int>(t_last);
    if (last < 0) return {0, 0};
    const uint32_t upto = static_cast<uint32_t>(last) / kChunkTile + 1;   // tiles of the cache below the last position seen
    Walk w{0, 0};
    uint32_t first = 0;   // the first of them, behind the sinks'
    if (p.window > 0) {
        const long long lowest = static_cast<long long>(span.base()) + t_first + 1 - p.window;
        first = lowest > 0 ? static_cast<uint32_t>(lowest) / kChunkTile : 0;
    }
    const uint32_t own0 = t.window0 / kChunkTile;   // the sequence's first tile behind its sinks' (0 without a gap)
    if (own0 == 0) {                                // the copy is the cache: the sinks' tiles come with the others
        const uint32_t sink = p.window > 0 ? (p.sinks + kChunkTile - 1) / kChunkTile : 0;
        if (first <= sink) return {upto, 0};
        return {sink + (upto > first ? upto - first : 0), first - sink};
    }
    w.skip = max(first, own0) - own0;
    w.tiles = t.sink_tiles + (upto > own0 + w.skip ? upto - own0 - w.skip : 0);
    return w;
}

// The same from a row tile's bounds.
__device__ __forceinline__ Walk walk_between(const PrepareParams& p, const uint2& b, const ChunkTiles& t) {
    const uint32_t upto = (b.y + kChunkTile - 1) / kChunkTile, sink = (min(p.sinks, b.y) + kChunkTile - 1) / kChunkTile;
    const uint32_t first = min(b.x / kChunkTile, upto), own0 = t.window0 / kChunkTile;   // (bounds of rows that see nothing: first == upto)
    if (own0 == 0) return first <= sink ? Walk{upto, 0} : Walk{sink + upto - first, first - sink};
    const uint32_t skip = max(first, own0) - own0;
    return {t.sink_tiles + (upto > own0 + skip ? upto - own0 - skip : 0), skip};
}

struct PlanScratch {
    Sums scan[kPrepareThreads / 32];
    uint32_t items[kCandidates], parts[kCandidates], longest, piece;
    unsigned long long work;   // 128ths of a tile: whole numbers, whose sum knows no order
};

// The list of the chunk kernel's CTAs; one block.
template <bool RANGED>
__device__ __forceinline__ void lay_out(const PrepareParams& p, const uint32_t* tile_starts, const uint32_t* scratch_starts, PlanScratch& sh) {
    const uint32_t tid = threadIdx.x, S = p.pool.batch.sequences, H = p.pool.view.kv_heads, row_tiles = tile_starts[S];
    if (tid == 0) p.plan->items = p.plan->groups = 0;
    if (static_cast<uint64_t>(row_tiles) * H > p.max_items || (RANGED && row_tiles > p.max_walks)) {   // starts that do not ascend: nothing of this is laid out
        if (tid == 0) report(p.pool, B200KV_STATUS_BAD_BOUND);
        return;
    }
    // ---- how far to split: candidate c has pieces of at most 3 longest / (c + 3) tiles.  The time is no less than a piece's, and about as many waves of average
    // pieces as there are: 152 pieces of one size on 148 SMs take twice as long as 148 (77 us for two chunks of 333 tokens over 5000).
    if (tid < kCandidates) sh.items[tid] = sh.parts[tid] = 0;
    if (tid == 0) { sh.longest = 0; sh.work = 0; }
    __syncthreads();
    if constexpr (RANGED) {   // row tiles differ by more than their place
        uint32_t most = 0;
        unsigned long long sum = 0;
        for (uint32_t i = tid; i < row_tiles; i += kPrepareThreads) {
            const uint32_t s = last_from(tile_starts, S, i);
            const Span span = span_of(p.pool, s);
            uint2 walk = p.tile_bounds[chunk_slot(span.first, p.group, s, tile_starts[s + 1] - 1 - i)];
            const uint32_t tiles = tiles_of<true>(p, span, s).tiles;
            walk.y = min(walk.y, tiles);           // (always so, but where starts do not ascend and two sequences have the same slot: nothing walks further than its copy)
            walk.x = min(walk.x, tiles - walk.y);
            p.walks[i] = walk;
            most = max(most, walk.x);
            sum += walk.x;
        }
        most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if ((tid & 31) == 0) {   // (an addition a thread to 64 bits that all share: 8 us)
            atomicMax(&sh.longest, most);
            atomicAdd(&sh.work, 128ull * sum * H);
        }
    } else {
        for (uint32_t s = tid; s < S; s += kPrepareThreads)
            if (const uint32_t n = scratch_starts[s + 1] - scratch_starts[s]; n > 0) atomicMax(&sh.longest, n);
    }
    __syncthreads();
    const uint32_t longest = sh.longest;
    const auto piece_of = [&](uint32_t c) { return max(3u, (3 * longest + c + 2) / (c + 3)); };
    if constexpr (RANGED) {
        // A warp has every eighth candidate and goes over all row tiles; quotients by a reciprocal, put right.  (All candidates by all threads, added up a warp at a time: 16 us for 348 row
        // tiles.)
        constexpr uint32_t kWarps = kPrepareThreads / 32, kEach = (kCandidates + kWarps - 1) / kWarps;
        const uint32_t warp = tid / 32;
        uint32_t items[kEach] = {}, parts[kEach] = {}, size[kEach];
        float over[kEach];
#pragma unroll
        for (uint32_t k = 0; k < kEach; ++k) {
            size[k] = warp + k * kWarps == 0 ? 0x7fffffffu : piece_of(warp + k * kWarps);
            over[k] = 1.0f / static_cast<float>(size[k]);
        }
        for (uint32_t i = tid & 31; i < row_tiles; i += 32) {
            const uint32_t tiles = p.walks[i].x;
#pragma unroll
            for (uint32_t k = 0; k < kEach; ++k) {
                uint32_t pieces = static_cast<uint32_t>(static_cast<float>(tiles) * over[k]);   // of up to a dozen: off by one at most
                if (static_cast<uint64_t>(pieces) * size[k] < tiles) ++pieces;
                else if (pieces > 0 && static_cast<uint64_t>(pieces - 1) * size[k] >= tiles) --pieces;
                pieces = max(pieces, 1u);
                items[k] += H * pieces;
                parts[k] += pieces > 1 ? H * pieces : 0;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kEach; ++k) {
            items[k] = __reduce_add_sync(0xffffffffu, items[k]);
            parts[k] = __reduce_add_sync(0xffffffffu, parts[k]);
            if ((tid & 31) == 0 && warp + k * kWarps < kCandidates) {
                sh.items[warp + k * kWarps] = items[k];
                sh.parts[warp + k * kWarps] = parts[k];
            }
        }
    } else {
        for (uint32_t s = tid; s < S; s += kPrepareThreads) {
            const uint32_t tiles = scratch_starts[s + 1] - scratch_starts[s], n = (tile_starts[s + 1] - tile_starts[s]) * H;
            if (n == 0) continue;
            atomicAdd(&sh.work, chunk_work(n, tiles, span_of(p.pool, s).tokens));
            for (uint32_t c = 0; c < kCandidates; ++c) {
                const uint32_t pieces = c == 0 ? 1 : max(1u, (tiles + piece_of(c) - 1) / piece_of(c));
                atomicAdd(&sh.items[c], n * pieces);
                if (pieces > 1) atomicAdd(&sh.parts[c], n * pieces);
            }
        }
    }
    __syncthreads();
    if (tid < 32) {
        float us = INFINITY;
        if (tid < kCandidates && (tid == 0 || (sh.items[tid] <= p.max_items && sh.parts[tid] <= p.max_parts))) {
            const float one = piece_of(tid) * p.costs.tile + p.costs.cta;
            const uint32_t n = sh.items[tid], full = n / p.sms, rest = n % p.sms;
            const float waves = full + (rest == 0 ? 0.0f : full == 0 ? 1.0f : p.costs.last_wave + (1.0f - p.costs.last_wave) * rest / p.sms);
            us = max(one, waves * (static_cast<float>(sh.work) / (128.0f * n) * p.costs.tile + p.costs.cta)) + (sh.parts[tid] > 0 ? p.costs.merge + p.costs.part * sh.parts[tid] : 0.0f);
        }
        const float best = -warp_max_redux(-us);
        const uint32_t which = __ffs(__ballot_sync(0xffffffffu, us == best)) - 1;
        if (tid == 0) sh.piece = which == 0 ? 0x7fffffffu : piece_of(which);
    }
    __syncthreads();
    const uint32_t piece = sh.piece;

    // ---- the list: a thread lays out a row tile, the longest of a sequence first
    uint32_t items = 0, parts = 0, groups = 0;
    for (uint32_t i0 = 0; i0 < row_tiles; i0 += kPrepareThreads) {
        const uint32_t i = i0 + tid;
        Sums v{0, 0, 0};
        ChunkItem item{};
        Walk walk{0, 0};
        uint32_t n = 1;
        if (i < row_tiles) {
            const uint32_t s = last_from(tile_starts, S, i);
            const Span span = span_of(p.pool, s);
            const ChunkTiles t = tiles_of<RANGED>(p, span, s);
            item.first = span.first;
            item.tokens = span.tokens;
            item.base = span.base();
            item.length = span.length;
            item.row_tile = tile_starts[s + 1] - 1 - i;
            if constexpr (RANGED) {
                const uint2 w = p.walks[i];
                walk = {w.x, w.y};
            } else {
                walk = walk_of(p, span, t, item.row_tile);
            }
            if (scratch_starts[s] + t.tiles > p.scratch_tiles) walk.tiles = 0;   // no room for the copy
            item.scratch_row = scratch_starts[s] * kChunkTile;
            const uint32_t sink = RANGED || p.window > 0 ? (p.sinks + kChunkTile - 1) / kChunkTile : 0;
            item.sink_tiles = t.window0 == 0 ? min(sink, walk.tiles) : t.sink_tiles;
            item.window0 = t.window0 == 0 ? item.sink_tiles * kChunkTile : t.window0;
            item.skip = walk.skip;
            n = max(1u, (walk.tiles + piece - 1) / piece);
            v = {H * n, n > 1 ? H * n : 0, n > 1 ? H : 0};
        }
        Sums total;
        const Sums before = scan(v, &total, sh.scan);
        if (i < row_tiles) {
            uint32_t at = items + before.a, part = parts + before.b, group = groups + before.c;
            for (uint32_t h = 0; h < H; ++h) {
                if (n > 1) p.groups[group++] = at;
                for (uint32_t z = 0; z < n; ++z, ++at) {
                    item.kv_head = h;
                    if (RANGED && n == 1) {   // (64-bit divisions: as long as all the rest)
                        item.tile0 = 0;
                        item.tiles = walk.tiles;
                    } else {
                        item.tile0 = static_cast<uint32_t>(static_cast<uint64_t>(walk.tiles) * z / n);
                        item.tiles = static_cast<uint32_t>(static_cast<uint64_t>(walk.tiles) * (z + 1) / n) - item.tile0;
                    }
                    item.part = n > 1 ? part++ : kNoPart;
                    item.parts = n;
                    p.items[at] = item;
                }
            }
        }
        items += total.a;
        parts += total.b;
        groups += total.c;
    }
    if (tid == 0) {
        p.plan->items = items;
        p.plan->groups = groups;
    }
}

// A unit of the gather: a tile of 64 positions of one side of one kv head.
template <int D, bool RANGED>
__device__ __forceinline__ void gather_unit(const PrepareParams& p, const uint32_t* scratch_starts, uint32_t unit) {
    constexpr uint32_t CPR = D / 8, kEach = kChunkTile * CPR / kPrepareThreads;   // 16-byte pieces of a row of the copy; a thread's of a tile
    const Paged& pool = p.pool;
    const uint32_t H = pool.view.kv_heads, c = threadIdx.x % CPR;
    const uint32_t side = unit & 1, head = (unit >> 1) % H, tile = (unit >> 1) / H;
    const uint32_t s = last_from(scratch_starts, pool.batch.sequences, tile);
    const Span span = span_of(pool, s);
    const ChunkTiles t = tiles_of<RANGED>(p, span, s);
    uint2 bounds = make_uint2(0, 0);
    if constexpr (RANGED) bounds = p.bounds[s];
    const uint32_t u = tile - scratch_starts[s];
    const uint32_t pos0 = u < t.sink_tiles ? u * kChunkTile : t.window0 + (u - t.sink_tiles) * kChunkTile;
    const bool q8 = side == 0 ? is_k_q8(pool.view.quant_mode) : is_v_q8(pool.view.quant_mode);
    const int8_t* q = side == 0 ? pool.view.key_q8 : pool.view.value_q8;
    const __half* scales = static_cast<const __half*>(side == 0 ? pool.view.key_scales : pool.view.value_scales);
    const __half* f16 = static_cast<const __half*>(side == 0 ? pool.view.key_f16 : pool.view.value_f16);
    const uint32_t blocks = D / pool.view.qblock;
    __half* out = p.out[side] + (static_cast<size_t>(head) * p.scratch_tiles + tile) * kChunkTile * D + c * 8;
    uint4 v[kEach];
    __half scale[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t j = pos0 + threadIdx.x / CPR + i * (kPrepareThreads / CPR);
        v[i] = make_uint4(0, 0, 0, 0);
        scale[i] = __ushort_as_half(0);
        bool seen;   // by any of the tokens
        if constexpr (RANGED) seen = j < bounds.y && (j >= bounds.x || j < p.sinks);
        else seen = j < span.length && (p.window == 0 || j < p.sinks || static_cast<int>(j + p.window) > span.base());
        const long long row = seen ? row_of(pool, s, head, j) : -1;
        if (row < 0) continue;   // zeros (a weight of 0 times what lies there would still be NaN where that is)
        const size_t at = static_cast<size_t>(row) * D + c * 8;
        if (q8) {
            const uint2 raw = *reinterpret_cast<const uint2*>(q + at);
            v[i].x = raw.x; v[i].y = raw.y;
            scale[i] = scales[static_cast<size_t>(row) * blocks + (blocks == 1 ? 0 : c / 4)];
        } else {
            v[i] = *reinterpret_cast<const uint4*>(f16 + at);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i)
        *reinterpret_cast<uint4*>(out + static_cast<size_t>(threadIdx.x / CPR + i * (kPrepareThreads / CPR)) * D) =
            q8 ? dequant8(make_uint2(v[i].x, v[i].y), scale[i]) : v[i];
}

// What the tokens of each row tile and of each sequence see, and what each row tile walks of it: a block a sequence, or several in turn, a warp four row tiles at a time, whose loads are under way
// together (one at a time: 12 us for 193 row tiles, a trip to L2 each).
constexpr int kBoundsThreads = 1024, kBoundsTiles = 4;
__global__ void __launch_bounds__(kBoundsThreads) paged_bounds_kernel(const __grid_constant__ PrepareParams p) {
    __shared__ uint32_t lowest, end;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t s = blockIdx.x; s < p.pool.batch.sequences; s += gridDim.x) {
        const Span span = span_of(p.pool, s);
        if (!p.mine(span)) continue;   // the same for all threads
        if (threadIdx.x == 0) { lowest = 0xffffffffu; end = 0; }
        __syncthreads();
        const uint32_t rows = span.tokens * p.group, row_tiles = p.row_tiles(span);
        uint2* const of_tiles = p.tile_bounds + chunk_slot(span.first, p.group, s, 0);
        for (uint32_t r0 = threadIdx.x / 32 * kBoundsTiles; r0 < row_tiles; r0 += kBoundsThreads / 32 * kBoundsTiles) {
            uint32_t low[kBoundsTiles], upto[kBoundsTiles];
#pragma unroll
            for (uint32_t i = 0; i < kBoundsTiles; ++i) {
                low[i] = 0xffffffffu;
                upto[i] = 0;
            }
            // of a row tile's tokens: where the heads are no whole fraction of it, those of its first and of its last token may both lie in two (44 tokens in 128 rows of three heads)
            for (uint32_t t0 = lane; t0 < (kChunkRows + 2 * (p.group - 1)) / p.group; t0 += 32) {
                Sight sight[kBoundsTiles];
#pragma unroll
                for (uint32_t i = 0; i < kBoundsTiles; ++i) {
                    const uint32_t r = r0 + i, t = r * kChunkRows / p.group + t0;
                    sight[i] = {0, 0};
                    if (r < row_tiles && t <= min((r + 1) * kChunkRows - 1, rows - 1) / p.group)
                        sight[i] = sight_of(p.ranges, static_cast<size_t>(span.first) + t, span.base() + static_cast<int>(t), p.window, span.length);
                }
#pragma unroll
                for (uint32_t i = 0; i < kBoundsTiles; ++i) {
                    if (!sight[i].empty()) low[i] = min(low[i], sight[i].low);
                    upto[i] = max(upto[i], sight[i].empty() ? min(sight[i].upto, p.sinks) : sight[i].upto);
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < kBoundsTiles; ++i) {
                low[i] = __reduce_min_sync(0xffffffffu, low[i]);
                upto[i] = __reduce_max_sync(0xffffffffu, upto[i]);
                if (lane == 0 && r0 + i < row_tiles) {
                    of_tiles[r0 + i] = make_uint2(low[i], upto[i]);
                    atomicMin(&lowest, low[i]);
                    atomicMax(&end, upto[i]);
                }
            }
        }
        __syncthreads();
        const ChunkTiles t = chunk_tiles_between(lowest, end, p.sinks);
        for (uint32_t r = threadIdx.x; r < row_tiles; r += kBoundsThreads) {
            const Walk walk = walk_between(p, of_tiles[r], t);
            of_tiles[r] = make_uint2(walk.tiles, walk.skip);
        }
        if (threadIdx.x == 0) p.bounds[s] = make_uint2(lowest, end);
        __syncthreads();   // the bounds are read
    }
}

template <int D, bool RANGED>
__global__ void __launch_bounds__(kPrepareThreads) paged_prepare_kernel(const __grid_constant__ PrepareParams p) {
    extern __shared__ uint32_t starts[];   // row tiles, then tiles of the copy, before every sequence
    __shared__ PlanScratch sh;
    pdl_launch_dependents();
    pdl_wait();   // lengths, starts and cache rows come from preceding kernels
    const uint32_t S = p.pool.batch.sequences;
    uint32_t* tile_starts = starts;
    uint32_t* scratch_starts = starts + S + 1;
    uint32_t row_tiles = 0, scratch_tiles = 0;
    for (uint32_t s0 = 0; s0 < S; s0 += kPrepareThreads) {
        const uint32_t s = s0 + threadIdx.x;
        Sums v{0, 0, 0};
        if (s < S) {
            const Span span = span_of(p.pool, s);
            if (p.mine(span)) {
                v.a = p.row_tiles(span);
                v.b = tiles_of<RANGED>(p, span, s).tiles;
            }
        }
        Sums total;
        const Sums before = scan(v, &total, sh.scan);
        if (s < S) {
            tile_starts[s] = row_tiles + before.a;
            scratch_starts[s] = min(scratch_tiles + before.b, p.scratch_tiles);
        }
        row_tiles += total.a;
        scratch_tiles += total.b;
    }
    if (threadIdx.x == 0) {
        if (blockIdx.x == 0 && scratch_tiles > p.scratch_tiles) report(p.pool, B200KV_STATUS_BAD_BOUND);
        tile_starts[S] = row_tiles;
        scratch_starts[S] = min(scratch_tiles, p.scratch_tiles);
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        lay_out<RANGED>(p, tile_starts, scratch_starts, sh);
        return;
    }
    const uint32_t units = scratch_starts[S] * p.pool.view.kv_heads * 2;
    for (uint32_t unit = blockIdx.x - 1; unit < units; unit += gridDim.x - 1) gather_unit<D, RANGED>(p, scratch_starts, unit);
}

struct ChunkMergeParams {
    const ChunkPlan* plan;
    const ChunkItem* items;
    const uint32_t* groups;
    const float* part_o;
    const float2* part_ml;
    const float* gate;
    void* out;
    int out_is_f16;
    float* lse;
    uint32_t query_heads, kv_heads;
};

// out = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), times sigmoid(gate).  A thread: four dims of a row of a shared row tile, four partials' loads under way
// together; blocks take a quarter or an eighth of a kilorow at a time in turn.  (All 16 partials' loads in flight took 108 registers: two blocks an SM, and a
// block's four pieces one behind the other: 34 us for 96 row tiles of three partials of 256 dims.)
template <int D>
__global__ void __launch_bounds__(256) paged_merge_kernel(const __grid_constant__ ChunkMergeParams p) {
    constexpr uint32_t VPR = D / 4, kBlocks = kChunkRows * VPR / 256;   // a row tile's
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t G = p.query_heads / p.kv_heads, units = p.plan->groups * kBlocks;
    for (uint32_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const ChunkItem item = p.items[p.groups[unit / kBlocks]];
        const uint32_t i = unit % kBlocks * 256 + threadIdx.x, r = i / VPR, c = i % VPR * 4, gr = item.row_tile * kChunkRows + r;
        if (gr >= item.tokens * G) continue;
        const size_t head_row = (static_cast<size_t>(item.first) + gr / G) * p.query_heads + item.kv_head * G + gr % G, at = head_row * D + c;
        float4 g4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p.gate != nullptr) g4 = *reinterpret_cast<const float4*>(p.gate + at);
        const float2* ml = p.part_ml + static_cast<size_t>(item.part) * kChunkRows + r;
        const float* part = p.part_o + (static_cast<size_t>(item.part) * kChunkRows + r) * D + c;
        float m = -INFINITY, l = 0.0f;
        bool poisoned = false;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t s0 = 0; s0 < item.parts; s0 += 4) {
            float2 x[4];
            float4 o[4];
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s) {
                x[s] = make_float2(-INFINITY, 0.0f);
                o[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (s0 + s >= item.parts) continue;
                x[s] = ml[(s0 + s) * kChunkRows];
                o[s] = *reinterpret_cast<const float4*>(part + static_cast<size_t>(s0 + s) * kChunkRows * D);
            }
            float m_new = m;
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s) {
                if (x[s].y != x[s].y) poisoned = true;
                if (x[s].y > 0.0f) m_new = fmaxf(m_new, x[s].x);
            }
            if (m_new > m) {
                const float f = m == -INFINITY ? 0.0f : exp2f(m - m_new);
                l *= f; acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
                m = m_new;
            }
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s) {
                if (!(x[s].y > 0.0f)) continue;
                const float w = exp2f(x[s].x - m);
                l += w * x[s].y;
                acc.x += w * o[s].x; acc.y += w * o[s].y; acc.z += w * o[s].z; acc.w += w * o[s].w;
            }
        }
        float f = l > 0.0f ? 1.0f / l : 0.0f;
        if (poisoned) f = __int_as_float(0x7fc00000);
        if (p.lse != nullptr && c == 0) p.lse[head_row] = poisoned ? f : l > 0.0f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
        acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
        if (p.gate != nullptr) {
            acc.x *= 1.0f / (1.0f + __expf(-g4.x)); acc.y *= 1.0f / (1.0f + __expf(-g4.y));
            acc.z *= 1.0f / (1.0f + __expf(-g4.z)); acc.w *= 1.0f / (1.0f + __expf(-g4.w));
        }
        if (p.out_is_f16) {
            const __half2 a = __floats2half2_rn(acc.x, acc.y), b = __floats2half2_rn(acc.z, acc.w);
            *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
            *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = acc;
        }
    }
}

// The chunk kernel multiplies queries rounded to fp16, which moves the statistics of fp32 ones by up to a few 1e-4 of a score's spread: more than the output, itself a
// mean over the rounded weights, shows, but 1e-5 and more of an lse.  To first order lse_i moves by scale (q_i - fp16(q_i)).(sum_j p_ij k_j), and the sum is what
// the chunk kernel gives for V = K; what is left is of the square of the rounding.  (That mean key is an fp16 output: 2^-11 of a correction which is 2^-11 itself.)
// Where both fp32 queries and statistics are asked for the chunks take twice the time for it (two sequences, 1668 new tokens under a window of 40, 24 / 4 heads of 256: 96 -> 148 us).
// Over int8 keys they do not: the copy has rounded those, which costs as much again and is not put back.  A warp: a head of a token of the chunk kernel's sequences, or several in turn.
struct LseParams {
    PrepareParams prepare;
    const float* q;
    const __half* mean_key;   // [total_tokens][query_heads][D]
    float* lse;
    uint32_t query_heads;
    float scale;
};
template <int D>
__global__ void __launch_bounds__(256) paged_lse_kernel(const __grid_constant__ LseParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const Paged& pool = p.prepare.pool;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t rows = static_cast<uint64_t>(pool.batch.total_tokens) * p.query_heads;
    for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * 8 + threadIdx.x / 32; row < rows; row += static_cast<uint64_t>(gridDim.x) * 8) {
        const uint32_t token = static_cast<uint32_t>(row / p.query_heads);
        const Span span = span_of(pool, sequence_of(pool, token));
        if (!p.prepare.mine(span) || token < span.first || token - span.first >= span.tokens) continue;
        float sum = 0.0f;
#pragma unroll
        for (int x = 0; x < D; x += 128) {
            const float4 q = *reinterpret_cast<const float4*>(p.q + row * D + x + lane * 4);
            const uint2 raw = *reinterpret_cast<const uint2*>(p.mean_key + row * D + x + lane * 4);
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
            const auto left = [](float v) { return v - __half2float(__float2half_rn(v)); };
            sum += left(q.x) * a.x + left(q.y) * a.y + left(q.z) * b.x + left(q.w) * b.y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) p.lse[row] += p.scale * sum;   // where nothing is seen: minus infinity and a sum of zeros
    }
}

// ---- the workspace of a call -----------------------------------------------------------------------------------------------------

struct Room {
    uint64_t scratch_tiles;    // of all sequences together
    uint64_t max_walks;        // row tiles of all sequences together, with ranges
    uint32_t max_items, max_parts;
    bool decode, chunks;       // which kernels the call may need
    size_t decode_parts, items, groups, k, v, part_o, part_ml, mean_key, tile_bounds, bounds, walks, bytes;   // offsets
};

uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

Room room_of(const b200kv_paged_view& view, const b200kv_paged_batch& batch, uint32_t query_heads, uint32_t window, uint32_t sinks, bool ranged, uint32_t sms) {
    Room r{};
    const uint64_t group = query_heads / view.kv_heads;
    // A single sequence goes by its bound: the chunk kernel takes a token as well, and the other's launch is saved.
    r.chunks = !decode_takes_all(batch, static_cast<uint32_t>(group));
    r.decode = !r.chunks || batch.sequences > 1;
    const uint64_t least = r.decode ? decode_rows(batch, static_cast<uint32_t>(group)) / group + 1 : 1;   // new tokens of a sequence of the chunk kernel
    const uint64_t sequences = std::min<uint64_t>(batch.sequences, batch.total_tokens / least);
    // a sequence's tiles: its length's, or those of its sinks and of the windows of its tokens
    uint64_t each = (static_cast<uint64_t>(batch.max_length) + kChunkTile - 1) / kChunkTile;
    if (window > 0) each = std::min<uint64_t>(each, (static_cast<uint64_t>(sinks) + kChunkTile - 1) / kChunkTile + (static_cast<uint64_t>(window) + batch.max_tokens + kChunkTile - 1) / kChunkTile + 1);
    r.scratch_tiles = sequences * each;
    if (batch.total_length > 0) r.scratch_tiles = std::min(r.scratch_tiles, batch.total_length / kChunkTile + sequences);
    r.scratch_tiles = std::max<uint64_t>(r.scratch_tiles, 1);   // lengths bounded by zero: the copy is a tile that nobody reads
    // every sequence's last row tile may be a partial one
    const uint64_t row_tiles = std::min<uint64_t>(batch.total_tokens * group / kChunkRows + sequences, sequences * ((batch.max_tokens * group + kChunkRows - 1) / kChunkRows));
    // (CTAs of the grid that turn out to have nothing to do cost a launch microseconds: row tiles are split where there are fewer of them than this)
    const uint64_t units = row_tiles * view.kv_heads, parts = 4ull * sms;
    r.max_items = static_cast<uint32_t>(std::min<uint64_t>(std::max(units, parts), 0x7fffffffu));
    r.max_parts = static_cast<uint32_t>(parts);
    size_t at = 256;                                     // the plan
    const auto take = [&](uint64_t bytes) { const size_t here = at; at += up(bytes, 1024); return here; };
    at = up(at, 1024);
    r.decode_parts = take(r.decode ? decode_part_bytes(view, sms) : 0);
    if (!r.chunks) {
        r.bytes = at + 1024;
        return r;
    }
    r.items = take(static_cast<uint64_t>(r.max_items) * sizeof(ChunkItem));
    r.groups = take(parts * 4);
    const uint64_t plane = r.scratch_tiles * kChunkTile * view.kv_heads * view.head_dim * sizeof(__half);
    r.k = take(plane);
    // the mean keys of the statistics (over fp16 keys) lie over V, which the second pass of the chunk kernel does not read
    r.v = r.mean_key = take(is_k_q8(view.quant_mode) ? plane : std::max(plane, static_cast<uint64_t>(batch.total_tokens) * query_heads * view.head_dim * sizeof(__half)));
    r.part_o = take(parts * kChunkRows * view.head_dim * sizeof(float));
    r.part_ml = take(parts * kChunkRows * sizeof(float2));
    if (ranged) {
        r.max_walks = batch.total_tokens * group / kChunkRows + batch.sequences + 1;
        r.tile_bounds = take(r.max_walks * sizeof(uint2));
        r.walks = take(r.max_walks * sizeof(uint2));
        r.bounds = take(static_cast<uint64_t>(batch.sequences) * sizeof(uint2));
    }
    r.bytes = at + 1024;                                 // the base is brought to a multiple of 1024
    return r;
}

}  // namespace

}  // namespace b200kv

using namespace b200kv;

namespace {

// Without scoring (null) nothing but the window cuts what a token sees.
void settle(const b200kv_paged_batch& batch, const b200kv_paged_scoring* scoring, uint32_t* window, uint32_t* sinks) {
    const uint32_t most = std::min(*sinks, batch.max_length);
    settle_window(batch, window, sinks);
    if (scoring != nullptr && scoring->ranges != nullptr) *sinks = most;
}

size_t workspace_of(const b200kv_paged_view* view, const b200kv_paged_batch* batch, const b200kv_paged_scoring* scoring, uint32_t query_heads, uint32_t window, uint32_t sinks) {
    if (view == nullptr || batch == nullptr || view->kv_heads == 0 || query_heads == 0 || query_heads % view->kv_heads != 0) return 0;
    settle(*batch, scoring, &window, &sinks);
    return room_of(*view, *batch, query_heads, window, sinks, scoring != nullptr && scoring->ranges != nullptr, kMostSms).bytes;
}

int attend(const b200kv_paged_view* view, const b200kv_paged_batch* batch, const b200kv_paged_scoring* scoring, const void* q, int q_dtype, const float* gate,
           void* output, int output_dtype, float* lse, uint32_t query_heads, float scale, uint32_t window, uint32_t sinks,
           void* workspace, size_t workspace_bytes, void* stream) {
    int rc = validate_paged(view, batch);
    if (rc != B200KV_OK) return rc;
    if (q == nullptr || output == nullptr || (q_dtype != B200KV_F16 && q_dtype != B200KV_F32) || (output_dtype != B200KV_F16 && output_dtype != B200KV_F32)) return B200KV_ERR_INVALID;
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(output) | reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(workspace)) & 15u) != 0 ||
        (reinterpret_cast<uintptr_t>(lse) & 3u) != 0)
        return B200KV_ERR_INVALID;
    if (query_heads == 0 || query_heads % view->kv_heads != 0 || !std::isfinite(scale) || !(scale > 0.0f)) return B200KV_ERR_INVALID;
    if (query_heads / view->kv_heads > 8) return B200KV_ERR_UNSUPPORTED;
    if (static_cast<uint64_t>(view->pages) * view->kv_heads * view->page_size > 0x7fffffffull) return B200KV_ERR_UNSUPPORTED;   // coordinates are 32-bit
    if (batch->sequences == 0 || batch->total_tokens == 0 || batch->max_tokens == 0) return B200KV_OK;
    settle(*batch, scoring, &window, &sinks);
    const bool capped = scoring != nullptr && scoring->cap > 0.0f, ranged = scoring != nullptr && scoring->ranges != nullptr;
    const uint32_t group = query_heads / view->kv_heads;
    if (scoring != nullptr) {   // read while results are written
        const uint64_t out_bytes = static_cast<uint64_t>(batch->total_tokens) * query_heads * view->head_dim * (output_dtype == B200KV_F32 ? 4 : 2), lse_bytes = static_cast<uint64_t>(batch->total_tokens) * query_heads * 4;
        for (const auto& [array, bytes] : {std::pair<const void*, uint64_t>{scoring->slopes, query_heads * 4ull}, std::pair<const void*, uint64_t>{scoring->ranges, batch->total_tokens * 8ull}})
            if (array != nullptr && (share(array, bytes, output, out_bytes) || (lse != nullptr && share(array, bytes, lse, lse_bytes)))) return B200KV_ERR_INVALID;
    }
    const bool again = lse != nullptr && q_dtype == B200KV_F32 && !is_k_q8(view->quant_mode) && !capped && !decode_takes_all(*batch, group);   // the queries are read once more when results are out
    const uint64_t rows = static_cast<uint64_t>(batch->total_tokens) * query_heads, q_bytes = rows * view->head_dim * 4;
    if (again && (share(q, q_bytes, output, output_dtype == B200KV_F32 ? q_bytes : q_bytes / 2) || share(q, q_bytes, lse, rows * 4))) return B200KV_ERR_INVALID;
    if (workspace == nullptr || workspace_bytes < workspace_of(view, batch, scoring, query_heads, window, sinks)) return B200KV_ERR_WORKSPACE;
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    const Room room = room_of(*view, *batch, query_heads, window, sinks, ranged, kMostSms);
    if (room.scratch_tiles * kChunkTile * view->kv_heads > 0x7fffffffull) return B200KV_ERR_UNSUPPORTED;
    uint8_t* ws = reinterpret_cast<uint8_t*>(up(reinterpret_cast<uintptr_t>(workspace), 1024));
    const Paged pool = paged_of(*view, *batch);
    const uint32_t sms = std::min(device_sms(), kMostSms);
    cudaStream_t s = static_cast<cudaStream_t>(stream);

    if (room.chunks) {
        const uint32_t few_rows = room.decode ? decode_rows(*batch, group) : 0;
        const PrepareParams pp{pool, reinterpret_cast<ChunkPlan*>(ws), reinterpret_cast<ChunkItem*>(ws + room.items), reinterpret_cast<uint32_t*>(ws + room.groups), room.max_items,
                               room.max_parts, static_cast<uint32_t>(room.scratch_tiles), group, window, sinks, sms, few_rows,
                               view->head_dim == 256 ? ChunkCosts{0.62f, 12.4f, 0.5f, 0.0f, 0.024f} : ChunkCosts{0.5f, 7.0f, 1.0f, 2.0f, 0.02f},
                               {reinterpret_cast<__half*>(ws + room.k), reinterpret_cast<__half*>(ws + room.v)}, ranged ? scoring->ranges : nullptr,
                               reinterpret_cast<uint2*>(ws + room.tile_bounds), reinterpret_cast<uint2*>(ws + room.bounds), reinterpret_cast<uint2*>(ws + room.walks),
                               static_cast<uint32_t>(room.max_walks)};
        const uint32_t blocks = 1 + static_cast<uint32_t>(std::min<uint64_t>(room.scratch_tiles * view->kv_heads * 2, 8ull * sms));
        const size_t smem = 2 * (static_cast<size_t>(batch->sequences) + 1) * 4;
        static std::atomic<uint64_t> done[4];
        const auto prepare = ranged ? (view->head_dim == 128 ? paged_prepare_kernel<128, true> : paged_prepare_kernel<256, true>)
                                    : (view->head_dim == 128 ? paged_prepare_kernel<128, false> : paged_prepare_kernel<256, false>);
        if (smem > 32 * 1024) B200KV_CUDA_TRY(opt_in_dynamic_smem(reinterpret_cast<const void*>(prepare), 2 * (kMostSequences + 1) * 4, done[(view->head_dim == 256) + 2 * ranged]));
        if (ranged) {
            B200KV_CUDA_TRY(launch_kernel(paged_bounds_kernel, dim3(std::min(batch->sequences, 2 * sms)), dim3(kBoundsThreads), 0, s, true, pp));
            B200KV_CUDA_TRY(launch_behind(prepare, dim3(blocks), dim3(kPrepareThreads), smem, s, pp));
        } else {
            B200KV_CUDA_TRY(launch_kernel(prepare, dim3(blocks), dim3(kPrepareThreads), smem, s, true, pp));
        }
        const ChunkLaunch cl{pp.items, pp.plan, room.max_items, pp.out[0], pp.out[1], static_cast<uint32_t>(room.scratch_tiles * kChunkTile), q, q_dtype == B200KV_F16, gate, output,
                             output_dtype == B200KV_F16, lse, query_heads, view->kv_heads, view->head_dim, window, sinks, scale * 1.4426950408889634f,
                             reinterpret_cast<float*>(ws + room.part_o), reinterpret_cast<float2*>(ws + room.part_ml), scoring != nullptr, capped ? scoring->cap : 0.0f, scale,
                             scoring != nullptr ? scoring->slopes : nullptr, pp.ranges};
        rc = launch_chunk(cl, s);
        if (rc != B200KV_OK) return rc;
        const ChunkMergeParams mp{pp.plan, pp.items, pp.groups, cl.part_o, cl.part_ml, gate, output, cl.out_is_f16, lse, query_heads, view->kv_heads};
        B200KV_CUDA_TRY(view->head_dim == 128 ? launch_behind(paged_merge_kernel<128>, dim3(5 * sms), dim3(256), 0, s, mp)
                                              : launch_behind(paged_merge_kernel<256>, dim3(5 * sms), dim3(256), 0, s, mp));
        if (again) {
            ChunkLaunch keys = cl;
            keys.v_scratch = cl.k_scratch;
            keys.gate = nullptr;
            keys.out = ws + room.mean_key;
            keys.out_is_f16 = 1;
            keys.lse = nullptr;
            rc = launch_chunk(keys, s);
            if (rc != B200KV_OK) return rc;
            const ChunkMergeParams km{pp.plan, pp.items, pp.groups, cl.part_o, cl.part_ml, nullptr, keys.out, 1, nullptr, query_heads, view->kv_heads};
            const LseParams lp{pp, static_cast<const float*>(q), reinterpret_cast<const __half*>(ws + room.mean_key), lse, query_heads, scale};
            const uint32_t blocks_of_rows = static_cast<uint32_t>(std::min<uint64_t>((static_cast<uint64_t>(batch->total_tokens) * query_heads + 7) / 8, 8ull * sms));
            B200KV_CUDA_TRY(view->head_dim == 128 ? launch_behind(paged_merge_kernel<128>, dim3(5 * sms), dim3(256), 0, s, km)
                                                  : launch_behind(paged_merge_kernel<256>, dim3(5 * sms), dim3(256), 0, s, km));
            B200KV_CUDA_TRY(view->head_dim == 128 ? launch_behind(paged_lse_kernel<128>, dim3(blocks_of_rows), dim3(256), 0, s, lp)
                                                  : launch_behind(paged_lse_kernel<256>, dim3(blocks_of_rows), dim3(256), 0, s, lp));
        }
    }
    if (room.decode) {
        PagedDecode dp{pool, q, q_dtype == B200KV_F16, gate, output, output_dtype == B200KV_F16, lse, query_heads, window, sinks, 0, scale * 1.4426950408889634f};
        if (scoring == nullptr) return launch_paged_decode(dp, ws + room.decode_parts, s, room.chunks);
        PagedDecodeScored scored{};
        static_cast<PagedDecode&>(scored) = dp;
        scored.cap_log2 = capped ? scoring->cap * 1.4426950408889634f : 0.0f;
        scored.cap_in = capped ? 1.0f / scored.cap_log2 : 0.0f;
        scored.slopes = scoring->slopes;
        scored.ranges = scoring->ranges;
        return launch_paged_decode_scored(scored, ws + room.decode_parts, s, room.chunks);
    }
    return B200KV_OK;
}

}  // namespace

extern "C" {

size_t b200kv_paged_attn_workspace_bytes(const b200kv_paged_view* view, const b200kv_paged_batch* batch, uint32_t query_heads, uint32_t window, uint32_t sinks) {
    return workspace_of(view, batch, nullptr, query_heads, window, sinks);
}

int b200kv_paged_attn(const b200kv_paged_view* view, const b200kv_paged_batch* batch, const void* q, int q_dtype, const float* gate,
                      void* output, int output_dtype, float* lse, uint32_t query_heads, float scale, uint32_t window, uint32_t sinks,
                      void* workspace, size_t workspace_bytes, void* stream) {
    return attend(view, batch, nullptr, q, q_dtype, gate, output, output_dtype, lse, query_heads, scale, window, sinks, workspace, workspace_bytes, stream);
}

size_t b200kv_paged_attn_scored_workspace_bytes(const b200kv_paged_view* view, const b200kv_paged_batch* batch, const b200kv_paged_scoring* scoring, uint32_t query_heads,
                                                uint32_t window, uint32_t sinks) {
    return scoring == nullptr ? 0 : workspace_of(view, batch, scoring, query_heads, window, sinks);
}

int b200kv_paged_attn_scored(const b200kv_paged_view* view, const b200kv_paged_batch* batch, const b200kv_paged_scoring* scoring, const void* q, int q_dtype, const float* gate,
                             void* output, int output_dtype, float* lse, uint32_t query_heads, float scale, uint32_t window, uint32_t sinks,
                             void* workspace, size_t workspace_bytes, void* stream) {
    if (scoring == nullptr || !std::isfinite(scoring->cap) || scoring->cap < 0.0f) return B200KV_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(scoring->slopes) & 3u) != 0 || (reinterpret_cast<uintptr_t>(scoring->ranges) & 7u) != 0) return B200KV_ERR_INVALID;
    // a cap's quotients with the scale, and its product with log2 e, are ordinary numbers
    if (scoring->cap > 0.0f && (scoring->cap < 1.0e-6f || scoring->cap > 1.0e6f)) return B200KV_ERR_UNSUPPORTED;
    const bool nothing = scoring->cap == 0.0f && scoring->slopes == nullptr && scoring->ranges == nullptr;
    return attend(view, batch, nothing ? nullptr : scoring, q, q_dtype, gate, output, output_dtype, lse, query_heads, scale, window, sinks, workspace, workspace_bytes, stream);
}

}  // extern "C"
