// The book of a paged cache's pages -- who holds which, and how many do -- and the copies that go with it: room for new tokens, sequences that go on from others', sequences
// that end, pages moved together, pages copied to another pool.
//
// A page is free where its count is 0.  Whoever needs pages gets the lowest free ones, in the order of the call's entries, so that a call has one result whatever the order of
// its threads is; counts are whole numbers, which atomics may add to in any order.  The book is device memory and a call needs bounds only, so it can be captured.
//
// Bound by latency in the book (one block finds the pages: a step over 16384 counts, a scan and a search an entry) and by HBM in the copies, which are all that takes time where
// there are many: a page of every layer is read once and written once.
#include "paged_common.cuh"

#include <algorithm>
#include <cstring>
#include <initializer_list>

namespace b200kv {

namespace {

constexpr uint32_t kMostLayers = 128;        // of a call
constexpr uint32_t kFewLayers = 16;          // kernels for so many have parameters an eighth of the size
constexpr int kBookThreads = 1024;
constexpr uint32_t kChunk = 4 * kBookThreads;   // counts that a block of the compaction looks at

// ---- copies of pages ---------------------------------------------------------------------------------------------------------------

constexpr int kCopyThreads = 256, kCopySteps = 8;
constexpr uint32_t kPiece = 32 * 16 * kCopySteps;   // bytes that a warp copies at a time

// The planes of the layers of two pools of one geometry: K, its scales, V, its scales, as far as there are any.
template <uint32_t LAYERS>
struct Planes {
    uint32_t layers, planes;          // of a layer: 2 to 4
    uint32_t bytes[4], pieces[4];     // a page's of each plane
    uint32_t layer_pieces;            // of all planes of a layer
    uint32_t from_pages, to_pages;
    uint32_t* status;
    const uint8_t* from[LAYERS][4];
    uint8_t* to[LAYERS][4];
};

// Pages sources[i] -> targets[i] for i < count, by all warps of the grid in turn: a piece of a plane of a layer each time, eight loads of 16 bytes a lane under way.
template <uint32_t LAYERS>
__device__ __forceinline__ void copy_pages(const Planes<LAYERS>& p, const int32_t* sources, const int32_t* targets, uint32_t count) {
    const uint32_t lane = threadIdx.x & 31, each = p.layers * p.layer_pieces;
    const uint32_t warps = gridDim.x * (kCopyThreads / 32), me = blockIdx.x * (kCopyThreads / 32) + threadIdx.x / 32;
    const uint32_t step_pairs = warps / each, step_rest = warps % each;
    uint32_t pair = me / each, rest = me % each;
    while (pair < count) {
        const int source = sources[pair], target = targets[pair];
        uint32_t layer = rest / p.layer_pieces, piece = rest % p.layer_pieces, plane = 0;
        while (piece >= p.pieces[plane]) piece -= p.pieces[plane++];
        if (static_cast<uint32_t>(source) < p.from_pages && static_cast<uint32_t>(target) < p.to_pages) {
            const uint32_t bytes = p.bytes[plane], at0 = piece * kPiece + lane * 16;
            const uint8_t* from = p.from[layer][plane] + static_cast<uint64_t>(source) * bytes;
            uint8_t* to = p.to[layer][plane] + static_cast<uint64_t>(target) * bytes;
            uint4 v[kCopySteps];
#pragma unroll
            for (int i = 0; i < kCopySteps; ++i)
                if (at0 + 512 * i < bytes) v[i] = __ldcs(reinterpret_cast<const uint4*>(from + at0 + 512 * i));
#pragma unroll
            for (int i = 0; i < kCopySteps; ++i)
                if (at0 + 512 * i < bytes) *reinterpret_cast<uint4*>(to + at0 + 512 * i) = v[i];
        } else if (lane == 0 && rest == 0 && target >= 0 && p.status != nullptr) {
            atomicOr(p.status, B200KV_STATUS_BAD_PAGE);
        }
        pair += step_pairs;
        rest += step_rest;
        if (rest >= each) { rest -= each; ++pair; }
    }
}

template <uint32_t LAYERS>
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const __grid_constant__ Planes<LAYERS> planes, const int32_t* sources, const int32_t* targets, uint32_t count) {
    pdl_wait();
    pdl_launch_dependents();   // behind the wait: it writes cache rows
    copy_pages(planes, sources, targets, count);
}

// ---- the book ----------------------------------------------------------------------------------------------------------------------

struct Book {
    b200kv_page_book b;
    uint32_t page_shift;
    uint32_t* status;
    __device__ __forceinline__ uint32_t pages_for(uint32_t length) const { return static_cast<uint32_t>((static_cast<uint64_t>(length) + b.page_size - 1) >> page_shift); }
    __device__ __forceinline__ uint32_t most() const { return static_cast<uint32_t>(min(static_cast<uint64_t>(b.max_pages) << page_shift, static_cast<uint64_t>(0x7fffffffu))); }
    __device__ __forceinline__ int32_t* row(uint32_t slot) const { return b.tables + static_cast<size_t>(slot) * b.max_pages; }
    __device__ __forceinline__ uint32_t length(uint32_t slot) const { return static_cast<uint32_t>(min(max(b.lengths[slot], 0), static_cast<int>(most()))); }
    __device__ __forceinline__ void report(uint32_t bit) const { if (status != nullptr) atomicOr(status, bit); }
    // Adds to a page's count, which stays 0 or more; false for a page outside the pool, or one that would go below.
    __device__ __forceinline__ bool count(int page, int by) const {
        if (static_cast<uint32_t>(page) < b.pages) {
            if (atomicAdd(b.refs + page, by) + by >= 0) return true;
            atomicSub(b.refs + page, by);
        }
        report(B200KV_STATUS_BAD_PAGE);
        return false;
    }
};

// Exclusive sums over a block of kBookThreads in order, and the total.
__device__ __forceinline__ uint32_t scan_block(uint32_t v, uint32_t* total, uint32_t* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();   // the scratch of the scan before is read
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    uint32_t sums = scratch[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, sums, o);
        if (lane >= o) sums += u;
    }
    *total = __shfl_sync(0xffffffffu, sums, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0));
    return (warp > 0 ? before : 0) + inc - v;
}
static_assert(kBookThreads == 32 * 32);

struct TakeParams {
    Book book;
    bool fork;
    const int32_t* slots;      // grow: the sequences; fork: the children
    const int32_t* add;        // grow: new tokens
    const int32_t* parents;    // fork
    const int32_t* at;         // fork: positions that are taken over; may be null
    uint32_t count;
    // workspace
    uint32_t* pairs;           // fork: how many pages there are to copy
    int32_t* sources;
    int32_t* targets;          // the fresh pages
    int32_t* done;             // fork: an entry's length, -1 where it was refused
};

// An entry of a call.  Everything is read as it was before the call: nothing of it changes until all entries are looked at.
struct Entry {
    int slot;              // -1: refused, or left out
    uint32_t length, held, need;   // its new length, the pages it has (fork: shares), those it needs
};
__device__ __forceinline__ Entry entry_of(const TakeParams& p, uint32_t e, int slot, const int* owner, uint32_t* bad) {
    const Book& book = p.book;
    Entry x{-1, 0, 0, 0};
    if (slot < 0) return x;
    if (static_cast<uint32_t>(slot) >= book.b.slots || owner[slot] != static_cast<int>(e)) { *bad |= B200KV_STATUS_BAD_SLOT; return x; }
    if (p.fork) {
        const int parent = p.parents[e];
        if (static_cast<uint32_t>(parent) >= book.b.slots || book.b.lengths[slot] != 0) { *bad |= B200KV_STATUS_BAD_SLOT; return x; }
        x.length = book.length(parent);
        if (p.at != nullptr) x.length = min(x.length, static_cast<uint32_t>(max(p.at[e], 0)));
        x.held = x.length >> book.page_shift;
        x.need = book.pages_for(x.length) - x.held;
    } else {
        const uint32_t length = book.length(slot);
        const int add = p.add[e];
        if (add < 0 || static_cast<uint64_t>(length) + add > book.most()) { *bad |= B200KV_STATUS_BAD_BOUND; return x; }
        x.length = length + add;
        x.held = book.pages_for(length);
        x.need = book.pages_for(x.length) - x.held;
    }
    x.slot = slot;
    return x;
}

// One block: which pages every entry gets.  A chain of trips to L2, so what does not depend on one another is asked for together, and an entry's numbers stay in shared memory (looked up
// again at each step: 8.5 us cold for eight entries over a pool of 64 pages, in place of 7.5).
__global__ void __launch_bounds__(kBookThreads) pages_take_kernel(const __grid_constant__ TakeParams p) {
    extern __shared__ uint32_t shared[];
    __shared__ uint32_t scratch[32];
    // of each entry: its sequence, its new length, the pages it has, and the fresh pages before its own, cut off above the pool's number; of each slot: the first entry that names it
    int* const slot_of = reinterpret_cast<int*>(shared);
    uint32_t *const length_of = shared + p.count, *const held_of = shared + 2 * p.count, *const first = shared + 3 * p.count;
    int* const owner = reinterpret_cast<int*>(shared + 4 * p.count);
    const Book& book = p.book;
    const uint32_t tid = threadIdx.x, pages = book.b.pages;
    for (uint32_t s = tid; s < book.b.slots; s += kBookThreads) owner[s] = 0x7fffffff;
    pdl_wait();
    pdl_launch_dependents();
    // A thread's sixteen counts from `at` on: a bit a free page.
    const auto free_bits = [&](uint32_t at) {
        uint32_t free = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (at + 4 * i + 4 <= pages) {
                const int4 r = *reinterpret_cast<const int4*>(book.b.refs + at + 4 * i);
                free |= ((r.x == 0) | (r.y == 0) << 1 | (r.z == 0) << 2 | (r.w == 0) << 3) << (4 * i);
            } else {
                for (uint32_t x = at + 4 * i; x < pages; ++x) free |= (book.b.refs[x] == 0 ? 1u : 0u) << (x - at);
            }
        }
        return free;
    };
    const uint32_t first_bits = free_bits(tid * 16);
    __syncthreads();
    for (uint32_t e = tid; e < p.count; e += kBookThreads) {
        const int slot = p.slots[e];
        slot_of[e] = slot;
        if (static_cast<uint32_t>(slot) < book.b.slots) atomicMin(&owner[slot], static_cast<int>(e));
    }
    __syncthreads();
    uint32_t bad = 0, wanted = 0;
    for (uint32_t e0 = 0; e0 < p.count; e0 += kBookThreads) {
        const uint32_t e = e0 + tid;
        Entry x{-1, 0, 0, 0};
        if (e < p.count) {
            x = entry_of(p, e, slot_of[e], owner, &bad);
            slot_of[e] = x.slot;
            length_of[e] = x.length;
            held_of[e] = x.held;
        }
        uint32_t total;
        const uint32_t before = scan_block(min(x.need, pages + 1), &total, scratch);   // at most max_pages, of which 1024 are counted in 32 bits
        if (e < p.count) first[e] = static_cast<uint32_t>(min(static_cast<uint64_t>(wanted) + before, static_cast<uint64_t>(pages) + 1));
        wanted = static_cast<uint32_t>(min(static_cast<uint64_t>(wanted) + total, static_cast<uint64_t>(pages) + 1));
    }
    if (bad != 0) book.report(bad);
    // ---- the lowest free pages, as many as are wanted or there are
    uint32_t found = 0;
    for (uint32_t base = 0; base < pages && found < wanted; base += 4 * kChunk) {
        const uint32_t at = base + tid * 16;
        uint32_t free = base == 0 ? first_bits : free_bits(at);
        uint32_t total;
        uint32_t rank = found + scan_block(__popc(free), &total, scratch);
        for (; free != 0 && rank < wanted; free &= free - 1, ++rank) p.targets[rank] = static_cast<int>(at) + __ffs(free) - 1;
        found += total;
    }
    __syncthreads();
    const uint32_t granted = min(found, wanted);
    const auto need_of = [&](uint32_t e) { return slot_of[e] < 0 ? 0 : book.pages_for(length_of[e]) - held_of[e]; };
    // ---- a thread a page: the entry it belongs to, all of whose pages are there or none
    for (uint32_t k = tid; k < granted; k += kBookThreads) {
        uint32_t lo = 0, hi = p.count;   // the last entry with first <= k
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (first[mid] <= k) lo = mid;
            else hi = mid;
        }
        const uint32_t held = held_of[lo];
        const int page = p.targets[k];
        int source = -1;
        if (static_cast<uint64_t>(first[lo]) + need_of(lo) <= granted) {
            book.row(slot_of[lo])[held + (k - first[lo])] = page;
            book.b.refs[page] = 1;
            if (p.fork) source = book.row(p.parents[lo])[held];
            if (p.fork && static_cast<uint32_t>(source) >= pages) book.report(B200KV_STATUS_BAD_PAGE);
        }
        if (p.fork) {
            p.sources[k] = source;
            if (source < 0) p.targets[k] = -1;
        }
    }
    // lengths: all have been read
    for (uint32_t e = tid; e < p.count; e += kBookThreads) {
        int slot = slot_of[e];
        const uint32_t need = need_of(e);
        if (need > 0 && static_cast<uint64_t>(first[e]) + need > granted) {
            book.report(B200KV_STATUS_NO_PAGE);
            slot = -1;
        }
        if (p.fork) p.done[e] = slot < 0 ? -1 : static_cast<int>(length_of[e]);
        if (slot >= 0) book.b.lengths[slot] = static_cast<int>(length_of[e]);
    }
    if (p.fork && tid == 0) *p.pairs = granted;
}

struct ForkParams {
    Book book;
    const int32_t* parents;
    const int32_t* children;
    uint32_t count;
    const uint32_t* pairs;
    const int32_t* sources;
    const int32_t* targets;
    const int32_t* done;
};
// The rest of a fork: the children's rows of the table, the counts of what they share, the copies of their last pages.
template <uint32_t LAYERS>
__global__ void __launch_bounds__(kCopyThreads) pages_fork_kernel(const __grid_constant__ ForkParams p, const __grid_constant__ Planes<LAYERS> planes) {
    pdl_wait();
    pdl_launch_dependents();
    const Book& book = p.book;
    for (uint32_t e = blockIdx.x; e < p.count; e += gridDim.x) {
        const int length = p.done[e];
        if (length < 0) continue;
        const uint32_t whole = static_cast<uint32_t>(length) >> book.page_shift, held = book.pages_for(length);
        const int32_t* from = book.row(p.parents[e]);
        int32_t* to = book.row(p.children[e]);
        for (uint32_t c = threadIdx.x; c < book.b.max_pages; c += kCopyThreads) {
            if (c < whole) {
                const int page = from[c];
                to[c] = page;
                book.count(page, 1);
            } else if (c >= held) {
                to[c] = -1;
            }
        }
    }
    copy_pages(planes, p.sources, p.targets, *p.pairs);
}

struct FreeParams {
    Book book;
    const int32_t* slots;
};
// A block an entry.  Whoever exchanges the length for 0 gives the pages back, so that a slot named twice is freed once.
__global__ void __launch_bounds__(128) pages_free_kernel(const __grid_constant__ FreeParams p) {
    __shared__ int length;
    pdl_wait();
    pdl_launch_dependents();
    const Book& book = p.book;
    const int slot = p.slots[blockIdx.x];
    if (slot < 0) return;
    if (static_cast<uint32_t>(slot) >= book.b.slots) {
        if (threadIdx.x == 0) book.report(B200KV_STATUS_BAD_SLOT);
        return;
    }
    if (threadIdx.x == 0) length = atomicExch(book.b.lengths + slot, 0);
    __syncthreads();
    const uint32_t held = book.pages_for(static_cast<uint32_t>(min(max(length, 0), static_cast<int>(book.most()))));
    int32_t* row = book.row(slot);
    for (uint32_t c = threadIdx.x; c < held; c += 128) {
        book.count(row[c], -1);
        row[c] = -1;
    }
}

// ---- compaction --------------------------------------------------------------------------------------------------------------------

struct CompactParams {
    Book book;
    int32_t* moved;        // of every page: where it is now, -1 for a free one
    uint32_t chunks;
    // workspace
    uint32_t* live;        // pages that are held, of every chunk
    uint32_t* pairs;       // how many move
    int32_t* movers;       // which, ascending
    int32_t* holes;        // and where to, ascending
    int32_t* ranks;        // of a page that moves: its number among them
};

// A thread's four counts of a chunk, a bit a page that is held.
__device__ __forceinline__ uint32_t held_bits(const Book& book, uint32_t at) {
    uint32_t held = 0;
    if (at + 4 <= book.b.pages) {
        const int4 r = *reinterpret_cast<const int4*>(book.b.refs + at);
        held = (r.x != 0) | (r.y != 0) << 1 | (r.z != 0) << 2 | (r.w != 0) << 3;
    } else {
        for (uint32_t x = at; x < book.b.pages; ++x) held |= (book.b.refs[x] != 0 ? 1u : 0u) << (x - at);
    }
    return held;
}

__global__ void __launch_bounds__(kBookThreads) pages_live_kernel(const __grid_constant__ CompactParams p) {
    __shared__ uint32_t scratch[32];
    pdl_wait();
    pdl_launch_dependents();
    uint32_t total;
    scan_block(__popc(held_bits(p.book, blockIdx.x * kChunk + threadIdx.x * 4)), &total, scratch);
    if (threadIdx.x == 0) p.live[blockIdx.x] = total;
}

// A block a chunk: with n pages held, the k-th free page below n takes the k-th held page at or above n.
__global__ void __launch_bounds__(kBookThreads) pages_rank_kernel(const __grid_constant__ CompactParams p) {
    __shared__ uint32_t scratch[32];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t tid = threadIdx.x, me = blockIdx.x, at = me * kChunk + tid * 4, held = held_bits(p.book, at);
    uint32_t mine = 0, all = 0, below = 0, before;   // held in the chunks before this one, in all, below page `all`, and before the thread's own
    const auto lower = [&](uint32_t from) { return from >= all ? 0u : all - from >= 4 ? 15u : (1u << (all - from)) - 1; };   // which of four pages lie below `all`
    if (p.chunks == 1) {
        __shared__ uint32_t below_all;
        before = scan_block(__popc(held), &all, scratch);
        if (at <= all && (all < at + 4 || tid == kBookThreads - 1)) below_all = before + __popc(held & lower(at));   // one thread's, the last one's where a whole chunk is held
        __syncthreads();
        below = below_all;
    } else {
        uint32_t total;
        for (uint32_t c0 = 0; c0 < p.chunks; c0 += kBookThreads) {
            const uint32_t c = c0 + tid, n = c < p.chunks ? p.live[c] : 0;
            scan_block(c < me ? n : 0, &total, scratch);
            mine += total;
            scan_block(n, &total, scratch);
            all += total;
        }
        // below page `all`: those of the chunks before it, and of its own
        const uint32_t edge = all / kChunk;
        for (uint32_t c0 = 0; c0 < p.chunks && c0 < edge; c0 += kBookThreads) {
            scan_block(c0 + tid < min(edge, p.chunks) ? p.live[c0 + tid] : 0, &total, scratch);
            below += total;
        }
        if (edge < p.chunks) {
            const uint32_t from = edge * kChunk + tid * 4;
            scan_block(__popc(held_bits(p.book, from) & lower(from)), &total, scratch);
            below += total;
        }
        before = mine + scan_block(__popc(held), &total, scratch);
    }
    for (uint32_t i = 0; i < 4 && at + i < p.book.b.pages; ++i) {
        const uint32_t page = at + i;
        if ((held >> i) & 1) {
            const uint32_t rank = before - below;
            if (page < all) {
                p.moved[page] = static_cast<int>(page);
            } else if (rank < p.book.b.pages) {   // (always, but for counts that somebody else changes meanwhile)
                p.movers[rank] = static_cast<int>(page);
                p.ranks[page] = static_cast<int>(rank);
            }
            ++before;
        } else {
            p.moved[page] = -1;
            if (page < all && page - before < p.book.b.pages) p.holes[page - before] = static_cast<int>(page);
        }
    }
    if (me == 0 && tid == 0) *p.pairs = min(all - below, p.book.b.pages / 2);   // no more than half of the pages can move
}

// The pages move, in all layers, and with them their counts and the table's entries.
template <uint32_t LAYERS>
__global__ void __launch_bounds__(kCopyThreads) pages_move_kernel(const __grid_constant__ CompactParams p, const __grid_constant__ Planes<LAYERS> planes) {
    pdl_wait();
    pdl_launch_dependents();
    const Book& book = p.book;
    const uint32_t pairs = *p.pairs;
    if (pairs == 0) return;
    // The counts of the pages that move are other words than those of the holes, and nothing else here reads either.  A page lies at or above the number of those held
    // and below the pool's exactly if it moves (a free one there is in no table).
    const uint32_t threads = gridDim.x * kCopyThreads, me = blockIdx.x * kCopyThreads + threadIdx.x;
    for (uint32_t k = me; k < pairs; k += threads) {
        const int source = p.movers[k], target = p.holes[k];
        if (static_cast<uint32_t>(source) >= book.b.pages || static_cast<uint32_t>(target) >= book.b.pages) continue;   // as above
        book.b.refs[target] = book.b.refs[source];
        book.b.refs[source] = 0;
        p.moved[source] = target;
    }
    const int first = p.movers[0];
    for (uint32_t s = blockIdx.x; s < book.b.slots; s += gridDim.x) {
        const uint32_t held = book.pages_for(book.length(s));
        int32_t* row = book.row(s);
        for (uint32_t c = threadIdx.x; c < held; c += kCopyThreads) {
            const int page = row[c];
            if (static_cast<uint32_t>(page) >= book.b.pages) { book.report(B200KV_STATUS_BAD_PAGE); continue; }
            if (page < first) continue;
            const uint32_t rank = static_cast<uint32_t>(p.ranks[page]);
            if (rank < pairs && p.movers[rank] == page) row[c] = p.holes[rank];
            else book.report(B200KV_STATUS_BAD_PAGE);   // a free page in a table
        }
    }
    copy_pages(planes, p.movers, p.holes, pairs);
}

// ---- host --------------------------------------------------------------------------------------------------------------------------

bool same_geometry(const b200kv_paged_view& a, const b200kv_paged_view& b) {
    return a.page_size == b.page_size && a.kv_heads == b.kv_heads && a.head_dim == b.head_dim && a.qblock == b.qblock && a.quant_mode == b.quant_mode;
}
int validate_views(const b200kv_paged_view* views, uint32_t layers) {
    if (views == nullptr || layers == 0) return B200KV_ERR_INVALID;
    if (layers > kMostLayers) return B200KV_ERR_UNSUPPORTED;
    const b200kv_paged_batch none{};
    for (uint32_t l = 0; l < layers; ++l) {
        const int rc = validate_paged(views + l, &none);
        if (rc != B200KV_OK) return rc;
        if (!same_geometry(views[l], views[0]) || views[l].pages != views[0].pages) return B200KV_ERR_INVALID;
    }
    // a page of a plane is counted in 32 bits
    return static_cast<uint64_t>(views[0].kv_heads) * views[0].page_size * views[0].head_dim * 2 > 0x7fffffffull ? B200KV_ERR_UNSUPPORTED : B200KV_OK;
}
int validate_book(const b200kv_page_book* b) {
    if (b == nullptr || b->pages == 0 || b->slots == 0 || b->max_pages == 0) return B200KV_ERR_INVALID;
    if (b->page_size < 16 || b->page_size > 256 || (b->page_size & (b->page_size - 1)) != 0) return B200KV_ERR_UNSUPPORTED;
    if (b->pages > 0x7ffffff0u || b->slots > kMostSequences || b->max_pages > 0x3fffffu) return B200KV_ERR_UNSUPPORTED;
    const auto given = [](const void* p, uintptr_t align) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (align - 1)) == 0; };
    if (!given(b->refs, 16) || !given(b->tables, 4) || !given(b->lengths, 4)) return B200KV_ERR_INVALID;
    return B200KV_OK;
}
int validate_book_views(const b200kv_page_book* book, const b200kv_paged_view* views, uint32_t layers) {
    int rc = validate_book(book);
    if (rc == B200KV_OK) rc = validate_views(views, layers);
    if (rc == B200KV_OK && (views[0].pages != book->pages || views[0].page_size != book->page_size)) rc = B200KV_ERR_INVALID;
    return rc;
}
Book book_of(const b200kv_page_book& b) {
    Book book{b, 0, current_status_word()};
    while ((1u << book.page_shift) < b.page_size) ++book.page_shift;
    return book;
}
bool words(const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
// Whether `count` words at p lie over any of the book's arrays.
bool over_book(const b200kv_page_book& b, const void* p, uint64_t count) {
    return p != nullptr && (share(p, count * 4, b.refs, b.pages * 4ull) || share(p, count * 4, b.lengths, b.slots * 4ull) ||
                            share(p, count * 4, b.tables, static_cast<uint64_t>(b.slots) * b.max_pages * 4));
}

template <uint32_t LAYERS>
Planes<LAYERS> planes_of(const b200kv_paged_view* from, const b200kv_paged_view* to, uint32_t layers) {
    Planes<LAYERS> p{};
    const b200kv_paged_view& v = from[0];
    const uint32_t rows = v.kv_heads * v.page_size, scales = rows * (v.head_dim / v.qblock) * 2;
    p.layers = layers;
    p.from_pages = v.pages;
    p.to_pages = to[0].pages;
    p.status = current_status_word();
    for (int side = 0; side < 2; ++side) {
        const bool q8 = side == 0 ? is_k_q8(v.quant_mode) : is_v_q8(v.quant_mode);
        p.bytes[p.planes] = rows * v.head_dim * (q8 ? 1 : 2);
        const uint32_t plane = p.planes++, plane_scales = q8 ? p.planes++ : 0;
        if (q8) p.bytes[plane_scales] = scales;
        for (uint32_t l = 0; l < layers; ++l)
            for (const bool target : {false, true}) {
                const b200kv_paged_view& x = target ? to[l] : from[l];
                uint8_t* data = static_cast<uint8_t*>(side == 0 ? (q8 ? x.key_q8 : x.key_f16) : (q8 ? x.value_q8 : x.value_f16));
                uint8_t* of_scales = static_cast<uint8_t*>(side == 0 ? x.key_scales : x.value_scales);
                if (target) {
                    p.to[l][plane] = data;
                    if (q8) p.to[l][plane_scales] = of_scales;
                } else {
                    p.from[l][plane] = data;
                    if (q8) p.from[l][plane_scales] = of_scales;
                }
            }
    }
    for (uint32_t i = 0; i < p.planes; ++i) p.layer_pieces += p.pieces[i] = (p.bytes[i] + kPiece - 1) / kPiece;
    return p;
}

// A grid for copies of up to `pages` pages: eight blocks an SM, or as many as there is work for.
template <uint32_t LAYERS>
uint32_t copy_grid(const Planes<LAYERS>& p, uint64_t pages) {
    const uint64_t warps = pages * p.layers * p.layer_pieces;
    return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>((warps + kCopyThreads / 32 - 1) / (kCopyThreads / 32), 8ull * device_sms())));
}

struct Room {
    size_t live, done, sources, targets, ranks, bytes;   // offsets, behind the number of pairs
};
Room room_of(const b200kv_page_book& b) {
    Room r{};
    size_t at = 256;
    const auto take = [&](uint64_t n) { const size_t here = at; at += (n * 4 + 255) / 256 * 256; return here; };
    r.live = take((b.pages + static_cast<uint64_t>(kChunk) - 1) / kChunk);
    r.done = take(b.slots);
    r.sources = take(b.pages);
    r.targets = take(b.pages);
    r.ranks = take(b.pages);
    r.bytes = at;
    return r;
}
// A call's workspace, which lies over none of the book's arrays, nor over its entries' (of `count` words each; may be null).
int check_workspace(const b200kv_page_book& book, const void* workspace, size_t bytes, std::initializer_list<const void*> entries = {}, uint64_t count = 0) {
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return B200KV_ERR_INVALID;
    const size_t room = room_of(book).bytes;
    if (workspace == nullptr || bytes < room) return B200KV_ERR_WORKSPACE;
    for (const void* array : entries)
        if (array != nullptr && share(workspace, room, array, count * 4)) return B200KV_ERR_INVALID;
    return over_book(book, workspace, room / 4) ? B200KV_ERR_INVALID : B200KV_OK;
}

int launch_take(const TakeParams& p, cudaStream_t stream) {
    const size_t smem = (4 * static_cast<size_t>(p.count) + p.book.b.slots) * 4;
    static std::atomic<uint64_t> done{0};
    if (smem > 40 * 1024) B200KV_CUDA_TRY(opt_in_dynamic_smem(reinterpret_cast<const void*>(pages_take_kernel), 5 * kMostSequences * 4, done));
    B200KV_CUDA_TRY(launch_kernel(pages_take_kernel, dim3(1), dim3(kBookThreads), smem, stream, true, p));
    return B200KV_OK;
}

template <uint32_t LAYERS>
int launch_copy(const b200kv_paged_view* from, const b200kv_paged_view* to, uint32_t layers, const int32_t* sources, const int32_t* targets, uint32_t count, cudaStream_t s) {
    const Planes<LAYERS> planes = planes_of<LAYERS>(from, to, layers);
    B200KV_CUDA_TRY(launch_kernel(pages_copy_kernel<LAYERS>, dim3(copy_grid(planes, count)), dim3(kCopyThreads), 0, s, true, planes, sources, targets, count));
    return B200KV_OK;
}
template <uint32_t LAYERS>
int launch_fork(const ForkParams& p, const b200kv_paged_view* views, uint32_t layers, cudaStream_t s) {
    const Planes<LAYERS> planes = planes_of<LAYERS>(views, views, layers);
    const uint32_t grid = std::max(copy_grid(planes, p.count), std::min(p.count, 8 * device_sms()));
    B200KV_CUDA_TRY(launch_behind(pages_fork_kernel<LAYERS>, dim3(grid), dim3(kCopyThreads), 0, s, p, planes));
    return B200KV_OK;
}
template <uint32_t LAYERS>
int launch_move(const CompactParams& p, const b200kv_paged_view* views, uint32_t layers, cudaStream_t s) {
    const Planes<LAYERS> planes = planes_of<LAYERS>(views, views, layers);
    const uint32_t grid = std::max(copy_grid(planes, p.book.b.pages / 2), std::min(p.book.b.slots, 8 * device_sms()));   // no more than half of the pages can move
    B200KV_CUDA_TRY(launch_behind(pages_move_kernel<LAYERS>, dim3(grid), dim3(kCopyThreads), 0, s, p, planes));
    return B200KV_OK;
}

}  // namespace

}  // namespace b200kv

using namespace b200kv;

extern "C" {

size_t b200kv_pages_workspace_bytes(const b200kv_page_book* book) { return validate_book(book) == B200KV_OK ? room_of(*book).bytes : 0; }

int b200kv_pages_copy(const b200kv_paged_view* from, const b200kv_paged_view* to, uint32_t layers, const int32_t* sources, const int32_t* targets, uint32_t count, void* stream) {
    int rc = validate_views(from, layers);
    if (rc == B200KV_OK) rc = validate_views(to, layers);
    if (rc != B200KV_OK) return rc;
    if (!same_geometry(from[0], to[0])) return B200KV_ERR_INVALID;
    if (count == 0) return B200KV_OK;
    if (!words(sources) || !words(targets) || count > 0x7fffffffu) return B200KV_ERR_INVALID;
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return layers <= kFewLayers ? launch_copy<kFewLayers>(from, to, layers, sources, targets, count, s) : launch_copy<kMostLayers>(from, to, layers, sources, targets, count, s);
}

int b200kv_pages_grow(const b200kv_page_book* book, const int32_t* slots, const int32_t* add, uint32_t count, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = validate_book(book);
    if (rc != B200KV_OK) return rc;
    if (count == 0) return B200KV_OK;
    if (!words(slots) || !words(add) || count > kMostSequences || over_book(*book, slots, count) || over_book(*book, add, count)) return B200KV_ERR_INVALID;
    rc = check_workspace(*book, workspace, workspace_bytes, {slots, add}, count);
    if (rc == B200KV_OK) rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    const Room room = room_of(*book);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    return launch_take(TakeParams{book_of(*book), false, slots, add, nullptr, nullptr, count, nullptr, nullptr, reinterpret_cast<int32_t*>(ws + room.targets), nullptr},
                       static_cast<cudaStream_t>(stream));
}

int b200kv_pages_fork(const b200kv_page_book* book, const b200kv_paged_view* views, uint32_t layers, const int32_t* parents, const int32_t* children, const int32_t* at,
                      uint32_t count, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = validate_book_views(book, views, layers);
    if (rc != B200KV_OK) return rc;
    if (count == 0) return B200KV_OK;
    // an entry's result lies in a place of its own in the workspace, which has as many as there are slots
    if (!words(parents) || !words(children) || (at != nullptr && !words(at)) || count > book->slots) return B200KV_ERR_INVALID;
    if (over_book(*book, parents, count) || over_book(*book, children, count) || over_book(*book, at, count)) return B200KV_ERR_INVALID;
    rc = check_workspace(*book, workspace, workspace_bytes, {parents, children, at}, count);
    if (rc == B200KV_OK) rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    const Room room = room_of(*book);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const auto ints = [&](size_t offset) { return reinterpret_cast<int32_t*>(ws + offset); };
    const TakeParams take{book_of(*book), true, children, nullptr, parents, at, count, reinterpret_cast<uint32_t*>(ws), ints(room.sources), ints(room.targets), ints(room.done)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    rc = launch_take(take, s);
    if (rc != B200KV_OK) return rc;
    const ForkParams p{take.book, parents, children, count, take.pairs, take.sources, take.targets, take.done};
    return layers <= kFewLayers ? launch_fork<kFewLayers>(p, views, layers, s) : launch_fork<kMostLayers>(p, views, layers, s);
}

int b200kv_pages_free(const b200kv_page_book* book, const int32_t* slots, uint32_t count, void* stream) {
    int rc = validate_book(book);
    if (rc != B200KV_OK) return rc;
    if (count == 0) return B200KV_OK;
    if (!words(slots) || count > 0x7fffffffu || over_book(*book, slots, count)) return B200KV_ERR_INVALID;
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    B200KV_CUDA_TRY(launch_kernel(pages_free_kernel, dim3(count), dim3(128), 0, static_cast<cudaStream_t>(stream), true, FreeParams{book_of(*book), slots}));
    return B200KV_OK;
}

int b200kv_pages_compact(const b200kv_page_book* book, const b200kv_paged_view* views, uint32_t layers, int32_t* moved, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = validate_book_views(book, views, layers);
    if (rc != B200KV_OK) return rc;
    if (!words(moved) || over_book(*book, moved, book->pages) || (workspace != nullptr && share(moved, book->pages * 4ull, workspace, room_of(*book).bytes))) return B200KV_ERR_INVALID;
    rc = check_workspace(*book, workspace, workspace_bytes);
    if (rc == B200KV_OK) rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    const Room room = room_of(*book);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const auto ints = [&](size_t offset) { return reinterpret_cast<int32_t*>(ws + offset); };
    const uint32_t chunks = (book->pages + kChunk - 1) / kChunk;
    const CompactParams p{book_of(*book), moved, chunks, reinterpret_cast<uint32_t*>(ws + room.live), reinterpret_cast<uint32_t*>(ws), ints(room.sources), ints(room.targets), ints(room.ranks)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (chunks == 1) {
        B200KV_CUDA_TRY(launch_kernel(pages_rank_kernel, dim3(1), dim3(kBookThreads), 0, s, true, p));
    } else {
        B200KV_CUDA_TRY(launch_kernel(pages_live_kernel, dim3(chunks), dim3(kBookThreads), 0, s, true, p));
        B200KV_CUDA_TRY(launch_behind(pages_rank_kernel, dim3(chunks), dim3(kBookThreads), 0, s, p));
    }
    return layers <= kFewLayers ? launch_move<kFewLayers>(p, views, layers, s) : launch_move<kMostLayers>(p, views, layers, s);
}

}  // extern "C"
