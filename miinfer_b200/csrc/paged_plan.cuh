// The work of one attention call over a paged cache, laid out on the device by the call's first kernel (paged_attn.cu) and read by the others: the host
// knows bounds only, the lengths are device memory.
#pragma once

#include "paged_common.cuh"

namespace b200kv {

constexpr uint32_t kChunkRows = 128;       // query rows of a row tile
constexpr uint32_t kChunkTile = 64;        // positions of a KV tile
constexpr uint32_t kNoPart = 0xffffffffu;

// What one CTA of the chunk kernel does: one row tile of one sequence and kv head, over some of its KV tiles.  A sequence's tiles are those of its
// copy in the scratch: first the tiles of the sinks, if the window leaves a gap behind them, then those from position `window0` on.
struct alignas(16) ChunkItem {   // written and read 16 bytes at a time
    uint32_t first, tokens;    // the sequence's rows of the activations
    int32_t base;              // place in the cache of its first new token
    uint32_t row_tile, kv_head;
    uint32_t scratch_row;      // of the sequence's first tile
    uint32_t sink_tiles, window0;
    uint32_t skip;             // tiles behind the sinks' that this row tile does not see
    uint32_t tile0, tiles;     // its tiles, counted without those
    uint32_t part;             // where its unnormalised partial goes; kNoPart: it writes the output itself
    uint32_t parts;            // how many share the row tile (a partial's own number is part - the first one's)
    uint32_t length;           // of the sequence
    uint32_t pad_[2];
};
static_assert(sizeof(ChunkItem) == 64);

struct ChunkPlan {
    uint32_t items, groups;
};

// Where a sequence's tiles lie in the cache.
struct ChunkTiles {
    uint32_t sink_tiles, window0;   // as in ChunkItem
    uint32_t tiles;                 // all of the sequence's
};
__host__ __device__ inline ChunkTiles chunk_tiles(int base, uint32_t length, uint32_t window, uint32_t sinks) {
    ChunkTiles t{0, 0, (length + kChunkTile - 1) / kChunkTile};
    if (window == 0) return t;
    const long long lowest = static_cast<long long>(base) + 1 - window;   // of the positions in the first token's window
    const uint32_t first = lowest > 0 ? static_cast<uint32_t>(lowest) / kChunkTile : 0, sink = (sinks + kChunkTile - 1) / kChunkTile;
    if (first <= sink) return t;
    t.sink_tiles = sink;
    t.window0 = first * kChunkTile;
    t.tiles = sink + (t.tiles > first ? t.tiles - first : 0);
    return t;
}

// The same where tokens have ranges of their own: all that any of them sees lies in [lowest, end) or is among the sinks below end.
__host__ __device__ inline ChunkTiles chunk_tiles_between(uint32_t lowest, uint32_t end, uint32_t sinks) {
    ChunkTiles t{0, 0, (end + kChunkTile - 1) / kChunkTile};
    const uint32_t first = lowest / kChunkTile, sink = ((sinks < end ? sinks : end) + kChunkTile - 1) / kChunkTile;
    if (first <= sink) return t;
    t.sink_tiles = sink;
    t.window0 = first * kChunkTile;
    t.tiles = sink + (t.tiles > first ? t.tiles - first : 0);
    return t;
}
// The slot of row tile r of sequence s among those of all sequences: as many as there can be, and each its own where the starts ascend.
__host__ __device__ inline size_t chunk_slot(uint32_t first, uint32_t group, uint32_t s, uint32_t r) { return static_cast<size_t>(static_cast<uint64_t>(first) * group / kChunkRows) + s + r; }

// Work of n row tiles of a sequence, in 128ths of a tile: tokens of a chunk see on average half of it.
__host__ __device__ inline unsigned long long chunk_work(uint32_t n, uint32_t tiles, uint32_t tokens) {
    const unsigned long long half = 64ull * tiles;
    return n * (2 * half - (half < tokens ? half : tokens));
}

// The chunk kernel's launch.
struct ChunkLaunch {
    const ChunkItem* items;
    const ChunkPlan* plan;
    uint32_t max_items;
    const __half* k_scratch;   // [kv_head][scratch_rows][head_dim]
    const __half* v_scratch;
    uint32_t scratch_rows;
    const void* q;
    int q_is_f16;
    const float* gate;
    void* out;
    int out_is_f16;
    float* lse;
    uint32_t query_heads, kv_heads, head_dim, window, sinks;
    float scale_log2;
    float* part_o;             // [part][kChunkRows][head_dim]
    float2* part_ml;           // [part][kChunkRows] {maximum in log2 units, sum}
    bool scored;               // with what follows
    float cap, scale;          // scores of at most cap; 0: any
    const float* slopes;       // [query_heads], may be null
    const int32_t* ranges;     // [total_tokens][2], may be null
};
int launch_chunk(const ChunkLaunch& c, cudaStream_t stream);

}  // namespace b200kv
