// The tokens-a-few attention over a paged cache (paged_decode.cu) as the entry point launches it.
#pragma once

#include "paged_tiles.cuh"

#include <cuda.h>

namespace b200kv {

constexpr uint32_t kDecodeRows = 8;        // query rows (tokens x heads of a kv head) of a sequence that this kernel takes

struct PagedDecode {
    Paged pool;
    const void* q;             // [total_tokens][query_heads][head_dim]
    int q_is_f16;
    const float* gate;         // may be null
    void* out;
    int out_is_f16;
    float* lse;                // may be null
    uint32_t query_heads, window, sinks;
    uint32_t rows;             // sequences of at most so many query rows are this launch's: 4 or 8
    float scale_log2;
    uint32_t ctas;             // of the launch: the tiles of all sequences are dealt to them in equal pieces
    float* part_o;             // [2 ctas][kDecodeRows][head_dim]: a CTA's piece begins and ends inside a kv head's tiles at most once each
    float2* part_ml;           // [2 ctas][kDecodeRows] {maximum in log2 units, sum}
    uint4* shared;             // [ctas]: the pair that begins in a CTA's piece and ends in another's: sequence, kv head, the other CTA, 1 (0: there is none)
    __device__ __forceinline__ Tiles tiles_of(const Span& span) const {
        if (span.tokens == 0 || span.tokens > kDecodeRows || span.tokens * (query_heads / pool.view.kv_heads) > rows) return {0, 0, 0};
        Tiles t = tiles_seen(span.base(), span.length, window, sinks);
        t.n = max(t.n, 1u);    // one tile where there is no position: the rows that see nothing come out as zeros
        return t;
    }
};

// Whether the sequences of a batch can all be of this kernel, and whether any can be.
inline bool decode_takes_all(const b200kv_paged_batch& b, uint32_t group) { return static_cast<uint64_t>(b.max_tokens) * group <= kDecodeRows; }
// The rows of the launch: four where they are enough for all sequences, or, beside the chunk kernel, for a token.  (Four rows leave room for two CTAs an SM of int8
// sides, 32 / 8 heads of 128: one token of 64 sequences of 4000 116 us with four, 153 with eight; beside a chunk of 40, of 39 129 and 145.  fp16 197 and 185, 170 and 168.)
inline uint32_t decode_rows(const b200kv_paged_batch& b, uint32_t group) { return group <= 4 && (b.max_tokens * static_cast<uint64_t>(group) <= 4 || !decode_takes_all(b, group)) ? 4 : kDecodeRows; }
uint32_t decode_ctas(const b200kv_paged_view& view, uint32_t sms);     // at most
size_t decode_part_bytes(const b200kv_paged_view& view, uint32_t sms);
int launch_paged_decode(PagedDecode p, void* parts, cudaStream_t stream, bool behind);

// A tensor map over a pool's plane as rows of head_dim: boxes of 128 bytes by `box_rows` rows, 128-byte swizzle.
bool encode_pool_map(CUtensorMap* map, const void* plane, bool f16, uint64_t rows, uint32_t head_dim, uint32_t box_rows);
// One over fp16 activations [tokens][heads][head_dim]: boxes of 64 dims of `box_heads` heads of `box_tokens` tokens, 128-byte swizzle.
bool encode_rows_map(CUtensorMap* map, const void* rows, uint32_t head_dim, uint32_t heads, uint32_t tokens, uint32_t box_heads, uint32_t box_tokens);

}  // namespace b200kv
