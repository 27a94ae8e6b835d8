// The list of tiles that the streaming kernels over a paged cache deal out to their CTAs: all tiles of 128 positions of all (sequence, kv head) pairs, in equal
// pieces.  Sequences and what they see are device memory, so every CTA finds its piece itself.
//
// A kernel's parameters P say what is in the list: P.pool, P.tiles_of(span) (a sequence's tiles, the same for each of its kv heads) and P.ctas.
#pragma once

#include "paged_common.cuh"

namespace b200kv {

constexpr uint32_t kDecodeTile = 128;      // positions of a tile
constexpr uint32_t kMostSms = 160;         // what workspaces are sized for, on any device; launches use no more

// A sequence's tiles: those of the sinks, if the window leaves a gap behind them, then those from tile `first` on.
struct Tiles {
    uint32_t n, sink, first;
    __device__ __forceinline__ uint32_t position(uint32_t j) const {   // first position of tile j of the list
        return (j < sink ? j : first + (j - sink)) * kDecodeTile;
    }
};
// What tokens from the one at cache place `place` on see of `length` positions.
__device__ __forceinline__ Tiles tiles_seen(long long place, uint32_t length, uint32_t window, uint32_t sinks) {
    const uint32_t all = (length + kDecodeTile - 1) / kDecodeTile;
    if (window == 0) return {all, 0, 0};
    const long long lowest = place + 1 - window;
    const uint32_t first = lowest > 0 ? static_cast<uint32_t>(lowest) / kDecodeTile : 0, sink = (sinks + kDecodeTile - 1) / kDecodeTile;
    if (first <= sink || first >= all) return {all, 0, 0};
    return {sink + all - first, sink, first};
}

// Tiles of all pairs before sequence s (up to the number of sequences: of all); a warp.
template <class P>
__device__ __forceinline__ uint64_t tiles_before(const P& p, uint32_t s, int lane) {
    uint64_t sum = 0;
    for (uint32_t i = lane; i < s; i += 32) sum += p.tiles_of(span_of(p.pool, i)).n;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum * p.pool.view.kv_heads;
}

// CTAs that have a piece, and where piece c begins: the first all % pieces of them have a tile more.
template <class P>
__device__ __forceinline__ uint32_t pieces_of(const P& p, uint64_t all) {
    return static_cast<uint32_t>(min(static_cast<uint64_t>(p.ctas), max(static_cast<uint64_t>(1), all)));
}
__device__ __forceinline__ uint64_t piece_begin(uint64_t all, uint32_t c, uint32_t pieces) {
    const uint64_t each = all / pieces, more = all % pieces;
    return c * each + min(static_cast<uint64_t>(c), more);
}

// The piece that holds tile w.
__device__ __forceinline__ uint32_t piece_with(uint64_t all, uint64_t w, uint32_t pieces) {
    const uint64_t each = all / pieces, more = all % pieces, bound = more * (each + 1);
    return static_cast<uint32_t>(w < bound ? w / (each + 1) : more + (w - bound) / each);
}

// CTA c's piece, by a warp: start = {sequence, kv head, tile, tiles of the piece (two words), tiles of the list (two words)}.
template <class P>
__device__ __forceinline__ void find_piece(const P& p, uint32_t c, int lane, uint32_t* start) {
    const uint32_t S = p.pool.batch.sequences, H = p.pool.view.kv_heads;
    constexpr uint32_t kOnce = 4;   // up to 128 sequences are looked up once, their loads together
    uint32_t mine_n[kOnce];
    uint64_t all = 0;
    if (S <= 32 * kOnce) {
        Span spans[kOnce];
#pragma unroll
        for (uint32_t x = 0; x < kOnce; ++x) spans[x] = span_of(p.pool, min(32 * x + lane, S - 1));
#pragma unroll
        for (uint32_t x = 0; x < kOnce; ++x) {
            mine_n[x] = 32 * x + lane < S ? p.tiles_of(spans[x]).n : 0;
            all += mine_n[x];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        all *= H;
    } else {
        all = tiles_before(p, S, lane);
    }
    const uint32_t pieces = pieces_of(p, all);
    uint64_t begin = 0, count = 0;
    if (all > 0 && c < pieces) {
        begin = piece_begin(all, c, pieces);
        count = piece_begin(all, c + 1, pieces) - begin;
    }
    if (count > 0) {
        uint64_t before = 0;   // the sequence in which it begins, 32 at a time
        for (uint32_t s0 = 0; s0 < S; s0 += 32) {
            const uint32_t s = s0 + lane;
            uint32_t n = 0;
            if (S <= 32 * kOnce) {
#pragma unroll
                for (uint32_t x = 0; x < kOnce; ++x)
                    if (s0 == 32 * x) n = mine_n[x];
            } else if (s < S) {
                n = p.tiles_of(span_of(p.pool, s)).n;
            }
            uint64_t inc = static_cast<uint64_t>(n) * H;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t u = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += u;
            }
            const uint64_t mine = before + inc - static_cast<uint64_t>(n) * H;
            if (n > 0 && begin >= mine && begin < before + inc) {
                start[0] = s;
                start[1] = static_cast<uint32_t>((begin - mine) / n);
                start[2] = static_cast<uint32_t>((begin - mine) % n);
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
            if (begin < before) break;
        }
    }
    if (lane == 0) {
        start[3] = static_cast<uint32_t>(count);
        start[4] = static_cast<uint32_t>(count >> 32);
        start[5] = static_cast<uint32_t>(all);
        start[6] = static_cast<uint32_t>(all >> 32);
    }
}

// A place in the list, and how much of the piece is left from there.
struct Cursor {
    uint32_t s, head, tile;
    uint64_t left;
    Span span;
    Tiles t;
    template <class P>
    __device__ __forceinline__ Cursor(const P& p, const uint32_t* start) : s(start[0]), head(start[1]), tile(start[2]), left(start[3] | static_cast<uint64_t>(start[4]) << 32) {
        if (left > 0) settle(p);
    }
    template <class P>
    __device__ __forceinline__ void settle(const P& p) {   // the pair's sequence
        span = span_of(p.pool, s);
        t = p.tiles_of(span);
    }
    __device__ __forceinline__ uint32_t take() const { return static_cast<uint32_t>(min(left, static_cast<uint64_t>(t.n - tile))); }   // tiles of this pair
    template <class P>
    __device__ __forceinline__ void advance(const P& p) {  // to the next pair that has tiles
        left -= take();
        tile = 0;
        if (left == 0 || ++head < p.pool.view.kv_heads) return;
        head = 0;
        do {
            ++s;
            settle(p);
        } while (t.n == 0 && s + 1 < p.pool.batch.sequences);
    }
};

}  // namespace b200kv
