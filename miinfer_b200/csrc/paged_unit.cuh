// What the streaming kernels over a paged cache put into shared memory for their MMAs: units of 128 cache rows, and the query rows of a pair.
#pragma once

#include "decode_common.cuh"
#include "paged_mma.cuh"
#include "paged_tiles.cuh"

namespace b200kv {

namespace {

template <int D, int FMT>
struct Unit {   // 128 rows of K or V: slabs of 128 bytes of every row, 128-byte swizzle; the scales in a place of their own
    static constexpr int kRow = FMT == F16 ? 2 * D : D, kSlabs = kRow / 128, kScale = FMT == F16 ? 0 : FMT == BLOCK ? D / 16 : 2;   // bytes
    static constexpr int kData = kDecodeTile * kRow, kScales = kDecodeTile * kScale;
};

// A tile's boxes, of which a lane has one: the rows of a page, or of 128 positions of a larger one.
struct Boxes {
    long long row;             // the lane's first row; negative where there is none
    uint32_t seg;              // rows of a box
    uint32_t found, missing;   // boxes to copy; mask of those whose page is outside the pool
};
// The page of a lane's box, looked up ahead of its tile: one behind the other, a lookup and the copies took 1.45 us a tile, whatever its bytes.
__device__ __forceinline__ int box_page(const Paged& pool, const int32_t* pages, uint32_t pos0, uint32_t length, int lane) {
    const uint32_t seg = min(pool.view.page_size, kDecodeTile), mine = pos0 + lane * seg;
    return lane * seg < kDecodeTile && mine < length ? pages[mine >> pool.page_shift] : 0;
}
__device__ __forceinline__ Boxes boxes_of(const Paged& pool, int page, uint32_t head, uint32_t pos0, uint32_t length, int lane) {
    Boxes b{-1, min(pool.view.page_size, kDecodeTile), 0, 0};
    const uint32_t mine = pos0 + lane * b.seg;
    const bool there = lane * b.seg < kDecodeTile && mine < length;
    if (there) {
        b.row = page_row(pool, page, head);
        if (b.row >= 0) b.row += mine & ((1u << pool.page_shift) - 1);
    }
    b.found = __popc(__ballot_sync(0xffffffffu, b.row >= 0));
    b.missing = __ballot_sync(0xffffffffu, there && b.row < 0);
    return b;
}

// One unit, by a warp: its copies complete on `full` -- or, where a box has no page, on `landed`, and the warp clears its rows and completes `full` itself.
// *fixes counts the uses of `landed`.  False if a wait ran out.
template <int D, int FMT>
__device__ __forceinline__ bool bring_unit(uint8_t* smem, uint32_t off, uint32_t scale_off, const CUtensorMap* map, const void* scales, const Boxes& b, uint32_t full, uint32_t landed,
                                           uint32_t* fixes, int lane) {
    using U = Unit<D, FMT>;
    const uint32_t sbase = smem_u32(smem);
    const bool fix = b.missing != 0;
    const uint32_t to = fix ? landed : full, bytes = b.found * b.seg * (U::kRow + U::kScale);
    if (lane == 0) {
        if (bytes > 0) mbar_expect_tx(to, bytes);
        else if (!fix) mbar_arrive(to);
    }
    __syncwarp();
    if (b.row >= 0) {
#pragma unroll
        for (int x = 0; x < U::kSlabs; ++x)
            tma_load_2d(sbase + off + x * (kDecodeTile * 128) + lane * b.seg * 128, map, x * (FMT == F16 ? 64 : 128), static_cast<int>(b.row), to);
        if constexpr (FMT != F16)
            bulk_load(sbase + scale_off + lane * b.seg * U::kScale, static_cast<const uint8_t*>(scales) + static_cast<size_t>(b.row) * U::kScale, b.seg * U::kScale, to);
    }
    if (!fix) return true;
    if (bytes > 0) {
        if (!wait_warp(to, *fixes & 1)) return false;
        ++*fixes;
    }
    for (uint32_t r = 0; r < kDecodeTile; ++r) {
        if (!((b.missing >> (r / b.seg)) & 1)) continue;
        for (int i = lane; i < U::kSlabs * 8; i += 32) *reinterpret_cast<uint4*>(smem + off + (i >> 3) * (kDecodeTile * 128) + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
        if (FMT != F16 && lane < U::kScale / 2) *reinterpret_cast<uint16_t*>(smem + scale_off + r * U::kScale + lane * 2) = 0;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(full);
    return true;
}

// ---- query rows: a warp, lane l the elements D/32 l .. of every row --------------------------------------------------------------------

// Rows r < rows of a pair: token r / G, head r % G of the kv head; the others are zeros.
template <int D, int ROWS>
__device__ __forceinline__ void load_query(float (&x)[ROWS][D / 32], const void* q, bool is_f16, uint32_t query_heads, uint32_t first_token, uint32_t head, uint32_t G, uint32_t rows, int lane) {
    constexpr int E = D / 32;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[r][e] = 0.0f;
        if (static_cast<uint32_t>(r) >= rows) continue;
        const size_t at = ((static_cast<size_t>(first_token) + r / G) * query_heads + head * G + r % G) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            if (is_f16) {
                const uint2 raw = *reinterpret_cast<const uint2*>(static_cast<const __half*>(q) + at + e);
                const float2 a = unpack2(raw.x), b = unpack2(raw.y);
                x[r][e] = a.x; x[r][e + 1] = a.y; x[r][e + 2] = b.x; x[r][e + 3] = b.y;
            } else {
                const float4 raw = *reinterpret_cast<const float4*>(static_cast<const float*>(q) + at + e);
                x[r][e] = raw.x; x[r][e + 1] = raw.y; x[r][e + 2] = raw.z; x[r][e + 3] = raw.w;
            }
        }
    }
}

// A K-major operand: `slab` bytes for each 128 bytes of a row, rows of 128 bytes, 128-byte swizzle.  Returns what a sum of products is to be multiplied by.
// One row as two fp16 terms, rows `row` and row + LOW: scaled by a power of two, the largest element to [2^13, 2^14).
template <int D, int LOW>
__device__ __forceinline__ float store_terms(uint8_t* q, int slab, int row, const float (&x)[D / 32], int lane) {
    constexpr int E = D / 32;
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) amax = fmaxf(amax, fabsf(x[e]));
    amax = warp_max(amax);
    const int exponent = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
    const int up = amax > 0.0f ? max(-100, min(100, 13 - exponent)) : 0;
    const float mult = exp2i(up);
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        const int dim = lane * E + e, chunk = (dim % 64) / 8;
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float a = x[e + 2 * i] * mult, b = x[e + 2 * i + 1] * mult;
            hi[i] = pack2(a, b);
            const float2 h = unpack2(hi[i]);
            lo[i] = pack2(a - h.x, b - h.y);
        }
        auto at = [&](int n) { return q + (dim / 64) * slab + n * 128 + ((chunk ^ (n & 7)) << 4) + (dim % 8) * 2; };
        *reinterpret_cast<uint2*>(at(row)) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(at(row + LOW)) = make_uint2(lo[0], lo[1]);
    }
    return exp2i(-up);
}
// One row as a whole number in PLANES int8 planes, the highest digit in row `row`, the next STRIDE rows on: 8 bits less one each.
// The largest magnitude is found on the bits, which order as magnitudes do, with NaN above infinity: a NaN anywhere in a row, of which its digits know nothing, is
// the row's factor and so its scores.
template <int D, int PLANES, int STRIDE>
__device__ __forceinline__ float store_planes(uint8_t* q, int slab, int row, const float (&x)[D / 32], int lane) {
    constexpr int E = D / 32;
    constexpr float kMost = PLANES == 3 ? 127.0f * 65536.0f : 127.0f * 256.0f;
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
    const float amax = __uint_as_float(__reduce_max_sync(0xffffffffu, most));
    const float inv = amax > 0.0f ? kMost / amax : 0.0f;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        const int dim = lane * E + e, chunk = (dim % 128) / 16;
        uint32_t w[PLANES] = {};   // from the lowest digit: signed bytes
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int v = __float2int_rn(x[e + i] * inv);
#pragma unroll
            for (int d = 0; d < PLANES; ++d) {
                const int digit = d + 1 < PLANES ? ((v + 128) & 255) - 128 : v;
                w[d] |= static_cast<uint32_t>(digit & 0xff) << (8 * i);
                v = (v - digit) >> 8;
            }
        }
#pragma unroll
        for (int d = 0; d < PLANES; ++d) {
            const int n = (PLANES - 1 - d) * STRIDE + row;
            *reinterpret_cast<uint32_t*>(q + (dim / 128) * slab + n * 128 + ((chunk ^ (n & 7)) << 4) + (dim % 16)) = w[d];
        }
    }
    return amax / kMost;
}

}  // namespace

}  // namespace b200kv
