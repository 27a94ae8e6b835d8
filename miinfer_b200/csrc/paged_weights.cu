// The weight that every cached position of a paged cache gets from a batch's new tokens, summed over tokens and query heads of the kv head:
// A[j] += sum over (token, head) of exp(scale q.k_j - lse), with the statistics lse that the attention call left.
//
// With the statistics known a weight needs nothing but its own score, so there is no running maximum and nothing to rescale: S^T = K Q^T with positions as
// rows of the tensor core's result and a thread for each of them that adds up its row.  A position belongs to one CTA, whose threads add to the
// account alone: no atomics, the same sums on every run.  The scores are those of fp32: against them weights are held to 1e-5.
//
// Both kernels take equal pieces of one list of tiles (paged_tiles.cuh); a sequence is of one or the other by its observed query rows.
//
//  * few_kernel, up to 8 rows: bound by HBM, the first half of the attention kernel (paged_decode.cu).  int8 keys go straight into kind::i8 MMAs, the
//    queries are whole numbers of 24 bits in three int8 planes; fp16 keys meet two fp16 terms of the queries.
//  * many_kernel, any number: K of a tile becomes the A operand in TMEM, as fp16: fp16 as it is, int8 with one scale a row as whole numbers (the scale
//    multiplies the score), int8 with a scale a block of 32 as two fp16 terms of the product, 22 bits.  The query rows that see any of the tile stream past it, 64 at a
//    time: fp16 ones by TMA, whole tokens' heads of the kv head as boxes of a map over the activations; fp32 ones split into two terms by nine warps.  Eight warps
//    convert K; four of them take the exponentials of the even groups, the others those of the odd ones, so that one set's are under way while the other
//    waits for its scores.  A from TMEM halves what an MMA reads from shared memory (K in shared memory: 78 clocks an MMA of 32).
//    The last 64 tokens of 300 over 7000 to 12000 positions, two sequences, 24 / 4 heads of 256, q8_0: 39.5 us (all eight on every group 56; the groups in
//    turn, but one warp that issues, 59).  Four sequences of 64 to 300 tokens over 5000 to 11000, all of them observed, 32 / 8 heads of 128, q8_0: 144 us; with fp32 queries
//    368 (two warps that split them 990, five with a division a row 590).
//    A group of 64 rows takes a CTA 0.6 us, of it 0.55 the MMAs of a K of two terms and 0.3 the exponentials; a tile 2.5 us more, K on its way and converted,
//    which nothing of the CTA covers (TMEM holds one tile's K and the scores).  fp32 queries are bound by their loads, L2's latency and the nine warps.
#include "paged_decode.cuh"
#include "paged_unit.cuh"

#include <algorithm>
#include <cmath>

namespace b200kv {

namespace {

struct WeightsParams {
    Paged pool;
    const void* q;             // [total_tokens][query_heads][D]
    int q_is_f16;
    const float* lse;          // [total_tokens][query_heads]
    float* weights;            // [sequences][kv_heads][stride]
    uint32_t stride, query_heads, window, sinks, observe;
    uint32_t from_rows, to_rows;   // this launch's sequences: from .. to observed query rows
    uint32_t ctas;
    float scale_log2;
    __device__ __forceinline__ uint32_t observed(const Span& span) const { return observe > 0 ? min(observe, span.tokens) : span.tokens; }
    __device__ __forceinline__ Tiles tiles_of(const Span& span) const {
        const uint32_t n = observed(span);
        const uint64_t rows = static_cast<uint64_t>(n) * (query_heads / pool.view.kv_heads);
        if (rows < from_rows || rows > to_rows) return {0, 0, 0};
        return tiles_seen(static_cast<long long>(span.length) - n, span.length, window, sinks);
    }
    __device__ __forceinline__ const float* lse_of(const Span& span, uint32_t token) const { return lse + (static_cast<size_t>(span.first) + token) * query_heads; }
};

// ---- up to 8 rows ------------------------------------------------------------------------------------------------------------------------

template <int D, int KF, int ROWS>   // ROWS: 4 or 8
struct FewLayout {
    using U = Unit<D, KF>;
    static constexpr int kPlanes = KF == F16 ? 2 : 3;
    static constexpr int kCols = kPlanes * ROWS <= 16 ? 16 : 32;                              // columns of an MMA
    static constexpr int kSCols = KF == BLOCK ? D / 32 * kCols : kCols;                        // of a score buffer
    static constexpr uint32_t kTmemCols = 2 * kSCols <= 32 ? 32 : 2 * kSCols <= 64 ? 64 : 2 * kSCols <= 128 ? 128 : 2 * kSCols <= 256 ? 256 : 512;
    static constexpr int kCtas = D == 128 && KF != F16 ? 2 : 1;                                // per SM
    static constexpr int kProducerWarp = 4, kSWarp = 5, kQWarp = 6, kThreads = 256;
    static constexpr int kQSlab = kCols * 128, kQBytes = kCols * D * (KF == F16 ? 2 : 1);
    static constexpr int kMisc = 1024;
    static constexpr int kFit = ((kCtas == 2 ? 115712 : 232448) - 1024 - kMisc - 2 * kQBytes) / (U::kData + U::kScales);
    static constexpr int kUnits = kFit > 8 ? 8 : kFit;
    static_assert(kUnits >= 2);
    static constexpr int kOffQ = kUnits * U::kData, kOffScales = kOffQ + 2 * kQBytes, kOffRows = kOffScales + kUnits * U::kScales;   // rows: [buffer][8] {factor, statistics}
    static constexpr int kOffBar = kOffRows + 2 * 8 * 8;
    static constexpr int FULL = 0, EMPTY = kUnits, LANDED = 2 * kUnits, S_FULL = LANDED + 1, S_EMPTY = S_FULL + 2, Q_FULL = S_EMPTY + 2, Q_EMPTY = Q_FULL + 2, kNumBars = Q_EMPTY + 2;
    static constexpr int kOffMisc = kOffBar + kNumBars * 8, kAlloc = kOffMisc + 48 + 1024;
    static_assert(kOffMisc + 48 - kOffRows <= kMisc);
};

template <int D, int KF, int ROWS>
__global__ void __launch_bounds__(256, FewLayout<D, KF, ROWS>::kCtas) few_kernel(const __grid_constant__ WeightsParams p, const __grid_constant__ CUtensorMap kmap) {
    using L = FewLayout<D, KF, ROWS>;
    using U = Unit<D, KF>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem), bar0 = sbase + L::kOffBar;
    auto bar = [&](int i) { return bar0 + i * 8; };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
    uint32_t* start = tmem_slot + 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t H = p.pool.view.kv_heads, G = p.query_heads / H;
    pdl_launch_dependents();
    if (warp == L::kProducerWarp && lane == 0) {
        for (int i = 0; i < L::kNumBars; ++i) mbar_init(bar(i), i >= L::EMPTY && i < L::LANDED ? 1 + 4 : i >= L::S_EMPTY && i < L::Q_FULL ? 128 : i >= L::Q_EMPTY ? 1 + 4 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    } else if (warp == L::kSWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    if (warp == L::kQWarp) find_piece(p, blockIdx.x, lane, start);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    Cursor c(p, start);

    if (warp == L::kProducerWarp) {
        uint32_t i = 0, fixes = 0, begun = 0;
        bool ok = true;
        for (; c.left > 0 && ok; c.advance(p)) {
            const int32_t* pages = pages_of(p.pool, c.s);
            const uint32_t n = c.take();
            int page = box_page(p.pool, pages, c.t.position(c.tile), c.span.length, lane);
            for (uint32_t j = 0; j < n && ok; ++j, ++i) {
                const uint32_t slot = i % L::kUnits;
                const Boxes boxes = boxes_of(p.pool, page, c.head, c.t.position(c.tile + j), c.span.length, lane);
                if (j + 1 < n) page = box_page(p.pool, pages, c.t.position(c.tile + j + 1), c.span.length, lane);
                ok = i < L::kUnits || wait_warp(bar(L::EMPTY + slot), ((i / L::kUnits) & 1) ^ 1);
                if (!ok) break;
                ++begun;
                ok = bring_unit<D, KF>(smem, slot * U::kData, L::kOffScales + slot * U::kScales, &kmap, p.pool.view.key_scales, boxes, bar(L::FULL + slot), bar(L::LANDED), &fixes, lane);
            }
        }
        last_phases(bar(L::FULL), L::kUnits, begun);
    } else if (warp == L::kQWarp) {
        for (uint32_t k = 0; c.left > 0; c.advance(p), ++k) {
            const uint32_t buf = k & 1, tokens = p.observed(c.span), t0 = c.span.tokens - tokens;
            float x[ROWS][D / 32];
            load_query<D, ROWS>(x, p.q, p.q_is_f16, p.query_heads, c.span.first + t0, c.head, G, tokens * G, lane);
            float lse = INFINITY;      // lane r: of row r; a row that does not exist, or sees nothing, has no weights
            if (lane < ROWS && static_cast<uint32_t>(lane) < tokens * G) {
                lse = p.lse_of(c.span, t0 + lane / G)[c.head * G + lane % G];
                lse = lse == -INFINITY ? INFINITY : lse * 1.4426950408889634f;
            }
            if (k >= 2 && !wait_warp(bar(L::Q_EMPTY + buf), ((k >> 1) & 1) ^ 1)) break;
            uint8_t* q = smem + L::kOffQ + buf * L::kQBytes;
            float2* rows = reinterpret_cast<float2*>(smem + L::kOffRows) + buf * 8;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                float unit;
                if constexpr (KF == F16) unit = store_terms<D, ROWS>(q, L::kQSlab, r, x[r], lane);
                else unit = store_planes<D, 3, ROWS>(q, L::kQSlab, r, x[r], lane);
                if (lane == r) rows[r] = make_float2(unit * p.scale_log2, lse);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(L::Q_FULL + buf));
        }
    } else if (warp == L::kSWarp) {
        const uint64_t k_desc = umma_desc(sbase, 16, 1024, 2), q_desc = umma_desc(sbase + L::kOffQ, 16, 1024, 2);
        uint32_t i = 0;
        bool ok = true;
        for (uint32_t k = 0; c.left > 0 && ok; c.advance(p), ++k) {
            const uint32_t n = c.take();
            ok = wait_warp(bar(L::Q_FULL + (k & 1)), (k >> 1) & 1);
            const uint64_t qd = q_desc + (((k & 1) * L::kQBytes) >> 4);
            for (uint32_t j = 0; j < n && ok; ++j, ++i) {
                const uint32_t buf = i & 1, slot = i % L::kUnits;
                ok = mbar_wait_both(bar(L::S_EMPTY + buf), ((i >> 1) & 1) ^ 1, bar(L::FULL + slot), (i / L::kUnits) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint64_t kd = k_desc + ((slot * U::kData) >> 4);
                const uint32_t d = tmem_base + buf * L::kSCols;
                if (elect_one()) {
                    if constexpr (KF == F16) {
                        constexpr uint32_t idesc = idesc_f16(128, L::kCols, 0, 0);
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            umma_f16(d, kd + (((kk >> 2) * (kDecodeTile * 128) + (kk & 3) * 32) >> 4), qd + (((kk >> 2) * L::kQSlab + (kk & 3) * 32) >> 4), idesc, kk > 0);
                    } else {
                        constexpr uint32_t idesc = idesc_i8(128, L::kCols, 1, 1, 0, 0);
#pragma unroll
                        for (int b = 0; b < D / 32; ++b)
                            umma_i8(d + (KF == BLOCK ? b * L::kCols : 0), kd + (((b >> 2) * (kDecodeTile * 128) + (b & 3) * 32) >> 4), qd + (((b >> 2) * L::kQSlab + (b & 3) * 32) >> 4), idesc,
                                    KF == ROW && b > 0);
                    }
                    umma_commit(bar(L::S_FULL + buf));
                    umma_commit(bar(L::EMPTY + slot));
                    if (j + 1 == n) umma_commit(bar(L::Q_EMPTY + (k & 1)));
                }
                __syncwarp();
            }
        }
        last_phases(bar(L::S_FULL), 2, i);
    } else if (warp < 4) {
        // =============================== a thread a position ===============================
        const uint32_t lane_addr = static_cast<uint32_t>(warp * 32) << 16;
        uint32_t i = 0;
        bool failed = false;
        auto wait = [&](uint32_t b, uint32_t parity) { if (!failed && !mbar_wait(b, parity)) failed = true; };
        for (uint32_t k = 0; c.left > 0; c.advance(p), ++k) {
            const uint32_t n = c.take(), tokens = p.observed(c.span);
            wait(bar(L::Q_FULL + (k & 1)), (k >> 1) & 1);
            float2 row[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) row[r] = reinterpret_cast<const float2*>(smem + L::kOffRows)[(k & 1) * 8 + r];
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(L::Q_EMPTY + (k & 1)));
            const int first = static_cast<int>(c.span.length) - static_cast<int>(tokens);   // place of the first observed token
            float* account = p.weights + (static_cast<size_t>(c.s) * H + c.head) * p.stride;
            for (uint32_t j = 0; j < n; ++j, ++i) {
                const uint32_t buf = i & 1, slot = i % L::kUnits, pos0 = c.t.position(c.tile + j), pos = pos0 + tid;
                const float before = pos < c.span.length ? account[pos] : 0.0f;
                if (!failed && !mbar_wait_both_lane(bar(L::FULL + slot), (i / L::kUnits) & 1, bar(L::S_FULL + buf), (i >> 1) & 1)) failed = true;
                __syncwarp();
                tc_fence_after();
                const uint32_t s_at = tmem_base + lane_addr + buf * L::kSCols;
                const uint8_t* scales = smem + L::kOffScales + slot * U::kScales + tid * U::kScale;
                float s[ROWS];
                if constexpr (KF == F16) {
                    int v[2][ROWS];
#pragma unroll
                    for (int d = 0; d < 2; ++d)
#pragma unroll
                        for (int r = 0; r < ROWS; r += 4) tmem_ld4(s_at + d * ROWS + r, reinterpret_cast<int(&)[4]>(v[d][r]));
                    tmem_ld_wait();
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) s[r] = terms(__int_as_float(v[0][r]), __int_as_float(v[1][r]));
                } else {
                    constexpr int B = KF == BLOCK ? D / 32 : 1;
                    float ks[B];
                    if constexpr (KF == BLOCK) {
                        uint32_t raw[B / 2];
                        if constexpr (B == 8) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(scales);
                        else *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(scales);
#pragma unroll
                        for (int b = 0; b < B; b += 2) { const float2 f = unpack2(raw[b / 2]); ks[b] = f.x; ks[b + 1] = f.y; }
                    } else {
                        ks[0] = __half2float(*reinterpret_cast<const __half*>(scales));
                    }
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) s[r] = 0.0f;
#pragma unroll
                    for (int b = 0; b < B; b += 2) {   // two blocks' sums at a time
                        int v[2][3][ROWS];
#pragma unroll
                        for (int x = 0; x < 2 && b + x < B; ++x)
#pragma unroll
                            for (int d = 0; d < 3; ++d)
#pragma unroll
                                for (int r = 0; r < ROWS; r += 4) tmem_ld4(s_at + (b + x) * L::kCols + d * ROWS + r, reinterpret_cast<int(&)[4]>(v[x][d][r]));
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 2 && b + x < B; ++x)
#pragma unroll
                            for (int r = 0; r < ROWS; ++r)
                                s[r] = fmaf(fmaf(static_cast<float>(v[x][0][r]), 65536.0f, static_cast<float>(v[x][1][r] * 256 + v[x][2][r])), ks[b + x], s[r]);
                    }
                }
                tc_fence_before();
                mbar_arrive(bar(L::S_EMPTY + buf));
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::EMPTY + slot));
                float sum = 0.0f;
                if (static_cast<int>(pos0) + static_cast<int>(kDecodeTile) <= first + 1 && (p.window == 0 || static_cast<long long>(pos0) + p.window >= c.span.length)) {   // all rows see all positions
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) sum += ex2(fmaf(s[r], row[r].x, -row[r].y));
                } else {
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        const int at = first + static_cast<int>(r / G);
                        const bool seen = static_cast<uint32_t>(r) < tokens * G && static_cast<int>(pos) <= at && (p.window == 0 || static_cast<long long>(pos) + p.window > at || pos < p.sinks);
                        const float w = ex2(fmaf(s[r], row[r].x, -row[r].y));
                        sum += seen ? w : 0.0f;
                    }
                }
                if (pos < c.span.length) account[pos] = before + (failed ? __int_as_float(0x7fc00000) : sum);
            }
        }
        if (failed && lane == 0) report(p.pool, B200KV_STATUS_PIPE_TIMEOUT);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == L::kSWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols) : "memory");
    }
}

// ---- any number of rows ----------------------------------------------------------------------------------------------------------------

// Two fp32 values in one instruction.
__device__ __forceinline__ Pair fma_pair(Pair a, Pair b, Pair c) { Pair r; asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ Pair add_pair(Pair a, Pair b) { Pair r; asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

constexpr int kTile = kDecodeTile;
constexpr int kGroup = 64;           // query rows of an MMA: as many whole tokens as fit
constexpr int kWorkers = 256, kProducerWarp = 8, kQWarp = 9;

template <int D, int KF, bool Q32>
struct ManyLayout {
    using U = Unit<D, KF>;
    static constexpr int kKTerms = KF == BLOCK ? 2 : 1, kQTerms = Q32 ? 2 : 1;
    static constexpr int kCtas = D == 128 && !Q32 ? 2 : 1;                                     // per SM
    static constexpr int kLoaders = Q32 ? 9 : 2, kMmaWarp = kQWarp + kLoaders;                 // warps that bring the queries, from kQWarp on
    static constexpr int kSBufs = kCtas == 2 ? 2 : 4;
    static constexpr uint32_t kColK = 0, kColS = kKTerms * D / 2, kTmemCols = kColS + kSBufs * kGroup <= 256 ? 256 : 512;   // K: two fp16 a column
    static_assert(kColS + kSBufs * kGroup <= 512 && (kCtas == 1 || kTmemCols == 256));
    static constexpr int kQTerm = kGroup * D * 2;
    static constexpr int kRaw = Q32 && D == 256 && KF == F16 ? 1 : 2;                                 // units of K on their way
    static constexpr int kMisc = 5120;
    static constexpr int kFit = ((kCtas == 2 ? 115712 : 232448) - 1024 - kMisc - kRaw * (U::kData + U::kScales)) / (kQTerms * kQTerm);
    static constexpr int kQBufs = kFit >= 4 ? 4 : 2;
    // An MMA of 64 columns takes the tensor core 32 clocks and a warp 60 to issue, so where an SM has one CTA two warps take the groups in turn.
    static constexpr int kIssuers = kCtas == 1 ? 2 : 1, kThreads = (kMmaWarp + kIssuers) * 32;
    static_assert(kFit >= 2 && kSBufs % 2 == 0, "warps that take the groups in turn see every phase of their buffers only if those are even in number");
    static constexpr int kOffQ = kRaw * U::kData, kOffScales = kOffQ + kQBufs * kQTerms * kQTerm;
    static constexpr int kOffRows = kOffScales + kRaw * U::kScales;                           // [buffer] statistics in log2 units [64], places of the tokens [64]
    static constexpr int kOffSum = kOffRows + kQBufs * kGroup * 8;                            // [parity][128]
    static constexpr int kOffBar = kOffSum + 2 * kTile * 4;
    static constexpr int RAW_FULL = 0, RAW_EMPTY = RAW_FULL + kRaw, LANDED = RAW_EMPTY + kRaw, K_FULL = LANDED + 1, Q_FULL = K_FULL + 2, Q_EMPTY = Q_FULL + kQBufs,
                         S_FULL = Q_EMPTY + kQBufs, S_EMPTY = S_FULL + kSBufs, kNumBars = S_EMPTY + kSBufs;
    static constexpr int kOffMisc = kOffBar + kNumBars * 8, kAlloc = kOffMisc + 48 + 1024;
    static_assert(kOffMisc + 48 - kOffRows <= kMisc);
};

// eight fp16 of a row as one 16-byte chunk of a K-major operand: slabs of 64 dims, kGroup rows of 128 bytes each, 128-byte swizzle
__device__ __forceinline__ uint32_t chunk_at(uint32_t row, uint32_t chunk) { return (chunk >> 3) * (kGroup * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }
__device__ __forceinline__ void umma_f16_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// A tile's first position, and the tokens [t0, t1) that see any of it.  The tiles of a pair come from both ends in turn: the first are seen by the most tokens
// of a chunk, the last by the fewest, and a piece is a few tiles.
struct Share { uint32_t pos0, t0, t1; };
__device__ __forceinline__ Share share_of(const WeightsParams& p, const Cursor& c, uint32_t j) {
    const uint32_t x = c.tile + j, turned = (x & 1) ? c.t.n - 1 - (x >> 1) : x >> 1;
    Share s{c.t.position(turned), c.span.tokens - p.observed(c.span), c.span.tokens};
    const long long base = c.span.base(), first = static_cast<long long>(s.pos0) - base;
    if (first > s.t0) s.t0 = static_cast<uint32_t>(min(first, static_cast<long long>(s.t1)));
    if (p.window > 0 && s.pos0 >= p.sinks) {
        const long long end = static_cast<long long>(s.pos0) + kTile - 1 + p.window - base;   // the first token whose window lies behind the tile
        s.t1 = end <= 0 ? 0 : static_cast<uint32_t>(min(static_cast<long long>(s.t1), end));
    }
    if (s.t1 < s.t0) s.t1 = s.t0;
    return s;
}

template <int D, int KF, bool Q32>
__global__ void __launch_bounds__(ManyLayout<D, KF, Q32>::kThreads, ManyLayout<D, KF, Q32>::kCtas)
many_kernel(const __grid_constant__ WeightsParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap qmap) {
    using L = ManyLayout<D, KF, Q32>;
    using U = Unit<D, KF>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem), bar0 = sbase + L::kOffBar;
    auto bar = [&](int i) { return bar0 + i * 8; };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
    uint32_t* start = tmem_slot + 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t H = p.pool.view.kv_heads, G = p.query_heads / H, group_tokens = kGroup / G, group_rows = group_tokens * G;
    pdl_launch_dependents();
    if (warp == kProducerWarp && lane == 0) {
        for (int i = 0; i < L::kNumBars; ++i) {
            uint32_t count = 1;
            if (i >= L::RAW_EMPTY && i < L::LANDED) count = kWorkers / 32;
            else if (i >= L::K_FULL && i < L::Q_FULL) count = kWorkers;
            else if (i >= L::Q_FULL && i < L::Q_EMPTY) count = Q32 ? L::kLoaders * 32 : 33;    // the warps that bring the rows; the statistics' warp and the copies
            else if (i >= L::Q_EMPTY && i < L::S_FULL) count = 1 + kWorkers / 64;          // the MMAs, and the set of warps that takes the group
            else if (i >= L::S_EMPTY) count = kWorkers / 64;
            mbar_init(bar(i), count);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    } else if (warp == L::kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp < kProducerWarp) {   // rows of a group that no token's head takes: zeros once, no copy reaches them
        const uint32_t spare = (kGroup - group_rows) * 8;
        for (uint32_t i = tid; i < L::kQBufs * L::kQTerms * (D / 64) * spare; i += kWorkers)
            *reinterpret_cast<uint4*>(smem + L::kOffQ + i / spare * (kGroup * 128) + group_rows * 128 + i % spare * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    pdl_wait();
    if (warp == kQWarp) find_piece(p, blockIdx.x, lane, start);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    Cursor c(p, start);
    // the tiles of the piece that some token sees, in order: f(share) until it says false
    auto each_tile = [&](auto f) {
        for (; c.left > 0; c.advance(p)) {
            const uint32_t n = c.take();
            for (uint32_t j = 0; j < n; ++j) {
                const Share s = share_of(p, c, j);
                if (s.t0 < s.t1 && !f(s)) return;
            }
        }
    };

    if (warp < kProducerWarp) {
        // =============================== K into TMEM, then the exponentials ===============================
        const int wg = warp >> 2, t128 = tid & 127;   // half of a row's dims, then every second group
        const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
        uint32_t i = 0, k = 0;   // tiles and groups so far
        bool failed = false;
        auto wait = [&](uint32_t b, uint32_t parity) { if (!failed && !mbar_wait(b, parity)) failed = true; };
        each_tile([&](const Share& sh) {
            const uint32_t raw = i % L::kRaw, mine = sh.pos0 + t128;
            float* account = p.weights + (static_cast<size_t>(c.s) * H + c.head) * p.stride + mine;
            const bool writes = wg == 0 && mine < c.span.length;
            const float before = writes ? *account : 0.0f;
            wait(bar(L::RAW_FULL + raw), (i / L::kRaw) & 1);
            __syncwarp();
            const uint8_t* scales = smem + L::kOffScales + raw * U::kScales + t128 * U::kScale;
            const uint8_t* src = smem + raw * U::kData + t128 * 128;
            constexpr int kChunks = U::kRow / 32;                            // 16-byte chunks of half a row
            float factor = p.scale_log2;
            [[maybe_unused]] __half2 even = __float2half2_rn(1.0f);
            if constexpr (KF == BLOCK) {   // a position's scales by a power of two, the largest to [2^7, 2^8), so that a product is in fp16's range whatever the scales are
                uint32_t words[D / 64], most = 0;
                if constexpr (D == 256) *reinterpret_cast<uint4*>(words) = *reinterpret_cast<const uint4*>(scales);
                else *reinterpret_cast<uint2*>(words) = *reinterpret_cast<const uint2*>(scales);
#pragma unroll
                for (int b = 0; b < D / 64; ++b) most = max(most, max(words[b] & 0x7fffu, (words[b] >> 16) & 0x7fffu));
                const int up = min(22 - static_cast<int>(most >> 10), 15);   // 7 less the exponent; subnormal ones by 2^15
                even = __half2half2(__ushort_as_half(static_cast<unsigned short>((up + 15) << 10)));
                factor *= exp2i(-up);
            }
#pragma unroll
            for (int x = 0; x < kChunks; x += KF == F16 ? 2 : 1) {
                const int chunk = wg * kChunks + x;
                auto piece = [&](int n) { return *reinterpret_cast<const uint4*>(src + (n >> 3) * (kTile * 128) + (((n & 7) ^ (t128 & 7)) << 4)); };
                const uint32_t col = tmem_base + lane_addr + L::kColK + chunk * (KF == F16 ? 4 : 8);   // 8 or 16 dims
                const uint4 a = piece(chunk);
                if constexpr (KF == F16) {
                    const uint4 b = piece(chunk + 1);
                    const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    tmem_st8(col, v);
                } else {
                    // int8 as exact fp16: 1024 + 128 + q beside the exponent of 1024, less 1152
                    const uint32_t w[4] = {a.x ^ 0x80808080u, a.y ^ 0x80808080u, a.z ^ 0x80808080u, a.w ^ 0x80808080u};
                    uint32_t hi[8];
                    [[maybe_unused]] uint32_t lo[8];
                    [[maybe_unused]] __half2 sc;
                    if constexpr (KF == BLOCK) sc = __hmul2(__half2half2(reinterpret_cast<const __half*>(scales)[chunk >> 1]), even);   // exact, but for what is 2^-30 of the largest
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t pair = __byte_perm(w[e >> 1], 0x64646464u, e & 1 ? 0x4342 : 0x4140);
                        const __half2 q2 = __hadd2(*reinterpret_cast<const __half2*>(&pair), __float2half2_rn(-1152.0f));
                        if constexpr (KF == ROW) {
                            hi[e] = *reinterpret_cast<const uint32_t*>(&q2);
                        } else {   // the product as two terms: rounded, and what the rounding left, which a fused multiply-add finds exactly
                            const __half2 product = __hmul2(q2, sc), rest = __hfma2(q2, sc, __hneg2(product));
                            hi[e] = *reinterpret_cast<const uint32_t*>(&product);
                            lo[e] = *reinterpret_cast<const uint32_t*>(&rest);
                        }
                    }
                    tmem_st8(col, hi);
                    if constexpr (KF == BLOCK) tmem_st8(col + D / 2, lo);
                }
            }
            if constexpr (KF == ROW) factor *= __half2float(*reinterpret_cast<const __half*>(scales));
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            mbar_arrive(bar(L::K_FULL + (i & 1)));
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(L::RAW_EMPTY + raw));
            const int base = c.span.base();
            const uint32_t groups = (sh.t1 - sh.t0 + group_tokens - 1) / group_tokens;
            Pair sum[2] = {0, 0}, before_group[2] = {0, 0};
            const Pair factor2 = pack_pair(factor, factor);
            // An fp32 query's element beyond fp16 (65504) has an infinite first term and a second one that takes infinity away again, so its row's scores are NaN.  Sums that a group
            // leaves NaN are taken again, row by row, in fp32: K from TMEM, the query as it is.  (1 to 3 us a row, a call whose rows are all like that 45 to 85 times as long.  Found
            // ahead of the products, by the warps that split the queries, such rows cost every call 4 to 12 %: those warps bound it.)
            [[maybe_unused]] auto again = [&](uint32_t first, const float* stats, const int* places) {
                const uint32_t rows = min(group_rows, (sh.t1 - first) * G);
                float total = 0.0f;
#pragma unroll 1
                for (uint32_t x = 0; x < rows; ++x) {
                    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + ((static_cast<size_t>(c.span.first) + first + x / G) * p.query_heads + c.head * G + x % G) * D);
                    float s[4] = {};
#pragma unroll 1
                    for (int col = 0; col < D / 2; col += 8) {
                        int hi[8], lo[8] = {};
                        tmem_ld8(tmem_base + lane_addr + L::kColK + col, hi);
                        if constexpr (KF == BLOCK) tmem_ld8(tmem_base + lane_addr + L::kColK + D / 2 + col, lo);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const float4 four = q[(col + e) / 2];
                            const float2 a = unpack2(hi[e]), b = unpack2(hi[e + 1]), a1 = unpack2(lo[e]), b1 = unpack2(lo[e + 1]);
                            s[0] = fmaf(four.x, a.x + a1.x, s[0]);
                            s[1] = fmaf(four.y, a.y + a1.y, s[1]);
                            s[2] = fmaf(four.z, b.x + b1.x, s[2]);
                            s[3] = fmaf(four.w, b.y + b1.y, s[3]);
                        }
                    }
                    const int at = places[x];
                    const bool seen = static_cast<int>(mine) <= at && (p.window == 0 || static_cast<long long>(mine) + p.window > at || mine < p.sinks);
                    if (seen) total += ex2(fmaf((s[0] + s[1]) + (s[2] + s[3]), factor, stats[x]));
                }
                return total;
            };
            for (uint32_t g = 0; g < groups; ++g, ++k) {
                if ((k & 1) != static_cast<uint32_t>(wg)) continue;
                const uint32_t sb = k % L::kSBufs, qb = k % L::kQBufs;
                if (!failed && !mbar_wait_both_lane(bar(L::Q_FULL + qb), (k / L::kQBufs) & 1, bar(L::S_FULL + sb), (k / L::kSBufs) & 1)) failed = true;
                __syncwarp();
                tc_fence_after();
                const float* stats = reinterpret_cast<const float*>(smem + L::kOffRows) + qb * 2 * kGroup;   // of the rows, negated; then their places
                const int* places = reinterpret_cast<const int*>(stats + kGroup);
                const uint32_t first = sh.t0 + g * group_tokens, last = first + group_tokens - 1;
                const bool whole = last < sh.t1 && static_cast<int>(sh.pos0) + kTile - 1 <= base + static_cast<int>(first) &&
                                   (p.window == 0 || static_cast<long long>(sh.pos0) + p.window > static_cast<long long>(base) + last);   // all rows see all positions
                if constexpr (Q32) { before_group[0] = sum[0]; before_group[1] = sum[1]; }
                constexpr int kStep = 16;
#pragma unroll
                for (int col0 = 0; col0 < kGroup; col0 += kStep) {
                    int x[kStep];
#pragma unroll
                    for (int e = 0; e < kStep; e += 8) tmem_ld8(tmem_base + lane_addr + L::kColS + sb * kGroup + col0 + e, reinterpret_cast<int(&)[8]>(x[e]));
                    tmem_ld_wait();
                    if (col0 + kStep == kGroup) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar(L::S_EMPTY + sb));
                    }
                    if (whole) {
#pragma unroll
                        for (int e = 0; e < kStep; e += 4) {
                            const float4 four = *reinterpret_cast<const float4*>(stats + col0 + e);
                            const float2 a = unpack_pair(fma_pair(pack_pair(__int_as_float(x[e]), __int_as_float(x[e + 1])), factor2, pack_pair(four.x, four.y)));
                            const float2 b = unpack_pair(fma_pair(pack_pair(__int_as_float(x[e + 2]), __int_as_float(x[e + 3])), factor2, pack_pair(four.z, four.w)));
                            sum[0] = add_pair(sum[0], pack_pair(ex2(a.x), ex2(a.y)));
                            sum[1] = add_pair(sum[1], pack_pair(ex2(b.x), ex2(b.y)));
                        }
                    } else {
                        const auto add_seen = [&](auto sees) {
#pragma unroll
                            for (int e = 0; e < kStep; e += 4) {
                                const float4 stat = *reinterpret_cast<const float4*>(stats + col0 + e);
                                const int4 at = *reinterpret_cast<const int4*>(places + col0 + e);   // -1: no row, which sees nothing
                                const auto weight = [&](int y, float of, int place) {
                                    const float w = ex2(fmaf(__int_as_float(x[e + y]), factor, of));
                                    return sees(place) ? w : 0.0f;
                                };
                                sum[0] = add_pair(sum[0], pack_pair(weight(0, stat.x, at.x), weight(1, stat.y, at.y)));
                                sum[1] = add_pair(sum[1], pack_pair(weight(2, stat.z, at.z), weight(3, stat.w, at.w)));
                            }
                        };
                        if (p.window == 0) add_seen([&](int at) { return static_cast<int>(mine) <= at; });
                        else add_seen([&](int at) { return static_cast<int>(mine) <= at && (static_cast<long long>(mine) + p.window > at || mine < p.sinks); });
                    }
                }
                if constexpr (Q32) {
                    const float2 now = unpack_pair(add_pair(sum[0], sum[1])), then = unpack_pair(add_pair(before_group[0], before_group[1]));
                    const bool mended = isnan(now.x + now.y) && !isnan(then.x + then.y);
                    if (__any_sync(0xffffffffu, mended && !failed)) {
                        const float group = again(first, stats, places);
                        if (mended) {
                            sum[0] = add_pair(before_group[0], pack_pair(group, 0.0f));
                            sum[1] = before_group[1];
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::Q_EMPTY + qb));
            }
            float* other = reinterpret_cast<float*>(smem + L::kOffSum) + (i & 1) * kTile;
            const float2 halves = unpack_pair(add_pair(sum[0], sum[1]));
            const float total = failed ? __int_as_float(0x7fc00000) : halves.x + halves.y;
            if (wg == 1) other[t128] = total;
            tc_fence_before();
            asm volatile("bar.sync 1, 256;" ::: "memory");   // and the tile is multiplied through: all its groups' scores have been seen
            tc_fence_after();
            if (writes) *account = before + (total + other[t128]);
            ++i;
            return true;
        });
        if (failed && lane == 0) report(p.pool, B200KV_STATUS_PIPE_TIMEOUT);
    } else if (warp == kProducerWarp) {
        // =============================== K as it lies in the pages ===============================
        uint32_t i = 0, fixes = 0;
        each_tile([&](const Share& sh) {
            const uint32_t raw = i % L::kRaw;
            const Boxes boxes = boxes_of(p.pool, box_page(p.pool, pages_of(p.pool, c.s), sh.pos0, c.span.length, lane), c.head, sh.pos0, c.span.length, lane);
            if (i >= L::kRaw && !wait_warp(bar(L::RAW_EMPTY + raw), ((i / L::kRaw) & 1) ^ 1)) return false;
            ++i;
            return bring_unit<D, KF>(smem, raw * U::kData, L::kOffScales + raw * U::kScales, &kmap, p.pool.view.key_scales, boxes, bar(L::RAW_FULL + raw), bar(L::LANDED), &fixes, lane);
        });
        last_phases(bar(L::RAW_FULL), L::kRaw, i);
    } else if (warp < L::kMmaWarp) {
        // =============================== the query rows, 64 at a time ===============================
        const uint32_t w = warp - kQWarp;
        uint32_t k = 0;
        // fp32: a lane's rows of a group, row r of it for every kStep x kLoaders-th r, and their elements from the group's first token and head on
        constexpr uint32_t kPieces = D / 8, kStep = 32 / kPieces, kSteps = (kGroup / kStep + L::kLoaders - 1) / L::kLoaders;   // 16-byte pieces of a row of the operand
        const uint32_t piece = lane % kPieces, row0 = w * kStep + lane / kPieces;
        [[maybe_unused]] uint32_t rel[kSteps];
        if constexpr (Q32) {
#pragma unroll
            for (uint32_t y = 0; y < kSteps; ++y) {
                const uint32_t r = row0 + y * (L::kLoaders * kStep);
                rel[y] = (r / G * p.query_heads + r % G) * D + piece * 8;
            }
        }
        each_tile([&](const Share& sh) {
            const uint32_t groups = (sh.t1 - sh.t0 + group_tokens - 1) / group_tokens;
            // statistics and places of a group's rows, by a warp: a lane's two rows
            static_assert(kGroup == 64);
            auto has_row = [&](uint32_t t0, uint32_t x) { return x < group_rows && t0 + x / G < sh.t1; };
            auto load_stats = [&](uint32_t t0, float (&lse)[2]) {
#pragma unroll
                for (uint32_t y = 0; y < 2; ++y) {
                    const uint32_t x = 32 * y + lane;
                    lse[y] = has_row(t0, x) ? p.lse_of(c.span, t0 + x / G)[c.head * G + x % G] : -INFINITY;
                }
            };
            auto store_stats = [&](uint32_t t0, uint32_t qb, const float (&lse)[2]) {
#pragma unroll
                for (uint32_t y = 0; y < 2; ++y) {
                    const uint32_t x = 32 * y + lane;
                    reinterpret_cast<float*>(smem + L::kOffRows)[qb * 2 * kGroup + x] = lse[y] == -INFINITY ? -INFINITY : lse[y] * -1.4426950408889634f;   // a row that sees nothing has no weights
                    reinterpret_cast<int*>(smem + L::kOffRows)[(qb * 2 + 1) * kGroup + x] = has_row(t0, x) ? c.span.base() + static_cast<int>(t0 + x / G) : -1;
                }
            };
            for (uint32_t g = 0; g < groups; ++g, ++k) {
                const uint32_t qb = k % L::kQBufs, t0 = sh.t0 + g * group_tokens;
                const auto free = [&] { return k < L::kQBufs || wait_warp(bar(L::Q_EMPTY + qb), ((k / L::kQBufs) & 1) ^ 1); };
                if constexpr (!Q32) {
                    float lse[2];
                    if (w == 1) load_stats(t0, lse);
                    if (!free()) return false;
                    if (w == 1) {
                        store_stats(t0, qb, lse);
                        mbar_arrive(bar(L::Q_FULL + qb));
                    } else if (lane == 0) {
                        mbar_expect_tx(bar(L::Q_FULL + qb), group_rows * D * 2);   // rows past the last token's, or of no tensor, come along: they are masked
#pragma unroll
                        for (int x = 0; x < D / 64; ++x)
                            tma_load_3d(sbase + L::kOffQ + qb * L::kQTerm + x * (kGroup * 128), &qmap, x * 64, static_cast<int>(c.head * G), static_cast<int>(c.span.first + t0), bar(L::Q_FULL + qb));
                    }
                } else {
                    constexpr uint32_t kHeld = 4;   // steps' loads under way together
                    uint8_t* dst = smem + L::kOffQ + qb * L::kQTerms * L::kQTerm;
                    const float* src = static_cast<const float*>(p.q) + ((static_cast<size_t>(c.span.first) + t0) * p.query_heads + c.head * G) * D;
                    const uint32_t rows = min(group_rows, (sh.t1 - t0) * G);
                    float lse[2];
                    if (w == 0) load_stats(t0, lse);
#pragma unroll
                    for (uint32_t y0 = 0; y0 < kSteps; y0 += kHeld) {
                        float4 a[kHeld], b[kHeld];
#pragma unroll
                        for (uint32_t y = y0; y < y0 + kHeld && y < kSteps; ++y) {
                            a[y - y0] = b[y - y0] = make_float4(0, 0, 0, 0);
                            if (row0 + y * (L::kLoaders * kStep) < rows) {
                                a[y - y0] = *reinterpret_cast<const float4*>(src + rel[y]);
                                b[y - y0] = *reinterpret_cast<const float4*>(src + rel[y] + 4);
                            }
                        }
                        if (y0 == 0 && !free()) return false;   // the first loads are under way while the buffer is still in use
#pragma unroll
                        for (uint32_t y = y0; y < y0 + kHeld && y < kSteps; ++y) {
                            const uint32_t r = row0 + y * (L::kLoaders * kStep);
                            const float4 &f0 = a[y - y0], &f1 = b[y - y0];
                            const float v[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                hi[x] = pack2(v[2 * x], v[2 * x + 1]);
                                const float2 f = unpack2(hi[x]);
                                lo[x] = pack2(v[2 * x] - f.x, v[2 * x + 1] - f.y);
                            }
                            if (r < group_rows) {
                                *reinterpret_cast<uint4*>(dst + chunk_at(r, piece)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                                *reinterpret_cast<uint4*>(dst + L::kQTerm + chunk_at(r, piece)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                            }
                        }
                    }
                    if (w == 0) store_stats(t0, qb, lse);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(bar(L::Q_FULL + qb));
                }
            }
            return true;
        });
        if (!Q32 && w == 0) last_phases(bar(L::Q_FULL), L::kQBufs, k);
    } else {
        // =============================== issuer of S^T = K Q^T ===============================
        constexpr uint32_t idesc = idesc_f16(kTile, kGroup, 0, 0);
        const uint64_t q_desc = umma_desc(sbase + L::kOffQ, 16, 1024, 2);
        uint32_t i = 0, k = 0;
        each_tile([&](const Share& sh) {
            const uint32_t groups = (sh.t1 - sh.t0 + group_tokens - 1) / group_tokens;
            // (two barriers in turn: a tile may be through before the warp that has no group of it looks)
            if (!wait_warp(bar(L::K_FULL + (i & 1)), (i >> 1) & 1)) return false;
            ++i;
            for (uint32_t g = 0; g < groups; ++g, ++k) {
                if (L::kIssuers == 2 && (k & 1) != static_cast<uint32_t>(warp - L::kMmaWarp)) continue;
                const uint32_t sb = k % L::kSBufs, qb = k % L::kQBufs;
                if (!mbar_wait_both(bar(L::Q_FULL + qb), (k / L::kQBufs) & 1, bar(L::S_EMPTY + sb), ((k / L::kSBufs) & 1) ^ 1)) return false;
                tc_fence_after();
                const uint32_t d = tmem_base + L::kColS + sb * kGroup;
                const uint64_t qd = q_desc + ((qb * L::kQTerms * L::kQTerm) >> 4);
                if (elect_one()) {
                    auto product = [&](uint32_t a, uint64_t b, bool first) {
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            umma_f16_a_tmem(d, a + kk * 8, b + (((kk >> 2) * (kGroup * 128) + (kk & 3) * 32) >> 4), idesc, !first || kk > 0);
                    };
                    const uint32_t a = tmem_base + L::kColK;
                    // the small terms first: what they add is not lost beside the large sums
                    if constexpr (L::kKTerms == 2) product(a + D / 2, qd, true);
                    if constexpr (L::kQTerms == 2) product(a, qd + (L::kQTerm >> 4), L::kKTerms == 1);
                    product(a, qd, L::kKTerms == 1 && L::kQTerms == 1);
                    umma_commit(bar(L::S_FULL + sb));
                    umma_commit(bar(L::Q_EMPTY + qb));
                }
                __syncwarp();
            }
            return true;
        });
        last_phases(bar(L::S_FULL), L::kSBufs, k);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == L::kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols) : "memory");
    }
}

// ---- launches --------------------------------------------------------------------------------------------------------------------------

bool key_map(CUtensorMap* map, const b200kv_paged_view& v) {
    const bool q8 = is_k_q8(v.quant_mode);
    return encode_pool_map(map, q8 ? static_cast<const void*>(v.key_q8) : v.key_f16, !q8, static_cast<uint64_t>(v.pages) * v.kv_heads * v.page_size, v.head_dim,
                           std::min(v.page_size, kDecodeTile));
}

template <int D, int KF, int ROWS>
int launch_few(WeightsParams p, cudaStream_t stream) {
    using L = FewLayout<D, KF, ROWS>;
    static std::atomic<uint64_t> done{0};
    B200KV_CUDA_TRY(opt_in_dynamic_smem(reinterpret_cast<const void*>(few_kernel<D, KF, ROWS>), L::kAlloc, done));
    CUtensorMap kmap;
    if (!key_map(&kmap, p.pool.view)) return B200KV_ERR_UNSUPPORTED;
    p.ctas = std::min(device_sms(), kMostSms) * L::kCtas;
    B200KV_CUDA_TRY(launch_kernel(few_kernel<D, KF, ROWS>, dim3(p.ctas), dim3(L::kThreads), L::kAlloc, stream, true, p, kmap));
    return B200KV_OK;
}
template <int D, int KF, bool Q32>
int launch_many(WeightsParams p, bool behind, cudaStream_t stream) {
    using L = ManyLayout<D, KF, Q32>;
    static std::atomic<uint64_t> done{0};
    const auto kernel = many_kernel<D, KF, Q32>;
    B200KV_CUDA_TRY(opt_in_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kAlloc, done));
    const uint32_t G = p.query_heads / p.pool.view.kv_heads;
    CUtensorMap kmap, qmap{};
    if (!key_map(&kmap, p.pool.view) || (!Q32 && !encode_rows_map(&qmap, p.q, D, p.query_heads, p.pool.batch.total_tokens, G, kGroup / G))) return B200KV_ERR_UNSUPPORTED;
    p.ctas = std::min(device_sms(), kMostSms) * L::kCtas;
    if (behind) B200KV_CUDA_TRY(launch_behind(kernel, dim3(p.ctas), dim3(L::kThreads), L::kAlloc, stream, p, kmap, qmap));
    else B200KV_CUDA_TRY(launch_kernel(kernel, dim3(p.ctas), dim3(L::kThreads), L::kAlloc, stream, true, p, kmap, qmap));
    return B200KV_OK;
}
template <int D, int KF>
int launch_both(WeightsParams p, uint64_t most_rows, uint32_t sequences, cudaStream_t stream) {
    // what the bounds allow; a single sequence goes by its bound
    const bool many = most_rows > kDecodeRows, few = !many || sequences > 1;
    if (few) {
        p.from_rows = 1;
        p.to_rows = kDecodeRows;
        const int rc = most_rows <= 4 ? launch_few<D, KF, 4>(p, stream) : launch_few<D, KF, 8>(p, stream);
        if (rc != B200KV_OK || !many) return rc;
    }
    p.from_rows = few ? kDecodeRows + 1 : 1;
    p.to_rows = 0xffffffffu;
    return p.q_is_f16 ? launch_many<D, KF, false>(p, few, stream) : launch_many<D, KF, true>(p, few, stream);
}
template <int D>
int launch_formats(const WeightsParams& p, uint64_t most_rows, uint32_t sequences, cudaStream_t stream) {
    const b200kv_paged_view& v = p.pool.view;
    if (!is_k_q8(v.quant_mode)) return launch_both<D, F16>(p, most_rows, sequences, stream);
    return v.qblock == D ? launch_both<D, ROW>(p, most_rows, sequences, stream) : launch_both<D, BLOCK>(p, most_rows, sequences, stream);
}

}  // namespace

}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_paged_weights(const b200kv_paged_view* view, const b200kv_paged_batch* batch, const void* q, int q_dtype, const float* lse,
                                    float* weights, uint32_t weights_stride, uint32_t query_heads, float scale, uint32_t window, uint32_t sinks,
                                    uint32_t observe, void* stream) {
    int rc = validate_paged(view, batch);
    if (rc != B200KV_OK) return rc;
    if (q == nullptr || lse == nullptr || weights == nullptr || (q_dtype != B200KV_F16 && q_dtype != B200KV_F32)) return B200KV_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(q) & 15u) != 0 || ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(weights)) & 3u) != 0) return B200KV_ERR_INVALID;
    if (query_heads == 0 || query_heads % view->kv_heads != 0 || !std::isfinite(scale) || !(scale > 0.0f)) return B200KV_ERR_INVALID;
    if (query_heads / view->kv_heads > 8) return B200KV_ERR_UNSUPPORTED;
    if (static_cast<uint64_t>(view->pages) * view->kv_heads * view->page_size > 0x7fffffffull) return B200KV_ERR_UNSUPPORTED;   // coordinates are 32-bit
    if (batch->sequences == 0 || batch->total_tokens == 0 || batch->max_tokens == 0 || batch->max_length == 0) return B200KV_OK;
    if (weights_stride < batch->max_length) return B200KV_ERR_INVALID;
    settle_window(*batch, &window, &sinks);
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    const WeightsParams p{paged_of(*view, *batch), q, q_dtype == B200KV_F16, lse, weights, weights_stride, query_heads, window, sinks, observe, 0, 0, 0, scale * 1.4426950408889634f};
    const uint64_t most_rows = static_cast<uint64_t>(observe > 0 ? std::min(observe, batch->max_tokens) : batch->max_tokens) * (query_heads / view->kv_heads);
    return view->head_dim == 128 ? launch_formats<128>(p, most_rows, batch->sequences, static_cast<cudaStream_t>(stream))
                                 : launch_formats<256>(p, most_rows, batch->sequences, static_cast<cudaStream_t>(stream));
}
