// Attention of a few query rows per sequence over a paged cache: a decode step of many sequences, one new token or a few each.
//
// Bound by HBM: every visible row of K and V is read once for all query rows of its kv head, and the kernel's work is to keep copies under way on every SM.
//
//  * The tiles of 128 positions of all (sequence, kv head) pairs form one list, and every CTA of a grid that fits the device at once takes an equal piece
//    of it, whatever the lengths are (sequences of 512 to 16384 positions in one launch end together).  A piece crosses from one pair to the next with its
//    copies running on; a pair that lies in several pieces leaves partials, two a CTA at most, and the CTA in whose piece it begins, of which there is one
//    such pair at most, leaves word of it for paged_decode_merge_kernel.  Nothing waits for another CTA.
//  * K and V come as units of 128 rows through tensor maps over the whole pool, a box a page (pages of less than 128 positions: several), each into a ring
//    of its own, the block scales beside them as bulk copies.  (One ring K0 V0 K1 V1 ... of an odd number of units would show an issuer, which reads one of
//    the two, every second phase of a slot only, and a parity does not tell those apart.)  The bytes are operands as they land:
//      S^T = K Q^T        M = 128 positions (a thread each), N = 16 or 32 columns
//      O^T = V^T P        M = 128 dims (a thread each, per half of 256), K = positions
//    int8 sides on kind::i8 -- the sums of a block of 32 dims are exact, so its scale multiplies the sum -- and fp16 sides on kind::f16.
//  * Against int8 keys a query is a whole number in three int8 planes, 24 bits (two, 16 bits, where that does not show: launch_of).  Against fp16 keys it is two fp16 terms.
//    Weights for int8 values are 16-bit fixed point relative to the tile's largest, times the position's value scale, in two uint8 planes (each is off by 2^-17 of the largest:
//    1e-5 of an output, below fp16's rounding, and what fits the columns and two CTAs an SM); for fp16 values two fp16 terms.  Sums of a tile are folded into fp32
//    registers.
//  * A softmax thread has four query rows of a position; with five to eight rows a second group of 128 threads has the others.
//  * Positions that no row sees weigh nothing and their values are cleared in shared memory where they are fp16 (0 x NaN is NaN), each by its own thread (by the warp that
//    brings them, ahead of the next copies: 18 us a ragged tile), tiles that nobody sees
//    (between the sinks and the window) are not in the list.
// Measured, us: one token of 64 sequences of 512 to 16383 positions, 32 / 8 heads of 128, q8_0, pages of 64: 176 to 188 (5.7 TB/s; a tile a CTA 1.46, two CTAs an SM);
// of 24 sequences under a window of 4096, 24 / 4 heads of 256, one scale a row, pages of 32: 53 (3.8 TB/s); of one sequence of 99: 10.2, of 74 of 100: 21, fp16 29.
// Every wait is bounded: one that runs out poisons the CTA's results with NaN, sets a status bit, and the CTA ends in the normal way.
#include "paged_decode.cuh"
#include "paged_unit.cuh"

#include <algorithm>

namespace b200kv {

namespace {

template <int D, int KF, int VF, int RG, int PLANES>   // RG: groups of four query rows; PLANES: of a query row, int8 planes or fp16 terms
struct Layout {
    static constexpr int kTile = kDecodeTile;
    static constexpr int kHalves = D / 128;
    static constexpr int kSoftmax = RG * 128;
    static constexpr int kProducerWarp = RG * 4, kSWarp = kProducerWarp + 1, kPvWarp = kSWarp + 1, kQWarp = kPvWarp + 1;
    static constexpr int kThreads = kSoftmax + 128;
    static constexpr int kCtas = D == 128 && KF != F16 && VF != F16 && RG == 1 ? 2 : 1;   // per SM
    static constexpr int kKData = Unit<D, KF>::kData, kVData = Unit<D, VF>::kData, kKScales = Unit<D, KF>::kScales, kVScales = Unit<D, VF>::kScales;
    // weights of a row group: rows of 32 bytes per position, one set per half of the dims where the halves' scales differ
    static constexpr int kPSets = VF == BLOCK ? kHalves : 1;
    static constexpr int kPBytes = kPSets * kTile * 32;
    static_assert(PLANES == 2 || (PLANES == 3 && KF != F16));
    static constexpr int kStride = PLANES == 3 ? RG * 4 : 8;                              // rows of the operand from a plane to the next
    static constexpr int kQCols = PLANES * RG * 4 <= 16 ? 16 : 32;                        // columns of a score MMA
    // Three planes of eight rows have 24 columns of sums, and the operand no more rows: what an MMA takes for the last eight is the next slab, or the scales behind the
    // last one, and nobody looks at their sums.
    static constexpr int kQRows = kQCols == 16 ? 16 : 24;
    static constexpr int kQSlab = kQRows * 128, kQBytes = kQRows * D * (KF == F16 ? 2 : 1);
    static constexpr int kSCols = KF == BLOCK ? D / 32 * kQCols : kQCols;                 // TMEM columns of a score buffer
    static constexpr int kOCols = RG * kHalves * 32;                                      // of a buffer of sums
    // Three planes of eight rows of 256 dims against block scales leave room for one buffer of scores: the next tile's follow once these are in registers.
    static constexpr int kSBufs = 2 * (kSCols + kOCols) <= 512 ? 2 : 1;
    static constexpr int kCols = kSBufs * kSCols + 2 * kOCols;
    static_assert(kCols <= 512);
    static constexpr uint32_t kTmemCols = kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
    static constexpr uint32_t kColS = 0, kColO = kSBufs * kSCols;
    static constexpr int kXchWords = 16;                                                  // 4 maxima of scores, up to 8 of value scales
    static constexpr int kMiscBytes = RG * 2 * 4 * kXchWords * 4 + RG * 64 + 2 * 8 * 4 + 12 * 16 + 24 * 8 + 80;
    static constexpr int kMostUnits = 6;
    static constexpr int kBudget = (kCtas == 2 ? 115712 : 232448) - 1024;                 // the base is brought to a multiple of 1024
    static constexpr int kFixed = 2 * RG * kPBytes + 2 * kQBytes + kMiscBytes;
    static constexpr int kKUnit = kKData + kKScales, kVUnit = kVData + kVScales, kRoom = kBudget - kFixed;
    // a V unit is held for longer, until its weights are there, so V has the odd one
    static constexpr int units(bool v) {
        int k = 1, n = 1;
        while (true) {
            if (n < kMostUnits && n <= k && k * kKUnit + (n + 1) * kVUnit <= kRoom) ++n;
            else if (k < kMostUnits && (k + 1) * kKUnit + n * kVUnit <= kRoom) ++k;
            else if (n < kMostUnits && k * kKUnit + (n + 1) * kVUnit <= kRoom) ++n;
            else return v ? n : k;
        }
    }
    static constexpr int kKUnits = units(false), kVUnits = units(true);
    static constexpr int kOffV = kKUnits * kKData;
    static constexpr int kOffP = kOffV + kVUnits * kVData;                                // [buffer][group]
    static constexpr int kOffQ = kOffP + 2 * RG * kPBytes;                                // [buffer]
    static constexpr int kOffKScales = kOffQ + 2 * kQBytes, kOffVScales = kOffKScales + kKUnits * kKScales;
    static constexpr int kOffXch = kOffVScales + kVUnits * kVScales;                      // [group][parity][warp][words]
    static constexpr int kOffSum = kOffXch + RG * 2 * 4 * kXchWords * 4;                  // [group][warp][4]
    static constexpr int kOffQmul = kOffSum + RG * 64;                                    // [buffer][8]
    static constexpr int kOffBar = kOffQmul + 2 * 8 * 4;
    static constexpr int K_FULL = 0, V_FULL = K_FULL + kKUnits, K_EMPTY = V_FULL + kVUnits, V_EMPTY = K_EMPTY + kKUnits, LANDED = V_EMPTY + kVUnits, S_FULL = LANDED + 1, S_EMPTY = S_FULL + 2, P_FULL = S_EMPTY + 2, P_EMPTY = P_FULL + 2 * RG,
                         Q_FULL = P_EMPTY + 2 * RG, Q_EMPTY = Q_FULL + 2, kNumBars = Q_EMPTY + 2;
    static constexpr int kOffMisc = kOffBar + kNumBars * 8;                               // tmem slot, fail flag, the piece
    static constexpr int kTotal = (kOffMisc + 48 + 15) / 16 * 16;
    static constexpr int kAlloc = kTotal + 1024;
    static_assert(kTotal <= kBudget && kOffQ + 2 * kQBytes + (kQCols - kQRows) * 128 <= kTotal);
};

template <int D, int KF, int VF, int RG, int PLANES>
__global__ void __launch_bounds__(Layout<D, KF, VF, RG, PLANES>::kThreads, Layout<D, KF, VF, RG, PLANES>::kCtas)
paged_decode_kernel(const __grid_constant__ PagedDecode p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using L = Layout<D, KF, VF, RG, PLANES>;
    constexpr int kHalves = L::kHalves;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem), bar0 = sbase + L::kOffBar;
    auto bar = [&](int i) { return bar0 + i * 8; };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
    volatile uint32_t* fail_flag = tmem_slot + 1;
    uint32_t* start = tmem_slot + 2;   // the piece: sequence, head, tile, and how many tiles (two words)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t H = p.pool.view.kv_heads, G = p.query_heads / H;

    // ---- set-up ---------------------------------------------------------------------------------------------
    pdl_launch_dependents();
    if (warp == L::kProducerWarp && lane == 0) {
        for (int i = 0; i < L::kNumBars; ++i) {
            uint32_t count = 1;
            if (i >= L::K_EMPTY && i < L::LANDED) count = 1 + RG * 4;                     // the MMAs that read it, and a lane of every softmax warp
            else if (i >= L::S_EMPTY && i < L::P_FULL) count = RG * 128;
            else if (i >= L::P_FULL && i < L::P_EMPTY) count = 128;
            else if (i >= L::Q_EMPTY) count = 1 + RG * 4;
            mbar_init(bar(i), count);
        }
        *fail_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    } else if (warp == L::kSWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();   // lengths, queries and cache rows come from preceding kernels
    if (warp == L::kPvWarp) find_piece(p, blockIdx.x, lane, start);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    Cursor c(p, start);
    if (c.left == 0 && tid == 0) p.shared[blockIdx.x] = make_uint4(0, 0, 0, 0);
    bool failed = false;

    if (warp == L::kProducerWarp) {
        // =============================== copies: K and V units, a page's rows each lane ===============================
        uint32_t i = 0, fixes = 0, begun_k = 0, begun_v = 0;
        for (; c.left > 0 && !failed; c.advance(p)) {
            const int32_t* pages = pages_of(p.pool, c.s);
            const uint32_t n = c.take(), length = c.span.length;
            int page = box_page(p.pool, pages, c.t.position(c.tile), length, lane);
            for (uint32_t j = 0; j < n && !failed; ++j, ++i) {
                const uint32_t pos0 = c.t.position(c.tile + j), ks = i % L::kKUnits, vs = i % L::kVUnits;
                const Boxes boxes = boxes_of(p.pool, page, c.head, pos0, length, lane);
                if (j + 1 < n) page = box_page(p.pool, pages, c.t.position(c.tile + j + 1), length, lane);
                failed = i >= L::kKUnits && !wait_warp(bar(L::K_EMPTY + ks), ((i / L::kKUnits) & 1) ^ 1);
                if (!failed) {
                    ++begun_k;
                    failed = !bring_unit<D, KF>(smem, ks * L::kKData, L::kOffKScales + ks * L::kKScales, &kmap, p.pool.view.key_scales, boxes, bar(L::K_FULL + ks), bar(L::LANDED), &fixes, lane);
                }
                failed = failed || (i >= L::kVUnits && !wait_warp(bar(L::V_EMPTY + vs), ((i / L::kVUnits) & 1) ^ 1));
                if (!failed) {
                    ++begun_v;
                    failed = !bring_unit<D, VF>(smem, L::kOffV + vs * L::kVData, L::kOffVScales + vs * L::kVScales, &vmap, p.pool.view.value_scales, boxes, bar(L::V_FULL + vs),
                                                bar(L::LANDED), &fixes, lane);
                }
            }
        }
        last_phases(bar(L::K_FULL), L::kKUnits, begun_k);
        last_phases(bar(L::V_FULL), L::kVUnits, begun_v);
    } else if (warp == L::kQWarp) {
        // =============================== the query rows of a pair, as the operand of its score MMAs ===============================
        // Rows of the operand: kStride plane + r.
        for (uint32_t k = 0; c.left > 0; c.advance(p), ++k) {
            const uint32_t buf = k & 1;
            float x[RG * 4][D / 32];
            load_query<D, RG * 4>(x, p.q, p.q_is_f16, p.query_heads, c.span.first, c.head, G, c.span.tokens * G, lane);
            if (k >= 2 && !wait_warp(bar(L::Q_EMPTY + buf), ((k >> 1) & 1) ^ 1)) break;
            uint8_t* q = smem + L::kOffQ + buf * L::kQBytes;
#pragma unroll
            for (int r = 0; r < RG * 4; ++r) {
                float unit;
                if constexpr (KF == F16) unit = store_terms<D, L::kStride>(q, L::kQSlab, r, x[r], lane);
                else unit = store_planes<D, PLANES, L::kStride>(q, L::kQSlab, r, x[r], lane);
                if (lane == 0) reinterpret_cast<float*>(smem + L::kOffQmul)[buf * 8 + r] = unit * p.scale_log2;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the MMAs read it through the async proxy
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(L::Q_FULL + buf));
        }
    } else if (warp == L::kSWarp) {
        // =============================== issuer of S^T = K Q^T ===============================
        const uint64_t k_desc = umma_desc(sbase, 16, 1024, 2), q_desc = umma_desc(sbase + L::kOffQ, 16, 1024, 2);
        uint32_t i = 0;
        bool ok = true;
        for (uint32_t k = 0; c.left > 0 && ok; c.advance(p), ++k) {
            const uint32_t n = c.take();
            ok = wait_warp(bar(L::Q_FULL + (k & 1)), (k >> 1) & 1);
            const uint64_t qd = q_desc + (((k & 1) * L::kQBytes) >> 4);
            for (uint32_t j = 0; j < n && ok; ++j, ++i) {
                const uint32_t buf = i % L::kSBufs, slot = i % L::kKUnits;
                ok = mbar_wait_both(bar(L::S_EMPTY + buf), ((i / L::kSBufs) & 1) ^ 1, bar(L::K_FULL + slot), (i / L::kKUnits) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint64_t kd = k_desc + ((slot * L::kKData) >> 4);
                const uint32_t d = tmem_base + L::kColS + buf * L::kSCols;
                if (elect_one()) {
                    if constexpr (KF == F16) {
                        constexpr uint32_t idesc = idesc_f16(128, 16, 0, 0);
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            umma_f16(d, kd + (((kk >> 2) * (kDecodeTile * 128) + (kk & 3) * 32) >> 4), qd + (((kk >> 2) * L::kQSlab + (kk & 3) * 32) >> 4), idesc, kk > 0);
                    } else {
                        constexpr uint32_t idesc = idesc_i8(128, L::kQCols, 1, 1, 0, 0);
#pragma unroll
                        for (int b = 0; b < D / 32; ++b)   // 32 dims each: a block's sums in columns of their own, or all in the same
                            umma_i8(d + (KF == BLOCK ? b * L::kQCols : 0), kd + (((b >> 2) * (kDecodeTile * 128) + (b & 3) * 32) >> 4), qd + (((b >> 2) * L::kQSlab + (b & 3) * 32) >> 4), idesc,
                                    KF == ROW && b > 0);
                    }
                    umma_commit(bar(L::S_FULL + buf));
                    umma_commit(bar(L::K_EMPTY + slot));
                    if (j + 1 == n) umma_commit(bar(L::Q_EMPTY + (k & 1)));
                }
                __syncwarp();
            }
        }
        last_phases(bar(L::S_FULL), L::kSBufs, i);
    } else if (warp == L::kPvWarp) {
        // =============================== issuer of O^T = V^T P ===============================
        const uint64_t v_desc = umma_desc(sbase + L::kOffV, kDecodeTile * 128, 1024, 2);
        const uint64_t p_desc = umma_desc(sbase + L::kOffP, 32, 256, 6);
        uint32_t begun = 0;
        bool ok = true;
        for (uint64_t i64 = 0; i64 < c.left && ok; ++i64) {
            const uint32_t i = static_cast<uint32_t>(i64), buf = i & 1, slot = i % L::kVUnits;
#pragma unroll
            for (int g = 0; g < RG; ++g) {
                const int pb = buf * RG + g;
                ok = mbar_wait_both(bar(L::P_FULL + pb), (i >> 1) & 1, bar(L::V_FULL + slot), (i / L::kVUnits) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint64_t vd = v_desc + ((slot * L::kVData) >> 4), pd = p_desc + ((pb * L::kPBytes) >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int half = 0; half < kHalves; ++half) {
                        const uint32_t d = tmem_base + L::kColO + buf * L::kOCols + (g * kHalves + half) * 32;
                        const uint64_t ph = pd + ((VF == BLOCK ? half * (kDecodeTile * 32) : 0) >> 4);
                        if constexpr (VF == F16) {
                            constexpr uint32_t idesc = idesc_f16(128, 16, 1, 1);
#pragma unroll
                            for (int kk = 0; kk < kDecodeTile / 16; ++kk)   // 16 positions; 128 dims are two slabs
                                umma_f16(d, vd + ((half * 2 * (kDecodeTile * 128) + kk * (16 * 128)) >> 4), ph + ((kk * (16 * 32)) >> 4), idesc, kk > 0);
                        } else {
                            constexpr uint32_t idesc = idesc_i8(128, 32, 1, 0, 1, 1);
#pragma unroll
                            for (int kk = 0; kk < kDecodeTile / 32; ++kk)   // 32 positions
                                umma_i8(d, vd + ((half * (kDecodeTile * 128) + kk * (32 * 128)) >> 4), ph + ((kk * (32 * 32)) >> 4), idesc, kk > 0);
                        }
                    }
                    umma_commit(bar(L::P_EMPTY + pb));
                    if (g + 1 == RG) umma_commit(bar(L::V_EMPTY + slot));
                }
                __syncwarp();
                ++begun;
            }
        }
        last_phases(bar(L::P_EMPTY), 2 * RG, begun);
    } else {
        // =============================== softmax: a thread has a position and four query rows ===============================
        const int g = warp >> 2, w4 = warp & 3, t128 = tid & 127;
        const uint32_t lane_addr = static_cast<uint32_t>(w4 * 32) << 16;
        const uint32_t p_flip = static_cast<uint32_t>((t128 >> 2) & 1) << 4;   // 32-byte swizzle: chunk c of row r at 32 r + ((c ^ ((r >> 2) & 1)) << 4)
        int* xch = reinterpret_cast<int*>(smem + L::kOffXch) + g * (2 * 4 * L::kXchWords);
        float* sums = reinterpret_cast<float*>(smem + L::kOffSum) + g * 16;
        auto group_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); };
        auto wait = [&](uint32_t b, uint32_t parity) { if (!failed && !mbar_wait(b, parity)) failed = true; };
        constexpr int NB = VF == BLOCK ? D / 32 : 1;     // value scales of a position
        uint32_t i = 0;
        for (uint32_t k = 0; c.left > 0; c.advance(p), ++k) {
            const uint32_t n = c.take(), rows = c.span.tokens * G;
            wait(bar(L::Q_FULL + (k & 1)), (k >> 1) & 1);
            float qmul[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) qmul[r] = reinterpret_cast<const volatile float*>(smem + L::kOffQmul)[(k & 1) * 8 + g * 4 + r];
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(L::Q_EMPTY + (k & 1)));
            uint32_t upto[4], low[4];                    // a row sees positions [low, upto) and the sinks below upto
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t row = g * 4 + r;
                const int at = row < rows ? c.span.base() + static_cast<int>(row / G) + 1 : 0;
                upto[r] = static_cast<uint32_t>(max(at, 0));
                low[r] = p.window > 0 && upto[r] > p.window ? upto[r] - p.window : 0;
            }
            const uint32_t first_upto = static_cast<uint32_t>(max(c.span.base() + 1, 0));                             // what every row sees: [.., first_upto)
            [[maybe_unused]] const uint32_t first_low = p.window > 0 && first_upto > p.window ? first_upto - p.window : 0;   // seen by nobody: below it, but for the sinks
            const uint32_t last_low = p.window > 0 && c.span.length > p.window ? c.span.length - p.window : 0;        // from here on
            float acc[kHalves][4], m_run[4], l_run[4], pend[2][kHalves][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                m_run[r] = -INFINITY;
                l_run[r] = 0.0f;
#pragma unroll
                for (int h = 0; h < kHalves; ++h) acc[h][r] = pend[0][h][r] = pend[1][h][r] = 0.0f;
            }
            auto fold = [&](auto buf_c) {                // the sums of a tile into the accumulators of this thread's dims
                constexpr int buf = decltype(buf_c)::value;
                int o[kHalves][8];
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < kHalves; ++h) tmem_ld8(tmem_base + lane_addr + L::kColO + buf * L::kOCols + (g * kHalves + h) * 32 + (VF == F16 ? 0 : w4 * 8), o[h]);
                tmem_ld_wait();
                tc_fence_before();
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = VF == F16 ? terms(__int_as_float(o[h][r]), __int_as_float(o[h][4 + r])) : static_cast<float>(o[h][r] * 256 + o[h][4 + r]);
                        acc[h][r] = fmaf(v, pend[buf][h][r], acc[h][r]);
                    }
            };
            auto step = [&](auto buf_c, uint32_t j) {
                constexpr int buf = decltype(buf_c)::value, sbuf = buf % L::kSBufs;
                const uint32_t slot = i % L::kKUnits, vslot = i % L::kVUnits;
                const uint32_t pos = c.t.position(c.tile + j) + t128;
                if (!failed && !mbar_wait_both_lane(bar(L::K_FULL + slot), (i / L::kKUnits) & 1, bar(L::S_FULL + sbuf), (i / L::kSBufs) & 1)) failed = true;
                __syncwarp();
                tc_fence_after();
                // ---- scores, in base-2 units ----
                float s[4];
                [[maybe_unused]] const uint8_t* kst = smem + L::kOffKScales + slot * L::kKScales;
                const uint32_t s_at = tmem_base + lane_addr + L::kColS + sbuf * L::kSCols;
                if constexpr (KF == F16) {
                    int hi[4], lo[4];
                    tmem_ld4(s_at + 4 * g, hi);
                    tmem_ld4(s_at + 8 + 4 * g, lo);
                    tmem_ld_wait();
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[r] = terms(__int_as_float(hi[r]), __int_as_float(lo[r]));
                } else {
                    constexpr int B = KF == BLOCK ? D / 32 : 1;
                    float ks[B];
                    if constexpr (KF == BLOCK) {
                        uint32_t raw[B / 2];
                        if constexpr (B == 8) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(kst + t128 * 16);
                        else *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(kst + t128 * 8);
#pragma unroll
                        for (int b = 0; b < B; b += 2) { const float2 f = unpack2(raw[b / 2]); ks[b] = f.x; ks[b + 1] = f.y; }
                    } else {
                        ks[0] = __half2float(*reinterpret_cast<const __half*>(kst + t128 * 2));
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[r] = 0.0f;
                    constexpr int kPart = RG == 2 && PLANES == 3 && B > 2 ? 2 : B;   // blocks' sums at a time (all 96 of a thread at once: 76.8 -> 78.8 us)
#pragma unroll
                    for (int b0 = 0; b0 < B; b0 += kPart) {
                        int v[kPart][PLANES][4];
#pragma unroll
                        for (int b = 0; b < kPart; ++b)
#pragma unroll
                            for (int d = 0; d < PLANES; ++d) tmem_ld4(s_at + (b0 + b) * L::kQCols + L::kStride * d + 4 * g, v[b][d]);
                        tmem_ld_wait();
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int b = 0; b < kPart; ++b) {
                                float x;
                                if constexpr (PLANES == 3) x = fmaf(static_cast<float>(v[b][0][r]), 65536.0f, static_cast<float>(v[b][1][r] * 256 + v[b][2][r]));
                                else x = static_cast<float>(v[b][0][r] * 256 + v[b][1][r]);
                                s[r] = fmaf(x, ks[b0 + b], s[r]);
                            }
                    }
                }
                tc_fence_before();
                mbar_arrive(bar(L::S_EMPTY + sbuf));
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::K_EMPTY + slot));      // the scales are read
                const uint32_t pos0 = pos - t128;
                bool any = true;
                if (pos0 + kDecodeTile <= first_upto && pos0 >= last_low) {   // every row sees all of the tile
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[r] *= qmul[r];
                } else {
                    any = false;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool seen = pos < upto[r] && (pos >= low[r] || pos < p.sinks);
                        s[r] = seen ? s[r] * qmul[r] : -INFINITY;
                        any |= seen;
                    }
                }
                // ---- the value scales, and the tile's maxima: inside the warp, then across the four ----
                wait(bar(L::V_FULL + vslot), (i / L::kVUnits) & 1);
                __syncwarp();
                if constexpr (VF == F16) {   // an fp16 value that none of the rows sees is cleared (int8 ones are finite whatever they are)
                    if (g == 0 && (pos >= c.span.length || (pos < first_low && pos >= p.sinks))) {
                        uint8_t* row = smem + L::kOffV + vslot * L::kVData + t128 * 128;
#pragma unroll 1
                        for (int x = 0; x < D / 64; ++x)
#pragma unroll
                            for (int y = 0; y < 8; ++y)   // lanes at different chunks: different banks
                                *reinterpret_cast<uint4*>(row + x * (kDecodeTile * 128) + ((y + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                }
                [[maybe_unused]] uint32_t vs_bits[NB];
                if constexpr (VF != F16) {
                    const uint8_t* vst = smem + L::kOffVScales + vslot * L::kVScales;
                    if constexpr (VF == ROW) {
                        vs_bits[0] = *reinterpret_cast<const uint16_t*>(vst + t128 * 2);
                    } else {
                        uint32_t raw[NB / 2];
                        if constexpr (NB == 8) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(vst + t128 * 16);
                        else *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(vst + t128 * 8);
#pragma unroll
                        for (int b = 0; b < NB; b += 2) { vs_bits[b] = raw[b / 2] & 0xffffu; vs_bits[b + 1] = raw[b / 2] >> 16; }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::V_EMPTY + vslot));
                float m_tile[4];
                [[maybe_unused]] float vs_max[NB];
                {
                    float mx[4];
                    [[maybe_unused]] uint32_t vmx[NB];
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx[r] = warp_max_redux(s[r]);
                    if constexpr (VF != F16) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) vmx[b] = __reduce_max_sync(0xffffffffu, any ? vs_bits[b] : 0u);   // positive fp16 order like integers
                    }
                    int* dst = xch + (buf * 4 + w4) * L::kXchWords;
                    if (lane == 0) {
                        *reinterpret_cast<float4*>(dst) = make_float4(mx[0], mx[1], mx[2], mx[3]);
                        if constexpr (VF != F16) {
#pragma unroll
                            for (int b = 0; b < NB; ++b) dst[4 + b] = static_cast<int>(vmx[b]);
                        }
                    }
                    group_sync();
#pragma unroll
                    for (int r = 0; r < 4; ++r) m_tile[r] = -INFINITY;
                    [[maybe_unused]] uint32_t vall[NB] = {};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int* src = xch + (buf * 4 + x) * L::kXchWords;
                        const float4 a = *reinterpret_cast<const float4*>(src);
                        m_tile[0] = fmaxf(m_tile[0], a.x); m_tile[1] = fmaxf(m_tile[1], a.y); m_tile[2] = fmaxf(m_tile[2], a.z); m_tile[3] = fmaxf(m_tile[3], a.w);
                        if constexpr (VF != F16) {
#pragma unroll
                            for (int b = 0; b < NB; ++b) vall[b] = max(vall[b], static_cast<uint32_t>(src[4 + b]));
                        }
                    }
                    if constexpr (VF != F16) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) vs_max[b] = __half2float(__ushort_as_half(static_cast<uint16_t>(vall[b])));
                    }
                }
                // ---- the running maxima; the branch is the group's ----
                if (m_tile[0] > m_run[0] || m_tile[1] > m_run[1] || m_tile[2] > m_run[2] || m_tile[3] > m_run[3]) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float m_new = fmaxf(m_run[r], m_tile[r]);
                        const float alpha = m_run[r] == -INFINITY ? 0.0f : ex2(m_run[r] - m_new);
                        l_run[r] *= alpha;
#pragma unroll
                        for (int h = 0; h < kHalves; ++h) { acc[h][r] *= alpha; pend[0][h][r] *= alpha; pend[1][h][r] *= alpha; }
                        m_run[r] = m_new;
                    }
                }
                // ---- weights ----
                uint32_t words[L::kPSets][8];            // this position's 32 bytes
                float scale_now[kHalves][4];             // what the tile's sums count for, relative to the running maxima
                if constexpr (VF == F16) {
                    float w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        w[r] = s[r] == -INFINITY ? 0.0f : ex2(s[r] - m_run[r]);
                        l_run[r] += w[r];
#pragma unroll
                        for (int h = 0; h < kHalves; ++h) scale_now[h][r] = 1.0f;
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        words[0][x] = pack2(w[2 * x], w[2 * x + 1]);
                        const float2 h = unpack2(words[0][x]);
                        words[0][2 + x] = pack2(w[2 * x] - h.x, w[2 * x + 1] - h.y);
                    }
                } else {
                    float wn[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float w = s[r] == -INFINITY ? 0.0f : ex2(s[r] - m_run[r]);
                        l_run[r] += w;
                        const float wmax = m_tile[r] == -INFINITY ? 0.0f : ex2(m_tile[r] - m_run[r]);
                        wn[r] = s[r] == -INFINITY || !(wmax > 0.0f) ? 0.0f : ex2(s[r] - m_tile[r]);   // relative to the tile's largest
#pragma unroll
                        for (int h = 0; h < kHalves; ++h) {
                            float own = vs_max[0];       // the largest value scale of this thread's block
                            if constexpr (VF == BLOCK) own = w4 == 0 ? vs_max[4 * h] : w4 == 1 ? vs_max[4 * h + 1] : w4 == 2 ? vs_max[4 * h + 2] : vs_max[4 * h + 3];
                            scale_now[h][r] = wmax * own * (1.0f / 65535.0f);
                        }
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const float wv = any && vs_max[b] > 0.0f ? __half2float(__ushort_as_half(static_cast<uint16_t>(vs_bits[b]))) * __fdividef(65535.0f, vs_max[b]) : 0.0f;
                        uint32_t pq[4];                  // beside 2^23 the products come rounded to whole numbers in the low 16 bits
#pragma unroll
                        for (int r = 0; r < 4; ++r) pq[r] = __float_as_uint(__fmaf_rn(wn[r], wv, 8388608.0f));
                        const uint32_t p01 = __byte_perm(pq[0], pq[1], 0x5410), p23 = __byte_perm(pq[2], pq[3], 0x5410);
                        const uint32_t hi = __byte_perm(p01, p23, 0x7531), lo = __byte_perm(p01, p23, 0x6420);
                        if constexpr (VF == BLOCK) {
                            words[b >> 2][2 * (b & 3)] = hi;
                            words[b >> 2][2 * (b & 3) + 1] = lo;
                        } else {
#pragma unroll
                            for (int x = 0; x < 4; ++x) { words[0][2 * x] = hi; words[0][2 * x + 1] = lo; }
                        }
                    }
                }
                // ---- the buffers were last used by the tile before the last: fold its sums, then hand the weights over ----
                if (j >= 2) {
                    wait(bar(L::P_EMPTY + buf * RG + g), ((i >> 1) & 1) ^ 1);
                    __syncwarp();
                    fold(buf_c);
                }
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) pend[buf][h][r] = scale_now[h][r];
                const uint32_t pt = sbase + L::kOffP + (buf * RG + g) * L::kPBytes + t128 * 32;
#pragma unroll
                for (int x = 0; x < L::kPSets; ++x) {
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(pt + x * (kDecodeTile * 32) + p_flip), "r"(words[x][0]), "r"(words[x][1]), "r"(words[x][2]), "r"(words[x][3]) : "memory");
                    if constexpr (VF != F16)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(pt + x * (kDecodeTile * 32) + (p_flip ^ 16u)), "r"(words[x][4]), "r"(words[x][5]), "r"(words[x][6]), "r"(words[x][7]) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(bar(L::P_FULL + buf * RG + g));
                ++i;
            };
            using Buf0 = std::integral_constant<int, 0>;
            using Buf1 = std::integral_constant<int, 1>;
            for (uint32_t j = 0; j < n; ++j) {
                if ((i & 1) == 0) step(Buf0{}, j);
                else step(Buf1{}, j);
            }
            // ---- the pair's end: row sums, the last two tiles' sums ----
#pragma unroll
            for (int r = 0; r < 4; ++r) l_run[r] = warp_sum(l_run[r]);
            if (lane == 0) *reinterpret_cast<float4*>(sums + w4 * 4) = make_float4(l_run[0], l_run[1], l_run[2], l_run[3]);
            for (uint32_t back = min(n, 2u); back > 0; --back) {
                const uint32_t x = i - back;
                wait(bar(L::P_EMPTY + (x & 1) * RG + g), (x >> 1) & 1);
                __syncwarp();
                if ((x & 1) == 0) fold(Buf0{});
                else fold(Buf1{});
            }
            if (failed) *fail_flag = 1;
            group_sync();
            float lt[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float4 a = *reinterpret_cast<const float4*>(sums + x * 4);
                lt[0] += a.x; lt[1] += a.y; lt[2] += a.z; lt[3] += a.w;
            }
            if (tid == 0 && c.left == n) {               // the piece's last pair
                uint4 word = make_uint4(c.s, c.head, 0, 0);
                if (c.tile == 0 && n < c.t.n) {
                    const uint64_t all = start[5] | static_cast<uint64_t>(start[6]) << 32;
                    const uint32_t pieces = pieces_of(p, all);
                    word.z = piece_with(all, piece_begin(all, blockIdx.x + 1, pieces) - n + c.t.n - 1, pieces);
                    word.w = 1;
                }
                p.shared[blockIdx.x] = word;
            }
            const bool poisoned = *fail_flag != 0;
            group_sync();                                // the sums are read: the next pair may write its own
            if (poisoned && t128 == 0) report(p.pool, B200KV_STATUS_PIPE_TIMEOUT);
            const float nan = __int_as_float(0x7fc00000);
            const bool whole = c.tile == 0 && n == c.t.n;
            const size_t part = (2 * static_cast<size_t>(blockIdx.x) + (c.tile > 0 ? 0 : 1)) * kDecodeRows;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t row = g * 4 + r;
                if (row >= rows) break;
                const size_t head_row = (static_cast<size_t>(c.span.first) + row / G) * p.query_heads + c.head * G + row % G;
                if (!whole) {
                    if (t128 == 0) p.part_ml[part + row] = make_float2(m_run[r], poisoned ? nan : lt[r]);
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) p.part_o[(part + row) * D + h * 128 + t128] = acc[h][r];
                    continue;
                }
                if (p.lse != nullptr && t128 == 0)
                    p.lse[head_row] = poisoned ? nan : m_run[r] == -INFINITY ? (lt[r] != lt[r] ? nan : -INFINITY) : (m_run[r] + log2f(lt[r])) * 0.69314718055994531f;
                const float f = poisoned || lt[r] != lt[r] ? nan : lt[r] > 0.0f ? 1.0f / lt[r] : 0.0f;
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    const size_t at = head_row * D + h * 128 + t128;
                    float v = acc[h][r] * f;
                    if (lt[r] == 0.0f) v = 0.0f;
                    if (p.gate != nullptr) v *= 1.0f / (1.0f + __expf(-p.gate[at]));
                    if (p.out_is_f16) static_cast<__half*>(p.out)[at] = __float2half_rn(v);
                    else static_cast<float*>(p.out)[at] = v;
                }
            }
        }
    }

    // ---- teardown: every role arrives here, with or without a timeout; TMEM is always released ----
    tc_fence_before();
    __syncthreads();
    if (warp == L::kSWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols) : "memory");
    }
}

// out = sum_c O_c 2^(m_c - M) / sum_c l_c 2^(m_c - M), times sigmoid(gate), over the CTAs whose pieces hold tiles of a pair.  A block: a query row of the pair that
// begins in piece blockIdx.y and ends in a later one, a thread a dim.  All other pairs have been written by their CTA.
template <int D>
__global__ void __launch_bounds__(D) paged_decode_merge_kernel(const __grid_constant__ PagedDecode p) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t c0 = blockIdx.y, row = blockIdx.x, tid = threadIdx.x, G = p.query_heads / p.pool.view.kv_heads;
    const uint4 word = p.shared[c0];
    if (word.w == 0) return;
    const Span span = span_of(p.pool, word.x);
    if (row >= span.tokens * G) return;
    auto part_of = [&](uint32_t c) { return (2 * static_cast<size_t>(c) + (c == c0 ? 1 : 0)) * kDecodeRows + row; };   // a later CTA's first partial
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    bool poisoned = false;
    for (uint32_t c = c0; c <= word.z; c += 8) {   // eight partials' loads under way together
        float2 ml[8];
        float o[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            ml[i] = make_float2(-INFINITY, 0.0f);
            o[i] = 0.0f;
            if (c + i > word.z) continue;
            ml[i] = p.part_ml[part_of(c + i)];
            o[i] = p.part_o[part_of(c + i) * D + tid];
        }
        float m_new = m;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            poisoned |= ml[i].y != ml[i].y;
            if (ml[i].y > 0.0f) m_new = fmaxf(m_new, ml[i].x);
        }
        const float f = m_new > m && m > -INFINITY ? ex2(m - m_new) : m_new > m ? 0.0f : 1.0f;
        l *= f;
        acc *= f;
        m = m_new;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            if (!(ml[i].y > 0.0f)) continue;
            const float w = ex2(ml[i].x - m);
            l = fmaf(w, ml[i].y, l);
            if (w > 0.0f) acc = fmaf(w, o[i], acc);
        }
    }
    const float nan = __int_as_float(0x7fc00000);
    const size_t head_row = (static_cast<size_t>(span.first) + row / G) * p.query_heads + word.y * G + row % G, at = head_row * D + tid;
    if (p.lse != nullptr && tid == 0) p.lse[head_row] = poisoned ? nan : l > 0.0f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
    float v = poisoned ? nan : l > 0.0f ? acc / l : 0.0f;
    if (p.gate != nullptr) v *= 1.0f / (1.0f + __expf(-p.gate[at]));
    if (p.out_is_f16) static_cast<__half*>(p.out)[at] = __float2half_rn(v);
    else static_cast<float*>(p.out)[at] = v;
}

template <int D, int KF, int VF, int RG, int PLANES>
int launch_planes(const PagedDecode& p, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream, bool behind) {
    using L = Layout<D, KF, VF, RG, PLANES>;
    const auto kernel = paged_decode_kernel<D, KF, VF, RG, PLANES>;
    static std::atomic<uint64_t> done{0};
    B200KV_CUDA_TRY(opt_in_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kAlloc, done));
    if (behind) B200KV_CUDA_TRY(launch_behind(kernel, dim3(p.ctas), dim3(L::kThreads), L::kAlloc, stream, p, kmap, vmap));
    else B200KV_CUDA_TRY(launch_kernel(kernel, dim3(p.ctas), dim3(L::kThreads), L::kAlloc, stream, true, p, kmap, vmap));
    return B200KV_OK;
}
// Three planes against int8 keys (a score to 2^-23 of its row's largest element), but for eight rows where the output alone is asked for, in fp16: two hold 2^-16, which that does not
// show, and are up to 12 % faster (24 sequences of 4000, 24 / 4 heads of 256: q8_0 66.6 and 75 us, where a tile has 96 sums a thread in place of 64 and one buffer of them; one scale a row 59.4
// and 61.4).
template <int D, int KF, int VF, int RG>
int launch_of(const PagedDecode& p, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream, bool behind) {
    if constexpr (KF == F16) return launch_planes<D, KF, VF, RG, 2>(p, kmap, vmap, stream, behind);
    if constexpr (KF != F16 && RG == 2) {
        if (p.lse == nullptr && p.out_is_f16) return launch_planes<D, KF, VF, RG, 2>(p, kmap, vmap, stream, behind);
    }
    if constexpr (KF != F16) return launch_planes<D, KF, VF, RG, 3>(p, kmap, vmap, stream, behind);
}
template <int D, int RG>
int launch_modes(const PagedDecode& p, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream, bool behind) {
    const bool blocks = p.pool.view.qblock != D;
    switch (p.pool.view.quant_mode) {
        case B200KV_F16_F16: return launch_of<D, F16, F16, RG>(p, kmap, vmap, stream, behind);
        case B200KV_Q8_F16: return blocks ? launch_of<D, BLOCK, F16, RG>(p, kmap, vmap, stream, behind) : launch_of<D, ROW, F16, RG>(p, kmap, vmap, stream, behind);
        case B200KV_F16_Q8: return blocks ? launch_of<D, F16, BLOCK, RG>(p, kmap, vmap, stream, behind) : launch_of<D, F16, ROW, RG>(p, kmap, vmap, stream, behind);
        default: return blocks ? launch_of<D, BLOCK, BLOCK, RG>(p, kmap, vmap, stream, behind) : launch_of<D, ROW, ROW, RG>(p, kmap, vmap, stream, behind);
    }
}

}  // namespace

uint32_t decode_ctas(const b200kv_paged_view& view, uint32_t sms) {
    return sms * (view.head_dim == 128 && view.quant_mode == B200KV_Q8_Q8 ? 2 : 1);
}
size_t decode_part_bytes(const b200kv_paged_view& view, uint32_t sms) {
    return decode_ctas(view, sms) * (2ull * kDecodeRows * (view.head_dim * sizeof(float) + sizeof(float2)) + sizeof(uint4));
}

int launch_paged_decode(PagedDecode p, void* parts, cudaStream_t stream, bool behind) {
    const b200kv_paged_view& v = p.pool.view;
    const b200kv_paged_batch& b = p.pool.batch;
    const uint64_t rows = static_cast<uint64_t>(v.pages) * v.kv_heads * v.page_size;
    const uint32_t box = std::min(v.page_size, kDecodeTile), group = p.query_heads / v.kv_heads;
    CUtensorMap kmap, vmap;
    if (!encode_pool_map(&kmap, is_k_q8(v.quant_mode) ? static_cast<const void*>(v.key_q8) : v.key_f16, !is_k_q8(v.quant_mode), rows, v.head_dim, box) ||
        !encode_pool_map(&vmap, is_v_q8(v.quant_mode) ? static_cast<const void*>(v.value_q8) : v.value_f16, !is_v_q8(v.quant_mode), rows, v.head_dim, box))
        return B200KV_ERR_UNSUPPORTED;
    p.rows = decode_rows(b, group);
    const bool few = p.rows == 4;
    const uint32_t sms = std::min(device_sms(), kMostSms), most = decode_ctas(v, sms);
    p.ctas = few ? most : sms;
    p.part_o = static_cast<float*>(parts);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + 2ull * most * kDecodeRows * v.head_dim);
    p.shared = reinterpret_cast<uint4*>(p.part_ml + 2ull * most * kDecodeRows);
    const int rc = v.head_dim == 128 ? (few ? launch_modes<128, 1>(p, kmap, vmap, stream, behind) : launch_modes<128, 2>(p, kmap, vmap, stream, behind))
                                     : (few ? launch_modes<256, 1>(p, kmap, vmap, stream, behind) : launch_modes<256, 2>(p, kmap, vmap, stream, behind));
    if (rc != B200KV_OK) return rc;
    // one tile a pair: no pair lies in two pieces
    if (b.max_length <= kDecodeTile) return B200KV_OK;
    const uint32_t most_rows = static_cast<uint32_t>(std::min<uint64_t>(p.rows, static_cast<uint64_t>(b.max_tokens) * group));
    const dim3 grid(most_rows, p.ctas);
    B200KV_CUDA_TRY(v.head_dim == 128 ? launch_behind(paged_decode_merge_kernel<128>, grid, dim3(128), 0, stream, p)
                                      : launch_behind(paged_decode_merge_kernel<256>, grid, dim3(256), 0, stream, p));
    return B200KV_OK;
}

}  // namespace b200kv
