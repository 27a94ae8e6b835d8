// A layer's queries, keys and values of a ragged batch on their way to the attention over a paged cache, in one launch: norms, rotary positions of any of the usual forms,
// the gate split off the queries, quantisation, and the write of K and V into their pages.
//
//   a' = m (a cos p f_i - b sin p f_i),  b' = m (a sin p f_i + b cos p f_i)   for pair i of the first `dims` elements of a head: (i, i + dims/2) or (2i, 2i + 1), position p
//
// Angles.  p f_i in fp32 is off by 2^-24 of itself, a tenth of a radian at a million.  A frequency comes as a 64-bit fraction of a turn instead: p times it modulo 2^64 is the
// angle's fraction of a turn, exact but for the table's own rounding (p 2^-65 turns).  Its upper 32 bits less the nearest quarter are the argument of a Taylor polynomial (to x^9 / x^8
// on |x| <= pi/4, 3e-8).
//
// A lane holds sixteen elements of a row, two runs of eight, so that the two halves of a pair are in one lane.  D/16 lanes are a row, a warp takes four rows of 128 or two of 256 at a time
// and a token's rows one step after the other; several warps share a token where there are few.  The next steps' rows come by cp.async into places of the lane's own, 8 KB a warp under
// way.  A token's sines and cosines are worked out once a warp, two or four of them a lane, and handed round.
// Bound by HBM for prompts with gates, by latency and instruction issue (16 warps an SM) without them and for a decode step.  Three prompts, 6100 tokens in all, fp16 to one scale a row, norms,
// halves, us: 24 / 4 heads of 256 with gates 79 (4.7 TB/s of 6.5; fp32 114, 5.8), 32 / 8 of 128 39 (3.4); 40 tokens 6.4.  With one run a lane, the other half by shuffles and the next step's
// loads in registers: 98 (142), 62; two runs a lane, loads in registers: 86 (115), 50; runs 2 l and 2 l + 1 of neighbours, every second 16 bytes an instruction: 47, in place of 35.
#include "append_row.cuh"
#include "paged_common.cuh"

#include <algorithm>
#include <cmath>
#include <utility>

namespace b200kv {

namespace {

constexpr int kRotaryWarps = 4;

struct RotaryParams {
    Paged pool;
    const uint64_t* turns;       // [dims / 2]
    uint32_t dims, neighbours;
    float magnitude, epsilon;
    const void* q;               // q, key, value: may be null (key and value both)
    const void* key;
    const void* value;
    uint64_t q_stride, key_stride, value_stride;   // elements from a token's rows to the next's
    const float* q_norm;
    const float* k_norm;
    const int32_t* positions;
    void* q_out;
    int q_out_is_f16;
    float* gate;                 // may be null; the heads of q are a query and its gate
    uint32_t query_heads;
    uint32_t share;              // warps to a token
};

// Sine and cosine of a fraction of a turn.
__device__ __forceinline__ void sincos_turns(uint64_t turns, float* s_out, float* c_out) {
    const uint32_t t = static_cast<uint32_t>(turns >> 32), quarter = (t + 0x20000000u) >> 30;
    const float x = static_cast<float>(static_cast<int>(t - (quarter << 30))) * 1.4629180792671596e-9f;   // 2 pi 2^-32
    const float z = x * x;
    const float s = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f), -1.0f / 6.0f), x);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 40320.0f, -1.0f / 720.0f), 1.0f / 24.0f), -0.5f), 1.0f);
    const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
    *s_out = quarter & 2 ? -a : a;
    *c_out = (quarter + 1) & 2 ? -b : b;
}

__device__ __forceinline__ Pair mul2(Pair a, Pair b) { Pair r; asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { Pair r; asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

// Eight elements as they lie in memory, and as pairs of fp32.
template <bool IN_F16> struct Run { uint4 v[IN_F16 ? 1 : 2]; };
// A lane's run on its way into its own places of shared memory, 32 pieces of 16 bytes of the warp one behind the other.
template <bool IN_F16>
__device__ __forceinline__ void bring_run(uint4* to, const void* src, size_t element) {
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(src) + element * (IN_F16 ? 2 : 4));
#pragma unroll
    for (int i = 0; i < (IN_F16 ? 1 : 2); ++i) {
        const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to + 32 * i));
        if constexpr (IN_F16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from + i) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from + i) : "memory");   // (half a sector each: the other half comes from L1)
    }
}
template <bool IN_F16>
__device__ __forceinline__ Run<IN_F16> brought_run(const uint4* at) {
    Run<IN_F16> r;
#pragma unroll
    for (int i = 0; i < (IN_F16 ? 1 : 2); ++i) r.v[i] = at[32 * i];
    return r;
}
template <bool IN_F16>
__device__ __forceinline__ void widen(const Run<IN_F16>& r, Pair (&x)[4]) {
    if constexpr (IN_F16) {
        const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[i] = pack_pair(f.x, f.y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[2 * i] = pack_pair(__uint_as_float(r.v[i].x), __uint_as_float(r.v[i].y));
            x[2 * i + 1] = pack_pair(__uint_as_float(r.v[i].z), __uint_as_float(r.v[i].w));
        }
    }
}
__device__ __forceinline__ uint4 as_halves(const Pair (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_pair(x[i]);
        const __half2 h = __floats2half2_rn(f.x, f.y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_floats(float* to, const Pair (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 a = unpack_pair(x[2 * i]), b = unpack_pair(x[2 * i + 1]);
        reinterpret_cast<float4*>(to)[i] = make_float4(a.x, a.y, b.x, b.y);
    }
}
// Largest magnitude; a NaN counts as 0, as in quantize_row.
__device__ __forceinline__ float amax_of(const Pair (&x)[4]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpack_pair(x[i]);
        asm("max.ftz.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(v.x)), "f"(fabsf(v.y)));
    }
    return m;
}
__device__ __forceinline__ uint2 quantize_eight(const Pair (&x)[4], float inv) {
    const Pair inv2 = pack_pair(inv, inv);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 a = unpack_pair(mul2(x[2 * i], inv2)), b = unpack_pair(mul2(x[2 * i + 1], inv2));
        asm("{ .reg .b32 t; cvt.pack.sat.s8.s32.b32 t, %4, %3, 0; cvt.pack.sat.s8.s32.b32 %0, %2, %1, t; }"
            : "=r"(w[i]) : "r"(__float2int_rn(a.x)), "r"(__float2int_rn(a.y)), "r"(__float2int_rn(b.x)), "r"(__float2int_rn(b.y)));
    }
    return make_uint2(w[0], w[1]);
}

// The rows of a step into the cache, runs ca and cb of each a lane.  The bits are quantize_row's.  The maxima of runs meet in `exchange`, [row of the step][run], a warp's own: sixteen
// lanes have a block each, or the rows' first ones a row, and work out its scale and the reciprocal, the two divisions of a block once.
template <int D>
__device__ __forceinline__ void store_rows(const b200kv_paged_view& view, bool is_k, long long row, const Pair (&a)[4], const Pair (&b)[4], uint32_t ca, uint32_t cb, uint32_t sub, bool there,
                                           float* exchange) {
    constexpr uint32_t kRuns = D / 8, kRows = 512 / D;
    const bool q8 = is_k ? is_k_q8(view.quant_mode) : is_v_q8(view.quant_mode);
    if (!q8) {
        __half* to = static_cast<__half*>(is_k ? view.key_f16 : view.value_f16) + row * D;
        if (there) {
            *reinterpret_cast<uint4*>(to + ca * 8) = as_halves(a);
            *reinterpret_cast<uint4*>(to + cb * 8) = as_halves(b);
        }
        return;
    }
    const uint32_t lane = threadIdx.x & 31;
    const bool rows = view.qblock == D;
    exchange[sub * kRuns + ca] = amax_of(a);
    exchange[sub * kRuns + cb] = amax_of(b);
    __syncwarp();
    float amax = 0.0f;
    if (rows) {
        const float4* of_row = reinterpret_cast<const float4*>(exchange + sub * kRuns);
#pragma unroll
        for (uint32_t i = 0; i < kRuns / 4; ++i) {
            const float4 m = of_row[i];
            amax = fmaxf(amax, fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w)));
        }
    } else {
        const float4 m = reinterpret_cast<const float4*>(exchange)[lane % (kRows * kRuns / 4)];   // block lane % 16: of row lane / (kRuns / 4)
        amax = fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
    }
    const float scale = amax > 0.0f ? __fdiv_rn(amax, 127.0f) : 1.0f;
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 1.0f;
    float inv_a = inv, inv_b = inv;
    if (!rows) {
        inv_a = __shfl_sync(0xffffffffu, inv, sub * (kRuns / 4) + ca / 4);
        inv_b = __shfl_sync(0xffffffffu, inv, sub * (kRuns / 4) + cb / 4);
    }
    // whose scale a lane stores: its own block's, or its row's
    const float scale_a = rows ? scale : __shfl_sync(0xffffffffu, scale, sub * (kRuns / 4) + ca / 4), scale_b = rows ? scale : __shfl_sync(0xffffffffu, scale, sub * (kRuns / 4) + cb / 4);
    __syncwarp();   // the maxima are read
    if (!there) return;
    int8_t* to = (is_k ? view.key_q8 : view.value_q8) + row * D;
    __half* scales = static_cast<__half*>(is_k ? view.key_scales : view.value_scales);
    *reinterpret_cast<uint2*>(to + ca * 8) = quantize_eight(a, inv_a);
    *reinterpret_cast<uint2*>(to + cb * 8) = quantize_eight(b, inv_b);
    if (rows) {
        if (ca == 0) scales[row] = __float2half_rn(scale_a);
    } else {
        if (ca % 4 == 0) scales[row * (D / 32) + ca / 4] = __float2half_rn(scale_a);
        if (cb % 4 == 0) scales[row * (D / 32) + cb / 4] = __float2half_rn(scale_b);
    }
}

template <int D, bool IN_F16>
__global__ void __launch_bounds__(kRotaryWarps * 32, 4) paged_rotary_kernel(const __grid_constant__ RotaryParams p) {
    constexpr uint32_t kLanes = D / 16, kRows = 32 / kLanes, kEach = 8 / kRows;   // lanes of a row, rows a step, angles a lane works out
    constexpr uint32_t kPieces = IN_F16 ? 1 : 2, kAhead = IN_F16 ? 4 : 2;   // 16-byte pieces of a run; steps whose loads are under way
    __shared__ __align__(16) float exchange[kRotaryWarps][kRows * D / 8];
    __shared__ uint4 ring[kRotaryWarps][kAhead][4 * kPieces * 32];   // a lane's two runs, and the gate's
    pdl_wait();
    pdl_launch_dependents();                             // behind the wait: it writes cache rows
    const Paged& pool = p.pool;
    const uint32_t lane = threadIdx.x & 31, l = lane % kLanes, sub = lane / kLanes;
    const uint64_t me = static_cast<uint64_t>(blockIdx.x) * kRotaryWarps + threadIdx.x / 32;
    if (me >= static_cast<uint64_t>(pool.batch.total_tokens) * p.share) return;
    const uint32_t token = static_cast<uint32_t>(me / p.share), part = static_cast<uint32_t>(me % p.share);

    // ---- where the token goes
    const uint32_t s = sequence_of(pool, token);
    const Span span = span_of(pool, s);
    if (token < span.first || token - span.first >= span.tokens) return;
    const int place = span.base() + static_cast<int>(token - span.first);
    const long long row0 = place >= 0 && p.key != nullptr ? row_of(pool, s, 0, static_cast<uint32_t>(place)) : -1;   // for kv head 0
    const uint64_t position = static_cast<uint32_t>(max(p.positions != nullptr ? p.positions[token] : place, 0));

    // ---- its rows: queries with their gates, keys, values, a step at a time
    const uint32_t H = pool.view.kv_heads, half = p.dims / 16;   // runs of a half
    const uint32_t k0 = p.q != nullptr ? (p.query_heads + kRows - 1) / kRows : 0, kv_steps = p.key != nullptr ? (H + kRows - 1) / kRows : 0, v0 = k0 + kv_steps, steps = v0 + kv_steps;
    const bool gated = p.gate != nullptr, in_halves = p.neighbours == 0 && l < half;
    // Halves are run l and run l + half; behind the rotated part, and of neighbours, lanes next to each other have runs next to each other as well.
    const uint32_t ca = p.neighbours ? l : in_halves ? l : l + half, cb = !p.neighbours && in_halves ? l + half : l + kLanes;
    const bool turns_a = ca * 8 < p.dims, turns_b = cb * 8 < p.dims;
    enum { QUERY, KEY, VALUE };
    struct Step { int kind; uint32_t head; bool there; };
    const auto step_of = [&](uint32_t t) {
        const int kind = t < k0 ? QUERY : t < v0 ? KEY : VALUE;
        const uint32_t head = (t - (kind == QUERY ? 0 : kind == KEY ? k0 : v0)) * kRows + sub;
        return Step{kind, head, t < steps && head < (kind == QUERY ? p.query_heads : H)};
    };
    uint4* const mine = ring[threadIdx.x / 32][0] + lane;
    constexpr uint32_t kRun = kPieces * 32, kStage = 4 * kRun;
    const auto fetch = [&](uint32_t t, uint32_t stage) {   // (a lane waits for its own copies only, and reads no others')
        const Step at = step_of(t);
        if (at.there) {
            const void* from = at.kind == QUERY ? p.q : at.kind == KEY ? p.key : p.value;
            const size_t element = token * (at.kind == QUERY ? p.q_stride : at.kind == KEY ? p.key_stride : p.value_stride) + static_cast<size_t>(at.head) * (at.kind == QUERY && gated ? 2 * D : D);
            uint4* to = mine + stage * kStage;
            bring_run<IN_F16>(to, from, element + ca * 8);
            bring_run<IN_F16>(to + kRun, from, element + cb * 8);
            if (at.kind == QUERY && gated) {
                bring_run<IN_F16>(to + 2 * kRun, from, element + D + ca * 8);
                bring_run<IN_F16>(to + 3 * kRun, from, element + D + cb * 8);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) fetch(part + i * p.share, i);

    // ---- its angles: eight a lane, of pair 8 l + i of halves, or of neighbours 4 ca + i and, from the fifth on, 4 cb + i - 4; a lane works out kEach of those that the lanes of its number share
    float cs[8], sn[8];
    {
        float c[kEach], n[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = sub * kEach + i, pair = p.neighbours ? (at < 4 ? 4 * ca + at : 4 * cb + at - 4) : 8 * l + at;
            c[i] = 1.0f;
            n[i] = 0.0f;
            if (2 * pair >= p.dims) continue;
            sincos_turns(position * p.turns[pair], &n[i], &c[i]);
            c[i] *= p.magnitude;
            n[i] *= p.magnitude;
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            cs[i] = __shfl_sync(0xffffffffu, c[i % kEach], i / kEach * kLanes + l);
            sn[i] = __shfl_sync(0xffffffffu, n[i % kEach], i / kEach * kLanes + l);
        }
    }

    Pair w[2][4];
    int weighed = -1;                                    // whose norm's weights these are
    uint32_t stage = 0;
    for (uint32_t t = part; t < steps; t += p.share, stage = stage + 1 == kAhead ? 0 : stage + 1) {
        const Step at = step_of(t);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        const uint4* from = mine + stage * kStage;
        Pair a[4], b[4];
        widen<IN_F16>(brought_run<IN_F16>(from), a);
        widen<IN_F16>(brought_run<IN_F16>(from + kRun), b);
        const size_t out = (static_cast<size_t>(token) * p.query_heads + at.head) * D;
        if (at.kind == QUERY && gated && at.there) {
            Pair g[4];
            widen<IN_F16>(brought_run<IN_F16>(from + 2 * kRun), g);
            store_floats(p.gate + out + ca * 8, g);
            widen<IN_F16>(brought_run<IN_F16>(from + 3 * kRun), g);
            store_floats(p.gate + out + cb * 8, g);
        }
        fetch(t + kAhead * p.share, stage);
        const long long row = row0 + (static_cast<long long>(at.head) << pool.page_shift);
        if (at.kind == VALUE) {
            store_rows<D>(pool.view, false, row, a, b, ca, cb, sub, at.there && row0 >= 0, exchange[threadIdx.x / 32]);
            continue;
        }
        const float* norm = at.kind == QUERY ? p.q_norm : p.k_norm;
        if (norm != nullptr) {
            if (weighed != at.kind) {
                weighed = at.kind;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[0][i] = pack_pair(norm[ca * 8 + 2 * i], norm[ca * 8 + 2 * i + 1]);
                    w[1][i] = pack_pair(norm[cb * 8 + 2 * i], norm[cb * 8 + 2 * i + 1]);
                }
            }
            Pair sums = mul2(a[0], a[0]), more = mul2(b[0], b[0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) {
                sums = fma2(a[i], a[i], sums);
                more = fma2(b[i], b[i], more);
            }
            const float2 x = unpack_pair(sums), y = unpack_pair(more);
            float sum = x.x + x.y + y.x + y.y;
#pragma unroll
            for (int o = 1; o < static_cast<int>(kLanes); o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = rsqrtf(fmaf(sum, 1.0f / D, p.epsilon));
            const Pair inv2 = pack_pair(inv, inv);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = mul2(mul2(a[i], inv2), w[0][i]);
                b[i] = mul2(mul2(b[i], inv2), w[1][i]);
            }
        }
        if (p.neighbours) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = unpack_pair(a[i]), y = unpack_pair(b[i]);   // (an infinity behind the rotated part stays one)
                if (turns_a) a[i] = pack_pair(fmaf(x.x, cs[i], -x.y * sn[i]), fmaf(x.x, sn[i], x.y * cs[i]));
                if (turns_b) b[i] = pack_pair(fmaf(y.x, cs[4 + i], -y.y * sn[4 + i]), fmaf(y.x, sn[4 + i], y.y * cs[4 + i]));
            }
        } else if (in_halves) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Pair c = pack_pair(cs[2 * i], cs[2 * i + 1]), n = pack_pair(sn[2 * i], sn[2 * i + 1]), minus = pack_pair(-sn[2 * i], -sn[2 * i + 1]);
                const Pair x = a[i], y = b[i];
                a[i] = fma2(y, minus, mul2(x, c));
                b[i] = fma2(x, n, mul2(y, c));
            }
        }
        if (at.kind == KEY) {
            store_rows<D>(pool.view, true, row, a, b, ca, cb, sub, at.there && row0 >= 0, exchange[threadIdx.x / 32]);
        } else if (at.there) {
            if (p.q_out_is_f16) {
                __half* to = static_cast<__half*>(p.q_out) + out;
                *reinterpret_cast<uint4*>(to + ca * 8) = as_halves(a);
                *reinterpret_cast<uint4*>(to + cb * 8) = as_halves(b);
            } else {
                store_floats(static_cast<float*>(p.q_out) + out + ca * 8, a);
                store_floats(static_cast<float*>(p.q_out) + out + cb * 8, b);
            }
        }
    }
}

template <int D>
int launch_rotary(const RotaryParams& p, bool f16, cudaStream_t stream) {
    const uint64_t warps = static_cast<uint64_t>(p.pool.batch.total_tokens) * p.share;
    const dim3 grid(static_cast<uint32_t>((warps + kRotaryWarps - 1) / kRotaryWarps)), block(kRotaryWarps * 32);
    B200KV_CUDA_TRY(f16 ? launch_kernel(paged_rotary_kernel<D, true>, grid, block, 0, stream, true, p) : launch_kernel(paged_rotary_kernel<D, false>, grid, block, 0, stream, true, p));
    return B200KV_OK;
}

// A frequency in radians a position as a 64-bit fraction of a turn.
uint64_t turns_of(long double radians) {
    long double f = radians / 6.283185307179586476925286766559005768L;
    f = std::ldexp(f - std::floor(f), 64);
    if (f >= 18446744073709551615.0L) return 0xffffffffffffffffull;
    const uint64_t whole = static_cast<uint64_t>(f);
    return whole + (f - static_cast<long double>(whole) >= 0.5L ? 1 : 0);
}

}  // namespace

}  // namespace b200kv

using namespace b200kv;

extern "C" {

int b200kv_rotary_turns_of(const double* radians, uint32_t count, uint64_t* turns) {
    if (radians == nullptr || turns == nullptr) return B200KV_ERR_INVALID;
    for (uint32_t i = 0; i < count; ++i)
        if (!std::isfinite(radians[i])) return B200KV_ERR_INVALID;
    for (uint32_t i = 0; i < count; ++i) turns[i] = turns_of(radians[i]);
    return B200KV_OK;
}

int b200kv_rotary_turns(uint32_t dims, double theta, const b200kv_rotary_scaling* scaling, uint64_t* turns, float* magnitude) {
    if (turns == nullptr || dims == 0 || dims > 256 || dims % 16 != 0 || !std::isfinite(theta) || !(theta > 1.0)) return B200KV_ERR_INVALID;
    const int kind = scaling != nullptr ? scaling->kind : B200KV_ROTARY_PLAIN;
    if (kind < B200KV_ROTARY_PLAIN || kind > B200KV_ROTARY_RAMP) return B200KV_ERR_INVALID;
    if (kind != B200KV_ROTARY_PLAIN && (!std::isfinite(scaling->factor) || !(scaling->factor > 0.0))) return B200KV_ERR_INVALID;
    const bool ranged = kind == B200KV_ROTARY_BANDS || kind == B200KV_ROTARY_RAMP;
    if (ranged && (!std::isfinite(scaling->original_length) || !(scaling->original_length > 0.0) || !std::isfinite(scaling->high) || !(scaling->low > 0.0) || !(scaling->high > scaling->low)))
        return B200KV_ERR_INVALID;
    constexpr long double kTurn = 6.283185307179586476925286766559005768L;
    const long double factor = kind == B200KV_ROTARY_PLAIN ? 1.0L : scaling->factor, n = dims;
    long double base = theta;
    if (kind == B200KV_ROTARY_BASE) base *= std::pow(factor, n / (n - 2));
    // the pair that turns so many times in the original length
    const auto pair_of = [&](double times) { return n * std::log(scaling->original_length / (times * kTurn)) / (2 * std::log(static_cast<long double>(theta))); };
    long double ramp0 = 0, ramp1 = 0;
    if (kind == B200KV_ROTARY_RAMP) {
        ramp0 = std::max(std::floor(pair_of(scaling->high)), 0.0L);
        ramp1 = std::min(std::ceil(pair_of(scaling->low)), n - 1);
        if (!(ramp1 > ramp0)) ramp1 = ramp0 + 0.001L;
    }
    for (uint32_t i = 0; i < dims / 2; ++i) {
        long double f = std::pow(base, -2.0L * i / n);
        const auto clamp = [](long double x) { return std::min(std::max(x, 0.0L), 1.0L); };
        if (kind == B200KV_ROTARY_LINEAR) f /= factor;
        if (kind == B200KV_ROTARY_BANDS) {
            const long double kept = clamp((scaling->original_length * f / kTurn - scaling->low) / (static_cast<long double>(scaling->high) - scaling->low));
            f = kept * f + (1 - kept) * f / factor;
        }
        if (kind == B200KV_ROTARY_RAMP) {
            const long double part = clamp((i - ramp0) / (ramp1 - ramp0));
            f = part * f / factor + (1 - part) * f;
        }
        turns[i] = turns_of(f);
    }
    if (magnitude != nullptr) *magnitude = kind == B200KV_ROTARY_RAMP && factor > 1 ? static_cast<float>(0.1L * std::log(factor) + 1) : 1.0f;
    return B200KV_OK;
}

int b200kv_paged_rotary(const b200kv_paged_view* view, const b200kv_paged_batch* batch, const b200kv_rotary* rotary, const void* q, uint64_t q_stride, const void* key,
                        uint64_t key_stride, const void* value, uint64_t value_stride, int dtype, const float* q_norm_weight, const float* k_norm_weight, float epsilon,
                        const int32_t* positions, uint32_t query_heads, void* q_out, int q_out_dtype, float* gate, void* stream) {
    int rc = validate_paged(view, batch);
    if (rc != B200KV_OK) return rc;
    if (rotary == nullptr || (dtype != B200KV_F16 && dtype != B200KV_F32) || !std::isfinite(epsilon) || epsilon < 0.0f) return B200KV_ERR_INVALID;
    if ((q == nullptr && key == nullptr) || (key == nullptr) != (value == nullptr) || (q == nullptr) != (q_out == nullptr)) return B200KV_ERR_INVALID;
    if (rotary->dims > view->head_dim || rotary->dims % 16 != 0) return B200KV_ERR_UNSUPPORTED;
    if (rotary->layout != B200KV_ROTARY_HALVES && rotary->layout != B200KV_ROTARY_NEIGHBOURS) return B200KV_ERR_INVALID;
    if (rotary->dims > 0 && (rotary->turns == nullptr || (reinterpret_cast<uintptr_t>(rotary->turns) & 7u) != 0 || !std::isfinite(rotary->magnitude))) return B200KV_ERR_INVALID;
    const auto aligned = [](const void* a, uintptr_t to) { return (reinterpret_cast<uintptr_t>(a) & (to - 1)) == 0; };
    const uint64_t size = dtype == B200KV_F16 ? 2 : 4, d = view->head_dim, tokens = batch->total_tokens, kv_width = view->kv_heads * d, q_width = query_heads * d * (gate != nullptr ? 2 : 1);
    if (!aligned(q, 16) || !aligned(key, 16) || !aligned(value, 16) || !aligned(q_out, 16) || !aligned(gate, 16) || !aligned(q_norm_weight, 4) || !aligned(k_norm_weight, 4) ||
        !aligned(positions, 4))
        return B200KV_ERR_INVALID;
    const auto rows_fit = [&](uint64_t stride, uint64_t width) { return stride >= width && stride * size % 16 == 0 && stride < 1ull << 32; };
    if (q != nullptr) {
        if (query_heads == 0 || query_heads > 65535u || (q_out_dtype != B200KV_F16 && q_out_dtype != B200KV_F32) || !rows_fit(q_stride, q_width)) return B200KV_ERR_INVALID;
    } else if (gate != nullptr) {
        return B200KV_ERR_INVALID;
    }
    if (key != nullptr && (!rows_fit(key_stride, kv_width) || !rows_fit(value_stride, kv_width))) return B200KV_ERR_INVALID;
    if (tokens == 0 || batch->sequences == 0) return B200KV_OK;
    if (q != nullptr) {
        // the queries may be rotated where they lie; no other row is written over before it is read
        const uint64_t out = tokens * query_heads * d, out_size = q_out_dtype == B200KV_F16 ? 2 : 4;
        const auto extent = [&](uint64_t stride, uint64_t width) { return ((tokens - 1) * stride + width) * size; };
        const bool in_place = q_out == q && q_out_dtype == dtype && gate == nullptr && q_stride == q_width;
        if (!in_place && share(q, extent(q_stride, q_width), q_out, out * out_size)) return B200KV_ERR_INVALID;
        if (gate != nullptr && (share(q, extent(q_stride, q_width), gate, out * 4) || share(q_out, out * out_size, gate, out * 4))) return B200KV_ERR_INVALID;
        if (key != nullptr)
            for (const auto& [rows, stride] : {std::pair{key, key_stride}, std::pair{value, value_stride}})
                if (share(rows, extent(stride, kv_width), q_out, out * out_size) || (gate != nullptr && share(rows, extent(stride, kv_width), gate, out * 4))) return B200KV_ERR_INVALID;
    }
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    RotaryParams p{paged_of(*view, *batch), rotary->turns, rotary->dims, rotary->layout == B200KV_ROTARY_NEIGHBOURS, rotary->magnitude, epsilon, q, key, value, q_stride, key_stride,
                   value_stride, q_norm_weight, k_norm_weight, positions, q_out, q_out_dtype == B200KV_F16, gate, q != nullptr ? query_heads : 0, 1};
    // Warps to a token: one, or as many as there are steps where the tokens alone do not occupy the device.
    const uint32_t at_once = view->head_dim == 128 ? 4 : 2;
    const uint64_t steps = (p.query_heads + at_once - 1) / at_once + (key != nullptr ? 2 * ((view->kv_heads + at_once - 1) / at_once) : 0);
    p.share = static_cast<uint32_t>(std::min<uint64_t>(steps, std::max<uint64_t>(1, 32ull * device_sms() / tokens)));
    if (tokens * p.share > 0x7fffffffull) return B200KV_ERR_RANGE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return view->head_dim == 128 ? launch_rotary<128>(p, dtype == B200KV_F16, s) : launch_rotary<256>(p, dtype == B200KV_F16, s);
}

}  // extern "C"
