// A layer's queries, keys and values of a ragged batch on their way to the attention over a paged cache, in one launch: norms, rotary positions of any of the usual forms,
// the gate split off the queries, quantisation, and the write of K and V into their pages.
//
//   a' = m (a cos p f_i - b sin p f_i),  b' = m (a sin p f_i + b cos p f_i)   for pair i of the first `dims` elements of a head: (i, i + dims/2) or (2i, 2i + 1), position p
//
// Angles.  p f_i in fp32 is off by 2^-24 of itself, a tenth of a radian at a million.  A frequency comes as a 64-bit fraction of a turn instead: p times it modulo 2^64 is the
// angle's fraction of a turn, exact but for the table's own rounding (p 2^-65 turns).  Its upper 32 bits less the nearest quarter are the argument of a Taylor polynomial (to x^9 / x^8
// on |x| <= pi/4, 3e-8).
//
// A lane holds eight consecutive elements, D/8 lanes a row (two rows a warp at head_dim 128).  Halves that are not in the lane come by shuffles.  A warp takes all rows of a token, or several share them where there are few tokens; the token's sines and cosines are worked out once a warp.
// Bound by HBM for prompts, by latency for a decode step.
#include "append_row.cuh"
#include "paged_common.cuh"

#include <algorithm>
#include <cmath>
#include <utility>

namespace b200kv {

namespace {

constexpr int kRotaryWarps = 4;
constexpr uint32_t kAhead = 2;   // steps

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

template <bool IN_F16> struct Eight { uint4 v[IN_F16 ? 1 : 2]; };   // a lane's elements as they lie in memory
template <bool IN_F16>
__device__ __forceinline__ Eight<IN_F16> load_eight(const void* src, size_t element) {
    Eight<IN_F16> r;
#pragma unroll
    for (int i = 0; i < (IN_F16 ? 1 : 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(src) + element * (IN_F16 ? 2 : 4))[i];
    return r;
}
template <bool IN_F16>
__device__ __forceinline__ void widen(const Eight<IN_F16>& r, float (&x)[8]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (IN_F16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + i));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        } else {
            x[2 * i] = __uint_as_float(w[2 * i]); x[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
        }
    }
}
__device__ __forceinline__ uint4 eight_halves(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_floats(float* to, const float (&x)[8]) {
    reinterpret_cast<float4*>(to)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(to)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// A row into the cache: eight elements a lane, `lanes` of the row.  The bits are quantize_row's.
template <int D>
__device__ __forceinline__ void store_row(const b200kv_paged_view& view, bool is_k, long long row, const float (&x)[8], int c, bool there) {
    const bool q8 = is_k ? is_k_q8(view.quant_mode) : is_v_q8(view.quant_mode);
    if (!q8) {
        if (there) *reinterpret_cast<uint4*>(static_cast<__half*>(is_k ? view.key_f16 : view.value_f16) + row * D + c * 8) = eight_halves(x);
        return;
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
    const bool rows = view.qblock == D;
    for (int o = 1; o < (rows ? D / 8 : 4); o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float scale = amax > 0.0f ? __fdiv_rn(amax, 127.0f) : 1.0f;
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 1.0f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i / 4] |= static_cast<uint32_t>(quantize_s8(__fmul_rn(x[i], inv)) & 0xff) << (8 * (i % 4));
    if (!there) return;
    *reinterpret_cast<uint2*>((is_k ? view.key_q8 : view.value_q8) + row * D + c * 8) = make_uint2(w[0], w[1]);
    __half* scales = static_cast<__half*>(is_k ? view.key_scales : view.value_scales);
    if (rows ? c == 0 : (c & 3) == 0) scales[rows ? row : row * (D / 32) + c / 4] = __float2half_rn(scale);
}

template <int D, bool IN_F16>
__global__ void __launch_bounds__(kRotaryWarps * 32) paged_rotary_kernel(const __grid_constant__ RotaryParams p) {
    constexpr int kLanes = D / 8, kRows = 32 / kLanes;   // of a row; rows a warp takes at a time
    pdl_wait();
    pdl_launch_dependents();                             // behind the wait: it writes cache rows
    const Paged& pool = p.pool;
    const uint32_t lane = threadIdx.x & 31, c = lane % kLanes, sub = lane / kLanes;
    const uint64_t me = static_cast<uint64_t>(blockIdx.x) * kRotaryWarps + threadIdx.x / 32;
    if (me >= static_cast<uint64_t>(pool.batch.total_tokens) * p.share) return;
    const uint32_t token = static_cast<uint32_t>(me / p.share), part = static_cast<uint32_t>(me % p.share);

    // ---- where the token goes, and its angles
    const uint32_t s = sequence_of(pool, token);
    const Span span = span_of(pool, s);
    if (token < span.first || token - span.first >= span.tokens) return;
    const int place = span.base() + static_cast<int>(token - span.first);
    const long long row0 = place >= 0 && p.key != nullptr ? row_of(pool, s, 0, static_cast<uint32_t>(place)) : -1;   // for kv head 0
    const uint64_t position = static_cast<uint32_t>(max(p.positions != nullptr ? p.positions[token] : place, 0));
    const bool turns = c * 8 < p.dims;
    const uint32_t half = p.dims / 16;                   // chunks of a half
    const uint32_t other = !turns || p.neighbours ? c : c < half ? c + half : c - half;   // the chunk of the elements' partners
    float cs[8], sn[8];                                  // x' = x cs + partner sn
#pragma unroll
    for (int i = 0; i < 8; ++i) { cs[i] = 1.0f; sn[i] = 0.0f; }
    if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (p.neighbours && (i & 1)) {
                cs[i] = cs[i - 1];
                sn[i] = -sn[i - 1];
                continue;
            }
            const uint32_t pair = p.neighbours ? c * 4 + i / 2 : (c < half ? c : c - half) * 8 + i;
            float sine, cosine;
            sincos_turns(position * p.turns[pair], &sine, &cosine);
            cs[i] = cosine * p.magnitude;
            sn[i] = (p.neighbours || c < half ? -sine : sine) * p.magnitude;
        }
    }

    // ---- its rows: queries with their gates, keys, values, a step at a time; kAhead steps' loads are under way
    const uint32_t H = pool.view.kv_heads;
    const uint32_t k0 = p.q != nullptr ? (p.query_heads + kRows - 1) / kRows : 0, kv_steps = p.key != nullptr ? (H + kRows - 1) / kRows : 0, v0 = k0 + kv_steps, steps = v0 + kv_steps;
    const bool gated = p.gate != nullptr;
    enum { QUERY, KEY, VALUE };
    struct Step { int kind; uint32_t head; bool there; };
    const auto step_of = [&](uint32_t t) {
        const int kind = t < k0 ? QUERY : t < v0 ? KEY : VALUE;
        const uint32_t head = (t - (kind == QUERY ? 0 : kind == KEY ? k0 : v0)) * kRows + sub;
        return Step{kind, head, t < steps && head < (kind == QUERY ? p.query_heads : H)};
    };
    using Raw = Eight<IN_F16>;
    Raw raw[kAhead], raw_gate[kAhead];
    const auto fetch = [&](uint32_t t, Raw& r, Raw& g) {
        const Step at = step_of(t);
        r = g = Raw{};
        if (!at.there) return;
        if (at.kind == QUERY) {
            const size_t element = token * p.q_stride + static_cast<size_t>(at.head) * (gated ? 2 * D : D) + c * 8;
            r = load_eight<IN_F16>(p.q, element);
            if (gated) g = load_eight<IN_F16>(p.q, element + D);
        } else {
            r = at.kind == KEY ? load_eight<IN_F16>(p.key, token * p.key_stride + at.head * D + c * 8) : load_eight<IN_F16>(p.value, token * p.value_stride + at.head * D + c * 8);
        }
    };
    float w[8];
    int weighed = -1;                                    // whose norm's weights these are
    const auto take = [&](uint32_t t, const Raw& now, const Raw& now_gate) {
        const Step at = step_of(t);
        float x[8];
        widen<IN_F16>(now, x);
        if (at.kind == VALUE) {
            store_row<D>(pool.view, false, row0 + (static_cast<long long>(at.head) << pool.page_shift), x, c, at.there && row0 >= 0);
            return;
        }
        const float* norm = at.kind == QUERY ? p.q_norm : p.k_norm;
        if (norm != nullptr) {
            if (weighed != at.kind) {
                weighed = at.kind;
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = norm[c * 8 + i];
            }
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = __frsqrt_rn(fmaf(sum, 1.0f / D, p.epsilon));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i];
        }
        float y[8];
        if (p.neighbours) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], static_cast<int>(sub * kLanes + other));
        }
        if (turns) {   // (an infinity in the rest of a head stays one)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], cs[i], y[i] * sn[i]);
        }
        if (at.kind == KEY) {
            store_row<D>(pool.view, true, row0 + (static_cast<long long>(at.head) << pool.page_shift), x, c, at.there && row0 >= 0);
        } else if (at.there) {
            const size_t out = (static_cast<size_t>(token) * p.query_heads + at.head) * D + c * 8;
            if (p.q_out_is_f16) *reinterpret_cast<uint4*>(static_cast<__half*>(p.q_out) + out) = eight_halves(x);
            else store_floats(static_cast<float*>(p.q_out) + out, x);
            if (gated) {
                float g[8];
                widen<IN_F16>(now_gate, g);
                store_floats(p.gate + out, g);
            }
        }
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) fetch(part + i * p.share, raw[i], raw_gate[i]);
    for (uint32_t t0 = part; t0 < steps; t0 += kAhead * p.share) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t t = t0 + i * p.share;
            if (t >= steps) break;
            const Raw now = raw[i], now_gate = raw_gate[i];
            fetch(t + kAhead * p.share, raw[i], raw_gate[i]);
            take(t, now, now_gate);
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
    const uint32_t at_once = view->head_dim == 128 ? 2 : 1;
    const uint64_t steps = (p.query_heads + at_once - 1) / at_once + (key != nullptr ? 2 * ((view->kv_heads + at_once - 1) / at_once) : 0);
    p.share = static_cast<uint32_t>(std::min<uint64_t>(steps, std::max<uint64_t>(1, 32ull * device_sms() / tokens)));
    if (tokens * p.share > 0x7fffffffull) return B200KV_ERR_RANGE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return view->head_dim == 128 ? launch_rotary<128>(p, dtype == B200KV_F16, s) : launch_rotary<256>(p, dtype == B200KV_F16, s);
}

}  // extern "C"
