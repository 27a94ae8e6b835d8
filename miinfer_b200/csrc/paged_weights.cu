// The weight that every cached position of a paged cache gets from a batch's new tokens, summed over tokens and query heads of the kv head:
// A[j] += sum over (token, head) of exp(scale q.k_j - lse), with the statistics lse that the attention call left.
#include "paged_common.cuh"

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
    float scale_log2;
};

constexpr int kPositions = 64, kRows = 8;

// A CTA takes 64 positions of a (sequence, kv head) and walks the observed rows, eight at a time; four threads share a position's dot products.
template <int D>
__global__ void __launch_bounds__(256) paged_weights_kernel(const __grid_constant__ WeightsParams p) {
    constexpr int KS = D + 4;
    extern __shared__ float smem[];
    float* k_s = smem;                       // [64][KS]
    float* q_s = smem + kPositions * KS;     // [8][D]
    __shared__ float lse_s[kRows];
    __shared__ int at_s[kRows];
    pdl_launch_dependents();
    pdl_wait();
    const Paged& pool = p.pool;
    const uint32_t s = blockIdx.z, head = blockIdx.y, tid = threadIdx.x;
    const Span span = span_of(pool, s);
    const uint32_t pos0 = blockIdx.x * kPositions, G = p.query_heads / pool.view.kv_heads;
    const uint32_t observed = p.observe > 0 ? min(p.observe, span.tokens) : span.tokens;
    if (pos0 >= span.length || observed == 0) return;
    const uint32_t t0 = span.tokens - observed;
    const bool q8 = is_k_q8(pool.view.quant_mode);
    for (uint32_t i = tid; i < kPositions * (D / 8); i += 256) {
        const uint32_t r = i / (D / 8), c = i % (D / 8);
        float v[8] = {};
        const long long row = pos0 + r < span.length ? row_of(pool, s, head, pos0 + r) : -1;
        if (row >= 0) {
            const size_t at = static_cast<size_t>(row) * D + c * 8;
            if (q8) {
                const uint32_t blocks = D / pool.view.qblock;
                const float scale = __half2float(static_cast<const __half*>(pool.view.key_scales)[static_cast<size_t>(row) * blocks + (blocks == 1 ? 0 : c / 4)]);
                for (int e = 0; e < 8; ++e) v[e] = scale * static_cast<float>(pool.view.key_q8[at + e]);
            } else {
                for (int e = 0; e < 8; ++e) v[e] = __half2float(static_cast<const __half*>(pool.view.key_f16)[at + e]);
            }
        }
        for (int e = 0; e < 8; ++e) k_s[r * KS + c * 8 + e] = v[e];
    }
    const uint32_t mine = tid / 4, part = tid % 4, j = pos0 + mine;
    float sum = 0.0f;
    for (uint32_t row0 = 0; row0 < observed * G; row0 += kRows) {
        __syncthreads();
        for (uint32_t i = tid; i < kRows * D; i += 256) {
            const uint32_t r = row0 + i / D;
            const size_t row = static_cast<size_t>(span.first + t0 + r / G) * p.query_heads + head * G + r % G;
            if (r >= observed * G) q_s[i] = 0.0f;
            else q_s[i] = p.q_is_f16 ? __half2float(static_cast<const __half*>(p.q)[row * D + i % D]) : static_cast<const float*>(p.q)[row * D + i % D];
        }
        if (tid < kRows) {
            const uint32_t r = row0 + tid;
            const bool in = r < observed * G;
            at_s[tid] = in ? span.base() + static_cast<int>(t0 + r / G) : -1;
            lse_s[tid] = in ? p.lse[static_cast<size_t>(span.first + t0 + r / G) * p.query_heads + head * G + r % G] : 0.0f;
        }
        __syncthreads();
        float dot[kRows] = {};
        for (int c = part; c < D / 4; c += 4) {
            const float4 k = *reinterpret_cast<const float4*>(k_s + mine * KS + 4 * c);
            for (int r = 0; r < kRows; ++r) {
                const float4 q = *reinterpret_cast<const float4*>(q_s + r * D + 4 * c);
                dot[r] += k.x * q.x + k.y * q.y + k.z * q.z + k.w * q.w;
            }
        }
        for (int r = 0; r < kRows; ++r) {
            dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], 1);
            dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], 2);
            const int at = at_s[r];
            const bool seen = static_cast<int>(j) <= at && (p.window == 0 || j + p.window > static_cast<uint32_t>(at) || j < p.sinks);
            if (seen && lse_s[r] != -INFINITY) sum += exp2f(dot[r] * p.scale_log2 - lse_s[r] * 1.4426950408889634f);
        }
    }
    if (part == 0 && j < span.length) p.weights[(static_cast<size_t>(s) * pool.view.kv_heads + head) * p.stride + j] += sum;
}

template <int D>
int launch_weights(const WeightsParams& p, cudaStream_t stream) {
    constexpr int kSmem = (kPositions * (D + 4) + kRows * D) * 4;
    static std::atomic<uint64_t> done{0};
    B200KV_CUDA_TRY(opt_in_dynamic_smem(reinterpret_cast<const void*>(paged_weights_kernel<D>), kSmem, done));
    const dim3 grid((p.pool.batch.max_length + kPositions - 1) / kPositions, p.pool.view.kv_heads, p.pool.batch.sequences);
    B200KV_CUDA_TRY(launch_kernel(paged_weights_kernel<D>, grid, dim3(256), kSmem, stream, true, p));
    return B200KV_OK;
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
    if (batch->sequences == 0 || batch->total_tokens == 0 || batch->max_length == 0) return B200KV_OK;
    if (weights_stride < batch->max_length) return B200KV_ERR_INVALID;
    settle_window(*batch, &window, &sinks);
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    const WeightsParams p{paged_of(*view, *batch), q, q_dtype == B200KV_F16, lse, weights, weights_stride, query_heads, window, sinks, observe,
                          scale * 1.4426950408889634f};
    return view->head_dim == 128 ? launch_weights<128>(p, static_cast<cudaStream_t>(stream)) : launch_weights<256>(p, static_cast<cudaStream_t>(stream));
}
