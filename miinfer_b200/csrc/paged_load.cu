// A paged cache on the host's side of a launch: checks of a view and a batch, what kernels are handed of them, and the gather that takes the rows of
// a ragged batch out of their pages as fp16.
#include "paged_common.cuh"
#include "dequant.cuh"

#include <algorithm>

namespace b200kv {

int validate_paged(const b200kv_paged_view* v, const b200kv_paged_batch* b) {
    if (v == nullptr || b == nullptr) return B200KV_ERR_INVALID;
    if (v->pages == 0 || v->kv_heads == 0 || v->quant_mode > B200KV_Q8_Q8) return B200KV_ERR_INVALID;
    if (v->page_size < 16 || v->page_size > 256 || (v->page_size & (v->page_size - 1)) != 0) return B200KV_ERR_UNSUPPORTED;
    if (v->head_dim != 128 && v->head_dim != 256) return B200KV_ERR_UNSUPPORTED;
    if (v->qblock != 32 && v->qblock != v->head_dim) return B200KV_ERR_UNSUPPORTED;
    if (v->pages > 0x7fffffffu || v->kv_heads > 65535u) return B200KV_ERR_UNSUPPORTED;   // page numbers are int32
    const auto given = [](const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    if (is_k_q8(v->quant_mode) ? !given(v->key_q8) || !given(v->key_scales) : !given(v->key_f16)) return B200KV_ERR_INVALID;
    if (is_v_q8(v->quant_mode) ? !given(v->value_q8) || !given(v->value_scales) : !given(v->value_f16)) return B200KV_ERR_INVALID;
    if (b->sequences == 0) return B200KV_OK;
    const auto word = [](const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
    if (!word(b->page_table) || !word(b->query_starts) || !word(b->lengths) || b->max_pages == 0) return B200KV_ERR_INVALID;
    if (b->sequences > kMostSequences) return B200KV_ERR_UNSUPPORTED;
    if (b->total_tokens > 0x7fffffffu || b->max_length > 0x7fffffffu || b->max_tokens > b->total_tokens) return B200KV_ERR_INVALID;
    if (b->max_length > static_cast<uint64_t>(b->max_pages) * v->page_size) return B200KV_ERR_RANGE;
    return B200KV_OK;
}

Paged paged_of(const b200kv_paged_view& view, const b200kv_paged_batch& batch) {
    Paged p{view, batch, 0, current_status_word()};
    while ((1u << p.page_shift) < view.page_size) ++p.page_shift;
    return p;
}

void settle_window(const b200kv_paged_batch& batch, uint32_t* window, uint32_t* sinks) {
    if (*window >= batch.max_length) *window = 0;
    *sinks = *window == 0 ? 0 : std::min(*sinks, batch.max_length);
}

namespace {

struct LoadParams {
    Paged pool;
    __half* key;
    __half* value;
    uint32_t tokens;   // of a warp: 1 or 4
};

// A warp takes a token of one side, or four where there are many: its first lanes look up where they lie, then all of it brings the rows of all kv heads, 16 bytes of output a lane and
// step, eight steps' loads under way together.  Bound by latency for few tokens, by HBM for many.
constexpr int kLoadThreads = 128, kLoadSteps = 8;
template <int D>
__global__ void __launch_bounds__(kLoadThreads) paged_load_kernel(const __grid_constant__ LoadParams p) {
    constexpr uint32_t CPR = D / 8;   // chunks of a row
    pdl_launch_dependents();
    pdl_wait();                       // the rows come from the store kernel just before
    const Paged& pool = p.pool;
    const uint32_t lane = threadIdx.x & 31, token0 = (blockIdx.x * (kLoadThreads / 32) + threadIdx.x / 32) * p.tokens, H = pool.view.kv_heads;
    const bool is_k = (blockIdx.y == 0) == (p.key != nullptr) || p.value == nullptr;
    // lane l < p.tokens: token token0 + l.  -2: not of any sequence; -1: of no page, zeros; else its row for kv head 0
    long long place = -2;
    if (lane < p.tokens && token0 + lane < pool.batch.total_tokens) {
        const uint32_t token = token0 + lane, s = sequence_of(pool, token);
        const Span span = span_of(pool, s);
        if (token >= span.first && token - span.first < span.tokens) {
            const int j = span.base() + static_cast<int>(token - span.first);
            place = j < 0 ? -1 : row_of(pool, s, 0, static_cast<uint32_t>(j));
        }
    }
    const bool q8 = is_k ? is_k_q8(pool.view.quant_mode) : is_v_q8(pool.view.quant_mode);
    const int8_t* q = is_k ? pool.view.key_q8 : pool.view.value_q8;
    const __half* scales = static_cast<const __half*>(is_k ? pool.view.key_scales : pool.view.value_scales);
    const __half* f16 = static_cast<const __half*>(is_k ? pool.view.key_f16 : pool.view.value_f16);
    __half* out = (is_k ? p.key : p.value) + static_cast<size_t>(token0) * H * D;
    const uint32_t blocks = D / pool.view.qblock, chunks = H * CPR;   // of a token
    for (uint32_t t = 0; t < p.tokens; ++t) {
        const long long at = __shfl_sync(0xffffffffu, place, t);
        if (at == -2) continue;
        for (uint32_t c0 = 0; c0 < chunks; c0 += 32 * kLoadSteps) {
            uint4 v[kLoadSteps];
            __half scale[kLoadSteps];
#pragma unroll
            for (int i = 0; i < kLoadSteps; ++i) {
                const uint32_t n = c0 + 32 * i + lane, head = n / CPR, c = n % CPR;
                v[i] = make_uint4(0, 0, 0, 0);
                scale[i] = __ushort_as_half(0);
                if (n >= chunks || at < 0) continue;
                const size_t row = static_cast<size_t>(at) + (static_cast<size_t>(head) << pool.page_shift);
                if (q8) {
                    const uint2 raw = *reinterpret_cast<const uint2*>(q + row * D + c * 8);
                    v[i].x = raw.x; v[i].y = raw.y;
                    scale[i] = scales[row * blocks + (blocks == 1 ? 0 : c / 4)];
                } else {
                    v[i] = *reinterpret_cast<const uint4*>(f16 + row * D + c * 8);
                }
            }
#pragma unroll
            for (int i = 0; i < kLoadSteps; ++i) {
                const uint32_t n = c0 + 32 * i + lane;
                if (n < chunks) *reinterpret_cast<uint4*>(out + (static_cast<size_t>(t) * chunks + n) * 8) = q8 ? dequant8(make_uint2(v[i].x, v[i].y), scale[i]) : v[i];
            }
        }
    }
}

}  // namespace

}  // namespace b200kv

using namespace b200kv;

extern "C" int b200kv_paged_load(const b200kv_paged_view* view, const b200kv_paged_batch* batch, void* key, void* value, void* stream) {
    int rc = validate_paged(view, batch);
    if (rc != B200KV_OK) return rc;
    if ((key == nullptr && value == nullptr) || ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15u) != 0) return B200KV_ERR_INVALID;
    if (batch->total_tokens == 0 || batch->sequences == 0) return B200KV_OK;
    rc = ensure_device();
    if (rc != B200KV_OK) return rc;
    // four where every SM has sixteen warps with work all the same: 48, 2000, 4700, 10000 and 40000 tokens of 8 heads of 128, q8_0, took 8.3, 11.2, 15.3, 21.5 and 62.3 us
    // with one a warp, 13.2, 13.2, 15.3, 21.7 and 54.3 with four
    const uint32_t tokens = batch->total_tokens >= 4 * 16 * device_sms() / 2 ? 4 : 1, of_block = kLoadThreads / 32 * tokens;
    const LoadParams p{paged_of(*view, *batch), static_cast<__half*>(key), static_cast<__half*>(value), tokens};
    const dim3 grid((batch->total_tokens + of_block - 1) / of_block, key != nullptr && value != nullptr ? 2 : 1);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    B200KV_CUDA_TRY(view->head_dim == 128 ? launch_kernel(paged_load_kernel<128>, grid, dim3(kLoadThreads), 0, s, true, p)
                                          : launch_kernel(paged_load_kernel<256>, grid, dim3(kLoadThreads), 0, s, true, p));
    return B200KV_OK;
}
