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
};

// One thread, 16 bytes of output: eight elements of a row of one side.  A block takes 256 of them of one token, its rows of all kv heads lying one behind the
// other in the output, and the token is looked up once.  Bound by latency for few tokens, by HBM for many.
template <int D>
__global__ void __launch_bounds__(256) paged_load_kernel(const __grid_constant__ LoadParams p) {
    constexpr uint32_t CPR = D / 8;   // chunks of a row
    pdl_launch_dependents();
    pdl_wait();                       // the rows come from the store kernel just before
    const Paged& pool = p.pool;
    const uint32_t token = blockIdx.x, c = threadIdx.x % CPR, head = blockIdx.y * (256 / CPR) + threadIdx.x / CPR;
    const bool is_k = (blockIdx.z == 0) == (p.key != nullptr) || p.value == nullptr;
    const uint32_t s = sequence_of(pool, token);
    const Span span = span_of(pool, s);
    const int j = span.base() + static_cast<int>(token - span.first);
    if (token < span.first || token - span.first >= span.tokens || head >= pool.view.kv_heads) return;
    uint4 v = make_uint4(0, 0, 0, 0);
    const long long row = j < 0 ? -1 : row_of(pool, s, head, static_cast<uint32_t>(j));
    if (row >= 0) {
        const size_t at = static_cast<size_t>(row) * D + c * 8;
        if (is_k ? is_k_q8(pool.view.quant_mode) : is_v_q8(pool.view.quant_mode)) {
            const uint32_t blocks = D / pool.view.qblock;
            const __half scale = static_cast<const __half*>(is_k ? pool.view.key_scales : pool.view.value_scales)[static_cast<size_t>(row) * blocks + (blocks == 1 ? 0 : c / 4)];
            v = dequant8(*reinterpret_cast<const uint2*>((is_k ? pool.view.key_q8 : pool.view.value_q8) + at), scale);
        } else {
            v = *reinterpret_cast<const uint4*>(static_cast<const __half*>(is_k ? pool.view.key_f16 : pool.view.value_f16) + at);
        }
    }
    *reinterpret_cast<uint4*>((is_k ? p.key : p.value) + (static_cast<size_t>(token) * pool.view.kv_heads + head) * D + c * 8) = v;
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
    const LoadParams p{paged_of(*view, *batch), static_cast<__half*>(key), static_cast<__half*>(value)};
    const uint32_t heads_per_block = 256 / (view->head_dim / 8);
    const dim3 grid(batch->total_tokens, (view->kv_heads + heads_per_block - 1) / heads_per_block, key != nullptr && value != nullptr ? 2 : 1);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    B200KV_CUDA_TRY(view->head_dim == 128 ? launch_kernel(paged_load_kernel<128>, grid, dim3(256), 0, s, true, p)
                                          : launch_kernel(paged_load_kernel<256>, grid, dim3(256), 0, s, true, p));
    return B200KV_OK;
}
