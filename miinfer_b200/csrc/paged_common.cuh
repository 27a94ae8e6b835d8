// What the kernels over a paged cache share: a sequence's part of a ragged batch, the way from a position to its row, and launches that follow one
// another within a call.
#pragma once

#include "kv_common.cuh"

namespace b200kv {

uint32_t* current_status_word();

constexpr uint32_t kMostSequences = 8192;   // of a batch

// Checks geometry, pointers and bounds.
int validate_paged(const b200kv_paged_view* view, const b200kv_paged_batch* batch);

// What every kernel needs of a call.  Rows are numbered over the whole pool, (page * kv_heads + head) * page_size + slot; all planes share the number.
struct Paged {
    b200kv_paged_view view;
    b200kv_paged_batch batch;
    uint32_t page_shift;       // log2 of the page size
    uint32_t* status;          // may be null
};
// Whether two arrays of so many bytes share any.
inline bool share(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}
// A window that reaches over every length is none, and without one there are no sinks.
void settle_window(const b200kv_paged_batch& batch, uint32_t* window, uint32_t* sinks);
Paged paged_of(const b200kv_paged_view& view, const b200kv_paged_batch& batch);

struct Span {
    uint32_t first;    // its first row of the activations
    uint32_t tokens;   // new tokens
    uint32_t length;   // cached positions, the new tokens among them
    // place in the cache of new token t: base() + t; negative where a length is smaller than the number of new tokens
    __device__ __forceinline__ int base() const { return static_cast<int>(length) - static_cast<int>(tokens); }
};

__device__ __forceinline__ void report(const Paged& p, uint32_t bit) {
    if (p.status != nullptr) atomicOr(p.status, bit);
}

// Sequence s, cut to the bounds of the launch (arrays that contradict them cost results, never an access out of range).
__device__ __forceinline__ Span span_of(const Paged& p, uint32_t s) {
    const b200kv_paged_batch& b = p.batch;
    const int total = static_cast<int>(b.total_tokens);
    const int q0 = b.query_starts[s], q1 = b.query_starts[s + 1], len = b.lengths[s];
    const int most = static_cast<int>(min(static_cast<uint64_t>(b.max_length), static_cast<uint64_t>(b.max_pages) << p.page_shift));
    const int first = min(max(q0, 0), total), end = min(max(q1, first), total);
    Span span{static_cast<uint32_t>(first), min(static_cast<uint32_t>(end - first), b.max_tokens), static_cast<uint32_t>(min(max(len, 0), most))};
    if (first != q0 || static_cast<int>(span.tokens) != q1 - q0 || static_cast<int>(span.length) != len) report(p, B200KV_STATUS_BAD_BOUND);
    return span;
}

// The sequence that row `row` of the activations belongs to: the last s < sequences with query_starts[s] <= row.  Its tokens may end before the row.
__device__ __forceinline__ uint32_t sequence_of(const Paged& p, uint32_t row) {
    uint32_t lo = 0, hi = p.batch.sequences;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (p.batch.query_starts[mid] <= static_cast<int>(row)) lo = mid;
        else hi = mid;
    }
    return lo;
}

// What a new token sees: positions [low, upto), and the first sinks below upto.
struct Sight {
    uint32_t low, upto;
    __device__ __forceinline__ bool empty() const { return low >= upto; }   // but for the sinks
};
// Of the token in row `row` of the activations, at place `place` of its sequence of `length` positions.  ranges (may be null): a token's own [low, upto) in place of [0, place + 1).
__device__ __forceinline__ Sight sight_of(const int32_t* ranges, size_t row, int place, uint32_t window, uint32_t length) {
    if (place < 0) return {0, 0};
    int low = 0, upto = place + 1;
    if (ranges != nullptr) {
        const int2 r = reinterpret_cast<const int2*>(ranges)[row];
        low = max(r.x, 0);
        upto = max(r.y, 0);
    }
    if (window > 0) low = max(low, place + 1 - static_cast<int>(window));
    return {static_cast<uint32_t>(low), min(static_cast<uint32_t>(upto), length)};
}

constexpr float kTanhSmall = 0.8f;
// tanh of any x: 1 - 2 / (e^2x + 1), off by a few roundings of numbers near 1, and so by up to 3e-7.
__device__ __forceinline__ float tanh_large(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 2.8853900817779268f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
    return fmaf(-2.0f, r, 1.0f);
}
// Of |x| <= kTanhSmall, by odd powers up to the eleventh: the polynomial with the smallest relative error, 5.8e-8 (Remez's exchange); 1e-7 in fp32.
__device__ __forceinline__ float tanh_small(float x) {
    const float k[6] = {0.99999994f, -0.333326757f, 0.13321048f, -0.0531143136f, 0.0190933011f, -0.00435529929f}, u = x * x;
    float r = k[5];
#pragma unroll
    for (int i = 4; i >= 0; --i) r = fmaf(r, u, k[i]);
    return x * r;
}

// The first row of page number `page` for a kv head, or -1 for a page outside the pool.
__device__ __forceinline__ long long page_row(const Paged& p, int page, uint32_t head) {
    if (static_cast<uint32_t>(page) >= p.view.pages) {
        report(p, B200KV_STATUS_BAD_PAGE);
        return -1;
    }
    return ((static_cast<long long>(page) * p.view.kv_heads + head) << p.page_shift);
}
__device__ __forceinline__ const int32_t* pages_of(const Paged& p, uint32_t s) { return p.batch.page_table + static_cast<size_t>(s) * p.batch.max_pages; }
// The row of position j of sequence s (j below its length), or -1.
__device__ __forceinline__ long long row_of(const Paged& p, uint32_t s, uint32_t head, uint32_t j) {
    const long long row = page_row(p, pages_of(p, s)[j >> p.page_shift], head);
    return row < 0 ? row : row + (j & ((1u << p.page_shift) - 1));
}

// A launch behind another of the same call: it may become resident early whatever the process-wide overlap is, since every kernel of a call waits for
// the one before it (griddepcontrol.wait, in every CTA) before it touches anything.
template <typename... KArgs, typename... Args>
cudaError_t launch_behind(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace b200kv
