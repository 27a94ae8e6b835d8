// CPython module under the Python mirror's per-token launchers: takes the tensors themselves, reads pointers, dtypes and
// the current stream through torch's C++ interface, and calls the C ABI through addresses handed over by _lib.py (so
// that the one loaded libb200kv.so serves both).  It holds no state of a call and does no arithmetic.
//
// Why it exists: through ctypes a launcher spent 10-14 us of Python time per call (argument conversion, three attribute
// calls per tensor, a Stream object per call), more than the kernels of a short-context step take; here it is about 1 us.
// The interpreter lock is released around every library call, as ctypes does: a launch can block when the stream's
// queue is full.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <initializer_list>
#include <utility>
#include <vector>

#include "b200kv.h"

namespace {

struct Api {
    decltype(&b200kv_append) append;
    decltype(&b200kv_q_split_norm_rope) q_split_norm_rope;
    decltype(&b200kv_decode_attn) decode_attn;
    decltype(&b200kv_decode_step) decode_step;
    decltype(&b200kv_decode_attn_batched) decode_attn_batched;
    decltype(&b200kv_prefill_attn_prepared) prefill_attn_prepared;
    decltype(&b200kv_paged_store) paged_store;
    decltype(&b200kv_paged_load) paged_load;
    decltype(&b200kv_paged_attn) paged_attn;
    decltype(&b200kv_paged_attn_scored) paged_attn_scored;
    decltype(&b200kv_paged_weights) paged_weights;
    decltype(&b200kv_paged_evict) paged_evict;
    decltype(&b200kv_paged_rotary) paged_rotary;
    decltype(&b200kv_pages_grow) pages_grow;
    decltype(&b200kv_pages_fork) pages_fork;
    decltype(&b200kv_pages_free) pages_free;
    decltype(&b200kv_pages_compact) pages_compact;
    decltype(&b200kv_pages_copy) pages_copy;
    decltype(&b200kv_pool_capture) pool_capture;
    decltype(&b200kv_pool_restore) pool_restore;
} g_api;
PyObject* g_view_type;   // the ctypes structure of a cache view
PyObject* g_paged_view_type;    // ... of a paged cache's view, and of a batch over it
PyObject* g_paged_batch_type;
PyObject* g_paged_scoring_type; // ... of what becomes of an attention call's scores
PyObject* g_rotary_type;        // ... of a table of rotary angles
PyObject* g_page_book_type;     // ... of the book of a paged cache's pages
PyObject* g_device_index;       // the name of their attribute

// One call's arguments, read left to right; the first failure sticks and leaves a Python exception set.
class Args {
public:
    Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t want) : args_(args) {
        if (n != want) {
            PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
            ok_ = false;
        }
    }
    ~Args() {
        for (int i = 0; i < held_; ++i) PyBuffer_Release(&buffers_[i]);
    }
    bool ok() const { return ok_; }

    void* tensor(int64_t* numel = nullptr, int* dtype = nullptr) {   // None = null pointer
        if (!ok_) return nullptr;
        PyObject* o = args_[i_++];
        if (numel) *numel = 0;
        if (o == Py_None) {
            if (dtype) fail(PyExc_ValueError, "a tensor is required");
            return nullptr;
        }
        if (!THPVariable_Check(o)) return fail(PyExc_TypeError, "a torch tensor is required");
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || !t.is_contiguous()) return fail(PyExc_ValueError, "expected a contiguous CUDA tensor");
        if (numel) *numel = t.numel();
        if (dtype) {
            const auto type = t.scalar_type();
            if (type == at::kHalf) *dtype = B200KV_F16;
            else if (type == at::kFloat) *dtype = B200KV_F32;
            else return fail(PyExc_ValueError, (std::string("unsupported dtype ") + c10::toString(type) + ": fp16 or fp32 expected").c_str());
        }
        return t.data_ptr();
    }
    template <typename T> T* tensor_as(int64_t* numel = nullptr, int* dtype = nullptr) { return static_cast<T*>(tensor(numel, dtype)); }

    uint32_t u32() {   // as a C unsigned conversion: higher bits are dropped
        if (!ok_) return 0;
        PyObject* o = args_[i_++];
        if (PyLong_Check(o)) return checked(static_cast<uint32_t>(PyLong_AsUnsignedLongMask(o)));
        PyObject* v = PyNumber_Index(o);
        if (v == nullptr) { ok_ = false; return 0; }
        const uint32_t r = static_cast<uint32_t>(PyLong_AsUnsignedLongMask(v));
        Py_DECREF(v);
        return checked(r);
    }
    float f32() {
        if (!ok_) return 0.0f;
        const double v = PyFloat_AsDouble(args_[i_++]);
        if (v == -1.0 && PyErr_Occurred()) ok_ = false;
        return static_cast<float>(v);
    }
    int rope() {   // an enum member, or anything else that int() takes
        if (!ok_) return 0;
        PyObject* v = PyNumber_Long(args_[i_++]);
        if (v == nullptr) { ok_ = false; return 0; }
        const uint32_t r = checked(static_cast<uint32_t>(PyLong_AsUnsignedLongMask(v)));
        Py_DECREF(v);
        return static_cast<int>(r);
    }
    // A cache view (the ctypes structure and nothing else): its memory, through the buffer protocol.
    const b200kv_view* view() {
        if (!ok_) return nullptr;
        const int is_view = PyObject_IsInstance(args_[i_], g_view_type);
        if (is_view <= 0) {
            if (is_view == 0) PyErr_Format(PyExc_TypeError, "expected a cache view, got %s", Py_TYPE(args_[i_])->tp_name);
            ok_ = false;
            return nullptr;
        }
        return views(1, false);
    }
    // A paged cache's view or a batch over it, likewise.
    template <typename T>
    const T* structure(PyObject* type, const char* what) {
        if (!ok_) return nullptr;
        PyObject* o = args_[i_++];
        if (!PyObject_TypeCheck(o, reinterpret_cast<PyTypeObject*>(type))) {   // (PyObject_IsInstance goes through the structures' metaclass: 0.1 us for each layer's view)
            PyErr_Format(PyExc_TypeError, "expected %s, got %s", what, Py_TYPE(o)->tp_name);
            ok_ = false;
            return nullptr;
        }
        if (PyObject_GetBuffer(o, &buffers_[held_], PyBUF_SIMPLE) != 0) { ok_ = false; return nullptr; }
        const Py_buffer& b = buffers_[held_++];
        if (static_cast<size_t>(b.len) < sizeof(T)) { fail(PyExc_ValueError, "a structure of another size"); return nullptr; }
        PyObject* device = PyObject_GetAttr(o, g_device_index);   // of the tensors it was built over; -1: it was not
        const long index = device == nullptr ? -1 : PyLong_AsLong(device);
        Py_XDECREF(device);
        if (PyErr_Occurred()) { ok_ = false; return nullptr; }
        if (index >= 0 && index != c10::cuda::current_device()) { fail(PyExc_ValueError, "a paged cache of another device than the current one"); return nullptr; }
        return static_cast<const T*>(b.buf);
    }
    const b200kv_paged_view* paged_view() { return structure<b200kv_paged_view>(g_paged_view_type, "a paged cache's view"); }
    const b200kv_paged_batch* paged_batch() { return structure<b200kv_paged_batch>(g_paged_batch_type, "a paged batch"); }
    const b200kv_paged_scoring* paged_scoring() {   // or None
        if (ok_ && args_[i_] == Py_None) { ++i_; return nullptr; }
        return structure<b200kv_paged_scoring>(g_paged_scoring_type, "a scoring");
    }
    const b200kv_rotary* rotary() { return structure<b200kv_rotary>(g_rotary_type, "a table of rotary angles"); }
    const b200kv_page_book* page_book() { return structure<b200kv_page_book>(g_page_book_type, "a page book"); }
    // A list or tuple of paged views, one behind the other in `to`.
    bool paged_views(std::vector<b200kv_paged_view>& to) {
        if (!ok_) return false;
        PyObject* list = args_[i_];
        if (!PyList_Check(list) && !PyTuple_Check(list)) { fail(PyExc_TypeError, "expected a list of paged views"); return false; }
        PyObject* const* const args = args_;
        const Py_ssize_t at = i_ + 1;
        for (Py_ssize_t k = 0; ok_ && k < PySequence_Fast_GET_SIZE(list); ++k) {
            PyObject* item = PySequence_Fast_GET_ITEM(list, k);
            args_ = &item;
            i_ = 0;
            if (const b200kv_paged_view* view = paged_view()) to.push_back(*view);
            if (ok_) PyBuffer_Release(&buffers_[--held_]);   // copied
        }
        args_ = args;
        i_ = at;
        return ok_;
    }
    // Rows [at least `rows`][exactly `width`] of fp16 or fp32 whose elements lie one behind the other, or None; *stride: elements from a row to the next.
    const void* strided(int* dtype, uint64_t rows, uint64_t width, uint64_t* stride, const char* text) {
        if (!ok_) return nullptr;
        PyObject* o = args_[i_++];
        if (o == Py_None) return nullptr;
        if (!THPVariable_Check(o)) return fail(PyExc_TypeError, "a torch tensor is required");
        const at::Tensor& t = THPVariable_Unpack(o);
        const auto type = t.scalar_type();
        if (!t.is_cuda() || (type != at::kHalf && type != at::kFloat)) return fail(PyExc_ValueError, "expected a CUDA tensor of fp16 or fp32");
        if (!here(o)) return nullptr;
        if (t.dim() != 2 || static_cast<uint64_t>(t.size(0)) < rows || static_cast<uint64_t>(t.size(1)) != width || t.stride(1) != 1 || (t.size(0) > 1 && t.stride(0) < t.size(1)))
            return fail(PyExc_ValueError, text);
        *dtype = type == at::kHalf ? B200KV_F16 : B200KV_F32;
        *stride = t.size(0) > 1 ? static_cast<uint64_t>(t.stride(0)) : width;
        return t.data_ptr();
    }
    // A tensor of one type and at least `least` elements, or None where that is allowed.
    template <typename T>
    T* exactly(at::ScalarType type, const char* text, uint64_t least, bool optional = false) {
        if (!ok_) return nullptr;
        PyObject* o = args_[i_];
        if (o == Py_None) {
            if (!optional) fail(PyExc_ValueError, "a tensor is required");
            ++i_;
            return nullptr;
        }
        int64_t n = 0;
        void* p = tensor(&n);
        if (!ok_) return nullptr;
        if (!here(o)) return nullptr;
        if (THPVariable_Unpack(o).scalar_type() != type || static_cast<uint64_t>(n) < least) return static_cast<T*>(fail(PyExc_ValueError, text));
        return static_cast<T*>(p);
    }
    // The same of a given shape [at least `rows`][shape...], where a number of the shape is exact, or, as the last one with `width`, the least, and *width what it is.  (An
    // account of more slots than the batch has sequences has the stride of its shape; its number of elements would say another.)
    template <typename T>
    T* shaped(at::ScalarType type, const char* text, uint64_t rows, std::initializer_list<uint64_t> shape, uint32_t* width = nullptr, bool optional = false) {
        PyObject* o = ok_ ? args_[i_] : Py_None;
        T* p = exactly<T>(type, text, 0, optional);
        if (!ok_ || o == Py_None || rows == 0) return p;
        const at::Tensor& t = THPVariable_Unpack(o);
        bool fits = static_cast<size_t>(t.dim()) == 1 + shape.size() && static_cast<uint64_t>(t.size(0)) >= rows;
        for (size_t i = 1; fits && i <= shape.size(); ++i) {
            const uint64_t want = shape.begin()[i - 1], n = static_cast<uint64_t>(t.size(i));
            fits = width != nullptr && i == shape.size() ? n >= want && n <= 0xffffffffu : n == want;
        }
        if (!fits) return static_cast<T*>(fail(PyExc_ValueError, text));
        if (width != nullptr) *width = static_cast<uint32_t>(t.size(t.dim() - 1));
        return p;
    }
    // An activation tensor of fp16 or fp32 with at least `least` elements.
    void* activation(int* dtype, uint64_t least, const char* text) {
        int64_t n = 0;
        PyObject* o = ok_ ? args_[i_] : nullptr;
        void* p = tensor(&n, dtype);
        if (!ok_ || !here(o)) return nullptr;
        if (static_cast<uint64_t>(n) < least) return fail(PyExc_ValueError, text);
        return p;
    }
    // An array of them (the caller has built it), or None.
    const b200kv_view* views(uint32_t count, bool optional) {
        if (!ok_) return nullptr;
        PyObject* o = args_[i_++];
        if (optional && o == Py_None) return nullptr;
        if (PyObject_GetBuffer(o, &buffers_[held_], PyBUF_SIMPLE) != 0) { ok_ = false; return nullptr; }
        const Py_buffer& b = buffers_[held_++];
        if (static_cast<size_t>(b.len) < sizeof(b200kv_view) * static_cast<size_t>(count)) {
            fail(PyExc_ValueError, "not a cache view");
            return nullptr;
        }
        return static_cast<const b200kv_view*>(b.buf);
    }
    void* stream() {   // None = torch's current stream
        if (!ok_) return nullptr;
        PyObject* o = args_[i_++];
        if (o == Py_None) return c10::cuda::getCurrentCUDAStream().stream();
        PyObject* h = PyObject_GetAttrString(o, "cuda_stream");
        if (h == nullptr) { ok_ = false; return nullptr; }
        void* s = PyLong_AsVoidPtr(h);
        Py_DECREF(h);
        if (s == nullptr && PyErr_Occurred()) ok_ = false;
        return s;
    }
    void* handle() {   // an address as an int, None = null
        if (!ok_) return nullptr;
        PyObject* o = args_[i_++];
        if (o == Py_None) return nullptr;
        void* p = PyLong_AsVoidPtr(o);
        if (p == nullptr && PyErr_Occurred()) ok_ = false;
        return p;
    }
    PyObject* object() { return ok_ ? args_[i_++] : nullptr; }
    void* fail(PyObject* type, const char* text) {
        if (ok_) PyErr_SetString(type, text);
        ok_ = false;
        return nullptr;
    }

private:
    bool here(PyObject* o) {   // on the current device, whose stream the launch goes to
        if (THPVariable_Unpack(o).get_device() == c10::cuda::current_device()) return true;
        fail(PyExc_ValueError, "a tensor of another device than the current one");
        return false;
    }
    uint32_t checked(uint32_t v) {
        if (v == 0xffffffffu && PyErr_Occurred()) ok_ = false;
        return v;
    }
    PyObject* const* args_;
    Py_ssize_t i_ = 0;
    bool ok_ = true;
    int held_ = 0;
    Py_buffer buffers_[4];
};

template <typename F>
PyObject* call(Args& a, F&& f) {
    if (!a.ok()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 12);
    int kd = 0, vd = 0;
    const b200kv_view* view = a.view();
    const void* key = a.tensor(nullptr, &kd);
    const void* value = a.tensor(nullptr, &vd);
    if (a.ok() && kd != vd) a.fail(PyExc_ValueError, "key and value must share a dtype");
    const float* w = a.tensor_as<const float>();
    const int rope = a.rope();
    const float theta = a.f32(), eps = a.f32();
    const uint32_t count = a.u32(), base = a.u32();
    const auto* ps = a.tensor_as<const b200kv_prefill_state>();
    const auto* ds = a.tensor_as<const b200kv_decode_state>();
    void* s = a.stream();
    return call(a, [&] { return g_api.append(view, key, value, kd, w, rope, theta, eps, count, base, ps, ds, s); });
}

PyObject* py_q_split_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 14);
    int id = 0, od = 0;
    const void* qfull = a.tensor(nullptr, &id);
    const float* w = a.tensor_as<const float>();
    void* query = a.tensor(nullptr, &od);
    float* gate = a.tensor_as<float>();
    const uint32_t count = a.u32(), base = a.u32(), heads = a.u32(), dim = a.u32();
    const int rope = a.rope();
    const float theta = a.f32(), eps = a.f32();
    const auto* ps = a.tensor_as<const b200kv_prefill_state>();
    const auto* ds = a.tensor_as<const b200kv_decode_state>();
    void* s = a.stream();
    return call(a, [&] { return g_api.q_split_norm_rope(qfull, id, w, query, od, gate, count, base, heads, dim, rope, theta, eps, ps, ds, s); });
}

PyObject* py_decode_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 13);
    int qd = 0;
    int64_t ws_bytes = 0;
    const b200kv_view* view = a.view();
    const void* q = a.tensor(nullptr, &qd);
    const float* gate = a.tensor_as<const float>();
    float* out = a.tensor_as<float>();
    float* gated = a.tensor_as<float>();
    auto* q8 = a.tensor_as<b200kv_q8_1_block>();
    const uint32_t heads = a.u32();
    const float scale = a.f32();
    const uint32_t length = a.u32();
    const auto* ds = a.tensor_as<const b200kv_decode_state>();
    void* ws = a.tensor(&ws_bytes);
    const uint32_t splits = a.u32();
    void* s = a.stream();
    return call(a, [&] {
        return g_api.decode_attn(view, q, qd, gate, out, gated, q8, heads, scale, length, ds, ws, static_cast<size_t>(ws_bytes), splits, s);
    });
}

PyObject* py_decode_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 19);
    int kd = 0, vd = 0, qd = 0;
    int64_t ws_bytes = 0;
    const b200kv_view* view = a.view();
    const void* key = a.tensor(nullptr, &kd);
    const void* value = a.tensor(nullptr, &vd);
    if (a.ok() && kd != vd) a.fail(PyExc_ValueError, "key and value must share a dtype");
    const float* w = a.tensor_as<const float>();
    const int rope = a.rope();
    const float theta = a.f32(), eps = a.f32();
    const void* q = a.tensor(nullptr, &qd);
    const float* gate = a.tensor_as<const float>();
    float* out = a.tensor_as<float>();
    float* gated = a.tensor_as<float>();
    auto* q8 = a.tensor_as<b200kv_q8_1_block>();
    const uint32_t heads = a.u32();
    const float scale = a.f32();
    const uint32_t position = a.u32();
    const auto* ds = a.tensor_as<const b200kv_decode_state>();
    void* ws = a.tensor(&ws_bytes);
    const uint32_t splits = a.u32();
    void* s = a.stream();
    return call(a, [&] {
        return g_api.decode_step(view, key, value, kd, w, rope, theta, eps, q, qd, gate, out, gated, q8, heads, scale, position, ds, ws,
                                 static_cast<size_t>(ws_bytes), splits, s);
    });
}

PyObject* py_decode_attn_batched(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 13);
    int qd = 0;
    int64_t ws_bytes = 0, sessions = 0;
    PyObject* views_arg = a.object();
    void* table = a.tensor();
    const uint32_t* lengths = a.tensor_as<const uint32_t>(&sessions);
    const uint32_t max_length = a.u32();
    const void* q = a.tensor(nullptr, &qd);
    const float* gate = a.tensor_as<const float>();
    float* out = a.tensor_as<float>();
    float* gated = a.tensor_as<float>();
    const uint32_t heads = a.u32();
    const float scale = a.f32();
    void* ws = a.tensor(&ws_bytes);
    const uint32_t splits = a.u32();
    void* s = a.stream();
    Args v(&views_arg, 1, 1);
    const b200kv_view* views = a.ok() ? v.views(static_cast<uint32_t>(sessions), true) : nullptr;
    if (a.ok() && !v.ok()) return nullptr;
    return call(a, [&] {
        return g_api.decode_attn_batched(views, table, lengths, static_cast<uint32_t>(sessions), max_length, q, qd, gate, out, gated, heads, scale,
                                         ws, static_cast<size_t>(ws_bytes), splits, s);
    });
}

PyObject* py_suffix_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 12);
    int qd = 0;
    int64_t ws_bytes = 0;
    const b200kv_view* view = a.view();
    const void* q = a.tensor(nullptr, &qd);
    const float* gate = a.tensor_as<const float>();
    float* gated = a.tensor_as<float>();
    const uint32_t count = a.u32(), base = a.u32(), heads = a.u32();
    const float scale = a.f32();
    const auto* ps = a.tensor_as<const b200kv_prefill_state>();
    void* ws = a.tensor(&ws_bytes);
    const uint32_t prepared = a.u32();
    void* s = a.stream();
    return call(a, [&] {
        return g_api.prefill_attn_prepared(view, q, qd, gate, gated, count, base, heads, scale, ps, ws, static_cast<size_t>(ws_bytes), prepared, s);
    });
}

// ---- the paged cache ------------------------------------------------------------------------------------------

constexpr const char* kSmall = "a tensor of another type, or with fewer elements than the batch has rows";

PyObject* py_paged_store(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 10);
    int kd = 0, vd = 0;
    const auto* view = a.paged_view();
    const auto* batch = a.paged_batch();
    const uint64_t tokens = a.ok() ? batch->total_tokens : 0, width = a.ok() ? static_cast<uint64_t>(view->kv_heads) * view->head_dim : 0;
    const void* key = a.activation(&kd, tokens * width, kSmall);
    const void* value = a.activation(&vd, tokens * width, kSmall);
    if (a.ok() && kd != vd) a.fail(PyExc_ValueError, "key and value must share a dtype");
    const float* w = a.exactly<const float>(at::kFloat, "the norm's weight: fp32 of head_dim elements", a.ok() ? view->head_dim : 0, true);
    const int rope = a.rope();
    const float theta = a.f32(), eps = a.f32();
    const int32_t* positions = a.exactly<const int32_t>(at::kInt, "positions: int32 of every token", tokens, true);
    void* s = a.stream();
    return call(a, [&] { return g_api.paged_store(view, batch, key, value, kd, w, rope, theta, eps, positions, s); });
}

PyObject* py_paged_load(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 5);
    const auto* view = a.paged_view();
    const auto* batch = a.paged_batch();
    const uint64_t least = a.ok() ? static_cast<uint64_t>(batch->total_tokens) * view->kv_heads * view->head_dim : 0;
    void* key = a.exactly<void>(at::kHalf, kSmall, least, true);
    void* value = a.exactly<void>(at::kHalf, kSmall, least, true);
    void* s = a.stream();
    return call(a, [&] { return g_api.paged_load(view, batch, key, value, s); });
}

PyObject* py_paged_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 13);
    int qd = 0, od = 0;
    int64_t ws_bytes = 0;
    const auto* view = a.paged_view();
    const auto* batch = a.paged_batch();
    const uint32_t heads = a.u32();
    const uint64_t rows = a.ok() ? static_cast<uint64_t>(batch->total_tokens) * heads : 0, dim = a.ok() ? view->head_dim : 0;
    const void* q = a.activation(&qd, rows * dim, kSmall);
    const float* gate = a.exactly<const float>(at::kFloat, kSmall, rows * dim, true);
    void* out = a.activation(&od, rows * dim, kSmall);
    float* lse = a.exactly<float>(at::kFloat, kSmall, rows, true);
    const float scale = a.f32();
    const uint32_t window = a.u32(), sinks = a.u32();
    void* ws = a.exactly<void>(at::kByte, "workspace: a uint8 tensor", 0, true);
    if (a.ok() && ws != nullptr) ws_bytes = THPVariable_Unpack(args[10]).numel();
    void* s = a.stream();
    const auto* scoring = a.paged_scoring();
    return call(a, [&] {
        if (scoring != nullptr)
            return g_api.paged_attn_scored(view, batch, scoring, q, qd, gate, out, od, lse, heads, scale, window, sinks, ws, static_cast<size_t>(ws_bytes), s);
        return g_api.paged_attn(view, batch, q, qd, gate, out, od, lse, heads, scale, window, sinks, ws, static_cast<size_t>(ws_bytes), s);
    });
}

PyObject* py_paged_weights(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 11);
    int qd = 0;
    const auto* view = a.paged_view();
    const auto* batch = a.paged_batch();
    const uint32_t heads = a.u32();
    const uint64_t rows = a.ok() ? static_cast<uint64_t>(batch->total_tokens) * heads : 0;
    const void* q = a.activation(&qd, rows * (a.ok() ? view->head_dim : 0), kSmall);
    const float* lse = a.exactly<const float>(at::kFloat, kSmall, rows);
    uint32_t stride = 0;
    float* weights = a.shaped<float>(at::kFloat, "weights: fp32 [sequences][kv_heads][at least max_length]", a.ok() ? batch->sequences : 0,
                                     {a.ok() ? view->kv_heads : 0, a.ok() ? batch->max_length : 0}, &stride);
    const float scale = a.f32();
    const uint32_t window = a.u32(), sinks = a.u32(), observe = a.u32();
    void* s = a.stream();
    return call(a, [&] { return g_api.paged_weights(view, batch, q, qd, lse, weights, stride, heads, scale, window, sinks, observe, s); });
}

PyObject* py_paged_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 11);
    const auto* view = a.paged_view();
    const auto* batch = a.paged_batch();
    const uint64_t sequences = a.ok() ? batch->sequences : 0, heads = a.ok() ? view->kv_heads : 0;
    const uint32_t keep = a.u32(), sinks = a.u32(), recent = a.u32();
    uint32_t pages = 0, stride = 0;
    const int32_t* target = a.shaped<const int32_t>(at::kInt, "target: int32 [sequences][pages]", sequences, {0}, &pages);
    const float* weights = a.shaped<const float>(at::kFloat, "weights: fp32 [sequences][kv_heads][at least max_length]", sequences, {heads, a.ok() ? batch->max_length : 0}, &stride);
    int32_t* kept = a.shaped<int32_t>(at::kInt, "kept: int32 [sequences][kv_heads][keep]", sequences, {heads, keep});
    float* new_weights = a.shaped<float>(at::kFloat, "new_weights: fp32 [sequences][kv_heads][keep]", sequences, {heads, keep}, nullptr, true);
    int32_t* new_lengths = a.exactly<int32_t>(at::kInt, "new_lengths: int32 [sequences]", sequences);
    void* s = a.stream();
    return call(a, [&] {
        return g_api.paged_evict(view, batch, target, pages, weights, stride, keep, sinks, recent, kept, new_weights,
                                 new_lengths, s);
    });
}

PyObject* py_paged_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 14);
    constexpr const char* kRows = "rows: [at least total_tokens][heads * head_dim, twice that for queries with gates], elements one behind the other";
    int dtypes[3] = {-1, -1, -1}, od = B200KV_F16;
    uint64_t strides[3] = {0, 0, 0};
    const auto* view = a.paged_view();
    const auto* batch = a.paged_batch();
    const auto* rotary = a.rotary();
    const uint32_t heads = a.u32();
    const uint64_t tokens = a.ok() ? batch->total_tokens : 0, dim = a.ok() ? view->head_dim : 0, width = a.ok() ? view->kv_heads * dim : 0;
    const void* key = a.strided(&dtypes[0], tokens, width, &strides[0], kRows);
    const void* value = a.strided(&dtypes[1], tokens, width, &strides[1], kRows);
    const void* q = a.strided(&dtypes[2], tokens, heads * dim * (a.ok() && args[7] != Py_None ? 2 : 1), &strides[2], kRows);
    float* gate = a.exactly<float>(at::kFloat, kSmall, tokens * heads * dim, true);
    void* out = nullptr;
    if (a.ok() && args[8] != Py_None) out = a.activation(&od, tokens * heads * dim, kSmall);
    else a.object();
    const float* q_norm = a.exactly<const float>(at::kFloat, "a norm's weight: fp32 of head_dim elements", dim, true);
    const float* k_norm = a.exactly<const float>(at::kFloat, "a norm's weight: fp32 of head_dim elements", dim, true);
    const float epsilon = a.f32();
    const int32_t* positions = a.exactly<const int32_t>(at::kInt, "positions: int32 of every token", tokens, true);
    void* s = a.stream();
    int dtype = -1;
    for (const int d : dtypes) {
        if (d < 0) continue;
        if (a.ok() && dtype >= 0 && d != dtype) a.fail(PyExc_ValueError, "queries, keys and values must share a dtype");
        dtype = d;
    }
    return call(a, [&] {
        return g_api.paged_rotary(view, batch, rotary, q, strides[2], key, strides[0], value, strides[1], dtype, q_norm, k_norm, epsilon, positions, heads, out, od, gate, s);
    });
}

// ---- the book of a paged cache's pages --------------------------------------------------------------------------

constexpr const char* kEntries = "an int32 tensor of every entry";

uint32_t entries(Args& a, PyObject* o) {   // of a call: the elements of its first array
    if (!a.ok()) return 0;
    if (!THPVariable_Check(o)) { a.fail(PyExc_TypeError, "a torch tensor is required"); return 0; }
    const int64_t n = THPVariable_Unpack(o).numel();
    if (n > 0x7fffffff) a.fail(PyExc_ValueError, "too many entries");
    return a.ok() ? static_cast<uint32_t>(n) : 0;
}
void* workspace(Args& a, PyObject* o, size_t* bytes) {
    void* ws = a.exactly<void>(at::kByte, "workspace: a uint8 tensor", 0, true);
    if (a.ok() && ws != nullptr) *bytes = static_cast<size_t>(THPVariable_Unpack(o).numel());
    return ws;
}

PyObject* py_pages_grow(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 5);
    size_t bytes = 0;
    const auto* book = a.page_book();
    const uint32_t count = a.ok() ? entries(a, args[1]) : 0;
    const int32_t* slots = a.exactly<const int32_t>(at::kInt, kEntries, count);
    const int32_t* add = a.exactly<const int32_t>(at::kInt, kEntries, count);
    void* ws = workspace(a, a.ok() ? args[3] : nullptr, &bytes);
    void* s = a.stream();
    return call(a, [&] { return g_api.pages_grow(book, slots, add, count, ws, bytes, s); });
}

PyObject* py_pages_fork(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 7);
    size_t bytes = 0;
    std::vector<b200kv_paged_view> views;
    const auto* book = a.page_book();
    a.paged_views(views);
    const uint32_t count = a.ok() ? entries(a, args[2]) : 0;
    const int32_t* parents = a.exactly<const int32_t>(at::kInt, kEntries, count);
    const int32_t* children = a.exactly<const int32_t>(at::kInt, kEntries, count);
    const int32_t* at = a.exactly<const int32_t>(at::kInt, kEntries, count, true);
    void* ws = workspace(a, a.ok() ? args[5] : nullptr, &bytes);
    void* s = a.stream();
    return call(a, [&] { return g_api.pages_fork(book, views.data(), static_cast<uint32_t>(views.size()), parents, children, at, count, ws, bytes, s); });
}

PyObject* py_pages_free(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 3);
    const auto* book = a.page_book();
    const uint32_t count = a.ok() ? entries(a, args[1]) : 0;
    const int32_t* slots = a.exactly<const int32_t>(at::kInt, kEntries, count);
    void* s = a.stream();
    return call(a, [&] { return g_api.pages_free(book, slots, count, s); });
}

PyObject* py_pages_compact(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 5);
    size_t bytes = 0;
    std::vector<b200kv_paged_view> views;
    const auto* book = a.page_book();
    a.paged_views(views);
    int32_t* moved = a.exactly<int32_t>(at::kInt, "moved: int32 of every page", a.ok() ? book->pages : 0);
    void* ws = workspace(a, a.ok() ? args[3] : nullptr, &bytes);
    void* s = a.stream();
    return call(a, [&] { return g_api.pages_compact(book, views.data(), static_cast<uint32_t>(views.size()), moved, ws, bytes, s); });
}

PyObject* py_pages_copy(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 5);
    std::vector<b200kv_paged_view> from, to;
    a.paged_views(from);
    a.paged_views(to);
    if (a.ok() && from.size() != to.size()) a.fail(PyExc_ValueError, "as many views on both sides");
    const uint32_t count = a.ok() ? entries(a, args[2]) : 0;
    const int32_t* sources = a.exactly<const int32_t>(at::kInt, kEntries, count);
    const int32_t* targets = a.exactly<const int32_t>(at::kInt, kEntries, count);
    void* s = a.stream();
    return call(a, [&] { return g_api.pages_copy(from.data(), to.data(), static_cast<uint32_t>(from.size()), sources, targets, count, s); });
}

// ---- the snapshot pool: token ids and storage objects in, one library call ------------------------------------

// Anything with a length that can be iterated over, as a list or tuple.
PyObject* items_of(PyObject* o, const char* text) { return PyObject_Size(o) < 0 ? nullptr : PySequence_Fast(o, text); }

bool read_tokens(PyObject* seq, std::vector<uint32_t>& out) {
    PyObject* fast = items_of(seq, "a sequence of token ids is required");
    if (fast == nullptr) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    PyObject** items = PySequence_Fast_ITEMS(fast);
    out.resize(static_cast<size_t>(n));
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (PyLong_Check(items[i])) {
            out[i] = static_cast<uint32_t>(PyLong_AsUnsignedLongMask(items[i]));
            continue;
        }
        PyObject* v = PyNumber_Index(items[i]);
        if (v == nullptr) { Py_DECREF(fast); return false; }
        out[i] = static_cast<uint32_t>(PyLong_AsUnsignedLongMask(v));
        Py_DECREF(v);
    }
    Py_DECREF(fast);
    return true;
}

enum Name { KEY, VALUE, KEY_Q8, KEY_SCALES, VALUE_Q8, VALUE_SCALES, CAPACITY, KV_HEADS, HEAD_DIM, QBLOCK, QUANT_MODE, VIEW, NAMES };
PyObject* g_names[NAMES];

bool plane(PyObject* o, Name name, void** out) {
    PyObject* t = PyObject_GetAttr(o, g_names[name]);
    if (t == nullptr) return false;
    *out = nullptr;
    if (t != Py_None) {
        if (!THPVariable_Check(t) || !THPVariable_Unpack(t).is_cuda() || !THPVariable_Unpack(t).is_contiguous()) {
            Py_DECREF(t);
            PyErr_SetString(PyExc_ValueError, "expected a contiguous CUDA tensor");
            return false;
        }
        *out = THPVariable_Unpack(t).data_ptr();
    }
    Py_DECREF(t);
    return true;
}
bool number(PyObject* o, Name name, uint64_t* out) {
    PyObject* v = PyObject_GetAttr(o, g_names[name]);
    if (v == nullptr) return false;
    *out = PyLong_AsUnsignedLongLongMask(v);
    Py_DECREF(v);
    return !(*out == ~0ull && PyErr_Occurred());
}

PyObject* g_storage_view;   // AttentionLayerKvCacheStorage.view

// The views of a sequence of cache storages: what their view() returns.  Where that is AttentionLayerKvCacheStorage's own, its
// result is read from the attributes it would take it from (a view() in Python costs 3 us a layer).
bool read_view(PyObject* o, b200kv_view& v) {
    PyObject* method = PyObject_GetAttr(o, g_names[VIEW]);
    if (method == nullptr) return false;
    const bool own = PyMethod_Check(method) && PyMethod_GET_FUNCTION(method) == g_storage_view && PyMethod_GET_SELF(method) == o;
    PyObject* result = own ? nullptr : PyObject_CallNoArgs(method);
    Py_DECREF(method);
    if (!own) {
        if (result == nullptr) return false;
        Args a(&result, 1, 1);
        const b200kv_view* view = a.view();
        if (view != nullptr) v = *view;
        Py_DECREF(result);
        return a.ok();
    }
    void *kq, *vq;
    uint64_t cap, heads, dim, qb, mode;
    if (!(plane(o, KEY, &v.key_f16) && plane(o, VALUE, &v.value_f16) && plane(o, KEY_Q8, &kq) && plane(o, KEY_SCALES, &v.key_scales) &&
          plane(o, VALUE_Q8, &vq) && plane(o, VALUE_SCALES, &v.value_scales) && number(o, CAPACITY, &cap) && number(o, KV_HEADS, &heads) &&
          number(o, HEAD_DIM, &dim) && number(o, QBLOCK, &qb) && number(o, QUANT_MODE, &mode)))
        return false;
    v.key_q8 = static_cast<int8_t*>(kq);
    v.value_q8 = static_cast<int8_t*>(vq);
    v.capacity = cap;
    v.kv_heads = static_cast<uint32_t>(heads);
    v.head_dim = static_cast<uint32_t>(dim);
    v.qblock = static_cast<uint32_t>(qb);
    v.quant_mode = static_cast<uint32_t>(mode);
    return true;
}
bool read_views(PyObject* storages, std::vector<b200kv_view>& out) {
    PyObject* fast = items_of(storages, "a sequence of cache storages is required");
    if (fast == nullptr) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    out.resize(static_cast<size_t>(n));
    bool ok = true;
    for (Py_ssize_t i = 0; i < n && ok; ++i) ok = read_view(PySequence_Fast_GET_ITEM(fast, i), out[i]);
    Py_DECREF(fast);
    return ok;
}

// (pool, tokens, storages, stream) -> (status, captured or matched length)
template <bool CAPTURE>
PyObject* py_pool(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Args a(args, n, 4);
    auto* pool = static_cast<b200kv_pool*>(a.handle());
    PyObject* tokens_arg = a.object();
    PyObject* storages = a.object();
    void* s = a.stream();
    if (!a.ok()) return nullptr;
    std::vector<uint32_t> tokens;
    std::vector<b200kv_view> views;
    if (!read_tokens(tokens_arg, tokens) || !read_views(storages, views)) return nullptr;
    const uint32_t count = static_cast<uint32_t>(tokens.size()), layers = static_cast<uint32_t>(views.size());
    static const uint32_t no_token = 0;   // an empty sequence still passes an address
    const uint32_t* ids = count ? tokens.data() : &no_token;
    const b200kv_view empty{};
    const b200kv_view* layer_views = layers ? views.data() : &empty;
    int rc, captured = 0;
    uint32_t matched = 0;
    Py_BEGIN_ALLOW_THREADS
    if (CAPTURE) rc = g_api.pool_capture(pool, ids, count, layer_views, layers, s, &captured);
    else rc = g_api.pool_restore(pool, ids, count, layer_views, layers, s, &matched);
    Py_END_ALLOW_THREADS
    return Py_BuildValue("iI", rc, CAPTURE ? static_cast<unsigned>(captured) : matched);
}

PyObject* py_bind(PyObject*, PyObject* arg) {   // {name: address}, and the structures "View", "PagedView", "PagedBatch", "PagedScoring", "Rotary" and "PageBook"
    PyObject* view = PyDict_GetItemString(arg, "View");
    if (view == nullptr || !PyType_Check(view)) return PyErr_Format(PyExc_KeyError, "View");
    Py_INCREF(view);
    Py_XSETREF(g_view_type, view);
    for (auto [name, slot] : {std::pair{"PagedView", &g_paged_view_type}, std::pair{"PagedBatch", &g_paged_batch_type}, std::pair{"PagedScoring", &g_paged_scoring_type}, std::pair{"Rotary", &g_rotary_type},
                              std::pair{"PageBook", &g_page_book_type}}) {
        PyObject* type = PyDict_GetItemString(arg, name);
        if (type == nullptr || !PyType_Check(type)) return PyErr_Format(PyExc_KeyError, "%s", name);
        Py_INCREF(type);
        Py_XSETREF(*slot, type);
    }
    struct { const char* name; void** slot; } table[] = {
        {"b200kv_append", reinterpret_cast<void**>(&g_api.append)},
        {"b200kv_q_split_norm_rope", reinterpret_cast<void**>(&g_api.q_split_norm_rope)},
        {"b200kv_decode_attn", reinterpret_cast<void**>(&g_api.decode_attn)},
        {"b200kv_decode_step", reinterpret_cast<void**>(&g_api.decode_step)},
        {"b200kv_decode_attn_batched", reinterpret_cast<void**>(&g_api.decode_attn_batched)},
        {"b200kv_prefill_attn_prepared", reinterpret_cast<void**>(&g_api.prefill_attn_prepared)},
        {"b200kv_paged_store", reinterpret_cast<void**>(&g_api.paged_store)},
        {"b200kv_paged_load", reinterpret_cast<void**>(&g_api.paged_load)},
        {"b200kv_paged_attn", reinterpret_cast<void**>(&g_api.paged_attn)},
        {"b200kv_paged_attn_scored", reinterpret_cast<void**>(&g_api.paged_attn_scored)},
        {"b200kv_paged_weights", reinterpret_cast<void**>(&g_api.paged_weights)},
        {"b200kv_paged_evict", reinterpret_cast<void**>(&g_api.paged_evict)},
        {"b200kv_paged_rotary", reinterpret_cast<void**>(&g_api.paged_rotary)},
        {"b200kv_pages_grow", reinterpret_cast<void**>(&g_api.pages_grow)},
        {"b200kv_pages_fork", reinterpret_cast<void**>(&g_api.pages_fork)},
        {"b200kv_pages_free", reinterpret_cast<void**>(&g_api.pages_free)},
        {"b200kv_pages_compact", reinterpret_cast<void**>(&g_api.pages_compact)},
        {"b200kv_pages_copy", reinterpret_cast<void**>(&g_api.pages_copy)},
        {"b200kv_pool_capture", reinterpret_cast<void**>(&g_api.pool_capture)},
        {"b200kv_pool_restore", reinterpret_cast<void**>(&g_api.pool_restore)},
    };
    for (auto& e : table) {
        PyObject* v = PyDict_GetItemString(arg, e.name);
        if (v == nullptr) return PyErr_Format(PyExc_KeyError, "%s", e.name);
        *e.slot = PyLong_AsVoidPtr(v);
        if (*e.slot == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "%s has no address", e.name);
    }
    Py_RETURN_NONE;
}

PyObject* py_bind_storage(PyObject*, PyObject* view) {   // AttentionLayerKvCacheStorage.view
    Py_INCREF(view);
    Py_XSETREF(g_storage_view, view);
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {   // no C++ exception reaches the interpreter
    try {
        return F(self, args, n);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}
#define ENTRY(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<f>)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {{"bind", py_bind, METH_O, nullptr},
                           {"bind_storage", py_bind_storage, METH_O, nullptr},
                           ENTRY("append", py_append),
                           ENTRY("q_split_norm_rope", py_q_split_norm_rope),
                           ENTRY("decode_attn", py_decode_attn),
                           ENTRY("decode_step", py_decode_step),
                           ENTRY("decode_attn_batched", py_decode_attn_batched),
                           ENTRY("suffix_attn", py_suffix_attn),
                           ENTRY("paged_store", py_paged_store),
                           ENTRY("paged_load", py_paged_load),
                           ENTRY("paged_attn", py_paged_attn),
                           ENTRY("paged_weights", py_paged_weights),
                           ENTRY("paged_evict", py_paged_evict),
                           ENTRY("paged_rotary", py_paged_rotary),
                           ENTRY("pages_grow", py_pages_grow),
                           ENTRY("pages_fork", py_pages_fork),
                           ENTRY("pages_free", py_pages_free),
                           ENTRY("pages_compact", py_pages_compact),
                           ENTRY("pages_copy", py_pages_copy),
                           ENTRY("pool_capture", py_pool<true>),
                           ENTRY("pool_restore", py_pool<false>),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) {
    const char* names[NAMES] = {"key_cache", "value_cache", "key_cache_q8", "key_scales", "value_cache_q8", "value_scales",
                                "capacity", "kv_heads", "head_dim", "qblock", "quant_mode", "view"};
    for (int i = 0; i < NAMES; ++i) {
        g_names[i] = PyUnicode_InternFromString(names[i]);
        if (g_names[i] == nullptr) return nullptr;
    }
    if ((g_device_index = PyUnicode_InternFromString("device_index")) == nullptr) return nullptr;
    return PyModule_Create(&g_module);
}
