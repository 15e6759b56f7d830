// The ragged operators' call path from Python to the C ABI: checks of arguments, outputs and
// workspaces from torch's allocator, the current stream.  These calls are made once or twice per
// layer and decode step, where the same steps in Python and ctypes took 8 to 13 us a call, as
// long as the kernels of a small batch.
//
// The C entries come as addresses (bind), from the one place that loads the library.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <optional>
#include <string>

#include "../../include/razorkv_b200.h"

namespace {

decltype(&rkv_ragged_page_tables) g_tables = nullptr;
decltype(&rkv_ragged_append) g_append = nullptr;
decltype(&rkv_ragged_decode_attention) g_decode = nullptr;
decltype(&rkv_ragged_decode_attention_workspace_size) g_decode_size = nullptr;
decltype(&rkv_status_string) g_status = nullptr;
PyObject* g_error = nullptr;                    // RazorKVError
std::atomic<unsigned long long> g_devices{0};   // devices that an operator has run on

// A Python exception on its way out of the checks.
struct Refused {
    PyObject* type;
    std::string text;
};

[[noreturn]] void refuse(PyObject* type, std::string text) { throw Refused{type, std::move(text)}; }

std::string shape_of(const at::Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + (t.dim() == 1 ? ",)" : ")");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o))
        refuse(PyExc_TypeError, std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}

const at::Tensor* tensor_or_none(PyObject* o, const char* name) {
    return o == Py_None ? nullptr : &tensor(o, name);
}

int64_t integer(PyObject* o, const char* name) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(PyExc_TypeError, std::string(name) + " must be an integer");
    }
    return v;
}

void want_int64(const at::Tensor& t, int64_t dim, const char* name) {
    if (t.scalar_type() != at::kLong)
        refuse(PyExc_TypeError, std::string(name) + " must be int64, got " + c10::toString(t.scalar_type()));
    if (t.dim() != dim)
        refuse(PyExc_ValueError, std::string(name) + " must have " + std::to_string(dim) +
                                     " dimension(s), got " + shape_of(t));
}

// A tensor that is updated in place cannot be copied into shape first.
void want_written(const at::Tensor& t, const char* name) {
    if (t.numel() && !t.is_contiguous())
        refuse(PyExc_ValueError, std::string(name) + " is updated in place and must be contiguous");
}

bool on_itself(const at::Tensor& t) { return at::has_internal_overlap(t) == at::MemOverlap::Yes; }
bool on_another(const at::Tensor& a, const at::Tensor& b) {
    const auto s = at::get_overlap_status(a, b);
    return s == at::MemOverlapStatus::Full || s == at::MemOverlapStatus::Partial;
}

int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return RKV_F32;
        case at::kHalf: return RKV_F16;
        case at::kBFloat16: return RKV_BF16;
        default:
            refuse(PyExc_TypeError, std::string("unsupported dtype ") + c10::toString(t) +
                                        "; expected float32, float16 or bfloat16");
    }
}

// The CUDA device of all tensors (null ones aside).
template <typename... T>
c10::DeviceIndex device_of(const at::Tensor& first, const T*... others) {
    const at::Tensor* all[] = {&first, others...};
    for (const at::Tensor* t : all)
        if (t && !t->is_cuda())
            refuse(PyExc_RuntimeError, "razorkv_b200 runs on CUDA tensors only; got a tensor on " +
                                           t->device().str() + " (there is no CPU path)");
    for (const at::Tensor* t : all)
        if (t && t->device() != first.device())
            refuse(PyExc_ValueError, "tensors on different devices: " + first.device().str() + " and " +
                                         t->device().str());
    return first.device().index();
}

rkv_kv_layout pool_layout(const at::Tensor& k, const at::Tensor& v) {
    if (k.dim() != 4 || v.sizes() != k.sizes())
        refuse(PyExc_ValueError, "key_pool and value_pool must both be [num_slots, Hkv, P, D], got " +
                                     shape_of(k) + " and " + shape_of(v));
    if (k.scalar_type() != v.scalar_type())
        refuse(PyExc_TypeError, "key_pool and value_pool must share a dtype");
    if (v.strides() != k.strides() || k.stride(3) != 1)
        refuse(PyExc_ValueError, "key_pool and value_pool must share their strides, with contiguous rows");
    if (!k.numel()) refuse(PyExc_ValueError, "the pool has an empty dimension: " + shape_of(k));
    rkv_kv_layout lay{};
    lay.k = k.data_ptr();
    lay.v = v.data_ptr();
    lay.dtype = dtype_code(k.scalar_type());
    lay.head_dim = (int32_t)k.size(3);
    lay.num_kv_heads = k.size(1);
    lay.stride_p = k.stride(0);
    lay.stride_h = k.stride(1);
    lay.stride_t = k.stride(2);
    lay.page_size = k.size(2);
    lay.num_slots = k.size(0);
    return lay;
}

// Makes the device current for a launch and notes that its error word may be set.
struct Launch {
    c10::cuda::OptionalCUDAGuard guard;
    void* stream;
    explicit Launch(c10::DeviceIndex index)
        : guard(c10::Device(c10::kCUDA, index)), stream(c10::cuda::getCurrentCUDAStream(index).stream()) {
        if (index < 64 && !(g_devices.load(std::memory_order_relaxed) >> index & 1))
            g_devices.fetch_or(1ull << index);
    }
    void check(int status, const char* what) const {
        if (status != RKV_OK)
            refuse(g_error, std::string(what) + ": " + g_status(status) + " (status " + std::to_string(status) + ")");
    }
};

PyObject* refused(const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
}

bool want_args(Py_ssize_t got, Py_ssize_t want) {
    if (got == want && g_decode) return true;
    PyErr_SetString(PyExc_TypeError, "ragged binding: wrong number of arguments, or not bound");
    return false;
}

// n elements of a contiguous tensor, from `offset` on, as a tensor of their own on its storage (a
// third of the time that an allocation or a view through the dispatcher takes).
at::Tensor carve(const at::Tensor& from, int64_t offset, int64_t n) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(from.storage()), from.key_set(), from.dtype());
    impl->set_storage_offset(offset);
    impl->set_sizes_contiguous({n});
    return at::Tensor(std::move(impl));
}

// tables(lengths, new_lengths, page_table, free_ring, free_state, page_size, max_new_tokens, inplace)
//   -> (lengths, slot_map, positions, token_starts, free_state)
PyObject* tables(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (!want_args(n_args, 8)) return nullptr;
    try {
        const at::Tensor &lengths = tensor(a[0], "lengths"), &wanted = tensor(a[1], "new_lengths"),
                         &table = tensor(a[2], "page_table"), &ring = tensor(a[3], "free_ring"),
                         &state = tensor(a[4], "free_state");
        const int64_t page = integer(a[5], "page_size"), most = integer(a[6], "max_new_tokens");
        const int inplace = PyObject_IsTrue(a[7]);
        if (inplace < 0) return nullptr;
        want_int64(lengths, 1, "lengths");
        want_int64(wanted, 1, "new_lengths");
        want_int64(table, 2, "page_table");
        want_int64(ring, 1, "free_ring");
        want_int64(state, 1, "free_state");
        const int64_t R = table.size(0), W = table.size(1);
        if (lengths.size(0) != R || wanted.size(0) != R)
            refuse(PyExc_ValueError, "lengths and new_lengths must be [" + std::to_string(R) +
                                         "] like page_table's rows, got " + shape_of(lengths) + " and " +
                                         shape_of(wanted));
        if (state.size(0) != 3 || ring.size(0) < 1)
            refuse(PyExc_ValueError,
                   "free_state must be [3] and free_ring [num_slots], as ragged_free_ring makes them");
        if (page < 1 || most < 0)
            refuse(PyExc_ValueError, "page_size " + std::to_string(page) + " and max_new_tokens " +
                                         std::to_string(most) + " must be positive");
        if (table.numel() && (table.stride(1) != 1 || (R > 1 && table.stride(0) < W)))
            refuse(PyExc_ValueError, "page_table is updated in place: its rows must be contiguous and apart");
        want_written(ring, "free_ring");
        want_written(state, "free_state");
        if (inplace) want_written(lengths, "lengths");
        const auto index = device_of(lengths, &wanted, &table, &ring, &state);
        const Launch launch(index);
        const at::Tensor n = lengths.contiguous(), m = wanted.contiguous();
        const auto options = n.options().requires_grad(false);
        // per token, and per request (which a caller may keep longer)
        const at::Tensor per_token = at::empty({2 * most}, options), per_request = at::empty({2 * R + 4}, options);
        at::Tensor slots = carve(per_token, 0, most), positions = carve(per_token, most, most);
        at::Tensor starts = carve(per_request, 0, R + 1);
        at::Tensor after = inplace ? lengths : carve(per_request, R + 1, R);
        at::Tensor state_after = inplace ? state : carve(per_request, 2 * R + 1, 3);
        launch.check(g_tables(n.data_ptr<int64_t>(), m.data_ptr<int64_t>(), R, page, table.data_ptr<int64_t>(),
                              std::max(table.stride(0), W), W,
                              ring.data_ptr<int64_t>(), ring.size(0), state.data_ptr<int64_t>(),
                              after.data_ptr<int64_t>(), state_after.data_ptr<int64_t>(), slots.data_ptr<int64_t>(),
                              positions.data_ptr<int64_t>(), most, starts.data_ptr<int64_t>(), launch.stream),
                     "rkv_ragged_page_tables");
        PyObject* out = PyTuple_New(5);
        if (!out) return nullptr;
        if (inplace) Py_INCREF(a[0]), Py_INCREF(a[4]);
        PyTuple_SET_ITEM(out, 0, inplace ? a[0] : THPVariable_Wrap(std::move(after)));
        PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(slots)));
        PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(positions)));
        PyTuple_SET_ITEM(out, 3, THPVariable_Wrap(std::move(starts)));
        PyTuple_SET_ITEM(out, 4, inplace ? a[4] : THPVariable_Wrap(std::move(state_after)));
        return out;
    } catch (const Refused& r) {
        return refused(r);
    }
    END_HANDLE_TH_ERRORS
}

// append(key, value, key_pool, value_pool, slot_map)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (!want_args(n_args, 5)) return nullptr;
    try {
        const at::Tensor &key = tensor(a[0], "key"), &value = tensor(a[1], "value"),
                         &kp = tensor(a[2], "key_pool"), &vp = tensor(a[3], "value_pool"),
                         &slots = tensor(a[4], "slot_map");
        want_int64(slots, 1, "slot_map");
        const rkv_kv_layout lay = pool_layout(kp, vp);
        const int64_t T = slots.size(0);
        if (key.sizes() != at::IntArrayRef({T, lay.num_kv_heads, (int64_t)lay.head_dim}) ||
            value.sizes() != key.sizes())
            refuse(PyExc_ValueError, "key and value must be [" + std::to_string(T) + ", " +
                                         std::to_string(lay.num_kv_heads) + ", " + std::to_string(lay.head_dim) +
                                         "], got " + shape_of(key) + " and " + shape_of(value));
        if (key.scalar_type() != kp.scalar_type() || value.scalar_type() != kp.scalar_type())
            refuse(PyExc_TypeError, std::string("key and value must have the pool's dtype ") +
                                        c10::toString(kp.scalar_type()));
        if (on_itself(kp) || on_itself(vp) || on_another(kp, vp))
            refuse(PyExc_ValueError, "the rows of key_pool and value_pool are written and must not overlap");
        const auto index = device_of(key, &value, &kp, &vp, &slots);
        if (T == 0) Py_RETURN_NONE;
        const Launch launch(index);
        const c10::AutoGradMode no_grad(false);
        at::Tensor k = key.stride(2) == 1 ? key : key.contiguous();
        at::Tensor v = value.stride(2) == 1 ? value : value.contiguous();
        if (k.strides() != v.strides()) k = k.contiguous(), v = v.contiguous();
        const at::Tensor s = slots.contiguous();
        launch.check(g_append(&lay, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), T, s.data_ptr<int64_t>(),
                              launch.stream),
                     "rkv_ragged_append");
        Py_RETURN_NONE;
    } catch (const Refused& r) {
        return refused(r);
    }
    END_HANDLE_TH_ERRORS
}

// Lengths, and the table entries of tokens that are attended, read back.
void validate(const at::Tensor& table, const at::Tensor& lengths, const at::Tensor* starts, const rkv_kv_layout& lay) {
    const int64_t lo = lengths.min().item<int64_t>(), hi = lengths.max().item<int64_t>();
    if (lo < 0 || hi > lay.num_tokens)
        refuse(PyExc_IndexError, "lengths must lie in [0, " + std::to_string(lay.num_tokens) + "], got [" +
                                     std::to_string(lo) + ", " + std::to_string(hi) + "]");
    if (starts && starts->min().item<int64_t>() < 0)
        refuse(PyExc_IndexError, "starts must not be negative, got " + std::to_string(starts->min().item<int64_t>()));
    if (!table.numel()) return;
    const at::Tensor first = (at::arange(table.size(1), table.options()) * lay.page_size).unsqueeze(0);
    at::Tensor used = first < lengths.unsqueeze(1);
    if (starts) used = used & (first + lay.page_size > starts->unsqueeze(1)) & (*starts < lengths).unsqueeze(1);
    if ((used & ((table < 0) | (table >= lay.num_slots))).any().item<bool>())
        refuse(PyExc_IndexError, "page_table entries must lie in [0, " + std::to_string(lay.num_slots) + ")");
}

// decode(query, key_pool, value_pool, page_table, lengths, scale, starts, return_lse, out, validate)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (!want_args(n_args, 10)) return nullptr;
    try {
        const at::Tensor &query = tensor(a[0], "query"), &kp = tensor(a[1], "key_pool"),
                         &vp = tensor(a[2], "value_pool"), &pages = tensor(a[3], "page_table"),
                         &lengths = tensor(a[4], "lengths");
        const at::Tensor *starts = tensor_or_none(a[6], "starts"), *given = tensor_or_none(a[8], "out");
        const int want_lse = PyObject_IsTrue(a[7]), want_checks = PyObject_IsTrue(a[9]);
        if (want_lse < 0 || want_checks < 0) return nullptr;
        if (query.dim() != 4) refuse(PyExc_ValueError, "query must be [B, H, 1, D], got " + shape_of(query));
        const int64_t B = query.size(0), H = query.size(1), D = query.size(3);
        if (query.size(2) != 1)
            refuse(PyExc_AssertionError, "ragged decode attention is defined for single-token decoding (q_len == 1).");
        want_int64(pages, 2, "page_table");
        want_int64(lengths, 1, "lengths");
        if (starts) want_int64(*starts, 1, "starts");
        rkv_kv_layout lay = pool_layout(kp, vp);
        if (lay.head_dim != D)
            refuse(PyExc_ValueError, "the pool's head_dim " + std::to_string(lay.head_dim) + " is not the query's " +
                                         std::to_string(D));
        if (H < 1 || H > INT32_MAX || H % lay.num_kv_heads)
            refuse(PyExc_ValueError, "num_heads " + std::to_string(H) + " is not a multiple of num_kv_heads " +
                                         std::to_string(lay.num_kv_heads));
        if (query.scalar_type() != kp.scalar_type())
            refuse(PyExc_TypeError, std::string("query ") + c10::toString(query.scalar_type()) + " and pool " +
                                        c10::toString(kp.scalar_type()) + " must share a dtype");
        if (pages.size(0) != B || lengths.size(0) != B || (starts && starts->size(0) != B))
            refuse(PyExc_ValueError, "page_table, lengths and starts must have one row per request (" +
                                         std::to_string(B) + ")");
        double scale = 0.0;
        if (a[5] != Py_None) {
            scale = PyFloat_AsDouble(a[5]);
            if (scale == -1.0 && PyErr_Occurred()) return nullptr;
            if (!(scale > 0.0 && std::isfinite((float)scale * 1.44269504f) && (float)scale > 0.f))   // (log2 e)
                refuse(PyExc_ValueError, "scale must be positive and below 2.35e38, got " + std::to_string(scale));
        }
        if (given) {
            if (given->sizes() != query.sizes() || given->scalar_type() != query.scalar_type() ||
                given->stride(3) != 1)
                refuse(PyExc_ValueError, "out must have the query's shape and dtype, with contiguous rows");
            if (B && given->data_ptr() == query.data_ptr()) refuse(PyExc_ValueError, "out must not be the query");
            if (on_itself(*given) || on_another(*given, query) || on_another(*given, kp) || on_another(*given, vp))
                refuse(PyExc_ValueError, "out's rows must not overlap each other, the query or the pools");
        }
        if (want_checks) {      // (on any device)
            lay.num_tokens = pages.size(1) * lay.page_size;
            if (B) validate(pages, lengths, starts, lay);
        }
        const auto index = device_of(query, &kp, &vp, &pages, &lengths, starts, given);
        const Launch launch(index);
        const c10::AutoGradMode no_grad(false);
        const auto options = query.options().requires_grad(false);
        at::Tensor out = given ? *given : at::empty({B, H, 1, D}, options);
        at::Tensor lse;
        if (want_lse) lse = at::empty({B, H}, options.dtype(at::kFloat));
        if (B) {
            const at::Tensor table = pages.stride(1) == 1 ? pages : pages.contiguous();
            const at::Tensor n = lengths.contiguous();
            std::optional<at::Tensor> first;
            if (starts) first = starts->contiguous();
            // rows in steps of 16 bytes, as the vector kernels read them
            at::Tensor q = query;
            const int64_t step = 16 / query.element_size();
            if (q.stride(3) != 1 || q.stride(0) % step || q.stride(1) % step || ((uintptr_t)q.data_ptr() & 15))
                q = at::empty({B, H, 1, D}, options).copy_(query);
            lay.batch = B;
            lay.page_table = table.data_ptr<int64_t>();
            lay.pt_stride_b = table.stride(0);
            lay.num_tokens = table.size(1) * lay.page_size;
            const rkv_query qs{q.data_ptr(), lay.dtype, (int32_t)H, 1, q.stride(0), q.stride(1), q.stride(2)};
            const rkv_output os{out.data_ptr(), lay.dtype, 0, out.stride(0), out.stride(1), out.stride(2)};
            const size_t bytes = g_decode_size(&qs, &lay);
            // of the caching allocator, so that each call and each captured graph has its own
            const at::Tensor ws = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
            launch.check(g_decode(&qs, &lay, n.data_ptr<int64_t>(), first ? first->data_ptr<int64_t>() : nullptr,
                                  (float)scale, &os, want_lse ? lse.data_ptr<float>() : nullptr, ws.data_ptr(), bytes,
                                  launch.stream),
                         "rkv_ragged_decode_attention");
        }
        PyObject* o;
        if (given) {
            o = a[8];
            Py_INCREF(o);
        } else {
            o = THPVariable_Wrap(std::move(out));
        }
        if (!want_lse || !o) return o;
        PyObject* pair = PyTuple_New(2);
        if (!pair) return nullptr;
        PyTuple_SET_ITEM(pair, 0, o);
        PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(lse)));
        return pair;
    } catch (const Refused& r) {
        return refused(r);
    }
    END_HANDLE_TH_ERRORS
}

// bind(error class, addresses of the five C entries below)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject* error;
    unsigned long long t, p, d, s, u;
    if (!PyArg_ParseTuple(args, "OKKKKK", &error, &t, &p, &d, &s, &u)) return nullptr;
    Py_INCREF(error);
    Py_XSETREF(g_error, error);
    g_tables = reinterpret_cast<decltype(g_tables)>(t);
    g_append = reinterpret_cast<decltype(g_append)>(p);
    g_decode_size = reinterpret_cast<decltype(g_decode_size)>(s);
    g_status = reinterpret_cast<decltype(g_status)>(u);
    g_decode = reinterpret_cast<decltype(g_decode)>(d);
    Py_RETURN_NONE;
}

// Bit mask of the devices that an operator has run on.
PyObject* devices(PyObject*, PyObject*) { return PyLong_FromUnsignedLongLong(g_devices.load()); }

PyMethodDef methods[] = {
    {"tables", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(tables)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(decode)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {"devices", devices, METH_NOARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ragged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ragged(void) { return PyModule_Create(&module); }
