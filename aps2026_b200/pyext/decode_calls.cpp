// The decode step's calls on torch tensors (_decode_calls, used by decode.py).
//
// A decode step makes dozens of calls whose kernels take a few microseconds,
// so what a call costs on the host is what a small step costs. Through ctypes,
// with the checks of some ten tensors in Python, a call took 8.4 us (4.2 us of
// checks, 1.5 us of converting arguments, the launch); here it is the launch
// and some tenths of a microsecond. Each function checks its tensors, raises
// ops.InvalidArgument for what it refuses, and returns the status of the C ABI
// call (include/aps2026_b200.h), which runs on the current torch stream.
#include <Python.h>

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>

#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/aps2026_b200.h"

namespace {

PyObject* invalid_argument = nullptr;  // ops.InvalidArgument

struct Refusal {
    std::string why;
};
struct PythonError {};  // the interpreter has it already

using At = at::Tensor;

const At& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) throw Refusal{std::string(what) + ": expected a tensor"};
    return THPVariable_Unpack(o);
}
std::size_t size(PyObject* o, const char* what) {
    const Py_ssize_t n = PyNumber_AsSsize_t(o, PyExc_OverflowError);
    if (n == -1 && PyErr_Occurred()) throw PythonError{};
    if (n < 0) throw Refusal{std::string(what) + " is negative"};
    return static_cast<std::size_t>(n);
}
float number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
    return static_cast<float>(v);
}
std::string list(std::initializer_list<std::int64_t> shape) {
    std::string s = "[";
    for (const std::int64_t n : shape) s += (s.size() > 1 ? ", " : "") + std::to_string(n);
    return s + "]";
}
bool has_shape(const At& t, std::initializer_list<std::int64_t> shape) {
    return t.sizes().equals(at::IntArrayRef(shape));
}
std::uint32_t dtype_code(const At& t, const char* what) {
    if (t.scalar_type() == at::kFloat) return B2_DTYPE_F32;
    if (t.scalar_type() == at::kBFloat16) return B2_DTYPE_BF16;
    throw Refusal{std::string(what) + ": expected float32 or bfloat16, got " + c10::toString(t.scalar_type())};
}
// The current stream of the tensors' device, which must be the current one.
b2_stream_t stream_of(int device) {
    if (device < 0) throw Refusal{"tensor is not on a CUDA device"};
    const int current = c10::cuda::current_device();
    if (device != current)
        throw Refusal{"tensors are on CUDA device " + std::to_string(device) + ", the current one is " +
                      std::to_string(current)};
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}
// n contiguous 32-bit indices.
const std::uint32_t* indices(PyObject* o, std::int64_t n, int device, const char* what) {
    const At& t = tensor(o, what);
    if ((t.scalar_type() != at::kInt && t.scalar_type() != at::kUInt32) || t.numel() != n || t.get_device() != device ||
        !t.is_contiguous())
        throw Refusal{std::string(what) + ": expected " + std::to_string(n) + " contiguous 32-bit indices on CUDA device " +
                      std::to_string(device)};
    return static_cast<const std::uint32_t*>(t.const_data_ptr());
}
// [rows, heads, dim] activations whose last dimension is contiguous (slices
// of a fused projection are).
struct Heads {
    const void* data = nullptr;
    std::size_t by_row = 0, by_head = 0;
};
Heads heads_of(const At& t, std::int64_t rows, std::int64_t heads, std::int64_t dim, int device, const char* what) {
    if (!has_shape(t, {rows, heads, dim}) || t.get_device() != device)
        throw Refusal{std::string(what) + ": expected " + list({rows, heads, dim}) + " on CUDA device " + std::to_string(device)};
    if (rows && t.stride(2) != 1) throw Refusal{std::string(what) + ": the last dimension must be contiguous"};
    return {t.const_data_ptr(), static_cast<std::size_t>(t.stride(0)), static_cast<std::size_t>(t.stride(1))};
}
// t, if it is contiguous and of this shape and type.
const At& whole(const At& t, std::initializer_list<std::int64_t> shape, at::ScalarType dtype, int device, const char* what) {
    if (t.scalar_type() != dtype || !has_shape(t, shape) || t.get_device() != device || !t.is_contiguous())
        throw Refusal{std::string(what) + ": expected a contiguous " + list(shape) + " " + c10::toString(dtype) +
                      " tensor on CUDA device " + std::to_string(device)};
    return t;
}
// Refuses a buffer that is not `bytes` adjacent bytes at least.
void bytes_of(const At& t, std::size_t bytes, const char* what) {
    if (!t.is_contiguous() || t.nbytes() < bytes)
        throw Refusal{std::string(what) + ": expected " + std::to_string(bytes) + " contiguous bytes, got " +
                      (t.is_contiguous() ? std::to_string(t.nbytes()) : "a tensor that is not contiguous")};
}

// Five arguments of a KVCache4 (data, pages, page_size, kv_heads, head_dim) and its page table.
b2_kv4_cache cache_of(PyObject* const* a, PyObject* page_table, bool writes, int* device) {
    const At &data = tensor(a[0], "cache"), &table = tensor(page_table, "page_table");
    *device = data.get_device();
    if (table.dim() != 2 || (table.scalar_type() != at::kInt && table.scalar_type() != at::kUInt32) ||
        table.get_device() != *device || !table.is_contiguous())
        throw Refusal{"page_table: expected contiguous 32-bit indices [seqs, max_pages] on the cache's device"};
    b2_kv4_cache c{};
    c.data = writes ? data.mutable_data_ptr() : const_cast<void*>(data.const_data_ptr());
    c.pages = size(a[1], "pages");
    c.page_size = size(a[2], "page_size");
    c.kv_heads = size(a[3], "kv_heads");
    c.head_dim = size(a[4], "head_dim");
    c.page_table = static_cast<const std::uint32_t*>(table.const_data_ptr());
    c.seqs = static_cast<std::size_t>(table.size(0));
    c.max_pages = static_cast<std::size_t>(table.size(1));
    // the kernels bound pages by c.pages alone (a description that has no page size is refused by the call itself)
    std::size_t page = 0;
    if (b2_kv4_page_bytes(c.page_size, c.kv_heads, c.head_dim, &page) == B2_OK)
        bytes_of(data, page && c.pages > SIZE_MAX / page ? SIZE_MAX : c.pages * page, "cache");
    return c;
}

// Runs f, which returns a status; errors become Python's. n: arguments wanted.
template <typename F>
PyObject* call(Py_ssize_t have, Py_ssize_t n, F f) {
    if (have != n) {
        PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", n, have);
        return nullptr;
    }
    try {
        return PyLong_FromLong(f());
    } catch (const Refusal& r) {
        PyErr_SetString(invalid_argument, r.why.c_str());
    } catch (const PythonError&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
// A launch may wait for room in the stream's queue: without the interpreter's lock.
template <typename F>
int unlocked(F f) {
    int rc = 0;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    return rc;
}

// k, v, row_seq, row_pos, cache x 5, page_table, q, q_out, cos, sin
PyObject* kv4_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 14, [&] {
        int device = -1;
        const b2_kv4_cache cache = cache_of(a + 4, a[9], true, &device);
        const b2_stream_t stream = stream_of(device);
        const At &k = tensor(a[0], "kv4_append k"), &v = tensor(a[1], "kv4_append v");
        const std::int64_t rows = k.dim() ? k.size(0) : 0, heads = static_cast<std::int64_t>(cache.kv_heads),
                           dim = static_cast<std::int64_t>(cache.head_dim);
        const std::uint32_t dtype = dtype_code(k, "kv4_append k");
        if (v.scalar_type() != k.scalar_type()) throw Refusal{"kv4_append: q, k and v must have one dtype"};
        const Heads kh = heads_of(k, rows, heads, dim, device, "kv4_append k");
        const Heads vh = heads_of(v, rows, heads, dim, device, "kv4_append v");
        Heads qh;
        void* q_out = nullptr;
        std::int64_t q_heads = 0;
        if (a[10] != Py_None) {
            const At& q = tensor(a[10], "kv4_append q");
            if (q.scalar_type() != k.scalar_type()) throw Refusal{"kv4_append: q, k and v must have one dtype"};
            if (a[11] == Py_None) throw Refusal{"kv4_append: q without q_out"};
            q_heads = q.dim() > 1 ? q.size(1) : 0;
            qh = heads_of(q, rows, q_heads, dim, device, "kv4_append q");
            q_out = whole(tensor(a[11], "kv4_append q_out"), {rows, q_heads, dim}, k.scalar_type(), device, "kv4_append q_out")
                        .mutable_data_ptr();
        }
        if ((a[12] == Py_None) != (a[13] == Py_None)) throw Refusal{"kv4_append: one rotation table without the other"};
        const float *cos = nullptr, *sin = nullptr;
        std::int64_t positions = 0;
        if (a[12] != Py_None) {
            const At &c = tensor(a[12], "kv4_append cos"), &s = tensor(a[13], "kv4_append sin");
            positions = c.dim() ? c.size(0) : 0;
            cos = static_cast<const float*>(whole(c, {positions, dim / 2}, at::kFloat, device, "kv4_append cos").const_data_ptr());
            sin = static_cast<const float*>(whole(s, {positions, dim / 2}, at::kFloat, device, "kv4_append sin").const_data_ptr());
        }
        const std::uint32_t *seq = indices(a[2], rows, device, "row_seq"), *pos = indices(a[3], rows, device, "row_pos");
        return unlocked([&] {
            return b2_kv4_append(qh.data, qh.by_row, qh.by_head, static_cast<std::size_t>(q_heads), q_out, kh.data,
                                 kh.by_row, kh.by_head, vh.data, vh.by_row, vh.by_head, dtype,
                                 static_cast<std::size_t>(rows), seq, pos, cos, sin,
                                 static_cast<std::size_t>(positions), &cache, stream);
        });
    });
}

// cache x 5, page_table, row_seq, row_pos, k_out, v_out
PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 10, [&] {
        int device = -1;
        const b2_kv4_cache cache = cache_of(a, a[5], false, &device);
        const b2_stream_t stream = stream_of(device);
        const std::int64_t rows = tensor(a[6], "row_seq").numel(), heads = static_cast<std::int64_t>(cache.kv_heads),
                           dim = static_cast<std::int64_t>(cache.head_dim);
        const std::uint32_t *seq = indices(a[6], rows, device, "row_seq"), *pos = indices(a[7], rows, device, "row_pos");
        const At &k = tensor(a[8], "kv4_read k_out"), &v = tensor(a[9], "kv4_read v_out");
        const std::uint32_t dtype = dtype_code(k, "kv4_read k_out");
        void* k_out = whole(k, {rows, heads, dim}, k.scalar_type(), device, "kv4_read k_out").mutable_data_ptr();
        void* v_out = whole(v, {rows, heads, dim}, k.scalar_type(), device, "kv4_read v_out").mutable_data_ptr();
        return unlocked([&] {
            return b2_kv4_read(&cache, seq, pos, static_cast<std::size_t>(rows), k_out, v_out, dtype, stream);
        });
    });
}

// q, cache x 5, page_table, lens, out, q_offsets, max_queries, max_len, scale,
// window, sinks, workspace, its bytes; max_len and scale may be None
PyObject* attention_kv4(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 17, [&] {
        int device = -1;
        const b2_kv4_cache cache = cache_of(a + 1, a[6], false, &device);
        const b2_stream_t stream = stream_of(device);
        const At &q = tensor(a[0], "attention_kv4 q"), &ws = tensor(a[15], "attention_kv4 workspace");
        if (q.dim() != 3) throw Refusal{"attention_kv4 q: expected [rows, q_heads, head_dim]"};
        const std::int64_t rows = q.size(0), q_heads = q.size(1), dim = static_cast<std::int64_t>(cache.head_dim);
        const std::int64_t seqs = static_cast<std::int64_t>(cache.seqs);
        const std::uint32_t dtype = dtype_code(q, "attention_kv4 q");
        const Heads qh = heads_of(q, rows, q_heads, dim, device, "attention_kv4 q");
        void* out = whole(tensor(a[8], "attention_kv4 out"), {rows, q_heads, dim}, q.scalar_type(), device, "attention_kv4 out")
                        .mutable_data_ptr();
        const std::uint32_t* offsets = a[9] == Py_None ? nullptr : indices(a[9], seqs + 1, device, "q_offsets");
        const std::uint32_t* lens = indices(a[7], seqs, device, "lens");
        const std::size_t max_queries = size(a[10], "attention_kv4: max_queries"),
                          max_len = a[11] == Py_None ? cache.max_pages * cache.page_size : size(a[11], "attention_kv4: max_len"),
                          window = size(a[13], "attention_kv4: window"), sinks = size(a[14], "attention_kv4: sinks"),
                          ws_bytes = size(a[16], "attention_kv4: workspace bytes");
        const float scale = a[12] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim))) : number(a[12]);
        if (ws.get_device() != device) throw Refusal{"attention_kv4: the workspace is on another device"};
        bytes_of(ws, ws_bytes, "attention_kv4 workspace");
        void* workspace = ws.mutable_data_ptr();
        return unlocked([&] {
            return b2_attention_kv4(qh.data, qh.by_row, qh.by_head, out, dtype, static_cast<std::size_t>(rows),
                                    static_cast<std::size_t>(q_heads), offsets, lens, max_queries, max_len, scale, window,
                                    sinks, &cache, workspace, ws_bytes, stream);
        });
    });
}

// x, logits, w_gate_up, w_down, out, quantum, tie_eps, gates (code), workspace, its bytes
PyObject* moe_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 10, [&] {
        const At &x = tensor(a[0], "moe_decode x"), &w_down = tensor(a[3], "moe_decode w_down");
        const At &out = tensor(a[4], "moe_decode out"), &ws = tensor(a[8], "moe_decode workspace");
        const int device = x.get_device();
        const b2_stream_t stream = stream_of(device);
        if (x.dim() != 2 || w_down.dim() != 3) throw Refusal{"moe_decode: expected x [T, H] and w_down [E, H, I]"};
        const std::int64_t T = x.size(0), H = x.size(1), E = w_down.size(0), I = w_down.size(2);
        if (!has_shape(out, {T, H}) || out.scalar_type() != x.scalar_type() || out.get_device() != device)
            throw Refusal{"moe_decode out: expected " + list({T, H}) + " " + c10::toString(x.scalar_type()) +
                          " on CUDA device " + std::to_string(device)};
        if (H > 1 && (x.stride(1) != 1 || out.stride(1) != 1))
            throw Refusal{"moe_decode: the last dimension of x and out must be contiguous"};
        const std::uint32_t x_dtype = dtype_code(x, "moe_decode x"), w_dtype = dtype_code(w_down, "moe_decode w_down");
        const at::ScalarType weights = w_down.scalar_type();
        const auto* logits = static_cast<const float*>(
            whole(tensor(a[1], "moe_decode logits"), {T, E}, at::kFloat, device, "moe_decode logits").const_data_ptr());
        const void* gate_up =
            whole(tensor(a[2], "moe_decode w_gate_up"), {E, 2 * I, H}, weights, device, "moe_decode w_gate_up").const_data_ptr();
        const void* down = whole(w_down, {E, H, I}, weights, device, "moe_decode w_down").const_data_ptr();
        if (ws.get_device() != device) throw Refusal{"moe_decode: the workspace is on another device"};
        const float quantum = number(a[5]), tie_eps = number(a[6]);
        const std::uint32_t gates = static_cast<std::uint32_t>(size(a[7], "moe_decode: gates"));
        const std::size_t ws_bytes = size(a[9], "moe_decode: workspace bytes");
        bytes_of(ws, ws_bytes, "moe_decode workspace");
        const std::size_t ld_x = static_cast<std::size_t>(T > 1 ? x.stride(0) : H),
                          ld_out = static_cast<std::size_t>(T > 1 ? out.stride(0) : H);
        void *to = out.mutable_data_ptr(), *workspace = ws.mutable_data_ptr();
        const void* from = x.const_data_ptr();
        return unlocked([&] {
            return b2_moe_decode(from, ld_x, x_dtype, logits, static_cast<std::size_t>(T), static_cast<std::size_t>(H),
                                 static_cast<std::size_t>(E), static_cast<std::size_t>(I), quantum, tie_eps, gates, gate_up,
                                 down, w_dtype, to, ld_out, workspace, ws_bytes, stream);
        });
    });
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<kv4_append>("kv4_append"), method<kv4_read>("kv4_read"),
                         method<attention_kv4>("attention_kv4"), method<moe_decode>("moe_decode"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decode_calls() {
    PyObject* ops = PyImport_ImportModule("aps2026_b200.ops");
    if (!ops) return nullptr;
    invalid_argument = PyObject_GetAttrString(ops, "InvalidArgument");
    Py_DECREF(ops);
    return invalid_argument ? PyModule_Create(&module) : nullptr;
}
