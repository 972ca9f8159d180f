// af_torch.cpp -- the paged operators for torch tensors (module
// atomflow_b200._torch_ops, called by atomflow_b200/ops.py).
//
// Argument checks, outputs and the call of the C ABI, in C++: a decode step calls
// these for every layer and its kernels take 3 to 6 us, while the same checks in
// Python took 10.  Positional arguments only; ops.py has the signatures and the
// documentation.  Bad arguments raise ValueError (TypeError where a tensor or a
// number is expected and something else given); a status of the C ABI other than
// AF_OK is returned as an int, for ops.py to raise.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <exception>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "atomflow_b200.h"

namespace {

struct ValueError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct TypeError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
struct PythonError : std::exception {};   // already set

[[noreturn]] void bad(const char* what) { throw ValueError(what); }

// These operators serve; a gradient asked for, backward or forward (a dual tensor's tangent), would be lost without a word.
// Outputs given by the caller too: what is written into them is not recorded.
void no_gradient(const at::Tensor& t) {
    if (t.requires_grad() && c10::GradMode::is_enabled()) bad("the paged operators have no gradient: detach the input, or call under torch.no_grad()");
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
        bad("the paged operators have no gradient: unpack the dual tensor, or call under torch.inference_mode()");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) throw TypeError(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o) {
    PyObject* i = PyNumber_Index(o);
    if (i == nullptr) throw PythonError();
    const long long v = PyLong_AsLongLong(i);
    Py_DECREF(i);
    if (v == -1 && PyErr_Occurred()) throw PythonError();
    return v;
}
int to_int(int64_t v, const char* what) {
    if (v < INT_MIN || v > INT_MAX) bad(what);
    return (int)v;
}
void no_gradient(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        if (t != nullptr) no_gradient(*t);
}
// Tells autograd that tensors were written in place, so that what saved one for its backward pass notices.  (Tensors made
// under inference mode have no version.)
void written(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
void* pointer(const at::Tensor& t) { return t.numel() == 0 ? nullptr : t.data_ptr(); }

// The C structures of a cache and a batch, checked (shapes, types, strides, one device), and the device's index.
struct Paged {
    af_paged_kv kv;
    af_paged_batch batch;
    int dev;
};
Paged paged(int64_t n_tokens, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& len,
            const at::Tensor& cu, const at::Tensor* ks, const at::Tensor* vs) {
    const char* one_device = "every tensor must be on one CUDA device";
    no_gradient({&k, &v, ks, vs});
    Paged p{};
    const at::ScalarType type = k.scalar_type();
    if (type == at::kHalf) p.kv.format = AF_KV_F16;
    else if (type == at::kFloat8_e4m3fn) p.kv.format = AF_KV_FP8_E4M3;
    else if (type == at::kChar) p.kv.format = AF_KV_INT8;
    else bad("k_pages and v_pages must both be float16, float8_e4m3fn or int8");
    if (v.scalar_type() != type) bad("k_pages and v_pages must both be float16, float8_e4m3fn or int8");
    if (k.dim() != 4 || v.sizes() != k.sizes() || v.strides() != k.strides())
        bad("k_pages and v_pages must be [n_pages, page_size, n_kv_heads, head_dim], strided alike");
    const int64_t n_pages = k.size(0), page = k.size(1), nkv = k.size(2), hd = k.size(3);
    if (k.stride(3) != 1 || k.stride(2) != hd || k.stride(1) != nkv * hd) bad("each page must be contiguous");
    const int dev = k.is_cuda() ? (int)k.get_device() : -1;
    if (p.kv.format == AF_KV_F16) {
        if (ks != nullptr || vs != nullptr) bad("float16 pages take no scales");
    } else {
        if (ks == nullptr || vs == nullptr) bad("8-bit pages need k_scale and v_scale");
        if (ks->scalar_type() != at::kHalf || vs->scalar_type() != at::kHalf || ks->dim() != 3 ||
            ks->sizes() != k.sizes().slice(0, 3) || vs->sizes() != ks->sizes() || vs->strides() != ks->strides() ||
            ks->stride(2) != 1 || ks->stride(1) != nkv)
            bad("scales must be float16 [n_pages, page_size, n_kv_heads], each page contiguous, alike");
        if (ks->get_device() != dev || vs->get_device() != dev) bad(one_device);
        p.kv.scale_stride = n_pages > 1 ? ks->stride(0) : page * nkv;
        p.kv.k_scale = pointer(*ks);
        p.kv.v_scale = pointer(*vs);
    }
    if (table.scalar_type() != at::kInt || len.scalar_type() != at::kInt || cu.scalar_type() != at::kInt || table.dim() != 2)
        bad("block_table must be int32 [n_seqs, max_pages], kv_len and the row offsets int32");
    const int64_t n = table.size(0), width = table.size(1);
    if (len.dim() != 1 || len.size(0) != n || cu.dim() != 1 || cu.size(0) != n + 1 || !len.is_contiguous() ||
        !cu.is_contiguous())
        bad("kv_len must be [n_seqs], the row offsets [n_seqs + 1], contiguous");
    if (width > 1 && table.stride(1) != 1) bad("block_table's rows must be contiguous");
    if (dev < 0 || v.get_device() != dev || table.get_device() != dev || len.get_device() != dev || cu.get_device() != dev)
        bad(one_device);
    const char* large = "a dimension does not fit in 32 bits";
    p.kv.n_pages = to_int(n_pages, large);
    p.kv.page_size = to_int(page, large);
    p.kv.n_kv_heads = to_int(nkv, large);
    p.kv.head_dim = to_int(hd, large);
    p.kv.k = pointer(k);
    p.kv.v = pointer(v);
    p.kv.page_stride = n_pages > 1 ? k.stride(0) : page * nkv * hd;
    p.batch.n_seqs = to_int(n, large);
    p.batch.n_tokens = to_int(n_tokens, large);
    p.batch.max_pages = to_int(width, large);
    p.batch.cu_rows = static_cast<const int*>(pointer(cu));
    p.batch.kv_len = static_cast<const int*>(pointer(len));
    p.batch.block_table = static_cast<const int*>(pointer(table));
    p.batch.table_stride = n > 1 ? table.stride(0) : width;
    p.dev = dev;
    return p;
}

// The distance between the rows of an FP16 tensor of the given shape, each row contiguous.
int64_t rows(const at::Tensor& t, const char* name, int dev, at::IntArrayRef shape) {
    if (t.scalar_type() != at::kHalf || t.sizes() != shape || t.get_device() != dev) {
        std::string s = std::string(name) + " must be a float16 tensor [";
        for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
        throw ValueError(s + "] on the pages' device");
    }
    int64_t inner = 1;
    for (int64_t d = (int64_t)shape.size() - 1; d > 0; --d) {
        if (t.stride(d) != inner && shape[d] != 1) throw ValueError(std::string(name) + "'s rows must be contiguous");
        inner *= shape[d];
    }
    return shape[0] > 1 ? t.stride(0) : inner;
}
// out, checked to be contiguous and of the given shape, or a new tensor like `model`.
at::Tensor output(const at::Tensor* out, const char* name, int dev, at::IntArrayRef shape, const at::Tensor& model) {
    if (out == nullptr) return at::empty(shape, model.options().dtype(at::kHalf));
    if (!out->is_contiguous()) throw ValueError(std::string(name) + " must be contiguous");
    rows(*out, name, dev, shape);
    return *out;
}

template <class F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& f) {
    try {
        if (got != want) throw TypeError("wrong number of arguments");
        return f();
    } catch (const PythonError&) {
    } catch (const ValueError& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const TypeError& e) {
        PyErr_SetString(PyExc_TypeError, e.what());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

// (qkv, k_pages, v_pages, block_table, kv_len, cu_rows, n_heads, cos, sin, k_scale, v_scale, q_out) -> q, or None
// without tables
PyObject* paged_kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&]() -> PyObject* {
        const at::Tensor& qkv = tensor(a[0], "qkv");
        const at::Tensor *cos = optional(a[7], "cos"), *sin = optional(a[8], "sin"), *q_out = optional(a[11], "q_out");
        if (qkv.dim() != 2) bad("qkv must be [T, (n_heads + 2 n_kv_heads) * head_dim]");
        no_gradient({&qkv, cos, sin, q_out});
        const int64_t T = qkv.size(0), nh = integer(a[6]);
        const at::Tensor &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages");
        const at::Tensor *ks = optional(a[9], "k_scale"), *vs = optional(a[10], "v_scale");
        Paged p = paged(T, k, v, tensor(a[3], "block_table"), tensor(a[4], "kv_len"), tensor(a[5], "cu_rows"), ks, vs);
        const int64_t hd = p.kv.head_dim;
        if (nh < 0 || nh > INT_MAX) bad("n_heads must be a count of heads");
        const int64_t stride = rows(qkv, "qkv", p.dev, {T, (nh + 2 * p.kv.n_kv_heads) * hd});
        const c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.dev);
        at::Tensor q;
        const float *c = nullptr, *s = nullptr;
        int64_t max_seq = 0;
        if (cos == nullptr || sin == nullptr) {
            if (cos != nullptr || sin != nullptr) bad("cos and sin come together");
            if (q_out != nullptr) bad("q_out needs cos and sin: without them q is left in qkv");
        } else {
            if (cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat || cos->dim() != 2 ||
                cos->size(1) * 2 != hd || sin->sizes() != cos->sizes() || cos->get_device() != p.dev ||
                sin->get_device() != p.dev || !cos->is_contiguous() || !sin->is_contiguous())
                bad("cos and sin must be contiguous float32 [max_seq, head_dim / 2] on the pages' device");
            max_seq = cos->size(0);
            c = static_cast<const float*>(pointer(*cos));
            s = static_cast<const float*>(pointer(*sin));
            if (c == nullptr) bad("cos and sin are empty");
            q = output(q_out, "q_out", p.dev, {T, nh, hd}, qkv);
        }
        const af_status st = af_paged_kv_write(&p.kv, &p.batch, pointer(qkv), stride, (int)nh, c, s,
                                               to_int(max_seq, "the tables are too long"), q.defined() ? pointer(q) : nullptr,
                                               c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)p.dev).stream());
        if (st != AF_OK) return PyLong_FromLong(st);
        written({&k, &v, ks, vs, q_out});
        if (!q.defined()) Py_RETURN_NONE;
        return THPVariable_Wrap(q);
    });
}

// (k_pages, v_pages, block_table, kv_len, cu_rows, n_rows, k_scale, v_scale, k_out, v_out) -> (k, v)
PyObject* paged_kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&]() -> PyObject* {
        const at::Tensor& pages = tensor(a[0], "k_pages");
        const at::Tensor *k_out = optional(a[8], "k_out"), *v_out = optional(a[9], "v_out");
        no_gradient({k_out, v_out});
        const int64_t T = integer(a[5]);
        if (T < 0) bad("n_rows must not be negative");
        Paged p = paged(T, pages, tensor(a[1], "v_pages"), tensor(a[2], "block_table"), tensor(a[3], "kv_len"),
                        tensor(a[4], "cu_rows"), optional(a[6], "k_scale"), optional(a[7], "v_scale"));
        const c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.dev);
        const int64_t shape[3] = {T, p.kv.n_kv_heads, p.kv.head_dim};
        const at::Tensor k = output(k_out, "k_out", p.dev, shape, pages);
        const at::Tensor v = output(v_out, "v_out", p.dev, shape, pages);
        const af_status st = af_paged_kv_read(&p.kv, &p.batch, pointer(k), pointer(v),
                                              c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)p.dev).stream());
        if (st != AF_OK) return PyLong_FromLong(st);
        written({k_out, v_out});
        PyObject *pk = THPVariable_Wrap(k), *pv = THPVariable_Wrap(v);
        PyObject* r = pk != nullptr && pv != nullptr ? PyTuple_Pack(2, pk, pv) : nullptr;
        Py_XDECREF(pk);
        Py_XDECREF(pv);
        return r;
    });
}

// (q, k_pages, v_pages, block_table, kv_len, cu_rows, scale, k_scale, v_scale, max_q, max_kv, out) -> out
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&]() -> PyObject* {
        const at::Tensor& q = tensor(a[0], "q");
        if (q.dim() != 3) bad("q must be [T, n_heads, head_dim]");
        const at::Tensor* given = optional(a[11], "out");
        no_gradient({&q, given});
        const int64_t T = q.size(0), nh = q.size(1);
        Paged p = paged(T, tensor(a[1], "k_pages"), tensor(a[2], "v_pages"), tensor(a[3], "block_table"),
                        tensor(a[4], "kv_len"), tensor(a[5], "cu_rows"), optional(a[7], "k_scale"), optional(a[8], "v_scale"));
        const int64_t hd = p.kv.head_dim;
        const int64_t stride = rows(q, "q", p.dev, {T, nh, hd});
        double scale = 1.0 / std::sqrt((double)hd);
        if (a[6] != Py_None) {
            scale = PyFloat_AsDouble(a[6]);
            if (scale == -1.0 && PyErr_Occurred()) throw PythonError();
        }
        // a bound past 32 bits bounds nothing
        auto bound = [](PyObject* o, const char* what) {
            const int64_t v = o == Py_None ? 0 : integer(o);
            if (v < 0) bad(what);
            return (int)(v > INT_MAX ? 0 : v);
        };
        const int max_q = bound(a[9], "max_q must not be negative"), max_kv = bound(a[10], "max_kv must not be negative");
        const c10::cuda::CUDAGuard guard((c10::DeviceIndex)p.dev);
        const at::Tensor out = output(given, "out", p.dev, {T, nh, hd}, q);
        const int heads = to_int(nh, "a dimension does not fit in 32 bits");
        // scratch of this call alone, from the stream's allocator: calls on several streams, or in several graphs,
        // share none
        at::Tensor ws;
        const size_t need = af_paged_attention_workspace_bytes(&p.kv, &p.batch, heads, max_q, max_kv);
        if (need != 0) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
        const af_status st = af_paged_attention(&p.kv, &p.batch, pointer(q), stride, heads, (float)scale, max_q, max_kv,
                                                pointer(out), need != 0 ? ws.data_ptr() : nullptr, need,
                                                c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)p.dev).stream());
        if (st != AF_OK) return PyLong_FromLong(st);
        written({given});
        return THPVariable_Wrap(out);
    });
}

PyMethodDef methods[] = {
    {"paged_kv_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_kv_write)), METH_FASTCALL, nullptr},
    {"paged_kv_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_kv_read)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
