// The Python side of the packed-batch calls (sme_gemm_b200/paged.py): reads the tensors, checks them, and calls the C ABI on torch's current stream.
//
// A call has five to eight tensors, and in Python reading and checking them takes as long as a small call's kernel (5 us for a rotation of one row whose kernel
// takes 2); here it is a few hundred nanoseconds.  What is wrong raises AssertionError with the message that the Python layer would have.
// The entry points of libsmeg_b200.so are handed over by address (bind), so that this module links against torch alone.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>

#include "../../include/smeg_api.h"
#include "rows.h"

namespace {

typedef int (*RotateFn)(const smeg_rotate_args*, void*);
typedef int (*AttendFn)(const smeg_paged_attend_args*, void*);
typedef size_t (*WorkspaceFn)(size_t, size_t, size_t, size_t, size_t, size_t, size_t);
typedef int (*PackedFn)(const smeg_attn_packed_args*, void*);
typedef int (*ReadFn)(const smeg_paged_read_args*, void*);
RotateFn f_rotate, f_append;
AttendFn f_attend;
WorkspaceFn f_workspace;
PackedFn f_packed;
ReadFn f_read;

struct Refused {};                                 // a Python exception is set

[[noreturn]] void refuse(const char* what, const char* message) {
    PyErr_Format(PyExc_AssertionError, "%s%s", what, message);
    throw Refused();
}
void require(bool ok, const char* what, const char* message) {
    if (!ok) refuse(what, message);
}

struct Rows {                                      // what the row tensors of a call have in common
    at::ScalarType type;
    int device;
    int64_t rows;
    bool bf16() const { return type == at::kBFloat16; }
};
const at::Tensor& tensor(PyObject* x, const char* what, const char* message) {
    require(THPVariable_Check(x), what, message);
    const at::Tensor& t = THPVariable_Unpack(x);
    require(t.is_cuda(), what, message);
    return t;
}
Rows first_rows(PyObject* x, const char* what) {
    const at::Tensor& t = tensor(x, what, " is a CUDA tensor");
    require(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, what, " is f16 or bf16");
    require(t.dim() == 2, what, " has rows");
    return {t.scalar_type(), (int)t.get_device(), t.size(0)};
}
// A tensor of rows of `width` values like the others: its address, and the rows' stride in elements.
uint16_t* rows_of(PyObject* x, const char* what, int64_t width, const Rows& like, size_t* stride) {
    const at::Tensor& t = tensor(x, what, " is a CUDA tensor");
    require(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, what, " is f16 or bf16");
    if (t.dim() != 2 || t.size(1) != width) {
        PyErr_Format(PyExc_AssertionError, "%s has rows of %lld values", what, (long long)width);
        throw Refused();
    }
    require(t.scalar_type() == like.type && t.get_device() == like.device, what, " has the same type and device as the other rows");
    require(t.size(0) == like.rows, what, " has as many rows as the others");
    const int64_t s = t.stride(0), one = t.stride(1);
    require(like.rows == 0 || ((one == 1 || width == 1) && (like.rows == 1 || s >= width)), what, " has its rows' values side by side");
    *stride = (size_t)(s >= width ? s : width);
    return static_cast<uint16_t*>(t.data_ptr());
}
// An output of rows may be the input that it comes from (own), and shares no memory with the others.
void apart(const smeg::RowsAt& out, const smeg::RowsAt& in, const Rows& like, const char* what, const char* from, bool own) {
    if ((own && smeg::same_rows(out, in, (size_t)like.rows)) || !smeg::rows_share(out, in, (size_t)like.rows)) return;
    PyErr_Format(PyExc_AssertionError, own ? "%s is %s, or shares no memory with it" : "%s shares no memory with %s", what, from);
    throw Refused();
}
// q_out and k_out of a rotation or an append.
void turned_apart(const smeg_rotate_args& a, const Rows& like) {
    const size_t q_len = a.heads * a.head_dim, kv_len = a.kv_heads * a.head_dim;
    const smeg::RowsAt q = {a.q, a.q_stride, q_len}, k = {a.k, a.k_stride, kv_len}, v = {a.v, a.v_stride, kv_len}, qo = {a.q_out, a.q_out_stride, q_len}, ko = {a.k_out, a.k_out_stride, kv_len};
    apart(qo, q, like, "q_out", "q", true);
    apart(ko, k, like, "k_out", "k", true);
    apart(qo, k, like, "q_out", "k", false);
    apart(qo, v, like, "q_out", "v", false);
    apart(ko, q, like, "k_out", "q", false);
    apart(ko, v, like, "k_out", "v", false);
    apart(qo, ko, like, "q_out", "k_out", false);
}
const int32_t* ints(PyObject* x, const char* what, int device, int64_t* n) {
    const at::Tensor& t = tensor(x, what, " is a contiguous int32 CUDA tensor");
    require(t.scalar_type() == at::kInt && t.is_contiguous(), what, " is a contiguous int32 CUDA tensor");
    require(t.get_device() == device, what, " is on the rows' device");
    *n = t.numel();
    return static_cast<const int32_t*>(t.data_ptr());
}
const float* head_norm(PyObject* w, const char* what, int64_t head_dim, int device) {
    if (w == Py_None) return nullptr;
    const at::Tensor& t = tensor(w, what, " has weights on a CUDA device");
    require(t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == head_dim, what, " has head_dim weights");
    require(t.get_device() == device, what, " is on the rows' device");
    return static_cast<const float*>(t.data_ptr());
}
unsigned long long whole(PyObject* x) {
    PyObject* index = PyNumber_Index(x);            // (a numpy integer is one too)
    if (!index) throw Refused();
    const unsigned long long v = PyLong_AsUnsignedLongLong(index);
    Py_DECREF(index);
    if (v == (unsigned long long)-1 && PyErr_Occurred()) throw Refused();
    return v;
}
double number(PyObject* x) {
    const double v = PyFloat_AsDouble(x);
    if (v == -1.0 && PyErr_Occurred()) throw Refused();
    return v;
}
unsigned long long at(PyObject* tuple, int i) { return whole(PyTuple_GET_ITEM(tuple, i)); }
template <class T>
T* ptr_at(PyObject* tuple, int i) { return reinterpret_cast<T*>(at(tuple, i)); }

// (pages of a batch: cu_rows, starts, table, sequences, columns, device) and (a cache: codes, scales, pages, page, heads, KV heads, depths, device, scale)
void same_device(PyObject* batch, PyObject* cache, const Rows& like) {
    require((int)at(cache, 7) == like.device, "", "the rows are on the cache's device");
    require(at(batch, 5) == at(cache, 7), "", "the batch is on the cache's device");
}
// A rotation: None, or (addresses by device, rotated depths, interleaved, factor).  False: not on this device yet.
bool rotation(PyObject* r, smeg_rotate_args& a, int device) {
    a.factor = 1.0f;
    if (r == Py_None) return true;
    PyObject* key = PyLong_FromLong(device);
    if (!key) throw Refused();
    PyObject* on = PyDict_GetItemWithError(PyTuple_GET_ITEM(r, 0), key);
    Py_DECREF(key);
    if (!on) {
        if (PyErr_Occurred()) throw Refused();
        return false;
    }
    a.turns = ptr_at<const double>(on, 0);
    a.steps = ptr_at<const float>(on, 1);
    a.rot = at(r, 1);
    a.interleaved = PyTuple_GET_ITEM(r, 2) == Py_True;
    a.factor = (float)number(PyTuple_GET_ITEM(r, 3));
    return true;
}
constexpr long kNotThere = -1000;                  // the rotation is not on the device: make it, and call again

// A call's device and stream.
struct On {
    c10::cuda::CUDAGuard guard;
    c10::cuda::CUDAStream stream;
    explicit On(int device) : guard((c10::DeviceIndex)device), stream(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device)) {}
    void* raw() const { return (void*)stream.stream(); }
};

template <class F>
PyObject* guarded(F f) {
    try {
        return PyLong_FromLong(f());
    } catch (const Refused&) {
        return nullptr;
    } catch (...) {
        torch::translate_exception_to_python(std::current_exception());   // (out of memory as torch's own exception)
        return nullptr;
    }
}
bool counted(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd wanted", n, want);
    return false;
}

PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (!counted(n, 6)) return nullptr;
    return guarded([&]() -> long {
        f_rotate = reinterpret_cast<RotateFn>(whole(v[0]));
        f_append = reinterpret_cast<RotateFn>(whole(v[1]));
        f_attend = reinterpret_cast<AttendFn>(whole(v[2]));
        f_workspace = reinterpret_cast<WorkspaceFn>(whole(v[3]));
        f_packed = reinterpret_cast<PackedFn>(whole(v[4]));
        f_read = reinterpret_cast<ReadFn>(whole(v[5]));
        return 0;
    });
}

// q, k, positions, q_out, k_out, q_norm weights, eps, k_norm weights, eps, rotation, head_dim
PyObject* rotate(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (!counted(n, 11)) return nullptr;
    return guarded([&]() -> long {
        smeg_rotate_args a;
        std::memset(&a, 0, sizeof(a));
        const bool has_q = v[0] != Py_None, has_k = v[1] != Py_None;
        require(has_q || has_k, "", "there are queries or keys");
        require(has_q == (v[3] != Py_None), "", "q and q_out come together");
        require(has_k == (v[4] != Py_None), "", "k and k_out come together");
        const Rows like = first_rows(has_q ? v[0] : v[1], has_q ? "q" : "k");
        const int64_t hd = (int64_t)whole(v[10]);
        auto heads_of = [&](PyObject* x, const char* what) {
            first_rows(x, what);
            const int64_t width = THPVariable_Unpack(x).size(1);
            require(width > 0 && width % hd == 0, what, " has rows of whole heads");
            return width / hd;
        };
        if (has_q) {
            a.heads = (size_t)heads_of(v[0], "q");
            a.q = rows_of(v[0], "q", (int64_t)a.heads * hd, like, &a.q_stride);
            a.q_out = rows_of(v[3], "q_out", (int64_t)a.heads * hd, like, &a.q_out_stride);
        }
        if (has_k) {
            a.kv_heads = (size_t)heads_of(v[1], "k");
            a.k = rows_of(v[1], "k", (int64_t)a.kv_heads * hd, like, &a.k_stride);
            a.k_out = rows_of(v[4], "k_out", (int64_t)a.kv_heads * hd, like, &a.k_out_stride);
        }
        if (THPVariable_Check(v[2])) {
            int64_t count;
            a.positions = ints(v[2], "positions", like.device, &count);
            require(count == like.rows, "", "positions has one value a row");
        } else {
            PyObject* index = PyNumber_Index(v[2]);
            if (!index) throw Refused();
            a.start = PyLong_AsLongLong(index);
            Py_DECREF(index);
            if (a.start == -1 && PyErr_Occurred()) throw Refused();
        }
        if (!rotation(v[9], a, like.device)) return kNotThere;
        a.q_norm = head_norm(v[5], "q_norm", hd, like.device);
        a.q_eps = (float)number(v[6]);
        a.k_norm = head_norm(v[7], "k_norm", hd, like.device);
        a.k_eps = (float)number(v[8]);
        a.bf16 = like.bf16();
        a.rows = (size_t)like.rows;
        a.head_dim = (size_t)hd;
        turned_apart(a, like);
        if (like.rows == 0) return 0;
        On on(like.device);
        return f_rotate(&a, on.raw());
    });
}

// k, v, k_out, q, q_out, q_norm weights, eps, k_norm weights, eps, rotation, batch, cache
PyObject* append(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (!counted(n, 12)) return nullptr;
    return guarded([&]() -> long {
        smeg_rotate_args a;
        std::memset(&a, 0, sizeof(a));
        PyObject *batch = v[10], *cache = v[11];
        const Rows like = first_rows(v[0], "k");
        same_device(batch, cache, like);
        a.heads = at(cache, 4);
        a.kv_heads = at(cache, 5);
        a.head_dim = at(cache, 6);
        const int64_t row = (int64_t)(a.kv_heads * a.head_dim), q_len = (int64_t)(a.heads * a.head_dim);
        a.k = rows_of(v[0], "k", row, like, &a.k_stride);
        a.v = rows_of(v[1], "v", row, like, &a.v_stride);
        if (v[2] != Py_None) a.k_out = rows_of(v[2], "k_out", row, like, &a.k_out_stride);
        require((v[3] != Py_None) == (v[4] != Py_None), "", "q and q_out come together");
        if (v[3] != Py_None) {
            a.q = rows_of(v[3], "q", q_len, like, &a.q_stride);
            a.q_out = rows_of(v[4], "q_out", q_len, like, &a.q_out_stride);
        }
        if (!rotation(v[9], a, like.device)) return kNotThere;
        a.q_norm = head_norm(v[5], "q_norm", (int64_t)a.head_dim, like.device);
        a.q_eps = (float)number(v[6]);
        a.k_norm = head_norm(v[7], "k_norm", (int64_t)a.head_dim, like.device);
        a.k_eps = (float)number(v[8]);
        a.bf16 = like.bf16();
        a.rows = (size_t)like.rows;
        a.cu_rows = ptr_at<const int32_t>(batch, 0);
        a.starts = ptr_at<const int32_t>(batch, 1);
        a.table = ptr_at<const int32_t>(batch, 2);
        a.seqs = at(batch, 3);
        a.table_cols = at(batch, 4);
        a.codes = ptr_at<uint8_t>(cache, 0);
        a.scales = ptr_at<float>(cache, 1);
        a.pages = at(cache, 2);
        a.page = at(cache, 3);
        turned_apart(a, like);
        if (like.rows == 0 || a.seqs == 0) return 0;
        On on(like.device);
        return f_append(&a, on.raw());
    });
}

// q, out, batch, cache
PyObject* attend(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (!counted(n, 4)) return nullptr;
    return guarded([&]() -> long {
        smeg_paged_attend_args a;
        std::memset(&a, 0, sizeof(a));
        PyObject *batch = v[2], *cache = v[3];
        const Rows like = first_rows(v[0], "q");
        same_device(batch, cache, like);
        a.heads = at(cache, 4);
        a.kv_heads = at(cache, 5);
        a.head_dim = at(cache, 6);
        const int64_t width = (int64_t)(a.heads * a.head_dim);
        a.q = rows_of(v[0], "q", width, like, &a.q_stride);
        a.out = rows_of(v[1], "out", width, like, &a.out_stride);
        apart({a.out, a.out_stride, (size_t)width}, {a.q, a.q_stride, (size_t)width}, like, "out", "q", false);
        a.codes = ptr_at<const uint8_t>(cache, 0);
        a.scales = ptr_at<const float>(cache, 1);
        a.pages = at(cache, 2);
        a.page = at(cache, 3);
        a.scale = (float)number(PyTuple_GET_ITEM(cache, 8));
        a.cu_rows = ptr_at<const int32_t>(batch, 0);
        a.starts = ptr_at<const int32_t>(batch, 1);
        a.table = ptr_at<const int32_t>(batch, 2);
        a.seqs = at(batch, 3);
        a.table_cols = at(batch, 4);
        a.rows = (size_t)like.rows;
        a.bf16 = like.bf16();
        if (like.rows == 0 || a.seqs == 0) return 0;
        On on(like.device);
        a.workspace_bytes = f_workspace(a.rows, a.seqs, a.table_cols, a.page, a.heads, a.kv_heads, a.head_dim);
        // the call's own memory, from the stream's pool of torch's allocator: two streams, or two captured graphs, never share it
        if (a.workspace_bytes) a.workspace = c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(a.workspace_bytes, on.stream.stream());
        const int rc = f_attend(&a, on.raw());
        if (a.workspace) c10::cuda::CUDACachingAllocator::raw_delete(a.workspace);
        return rc;
    });
}

// ids, out, cache
PyObject* read_pages(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (!counted(n, 3)) return nullptr;
    return guarded([&]() -> long {
        smeg_paged_read_args a;
        std::memset(&a, 0, sizeof(a));
        PyObject* cache = v[2];
        const int device = (int)at(cache, 7);
        int64_t count;
        a.ids = ints(v[0], "ids", device, &count);
        const at::Tensor& out = tensor(v[1], "out", " is contiguous f16 or bf16");
        require(out.get_device() == device && (out.scalar_type() == at::kHalf || out.scalar_type() == at::kBFloat16) && out.is_contiguous(), "out", " is contiguous f16 or bf16");
        a.pages = at(cache, 2);
        a.page = at(cache, 3);
        a.kv_heads = at(cache, 5);
        a.head_dim = at(cache, 6);
        require(out.numel() == count * (int64_t)(a.kv_heads * 2 * a.page * a.head_dim), "out", " holds n pages");
        a.out = static_cast<uint16_t*>(out.data_ptr());
        a.codes = ptr_at<const uint8_t>(cache, 0);
        a.scales = ptr_at<const float>(cache, 1);
        a.n = (size_t)count;
        a.bf16 = out.scalar_type() == at::kBFloat16;
        if (count == 0) return 0;
        On on(device);
        return f_read(&a, on.raw());
    });
}

// q, k, v, cu_rows, out, heads, KV heads, scale (None: 1 / sqrt(head_dim))
PyObject* packed(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (!counted(n, 8)) return nullptr;
    return guarded([&]() -> long {
        smeg_attn_packed_args a;
        std::memset(&a, 0, sizeof(a));
        const Rows like = first_rows(v[0], "q");
        a.heads = whole(v[5]);
        a.kv_heads = whole(v[6]);
        const int64_t width = THPVariable_Unpack(v[0]).size(1), hd = width / (int64_t)a.heads;
        require(hd * (int64_t)a.heads == width, "q", " has rows of heads * head_dim values");
        require(hd % 8 == 0 && hd >= 8 && hd <= 256, "", "head_dim must be a multiple of 8 in 8..=256");
        a.head_dim = (size_t)hd;
        const int64_t row = (int64_t)a.kv_heads * hd;
        a.q = rows_of(v[0], "q", width, like, &a.q_stride);
        a.k = rows_of(v[1], "k", row, like, &a.k_stride);
        a.v = rows_of(v[2], "v", row, like, &a.v_stride);
        a.out = rows_of(v[4], "out", width, like, &a.out_stride);
        const smeg::RowsAt out = {a.out, a.out_stride, (size_t)width};
        for (const smeg::RowsAt& in : {smeg::RowsAt{a.q, a.q_stride, (size_t)width}, smeg::RowsAt{a.k, a.k_stride, (size_t)row}, smeg::RowsAt{a.v, a.v_stride, (size_t)row}})
            require(!smeg::rows_share(out, in, (size_t)like.rows), "out", " is none of the inputs, and shares no memory with them");
        int64_t count;
        a.cu_rows = ints(v[3], "cu_rows", like.device, &count);
        require(count >= 1, "", "cu_rows has one value more than there are sequences");
        a.seqs = (size_t)(count - 1);
        a.rows = (size_t)like.rows;
        a.scale = v[7] == Py_None ? 1.0f / std::sqrt((float)hd) : (float)number(v[7]);
        a.bf16 = like.bf16();
        if (like.rows == 0 || a.seqs == 0) return 0;
        On on(like.device);
        return f_packed(&a, on.raw());
    });
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, "The addresses of the library's entry points."},
    {"rotate", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotate)), METH_FASTCALL, "smeg_rotate_heads_dev on tensors."},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, "smeg_paged_append_dev on tensors."},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, "smeg_paged_attend_dev on tensors."},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(read_pages)), METH_FASTCALL, "smeg_paged_read_dev on tensors."},
    {"packed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(packed)), METH_FASTCALL, "smeg_attn_packed_dev on tensors."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "Packed-batch calls on torch tensors.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
