// The Python side of piton_b200.decode's calls: checks of the arguments, outputs from torch's allocator and the
// C entry points' argument structs, which in Python took longer than the kernels of a decode step (a call of
// kv_append 17 us, of which the launch 4).  Nothing is kept from one call to the next.
//
// Each function returns the result, or None where an argument is not what it has to be (piton_b200.decode then
// says which), or the entry point's status code where that is not 0.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "piton_b200.h"

namespace {

int (*append_entry)(const piton_kv_append_args *, void *);
int (*attention_entry)(const piton_kv_attention_args *, void *);
size_t (*attention_workspace)(const piton_kv_attention_args *);
int (*matvec_entry)(const piton_matvec_w4_args *, void *);
size_t (*matvec_workspace)(const piton_matvec_w4_args *);
PyObject *out_of_memory;      // torch.OutOfMemoryError

const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
uint64_t address(const at::Tensor &t) { return reinterpret_cast<uint64_t>(t.data_ptr()); }
bool is_a(const at::Tensor *t, at::ScalarType type, int device, int64_t dim) {
    return t && t->scalar_type() == type && t->is_cuda() && t->get_device() == device && t->dim() == dim;
}
int type_of(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PITON_B200_TYPE_F32;
        case at::kHalf: return PITON_B200_TYPE_F16;
        case at::kBFloat16: return PITON_B200_TYPE_BF16;
        default: return -1;
    }
}

// Whether an output would have to carry a gradient, which these operators have none of.
template <typename... T> bool wants_gradient(const T *...t) { return c10::GradMode::is_enabled() && (... || (t && t->requires_grad())); }

// The four tensors of a cache, of `device`.
struct Cache {
    const at::Tensor *t[4];
    int64_t pages, heads, page, dim;
    bool take(PyObject *o, int device) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
        for (int i = 0; i < 4; ++i)
            if (!(t[i] = tensor(PyTuple_GET_ITEM(o, i))) || !t[i]->is_cuda() || t[i]->get_device() != device || !t[i]->is_contiguous())
                return false;
        for (int i = 0; i < 2; ++i)
            if ((t[i]->scalar_type() != at::kFloat8_e4m3fn && t[i]->scalar_type() != at::kByte) || t[i]->dim() != 4 ||
                t[i]->sizes() != t[0]->sizes() || t[2 + i]->scalar_type() != at::kFloat || t[2 + i]->sizes() != t[0]->sizes().slice(0, 2))
                return false;
        pages = t[0]->size(0), heads = t[0]->size(1), page = t[0]->size(2), dim = t[0]->size(3);
        return true;
    }
};

// The page table, the int32 vector of the sequences and the offsets (None: the same number of tokens each).
struct Sequences {
    const at::Tensor *table, *vector, *cu;
    int64_t batch;
    bool take(PyObject *table_o, PyObject *vector_o, PyObject *cu_o, int64_t tokens, int device) {
        table = tensor(table_o), vector = tensor(vector_o), cu = cu_o == Py_None ? nullptr : tensor(cu_o);
        if (!is_a(table, at::kInt, device, 2) || (table->size(1) > 1 && table->stride(1) != 1)) return false;
        batch = table->size(0);
        if (!is_a(vector, at::kInt, device, 1) || vector->size(0) != batch || !vector->is_contiguous()) return false;
        if (cu_o == Py_None) return batch ? tokens % batch == 0 : tokens == 0;
        return is_a(cu, at::kInt, device, 1) && cu->size(0) == batch + 1 && cu->is_contiguous();
    }
};

// Whether t is [tokens, heads, dim] (heads < 0: any number) of this type with unit stride along dim.
bool rows(const at::Tensor *t, at::ScalarType type, int device, int64_t tokens, int64_t heads, int64_t dim) {
    return is_a(t, type, device, 3) && t->size(0) == tokens && (heads < 0 || t->size(1) == heads) && t->size(2) == dim && t->stride(2) == 1;
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like) {
    return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

// Makes `device` current while it lives: a workspace's size and the launch that checks it are made of the same device's SM count.
struct On {
    c10::cuda::OptionalCUDAGuard guard;
    explicit On(int device) {
        if (c10::cuda::current_device() != device) guard.set_index((c10::DeviceIndex)device);
    }
};

// Runs an entry point on the current stream of `device`; its status.
template <typename Entry, typename Args> int enter(Entry entry, const Args &a, int device) {
    return entry(&a, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream());
}

PyObject *wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

// C++ exceptions (an allocation that fails, say) become Python's.
template <typename F> PyObject *guarded(F f) {
    try {
        return f();
    } catch (const c10::OutOfMemoryError &e) {
        PyErr_SetString(out_of_memory, e.what_without_backtrace());
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// kv_append(k, v, cache, table, starts, cu, cos, sin, interleaved, q)
PyObject *kv_append(PyObject *, PyObject *const *o, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 10) Py_RETURN_NONE;
        const at::Tensor *k = tensor(o[0]), *v = tensor(o[1]), *cos = nullptr, *sin = nullptr, *q = nullptr;
        if (!k || !k->is_cuda() || k->dim() != 3 || type_of(*k) < 0) Py_RETURN_NONE;
        const int device = k->get_device();
        const at::ScalarType type = k->scalar_type();
        const int64_t tokens = k->size(0);
        Cache c;
        Sequences s;
        if (!c.take(o[2], device) || !rows(k, type, device, tokens, c.heads, c.dim) || !rows(v, type, device, tokens, c.heads, c.dim) ||
            !s.take(o[3], o[4], o[5], tokens, device))
            Py_RETURN_NONE;
        if (o[6] != Py_None || o[7] != Py_None) {
            cos = tensor(o[6]), sin = tensor(o[7]);
            if (!is_a(cos, at::kFloat, device, 2) || !is_a(sin, at::kFloat, device, 2) || cos->sizes() != sin->sizes() ||
                2 * cos->size(1) > c.dim || !cos->is_contiguous() || !sin->is_contiguous())
                Py_RETURN_NONE;
        }
        if (o[9] != Py_None && !rows(q = tensor(o[9]), type, device, tokens, -1, c.dim)) Py_RETURN_NONE;
        if (wants_gradient(k, v, q, cos, sin, c.t[2], c.t[3])) Py_RETURN_NONE;
        const On on(device);
        const int interleaved = PyObject_IsTrue(o[8]);
        if (interleaved < 0) return nullptr;
        at::Tensor out, lengths = empty({s.batch}, at::kInt, *k);
        piton_kv_append_args a = {};
        a.k = address(*k), a.v = address(*v);
        if (q) {
            out = empty(q->sizes(), type, *k);
            a.q = address(*q), a.q_out = address(out), a.q_heads = q->size(1);
            a.stride_qt = q->stride(0), a.stride_qh = q->stride(1), a.stride_ot = a.q_heads * c.dim, a.stride_oh = c.dim;
        }
        a.k_codes = address(*c.t[0]), a.v_codes = address(*c.t[1]), a.k_scale = address(*c.t[2]), a.v_scale = address(*c.t[3]);
        a.table = address(*s.table), a.starts = address(*s.vector), a.cu = s.cu ? address(*s.cu) : 0, a.lengths = address(lengths);
        if (cos) a.cos_table = address(*cos), a.sin_table = address(*sin), a.rot_dim = 2 * cos->size(1), a.rope_len = cos->size(0);
        a.batch = s.batch, a.tokens = tokens, a.kv_heads = c.heads, a.head_dim = c.dim, a.page_size = c.page, a.num_pages = c.pages;
        a.table_width = s.table->size(1), a.table_stride = s.table->stride(0);
        a.stride_kt = k->stride(0), a.stride_kh = k->stride(1), a.stride_vt = v->stride(0), a.stride_vh = v->stride(1);
        a.type = type_of(*k), a.interleaved = interleaved;
        if (const int rc = enter(append_entry, a, device)) return PyLong_FromLong(rc);
        PyObject *first = q ? wrap(std::move(out)) : Py_NewRef(Py_None), *second = wrap(std::move(lengths));
        PyObject *both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
        Py_XDECREF(first);
        Py_XDECREF(second);
        return both;
    });
}

// kv_attention(q, cache, table, lengths, cu, scale, window, max_length, max_new, return_lse)
PyObject *kv_attention(PyObject *, PyObject *const *o, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 10) Py_RETURN_NONE;
        const at::Tensor *q = tensor(o[0]);
        if (!q || !q->is_cuda() || q->dim() != 3 || type_of(*q) < 0) Py_RETURN_NONE;
        const int device = q->get_device();
        Cache c;
        Sequences s;
        if (!c.take(o[1], device) || !rows(q, q->scalar_type(), device, q->size(0), -1, c.dim) ||
            !s.take(o[2], o[3], o[4], q->size(0), device) || wants_gradient(q, c.t[2], c.t[3]))
            Py_RETURN_NONE;
        const On on(device);
        piton_kv_attention_args a = {};
        a.sm_scale = o[5] == Py_None ? 1.0 / std::sqrt((double)c.dim) : PyFloat_AsDouble(o[5]);
        a.window = PyLong_AsLongLong(o[6]), a.max_length = PyLong_AsLongLong(o[7]), a.max_new = PyLong_AsLongLong(o[8]);
        const int with_lse = PyObject_IsTrue(o[9]);
        if (PyErr_Occurred()) return nullptr;
        if (a.window < 0 || a.max_length < 0 || a.max_new < 0) Py_RETURN_NONE;
        a.tokens = q->size(0), a.q_heads = q->size(1);
        at::Tensor out = empty(q->sizes(), q->scalar_type(), *q), lse, scratch;
        if (with_lse) lse = empty({a.tokens, a.q_heads}, at::kFloat, *q);
        a.q = address(*q), a.out = address(out), a.lse = with_lse ? address(lse) : 0;
        a.k_codes = address(*c.t[0]), a.v_codes = address(*c.t[1]), a.k_scale = address(*c.t[2]), a.v_scale = address(*c.t[3]);
        a.table = address(*s.table), a.lengths = address(*s.vector), a.cu = s.cu ? address(*s.cu) : 0;
        a.batch = s.batch, a.kv_heads = c.heads, a.head_dim = c.dim, a.page_size = c.page, a.num_pages = c.pages;
        a.table_width = s.table->size(1), a.table_stride = s.table->stride(0);
        a.stride_qt = q->stride(0), a.stride_qh = q->stride(1), a.stride_ot = a.q_heads * c.dim, a.stride_oh = c.dim;
        a.type = type_of(*q);
        if (const size_t need = attention_workspace(&a)) {      // of this call's stream, so calls never share it
            scratch = empty({(int64_t)need}, at::kByte, *q);
            a.workspace = address(scratch), a.workspace_bytes = need;
        }
        if (const int rc = enter(attention_entry, a, device)) return PyLong_FromLong(rc);
        if (!with_lse) return wrap(std::move(out));
        PyObject *first = wrap(std::move(out)), *second = wrap(std::move(lse));
        PyObject *both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
        Py_XDECREF(first);
        Py_XDECREF(second);
        return both;
    });
}

// matvec_w4(x, codes, scales, group, zeros, bias)
PyObject *matvec_w4(PyObject *, PyObject *const *o, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 6) Py_RETURN_NONE;
        const at::Tensor *x = tensor(o[0]), *codes = tensor(o[1]), *scales = tensor(o[2]), *zeros = nullptr, *bias = nullptr;
        if (!x || !x->is_cuda() || (x->dim() != 1 && x->dim() != 2) || type_of(*x) < 0) Py_RETURN_NONE;
        const int device = x->get_device();
        const int64_t group = PyLong_AsLongLong(o[3]);
        if (PyErr_Occurred()) return nullptr;
        if (group != 32 && group != 64 && group != 128) Py_RETURN_NONE;
        const bool flat = x->dim() == 1;
        const int64_t inner = x->size(-1), groups = (inner + group - 1) / group;
        auto lines = [](const at::Tensor &t) { return t.size(1) <= 1 || t.stride(1) == 1; };
        if ((inner > 1 && x->stride(-1) != 1) || !is_a(codes, at::kByte, device, 2) || codes->size(1) != (inner + 1) / 2 || !lines(*codes))
            Py_RETURN_NONE;
        const int64_t outer = codes->size(0);
        auto by_group = [&](const at::Tensor *t) { return t->size(0) == outer && t->size(1) == groups && lines(*t); };
        if (!scales || type_of(*scales) < 0 || !is_a(scales, scales->scalar_type(), device, 2) || !by_group(scales)) Py_RETURN_NONE;
        if (o[4] != Py_None && (!is_a(zeros = tensor(o[4]), at::kByte, device, 2) || !by_group(zeros))) Py_RETURN_NONE;
        if (o[5] != Py_None && (!is_a(bias = tensor(o[5]), x->scalar_type(), device, 1) || bias->size(0) != outer ||
                                (outer > 1 && bias->stride(0) != 1)))
            Py_RETURN_NONE;
        if (wants_gradient(x, scales, bias)) Py_RETURN_NONE;
        const On on(device);
        piton_matvec_w4_args a = {};
        a.rows = flat ? 1 : x->size(0), a.inner = inner, a.outer = outer;
        at::Tensor y = flat ? empty({outer}, x->scalar_type(), *x) : empty({a.rows, outer}, x->scalar_type(), *x);
        a.x = address(*x), a.codes = address(*codes), a.scales = address(*scales), a.zeros = zeros ? address(*zeros) : 0;
        a.bias = bias ? address(*bias) : 0, a.y = address(y);
        a.stride_x = flat ? 0 : x->stride(0), a.stride_codes = codes->stride(0), a.stride_scales = scales->stride(0);
        a.stride_zeros = zeros ? zeros->stride(0) : 0, a.stride_y = outer;
        a.group = (int32_t)group, a.type = type_of(*x), a.scale_type = type_of(*scales);
        at::Tensor scratch;
        if (const size_t need = matvec_workspace(&a)) {
            scratch = empty({(int64_t)need}, at::kByte, *x);
            a.workspace = address(scratch), a.workspace_bytes = need;
        }
        if (const int rc = enter(matvec_entry, a, device)) return PyLong_FromLong(rc);
        return wrap(std::move(y));
    });
}

// bind(addresses of the entry points in the library that the package has loaded, in the order below, torch.OutOfMemoryError).
PyObject *bind(PyObject *, PyObject *args) {
    unsigned long long f[5];
    PyObject *oom;
    if (!PyArg_ParseTuple(args, "KKKKKO", &f[0], &f[1], &f[2], &f[3], &f[4], &oom)) return nullptr;
    Py_XSETREF(out_of_memory, Py_NewRef(oom));
    append_entry = reinterpret_cast<decltype(append_entry)>(f[0]);
    attention_entry = reinterpret_cast<decltype(attention_entry)>(f[1]);
    attention_workspace = reinterpret_cast<decltype(attention_workspace)>(f[2]);
    matvec_workspace = reinterpret_cast<decltype(matvec_workspace)>(f[3]);
    matvec_entry = reinterpret_cast<decltype(matvec_entry)>(f[4]);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"kv_append", (PyCFunction)(void *)kv_append, METH_FASTCALL, nullptr},
    {"kv_attention", (PyCFunction)(void *)kv_attention, METH_FASTCALL, nullptr},
    {"matvec_w4", (PyCFunction)(void *)matvec_w4, METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__decode_calls() { return PyModule_Create(&module); }
