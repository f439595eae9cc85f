// paged_torch.cpp -- neurons_b200._paged: the paged cache's calls with torch
// tensors, as a CPython module over the C ABI (nq_paged_*, nq_pages_*).
//
// A decode step makes these calls once per layer or step with microseconds of
// GPU work each.  Reading a tensor's properties one by one from Python and
// passing them through ctypes takes 5 to 10 us a call; here the same checks, the
// outputs and the workspace take about 2.  The functions take their arguments
// by position and are wrapped, with their documentation, in paged.py.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "nq.h"

namespace {

// A refused argument; becomes NQError(InvalidInput).
struct Refused {
    std::string why;
};

[[noreturn]] void refuse(const std::string &why) { throw Refused{why}; }

PyObject *raise(int status, const std::string &message) {
    static PyObject *error = nullptr;  // (kept for the process; the GIL is held)
    if (!error) {
        PyObject *m = PyImport_ImportModule("neurons_b200._lib");
        if (!m) return nullptr;
        error = PyObject_GetAttrString(m, "NQError");
        Py_DECREF(m);
        if (!error) return nullptr;
    }
    if (PyObject *args = Py_BuildValue("(is)", status, message.c_str())) {
        PyErr_SetObject(error, args);
        Py_DECREF(args);
    }
    return nullptr;
}

const at::Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

int cuda_device(const at::Tensor &t) { return t.is_cuda() ? t.get_device() : -1; }

int64_t integer(PyObject *o, const char *name) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(std::string(name) + " must be an integer");
    }
    return v;
}

// An int32 vector on `device`, of n entries when n >= 0.
const int32_t *index(PyObject *o, const char *name, int device, int64_t n = -1) {
    const at::Tensor &t = tensor(o, name);
    if (t.scalar_type() != at::kInt || cuda_device(t) != device || t.dim() != 1 || !t.is_contiguous())
        refuse(std::string(name) + " must be a contiguous int32 vector on the cache's device");
    if (n >= 0 && t.size(0) != n)
        refuse(std::string(name) + " must have " + std::to_string(n) + " entries");
    return static_cast<const int32_t *>(t.data_ptr());
}

struct Table {
    int32_t *data;
    int64_t rows, width, ld;
};
Table table_of(PyObject *o, int device) {
    const at::Tensor &t = tensor(o, "table");
    if (t.scalar_type() != at::kInt || cuda_device(t) != device || t.dim() != 2)
        refuse("table must be an int32 matrix on the cache's device");
    if (t.stride(1) != 1 && t.size(1) > 1)
        refuse("the entries of a table row must lie one after another");
    return Table{static_cast<int32_t *>(t.data_ptr()), t.size(0), t.size(1),
                 t.size(0) > 1 ? t.stride(0) : t.size(1)};
}

// Rows [tokens, heads, dim] whose heads lie one after another.
struct Rows {
    uint16_t *data;
    int64_t tokens, heads, ld;
};
Rows rows_of(PyObject *o, const char *name, int64_t heads, int64_t dim, at::ScalarType dtype,
             int device) {
    const at::Tensor &t = tensor(o, name);
    if (t.scalar_type() != dtype || cuda_device(t) != device || t.dim() != 3)
        refuse(std::string(name) +
               " must be [tokens, heads, head dim], of the cache's type and on its device");
    if (t.size(2) != dim || (heads >= 0 && t.size(1) != heads))
        refuse(std::string(name) + ": wrong number of heads or head dim");
    if (t.stride(2) != 1 || (t.size(1) > 1 && t.stride(1) != dim))
        refuse(std::string(name) + ": the heads of a token must lie one after another");
    return Rows{static_cast<uint16_t *>(t.data_ptr()), t.size(0), t.size(1),
                t.size(0) > 1 ? t.stride(0) : t.size(1) * dim};
}

struct Cache {
    nq_paged_cache_t c;
    at::ScalarType dtype;
    int device;
};
Cache cache_of(PyObject *ko, PyObject *vo) {
    const at::Tensor &k = tensor(ko, "k_pages"), &v = tensor(vo, "v_pages");
    const at::ScalarType dtype = k.scalar_type();
    const int device = cuda_device(k);
    if ((dtype != at::kBFloat16 && dtype != at::kHalf) || k.dim() != 4 || device < 0)
        refuse("k_pages must be a bf16 or fp16 CUDA tensor [pages, kv heads, page size, head dim]");
    if (v.scalar_type() != dtype || cuda_device(v) != device || v.sizes() != k.sizes() ||
        v.strides() != k.strides())
        refuse("v_pages must match k_pages in type, shape, strides and device");
    const int64_t n = k.size(0), heads = k.size(1), size = k.size(2), dim = k.size(3);
    if (k.numel() > 0 && (k.stride(3) != 1 || k.stride(2) != dim ||
                          (heads > 1 && k.stride(1) != size * dim)))
        refuse("a page must be contiguous");
    if (heads > INT32_MAX || size > INT32_MAX || dim > INT32_MAX) refuse("a size is too large");
    if (device != c10::cuda::current_device()) refuse("the cache is not on the current device");
    return Cache{{k.data_ptr(), v.data_ptr(), n, n > 1 ? k.stride(0) : heads * size * dim, (int)heads,
                  (int)size, (int)dim, dtype == at::kHalf ? NQ_DTYPE_F16 : NQ_DTYPE_BF16},
                 dtype,
                 device};
}

nq_paged_batch_t batch_of(PyObject *table, PyObject *lens, PyObject *seqs, PyObject *starts,
                          int64_t tokens, int device) {
    const Table t = table_of(table, device);
    nq_paged_batch_t b{};
    b.table = t.data;
    b.table_ld = t.ld;
    b.table_width = t.width;
    b.n_rows = t.rows;
    b.kv_lens = index(lens, "kv_lens", device, t.rows);
    b.n_tokens = tokens;
    if (seqs != Py_None) {
        b.seqs = index(seqs, "seqs", device);
        b.n_seqs = THPVariable_Unpack(seqs).size(0);
        if (starts != Py_None) b.q_starts = index(starts, "q_starts", device, b.n_seqs + 1);
    } else if (starts != Py_None) {
        b.q_starts = index(starts, "q_starts", device);
        b.n_seqs = THPVariable_Unpack(starts).size(0) - 1;
    } else {
        b.n_seqs = std::min(t.rows, tokens);
    }
    return b;
}

// The caller's workspace, or a new one of `need` bytes.
struct Workspace {
    at::Tensor keep;
    void *data = nullptr;
    size_t bytes = 0;
    Workspace(PyObject *o, size_t need, int device) {
        if (o != Py_None) {
            const at::Tensor &t = tensor(o, "workspace");
            if (cuda_device(t) != device || !t.is_contiguous())
                refuse("workspace must be contiguous, on the cache's device");
            data = t.data_ptr();
            bytes = t.numel() * t.element_size();
        } else if (need > 0) {
            keep = at::empty({(int64_t)need},
                             at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
            data = keep.data_ptr();
            bytes = need;
        }
    }
};

void *stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

// Runs a call's body, its refusals and exceptions as Python ones.
template <typename F>
PyObject *guarded(Py_ssize_t got, Py_ssize_t want, const char *name, F &&body) {
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
        return nullptr;
    }
    try {
        return body();
    } catch (const Refused &r) {
        return raise(NQ_INVALID_INPUT, r.why);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}

PyObject *done(int rc) {
    if (rc) return raise(rc, nq_last_error());
    Py_RETURN_NONE;
}

// q, k_pages, v_pages, table, kv_lens, q_starts, max_q, window, scale, seqs, out, workspace
PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 12, "attention", [&]() -> PyObject * {
        const Cache c = cache_of(a[1], a[2]);
        const int64_t dim = c.c.head_dim;
        const Rows q = rows_of(a[0], "q", -1, dim, c.dtype, c.device);
        const nq_paged_batch_t b = batch_of(a[3], a[4], a[9], a[5], q.tokens, c.device);
        int64_t max_q = a[6] == Py_None ? 0 : integer(a[6], "max_q");
        if (a[5] == Py_None) max_q = 1;
        if (max_q == 0) max_q = q.tokens;
        const int64_t window = integer(a[7], "window");
        double scale = 1.0 / std::sqrt((double)dim);
        if (a[8] != Py_None) {
            scale = PyFloat_AsDouble(a[8]);
            if (PyErr_Occurred()) return nullptr;
        }
        at::Tensor fresh;
        Rows out;
        if (a[10] == Py_None) {
            fresh = at::empty({q.tokens, q.heads, dim},
                              at::TensorOptions().dtype(c.dtype).device(at::kCUDA, c.device));
            out = Rows{static_cast<uint16_t *>(fresh.data_ptr()), q.tokens, q.heads, q.heads * dim};
        } else {
            out = rows_of(a[10], "out", q.heads, dim, c.dtype, c.device);
            if (out.tokens != q.tokens) refuse("out must have q's shape");
        }
        if (q.heads > INT32_MAX) refuse("a size is too large");
        const Workspace ws(a[11],
                           nq_paged_attention_workspace_size((int)q.heads, c.c.n_kv_heads, (int)dim,
                                                             max_q, b.table_width * c.c.page_size),
                           c.device);
        const int rc = nq_paged_attention(q.data, q.ld, (int)q.heads, &c.c, &b, max_q, (float)scale,
                                          window, ws.data, ws.bytes, out.data, out.ld,
                                          stream_of(c.device));
        if (rc) return raise(rc, nq_last_error());
        if (a[10] == Py_None) return THPVariable_Wrap(std::move(fresh));
        Py_INCREF(a[10]);
        return a[10];
    });
}

// q, k, v, k_pages, v_pages, table, kv_lens, q_starts, freqs, seqs, q_out
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 11, "append", [&]() -> PyObject * {
        const Cache c = cache_of(a[3], a[4]);
        const int64_t dim = c.c.head_dim;
        const Rows q = rows_of(a[0], "q", -1, dim, c.dtype, c.device);
        const Rows k = rows_of(a[1], "k", c.c.n_kv_heads, dim, c.dtype, c.device);
        const Rows v = rows_of(a[2], "v", c.c.n_kv_heads, dim, c.dtype, c.device);
        if (k.tokens != q.tokens || v.tokens != q.tokens) refuse("q, k and v differ in tokens");
        const nq_paged_batch_t b = batch_of(a[5], a[6], a[9], a[7], q.tokens, c.device);
        const float *freqs = nullptr;
        int64_t nf = 0;
        if (a[8] != Py_None) {
            const at::Tensor &f = tensor(a[8], "freqs");
            if (f.scalar_type() != at::kFloat || f.dim() != 1 || cuda_device(f) != c.device ||
                !f.is_contiguous() || f.size(0) > INT32_MAX)
                refuse("freqs must be a contiguous fp32 vector on the cache's device");
            freqs = static_cast<const float *>(f.data_ptr());
            nf = f.size(0);
        }
        at::Tensor fresh;
        Rows out;
        if (a[10] == Py_None) {
            fresh = at::empty({q.tokens, q.heads, dim},
                              at::TensorOptions().dtype(c.dtype).device(at::kCUDA, c.device));
            out = Rows{static_cast<uint16_t *>(fresh.data_ptr()), q.tokens, q.heads, q.heads * dim};
        } else {
            out = rows_of(a[10], "q_out", q.heads, dim, c.dtype, c.device);
            if (out.tokens != q.tokens) refuse("q_out must have q's shape");
        }
        if (q.heads > INT32_MAX) refuse("a size is too large");
        const int rc = nq_paged_append(q.data, q.ld, k.data, k.ld, v.data, v.ld, (int)q.heads, &c.c,
                                       &b, freqs, (int)nf, out.data, out.ld, stream_of(c.device));
        if (rc) return raise(rc, nq_last_error());
        if (a[10] == Py_None) return THPVariable_Wrap(std::move(fresh));
        Py_INCREF(a[10]);
        return a[10];
    });
}

// refs, table and lens (None: not used) as the C ABI's page table
struct Pages {
    nq_page_table_t t;
    int device;
};
Pages pages_of(PyObject *refs, PyObject *table, PyObject *lens, int64_t page_size) {
    const at::Tensor &r = tensor(refs, "refs");
    const int device = cuda_device(r);
    if (device < 0 || device != c10::cuda::current_device())
        refuse("refs must be a CUDA tensor on the current device");
    index(refs, "refs", device);
    const Table t = table_of(table, device);
    int32_t *ref = static_cast<int32_t *>(r.data_ptr());
    if (page_size > INT32_MAX) refuse("a size is too large");
    return Pages{{ref, t.data,
                  lens == Py_None ? ref
                                  : const_cast<int32_t *>(index(lens, "lens", device, t.rows)),
                  r.size(0), t.rows, t.ld, t.width, (int)page_size},
                 device};
}

nq_page_pool_t pool_of(PyObject *o, int device) {
    const at::Tensor &p = tensor(o, "pool");
    if (cuda_device(p) != device || p.dim() < 4 || !p.is_contiguous())
        refuse("pool must be a contiguous CUDA tensor [..., pages, kv heads, page size, head dim] "
               "on the current device");
    if (p.numel() == 0) refuse("the pool is empty");
    const int64_t pages = p.size(-4), page = p.size(-3) * p.size(-2) * p.size(-1);
    return nq_page_pool_t{p.data_ptr(), p.numel() / (pages * page), pages, page * p.element_size()};
}

int64_t page_size_of(PyObject *pool) {
    const at::Tensor &p = tensor(pool, "pool");
    return p.dim() < 4 ? 0 : p.size(-2);
}

// refs, table, lens, seqs
PyObject *free_(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 4, "free", [&] {
        const Pages p = pages_of(a[0], a[1], a[2], 1);
        const int32_t *seqs = index(a[3], "seqs", p.device);
        return done(nq_pages_free(&p.t, seqs, THPVariable_Unpack(a[3]).size(0), stream_of(p.device)));
    });
}

// refs, table, lens, parents, children
PyObject *fork_(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 5, "fork", [&] {
        const Pages p = pages_of(a[0], a[1], a[2], 1);
        const int32_t *parents = index(a[3], "parents", p.device);
        const int64_t count = THPVariable_Unpack(a[3]).size(0);
        const int32_t *children = index(a[4], "children", p.device, count);
        return done(nq_pages_fork(&p.t, parents, children, count, stream_of(p.device)));
    });
}

// pool, refs, table, lens, seqs, new_lens, workspace
PyObject *reserve(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 7, "reserve", [&] {
        const Pages p = pages_of(a[1], a[2], a[3], page_size_of(a[0]));
        const nq_page_pool_t pool = pool_of(a[0], p.device);
        const int32_t *seqs = index(a[4], "seqs", p.device);
        const int64_t count = THPVariable_Unpack(a[4]).size(0);
        const int32_t *lens = index(a[5], "new_lens", p.device, count);
        const Workspace ws(a[6], nq_pages_workspace_size(0, count), p.device);
        return done(nq_pages_reserve(&p.t, &pool, seqs, lens, count, ws.data, ws.bytes,
                                     stream_of(p.device)));
    });
}

// pool, refs, table, workspace
PyObject *compact(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 4, "compact", [&] {
        const Pages p = pages_of(a[1], a[2], Py_None, page_size_of(a[0]));
        const nq_page_pool_t pool = pool_of(a[0], p.device);
        const Workspace ws(a[3], nq_pages_workspace_size(p.t.n_pages, 0), p.device);
        return done(nq_pages_compact(&p.t, &pool, ws.data, ws.bytes, stream_of(p.device)));
    });
}

// pool, src, dst
PyObject *copy(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded(n, 3, "copy", [&] {
        const int device = c10::cuda::current_device();
        const nq_page_pool_t pool = pool_of(a[0], device);
        const int32_t *src = index(a[1], "src", device);
        const int64_t count = THPVariable_Unpack(a[1]).size(0);
        const int32_t *dst = index(a[2], "dst", device, count);
        return done(nq_pages_copy(&pool, src, dst, count, stream_of(device)));
    });
}

PyMethodDef methods[] = {
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(attention)), METH_FASTCALL,
     nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(append)), METH_FASTCALL,
     nullptr},
    {"free", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(free_)), METH_FASTCALL, nullptr},
    {"fork", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(fork_)), METH_FASTCALL, nullptr},
    {"reserve", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(reserve)), METH_FASTCALL,
     nullptr},
    {"compact", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(compact)), METH_FASTCALL,
     nullptr},
    {"copy", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(copy)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, methods, nullptr, nullptr,
                      nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged(void) { return PyModule_Create(&module); }
