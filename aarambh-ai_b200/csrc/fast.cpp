// The host side of the operators of a serving step (dispatch.py) for their plain calls: CUDA tensors on the current device, contiguous, of types and
// shapes that match, results freshly allocated.  A step of a few sessions runs some microseconds on the GPU; looking the tensors over in Python and
// ctypes took 8 to 10 of the 12 to 15 that a call took.  Each function answers None where a call is anything else: dispatch.py then looks at it, and makes it or
// says what is wrong.  A number is the status of a refused call; results otherwise.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "aarambh_b200.h"

namespace {

// A tensor or None (null); `plain` falls where it is neither, or not contiguous on the current device.
struct Args {
    PyObject *const *args;
    c10::DeviceIndex device = -1;
    bool plain = true;
    const at::Tensor *operator()(int i, bool optional = false) {
        PyObject *o = args[i];
        if (optional && o == Py_None) return nullptr;
        if (!THPVariable_CheckExact(o)) { plain = false; return nullptr; }
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!t.is_cuda() || !t.is_contiguous() || t.layout() != at::kStrided) { plain = false; return nullptr; }
        if (device < 0) {
            device = t.get_device();
            plain = plain && device == c10::cuda::current_device();
        } else if (t.get_device() != device) {
            plain = false;
        }
        return &t;
    }
};

int dtype_of(const at::Tensor &t) {
    switch (t.scalar_type()) {
    case at::kFloat: return AB2_F32;
    case at::kHalf: return AB2_F16;
    case at::kBFloat16: return AB2_BF16;
    default: return -1;
    }
}
int layout_of(PyObject *o) {
    const char *s = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    if (!s) PyErr_Clear();   // of a text that has no UTF-8
    return s && !strcmp(s, "half") ? AB2_ROTARY_HALF : s && !strcmp(s, "interleaved") ? AB2_ROTARY_INTERLEAVED : -1;
}
bool is(const at::Tensor *t, at::ScalarType type, std::initializer_list<int64_t> shape) { return t->scalar_type() == type && t->sizes().equals(shape); }
bool number(PyObject *o, double &x) {
    if (PyFloat_CheckExact(o)) { x = PyFloat_AS_DOUBLE(o); return true; }
    if (PyLong_CheckExact(o)) {
        x = PyLong_AsDouble(o);
        if (!PyErr_Occurred()) return true;
        PyErr_Clear();
    }
    return false;
}
bool fits(int64_t n) { return n >= 0 && n <= 0x7fffffff; }
void *ptr(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }
PyObject *none() { Py_RETURN_NONE; }

// What tensors' own functions throw becomes a Python error.
template <class F> PyObject *guarded(F f) {
    try {
        return f();
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "an exception of unknown type");
        return nullptr;
    }
}

// rotary(q, k, positions, frequencies, layout, magnitude)
PyObject *rotary(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 6) return none();
        Args a{args};
        const at::Tensor *q = a(0), *k = a(1, true), *pos = a(2), *f = a(3);
        const int layout = layout_of(args[4]);
        double magnitude;
        if (!a.plain || layout < 0 || !number(args[5], magnitude) || q->dim() != 3 || (k && k->dim() != 3) || f->dim() != 1) return none();
        const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), kv = k ? k->size(1) : 0;
        if (!fits(tokens) || !fits(heads) || !fits(dim) || !fits(kv) || dtype_of(*q) < 0) return none();
        if (k && (k->scalar_type() != q->scalar_type() || k->size(0) != tokens || k->size(2) != dim)) return none();
        const bool wide = pos->scalar_type() == at::kLong;
        if (!is(pos, wide ? at::kLong : at::kInt, {tokens}) || f->scalar_type() != at::kDouble || 2 * f->size(0) > dim) return none();
        at::Tensor qo = at::empty_like(*q), ko;
        if (k) ko = at::empty_like(*k);
        const int rc = ab2_rotary_apply(ptr(q), heads * dim, (int)heads, ptr(k), kv * dim, (int)kv, (int)dim, ptr(pos), wide, (int)tokens, (const double *)ptr(f), (int)(2 * f->size(0)), layout,
                                        (float)magnitude, qo.data_ptr(), heads * dim, k ? ko.data_ptr() : nullptr, kv * dim, (ab2_dtype)dtype_of(*q), c10::cuda::getCurrentCUDAStream().stream());
        if (rc != AB2_OK) return PyLong_FromLong(rc);
        PyObject *first = THPVariable_Wrap(qo), *second = k ? THPVariable_Wrap(ko) : Py_NewRef(Py_None), *both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
        Py_XDECREF(first);
        Py_XDECREF(second);
        return both;
    });
}

// ab2_paged of the arguments from `at` on: k_pages, v_pages, table, lens, starts
bool paged_of(Args &a, int kp, int tab, int len, int st, int64_t tokens, ab2_paged &c, const at::Tensor *&pages) {
    const at::Tensor *k = a(kp), *v = a(kp + 1), *table = a(tab), *lens = a(len), *starts = a(st, true);
    if (!a.plain || k->dim() != 4 || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() || table->dim() != 2 || table->scalar_type() != at::kInt) return false;
    const int64_t rows = table->size(0), width = table->size(1);
    if (!is(lens, at::kInt, {rows}) || (starts && !is(starts, at::kInt, {rows + 1}))) return false;
    if (!fits(rows) || !fits(width) || !fits(tokens) || !fits(k->size(0)) || !fits(k->size(1)) || !fits(k->size(2)) || !fits(k->size(3))) return false;
    c.k_pages = ptr(k); c.v_pages = ptr(v);
    c.table = (const int *)ptr(table); c.lens = (const int *)ptr(lens); c.starts = (const int *)ptr(starts);
    c.pages = (int)k->size(0); c.kv_heads = (int)k->size(1); c.page_size = (int)k->size(2); c.head_dim = (int)k->size(3);
    c.table_width = (int)width; c.rows = (int)rows; c.tokens = (int)tokens; c.table_stride = width;
    pages = k;
    return true;
}

// The scales of pages of 8 bits, a pair (or None: neither); false where they and the pages do not belong together.
bool scales_of(Args &a, PyObject *pair, const at::Tensor &pages, const float *&ks, const float *&vs) {
    ks = vs = nullptr;
    const bool codes = pages.scalar_type() == at::kFloat8_e4m3fn;
    if (pair == Py_None) return !codes;
    if (!codes || !PyTuple_CheckExact(pair) || PyTuple_GET_SIZE(pair) != 2) return false;
    PyObject *both[2] = {PyTuple_GET_ITEM(pair, 0), PyTuple_GET_ITEM(pair, 1)};
    Args s{both, a.device};
    const at::Tensor *k = s(0), *v = s(1);
    if (!s.plain) return false;
    for (const at::Tensor *t : {k, v})
        if (!is(t, at::kFloat, {pages.size(0), pages.size(1), pages.size(2) / 16})) return false;
    ks = (const float *)ptr(k);
    vs = (const float *)ptr(v);
    return true;
}

// append(k_pages, v_pages, k, v, table, lens, starts, q, frequencies, layout, magnitude[, scales])
PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 11 && n != 12) return none();
        PyObject *scales = n > 11 ? args[11] : Py_None;
        Args a{args};
        const at::Tensor *k = a(2), *v = a(3), *q = a(7, true), *f = a(8, true), *pages;
        const int layout = layout_of(args[9]);
        double magnitude;
        if (!a.plain || layout < 0 || !number(args[10], magnitude) || k->dim() != 3 || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type()) return none();
        const int64_t tokens = k->size(0), kv = k->size(1), dim = k->size(2), heads = q && q->dim() == 3 ? q->size(1) : 0;
        ab2_paged c;
        if (!paged_of(a, 0, 4, 5, 6, tokens, c, pages) || (scales == Py_None && pages->scalar_type() != k->scalar_type()) || kv != c.kv_heads || dim != c.head_dim || dtype_of(*k) < 0 || !fits(heads)) return none();
        if (q && (q->dim() != 3 || q->scalar_type() != k->scalar_type() || q->size(0) != tokens || q->size(2) != dim)) return none();
        if (f && (f->dim() != 1 || f->scalar_type() != at::kDouble || 2 * f->size(0) > dim)) return none();
        const float *ks, *vs;
        if (!a.plain || !scales_of(a, scales, *pages, ks, vs)) return none();
        at::Tensor out;
        if (q) out = at::empty_like(*q);
        if (ks) {
            const int rc = ab2_paged_append_e4m3(&c, (float *)ks, (float *)vs, ptr(k), kv * dim, ptr(v), kv * dim, ptr(q), heads * dim, (int)heads, q ? out.data_ptr() : nullptr, heads * dim,
                                                 (const double *)ptr(f), f ? (int)(2 * f->size(0)) : 0, layout, (float)magnitude, (ab2_dtype)dtype_of(*k), c10::cuda::getCurrentCUDAStream().stream());
            if (rc != AB2_OK) return PyLong_FromLong(rc);
            return q ? THPVariable_Wrap(out) : Py_NewRef(Py_True);
        }
        const int rc = ab2_paged_append(&c, ptr(k), kv * dim, ptr(v), kv * dim, ptr(q), heads * dim, (int)heads, q ? out.data_ptr() : nullptr, heads * dim, (const double *)ptr(f),
                                        f ? (int)(2 * f->size(0)) : 0, layout, (float)magnitude, (ab2_dtype)dtype_of(*k), c10::cuda::getCurrentCUDAStream().stream());
        if (rc != AB2_OK) return PyLong_FromLong(rc);
        return q ? THPVariable_Wrap(out) : Py_NewRef(Py_True);
    });
}

// attention(q, k_pages, v_pages, table, lens, scale, starts, max_new[, scales, window, sinks])
PyObject *attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 8 && n != 11) return none();
        PyObject *scales = n > 8 ? args[8] : Py_None;
        Args a{args};
        const at::Tensor *q = a(0), *pages;
        double scale, most = -1, window = 0, sinks = 0;
        if (!a.plain || q->dim() != 3 || !number(args[5], scale) || (args[7] != Py_None && (!PyLong_CheckExact(args[7]) || !number(args[7], most) || most > 0x7fffffff)) ||
            (n > 8 && (!PyLong_CheckExact(args[9]) || !number(args[9], window) || !PyLong_CheckExact(args[10]) || !number(args[10], sinks))) || window < 0 || window > 0x7fffffff || sinks < 0 || sinks > 0x7fffffff)
            return none();
        const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2);
        ab2_paged c;
        if (!paged_of(a, 1, 3, 4, 6, tokens, c, pages) || (scales == Py_None && pages->scalar_type() != q->scalar_type()) || dim != c.head_dim || dtype_of(*q) < 0 || !fits(heads)) return none();
        const float *ks, *vs;
        if (!a.plain || !scales_of(a, scales, *pages, ks, vs)) return none();
        if (((uintptr_t)q->data_ptr() | (uintptr_t)(heads * dim * q->element_size())) & 15) return none();
        if (args[7] == Py_None) most = c.starts ? (double)std::max<int64_t>(tokens, 1) : 1;
        size_t bytes = 0;
        if (c.table_width * (int64_t)c.page_size > AB2_PAGED_UNCUT && ab2_paged_workspace(c.head_dim, &bytes) != AB2_OK) return none();
        at::Tensor out = at::empty_like(*q), work;
        if (bytes > 0) work = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte));
        void *room = bytes > 0 ? work.data_ptr() : nullptr;
        ab2_stream stream = c10::cuda::getCurrentCUDAStream().stream();
        const ab2_dtype type = (ab2_dtype)dtype_of(*q);
        const long long row = heads * dim;
        const int rc = ks       ? ab2_paged_attention_e4m3(&c, ks, vs, (int)window, (int)sinks, q->data_ptr(), row, (int)heads, out.data_ptr(), row, (int)most, (float)scale, room, bytes, type, stream)
                       : window || sinks ? ab2_paged_attention_window(&c, (int)window, (int)sinks, q->data_ptr(), row, (int)heads, out.data_ptr(), row, (int)most, (float)scale, room, bytes, type, stream)
                                : ab2_paged_attention(&c, q->data_ptr(), row, (int)heads, out.data_ptr(), row, (int)most, (float)scale, room, bytes, type, stream);
        return rc == AB2_OK ? THPVariable_Wrap(out) : PyLong_FromLong(rc);
    });
}

// logits(logits, history, lengths, rules, bias_ids, bias_values, allowed)
PyObject *logits(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 7) return none();
        Args a{args};
        const at::Tensor *z = a(0), *h = a(1, true), *len = a(2, true), *rules = a(3, true), *ids = a(4, true), *values = a(5, true), *allowed = a(6, true);
        if (!a.plain || z->dim() != 2 || dtype_of(*z) < 0) return none();
        const int64_t rows = z->size(0), vocab = z->size(1);
        if (!fits(rows) || !fits(vocab)) return none();
        int64_t width = 0, biases = 0;
        if (h) {
            if (!rules || h->dim() != 2 || h->size(0) != rows || h->scalar_type() != at::kInt || !is(rules, at::kFloat, {rows, 3}) || (len && !is(len, at::kInt, {rows}))) return none();
            width = h->size(1);
        } else if (len || rules) {
            return none();
        }
        if (!ids != !values) return none();
        if (ids) {
            if (ids->dim() != 2) return none();
            biases = ids->size(1);
            if (!is(ids, at::kInt, {rows, biases}) || !is(values, at::kFloat, {rows, biases})) return none();
        }
        if ((allowed && !is(allowed, at::kInt, {rows, (vocab + 31) / 32})) || !fits(width) || !fits(biases)) return none();
        at::Tensor out = at::empty_like(*z);
        const int rc = ab2_adjust_logits(z->data_ptr(), vocab, (int)rows, (int)vocab, (const int *)ptr(h), width, (int)width, (const int *)ptr(len), (const float *)ptr(rules), (const int *)ptr(ids),
                                         (const float *)ptr(values), (int)biases, (const uint32_t *)ptr(allowed), out.data_ptr(), (ab2_dtype)dtype_of(*z), c10::cuda::getCurrentCUDAStream().stream());
        return rc == AB2_OK ? THPVariable_Wrap(out) : PyLong_FromLong(rc);
    });
}

// sample(logits, uniforms, temperature, top_k, top_p, min_p)
PyObject *sample(PyObject *, PyObject *const *args, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        if (n != 6) return none();
        Args a{args};
        const at::Tensor *z = a(0), *u = a(1), *temperature = a(2, true), *top_k = a(3, true), *top_p = a(4, true), *min_p = a(5, true);
        if (!a.plain || z->dim() != 2 || dtype_of(*z) < 0) return none();
        const int64_t rows = z->size(0), vocab = z->size(1);
        const bool wide = u->scalar_type() == at::kDouble;
        if (!fits(rows) || !fits(vocab) || !is(u, wide ? at::kDouble : at::kFloat, {rows})) return none();
        for (const at::Tensor *t : {temperature, top_p, min_p})
            if (t && !is(t, at::kFloat, {rows})) return none();
        if (top_k && !is(top_k, at::kInt, {rows})) return none();
        at::Tensor out = at::empty({rows}, z->options().dtype(at::kInt));
        const int rc = ab2_sample(z->data_ptr(), vocab, (int)rows, (int)vocab, u->data_ptr(), wide, (const float *)ptr(temperature), (const int *)ptr(top_k), (const float *)ptr(top_p),
                                  (const float *)ptr(min_p), out.data_ptr<int>(), (ab2_dtype)dtype_of(*z), c10::cuda::getCurrentCUDAStream().stream());
        return rc == AB2_OK ? THPVariable_Wrap(out) : PyLong_FromLong(rc);
    });
}

PyMethodDef methods[] = {{"rotary", (PyCFunction)(void (*)(void))rotary, METH_FASTCALL, nullptr},
                         {"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, nullptr},
                         {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, nullptr},
                         {"logits", (PyCFunction)(void (*)(void))logits, METH_FASTCALL, nullptr},
                         {"sample", (PyCFunction)(void (*)(void))sample, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast() { return PyModule_Create(&module); }
