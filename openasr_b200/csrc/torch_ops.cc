// torch_ops.cc -- the Python binding's short way to the operators of the paged cache
// (openasr_b200/_torch_ops.so): torch tensors in, one C call, its status out.
//
// A step calls these once per layer with up to twelve tensors.  Describing a tensor through its
// Python attributes takes 0.3 us and a call through ctypes more than 1 us, together longer than
// the kernels run; here a tensor's pointer, sizes and strides are read from the tensor itself.
#include <torch/csrc/autograd/python_variable.h>

#include <exception>

#include "oasr_b200.h"

namespace {

PyObject *s_unsupported;  // callable(what, reason or None for a dtype): raises
decltype(&oasr_b200_qk_norm_rope) s_qk_norm_rope;
decltype(&oasr_b200_flash_attn_tree) s_flash_attn_tree;
decltype(&oasr_b200_tree_commit) s_tree_commit;
decltype(&oasr_b200_kv_pages_copy) s_kv_pages_copy;
decltype(&oasr_b200_tree_sample) s_tree_sample;
decltype(&oasr_b200_attn_weights) s_attn_weights;
decltype(&oasr_b200_kv_evict) s_kv_evict;

// The descriptor of a torch tensor (ne = reversed sizes, nb = reversed byte strides), of a ready
// one (any object whose buffer is an oasr_tensor), or nothing for None.
//
// The kernels read all of them on the backend's device: a tensor elsewhere (a page table still on the
// host) would be an illegal access there, so it is refused here.
struct Arg {
    oasr_tensor d;
    oasr_tensor *p = nullptr;

    static bool refuse(PyObject *what, const char *reason) {
        if (what) Py_XDECREF(PyObject_CallFunction(s_unsupported, "Oz", what, reason));
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "unsupported tensor");
        return false;
    }

    bool take(PyObject *o, int device) {
        if (o == Py_None) return true;
        p = &d;
        if (!THPVariable_Check(o)) {
            Py_buffer view;
            if (PyObject_GetBuffer(o, &view, PyBUF_SIMPLE)) return false;
            const bool ok = view.len == (Py_ssize_t)sizeof d;
            if (ok) d = *static_cast<const oasr_tensor *>(view.buf);
            else PyErr_SetString(PyExc_TypeError, "a tensor, a descriptor or None");
            PyBuffer_Release(&view);
            return ok;
        }
        const at::Tensor &t = THPVariable_Unpack(o);
        int64_t size = 4;
        switch (t.scalar_type()) {
            case at::kFloat: d.type = OASR_TYPE_F32; break;
            case at::kHalf: d.type = OASR_TYPE_F16, size = 2; break;
            case at::kInt: d.type = OASR_TYPE_I32; break;
            case at::kLong: d.type = OASR_TYPE_I64, size = 8; break;
            default: {
                PyObject *dtype = PyObject_GetAttrString(o, "dtype");
                const bool taken = refuse(dtype, nullptr);
                Py_XDECREF(dtype);
                return taken;
            }
        }
        if (device >= 0 && t.numel() != 0 && !(t.is_cuda() && t.get_device() == device)) {
            PyObject *where = PyObject_GetAttrString(o, "device");
            const bool taken = refuse(where, "a tensor on another device than the backend's:");
            Py_XDECREF(where);
            return taken;
        }
        try {
            const auto sizes = t.sizes(), strides = t.strides();
            const int64_t dims = t.dim();
            if (dims > 4) {
                PyObject *n = PyLong_FromLongLong(dims);
                const bool taken = refuse(n, "a tensor has at most 4 dimensions, not");
                Py_XDECREF(n);
                return taken;
            }
            for (int i = 0; i < 4; ++i) {
                d.ne[i] = i < dims ? sizes[dims - 1 - i] : 1;
                d.nb[i] = i < dims ? strides[dims - 1 - i] * size : i ? d.nb[i - 1] * d.ne[i - 1] : size;
            }
            d.flags = 0;
            d.data = t.data_ptr();
        } catch (const std::exception &e) {
            PyErr_SetString(PyExc_ValueError, e.what());
            return false;
        }
        return true;
    }
};

bool count(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", want, n);
    return n == want;
}

// The backend: its address, or (address, device) to have the tensors' device checked.
struct Where {
    oasr_backend *be = nullptr;
    int device = -1;

    explicit Where(PyObject *o) {
        if (PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2) {
            device = (int)PyLong_AsLong(PyTuple_GET_ITEM(o, 1));
            o = PyTuple_GET_ITEM(o, 0);
        }
        if (!PyErr_Occurred()) be = static_cast<oasr_backend *>(PyLong_AsVoidPtr(o));
    }
};

// args[i] to t[i]
template <int N>
bool take(Arg (&t)[N], PyObject *const *args, const Where &at) {
    if (PyErr_Occurred()) return false;
    for (int i = 0; i < N; ++i)
        if (!t[i].take(args[i], at.device)) return false;
    return true;
}

// The status of call(f).
template <class Fn, class F>
PyObject *status(Fn *f, F &&call) {
    if (!f) {
        PyErr_SetString(PyExc_RuntimeError, "this function has not been bound");
        return nullptr;
    }
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = call(f);
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(rc);
}

PyObject *qk_norm_rope(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Arg x[3], y[8];
    if (!count(n, 13)) return nullptr;
    const Where at(a[0]);
    if (!take(x, a + 1, at) || !take(y, a + 5, at)) return nullptr;
    const float eps = (float)PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) return nullptr;
    return status(s_qk_norm_rope, [&](auto f) {
        return f(at.be, x[0].p, x[1].p, x[2].p, eps, y[0].p, y[1].p, y[2].p, y[3].p, y[4].p, y[5].p, y[6].p, y[7].p);
    });
}

PyObject *flash_attn_tree(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Arg x[7], y[1];
    if (!count(n, 10)) return nullptr;
    const Where at(a[0]);
    if (!take(x, a + 1, at) || !take(y, a + 9, at)) return nullptr;
    const float scale = (float)PyFloat_AsDouble(a[8]);
    if (PyErr_Occurred()) return nullptr;
    return status(s_flash_attn_tree, [&](auto f) {
        return f(at.be, x[0].p, x[1].p, x[2].p, x[3].p, x[4].p, x[5].p, x[6].p, scale, y[0].p);
    });
}

bool int32(PyObject *o, int32_t *v) {
    const long x = PyLong_AsLong(o);
    if (x == -1 && PyErr_Occurred()) return false;
    if (x < INT32_MIN || x > INT32_MAX) {
        PyErr_SetString(PyExc_OverflowError, "out of range");
        return false;
    }
    *v = (int32_t)x;
    return true;
}

PyObject *tree_commit(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Arg x[8], y[4];
    int32_t layers;
    if (!count(n, 14)) return nullptr;
    const Where at(a[0]);
    if (!take(x, a + 1, at) || !int32(a[9], &layers) || !take(y, a + 10, at)) return nullptr;
    return status(s_tree_commit, [&](auto f) {
        return f(at.be, x[0].p, x[1].p, x[2].p, x[3].p, x[4].p, x[5].p, x[6].p, x[7].p, layers, y[0].p, y[1].p, y[2].p, y[3].p);
    });
}

PyObject *kv_pages_copy(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Arg x[2], y[1];
    int32_t layers;
    if (!count(n, 5)) return nullptr;
    const Where at(a[0]);
    if (!take(x, a + 1, at) || !int32(a[3], &layers) || !take(y, a + 4, at)) return nullptr;
    return status(s_kv_pages_copy, [&](auto f) { return f(at.be, x[0].p, x[1].p, layers, y[0].p); });
}

PyObject *tree_sample(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Arg x[9];
    if (!count(n, 10)) return nullptr;
    const Where at(a[0]);
    if (!take(x, a + 1, at)) return nullptr;
    return status(s_tree_sample, [&](auto f) {
        return f(at.be, x[0].p, x[1].p, x[2].p, x[3].p, x[4].p, x[5].p, x[6].p, x[7].p, x[8].p);
    });
}

PyObject *attn_weights(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Arg x[5], y[1];
    if (!count(n, 9)) return nullptr;
    const Where at(a[0]);
    if (!take(x, a + 1, at) || !take(y, a + 8, at)) return nullptr;
    const float scale = (float)PyFloat_AsDouble(a[6]), decay = (float)PyFloat_AsDouble(a[7]);
    if (PyErr_Occurred()) return nullptr;
    return status(s_attn_weights, [&](auto f) { return f(at.be, x[0].p, x[1].p, x[2].p, x[3].p, x[4].p, scale, decay, y[0].p); });
}

PyObject *kv_evict(PyObject *, PyObject *const *a, Py_ssize_t n) {
    Arg x[4], y[2], z[1];
    int32_t sink, recent, layers;
    if (!count(n, 11)) return nullptr;
    const Where at(a[0]);
    if (!take(x, a + 1, at) || !int32(a[5], &sink) || !int32(a[6], &recent) || !take(y, a + 7, at) || !int32(a[9], &layers) ||
        !take(z, a + 10, at))
        return nullptr;
    return status(s_kv_evict, [&](auto f) { return f(at.be, x[0].p, x[1].p, x[2].p, x[3].p, sink, recent, y[0].p, y[1].p, layers, z[0].p); });
}

// bind(unsupported, addresses of the C functions in the order below: the first four, or all); what has no address raises
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    constexpr int FEW = 4, ALL = 7;
    if (n != 1 + FEW && !count(n, 1 + ALL)) return nullptr;
    void *f[ALL] = {};
    for (int i = 0; i < n - 1; ++i) f[i] = PyLong_AsVoidPtr(a[1 + i]);
    if (PyErr_Occurred()) return nullptr;
    Py_INCREF(a[0]);
    Py_XSETREF(s_unsupported, a[0]);
    s_qk_norm_rope = reinterpret_cast<decltype(s_qk_norm_rope)>(f[0]);
    s_flash_attn_tree = reinterpret_cast<decltype(s_flash_attn_tree)>(f[1]);
    s_tree_commit = reinterpret_cast<decltype(s_tree_commit)>(f[2]);
    s_kv_pages_copy = reinterpret_cast<decltype(s_kv_pages_copy)>(f[3]);
    s_tree_sample = reinterpret_cast<decltype(s_tree_sample)>(f[4]);
    s_attn_weights = reinterpret_cast<decltype(s_attn_weights)>(f[5]);
    s_kv_evict = reinterpret_cast<decltype(s_kv_evict)>(f[6]);
    Py_RETURN_NONE;
}

#define FAST(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(qk_norm_rope), FAST(flash_attn_tree), FAST(tree_commit), FAST(kv_pages_copy),
                         FAST(tree_sample), FAST(attn_weights), FAST(kv_evict),
                         {nullptr, nullptr, 0, nullptr}};
#undef FAST
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) { return PyModule_Create(&module_def); }
