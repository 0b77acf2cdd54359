// Host code of the calls whose time is the host's (CPython module stratum_amd._fast): reading
// a list of tensors into an address table, and the gated block's call in its plain form.
// 448 tensors, us: dtype, device, size, layout and address of each read from Python
// 110, here 6; a call of the gated block on one row 10.4, here 6.
//
// Nothing is decided here that the Python layer does not decide as well: what is not the
// plain form is handed back (None, or the index of the tensor), and Python converts it or
// names what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstdint>
#include <exception>
#include <vector>

#include "../../include/stratum_nf4.h"

namespace {

int dtype_tag(at::ScalarType t) {
    return t == at::kHalf ? STM_F16 : t == at::kBFloat16 ? STM_BF16 : t == at::kFloat ? STM_F32 : -1;  // -1: any other
}

bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// collect(tensors, addresses, stride, sizes_in, sizes_out) -> (dtype tag, device index, tensors that are not None, bad)
// Writes the address of tensors[i] (None: 0) to ((int64 *)addresses)[i * stride], and, where sizes_out is
// not 0, its size there. bad: the first tensor that is not contiguous, on the first one's GPU, of its
// type (of 16 or 32 bits, or uint8: tag -1) and, where sizes_in is not 0, of that size; -1: none.
struct Collected {
    long long tag = -1, device = -1, count = 0, bad = -1;
};

Collected collect(PyObject* list, int64_t* out, int64_t stride, const int64_t* want, int64_t* sizes) {
    Collected c;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    at::ScalarType type = at::kByte;
    for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* item = PyList_GET_ITEM(list, i);
        if (item == Py_None) {
            out[i * stride] = 0;
            if (sizes) sizes[i] = 0;
            continue;
        }
        c.bad = i;
        if (!THPVariable_Check(item)) return c;
        const at::Tensor& t = THPVariable_Unpack(item);
        if (t.layout() != at::kStrided || !t.is_cuda()) return c;
        if (c.count == 0) {
            type = t.scalar_type();
            c.tag = dtype_tag(type);
            c.device = t.get_device();
        }
        if ((c.tag < 0 && type != at::kByte) || t.scalar_type() != type || t.get_device() != c.device ||
            !t.is_contiguous() || (want && t.numel() != want[i]))
            return c;
        out[i * stride] = reinterpret_cast<int64_t>(t.data_ptr());
        if (sizes) sizes[i] = t.numel();
        ++c.count;
        c.bad = -1;
    }
    return c;
}

PyObject* py_collect(PyObject*, PyObject* args) {
    PyObject* list;
    long long addresses, stride, sizes_in, sizes_out;
    if (!PyArg_ParseTuple(args, "O!LLLL", &PyList_Type, &list, &addresses, &stride, &sizes_in, &sizes_out)) return nullptr;
    try {
        const Collected c = collect(list, reinterpret_cast<int64_t*>(addresses), stride,
                                    reinterpret_cast<const int64_t*>(sizes_in), reinterpret_cast<int64_t*>(sizes_out));
        return Py_BuildValue("LLLL", c.tag, c.device, c.count, c.bad);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// Whether `device` is the current GPU.
bool is_current(const c10::Device& device) {
    return c10::impl::getDeviceGuardImpl(device.type())->getDevice() == device;
}

typedef int64_t (*NormBytes)(int, const int64_t*);
typedef int (*Norm)(int, const void* const*, const int64_t*, int, double, double, float*, void*, int64_t, void*);

// grad_norm(function, workspace function, gradients, max_norm, loss_scale, raw stream of a GPU)
//   -> the two values; None where a gradient has to be copied or refused, or the list is empty.
PyObject* grad_norm(PyObject*, PyObject* args) {
    long long fn, ws_fn;
    PyObject *list, *stream_of;
    double max_norm, loss_scale;
    if (!PyArg_ParseTuple(args, "LLO!ddO", &fn, &ws_fn, &PyList_Type, &list, &max_norm, &loss_scale, &stream_of))
        return nullptr;
    try {
        const Py_ssize_t n = PyList_GET_SIZE(list);
        std::vector<int64_t> addresses(n), sizes(n);
        const Collected c = collect(list, addresses.data(), 1, nullptr, sizes.data());
        if (c.bad >= 0 || c.count == 0 || c.tag < 0 || n > INT_MAX) Py_RETURN_NONE;
        const c10::Device device(c10::DeviceType::CUDA, (c10::DeviceIndex)c.device);
        if (!is_current(device)) Py_RETURN_NONE;
        PyObject* raw = PyObject_CallFunction(stream_of, "L", c.device);
        if (!raw) return nullptr;
        void* stream = PyLong_AsVoidPtr(raw);
        Py_DECREF(raw);
        const int64_t bytes = reinterpret_cast<NormBytes>(ws_fn)((int)n, sizes.data());
        if (bytes < 0) return PyLong_FromLongLong(bytes);
        const auto options = at::TensorOptions().device(device);
        at::Tensor out = at::empty({2}, options.dtype(at::kFloat)), ws = at::empty({bytes / 8}, options.dtype(at::kDouble));
        const int rc = reinterpret_cast<Norm>(fn)((int)n, reinterpret_cast<const void* const*>(addresses.data()),
                                                  sizes.data(), (int)c.tag, max_norm, loss_scale, out.data_ptr<float>(),
                                                  ws.data_ptr(), bytes, stream);
        if (rc != STM_OK) return PyLong_FromLong(rc);
        return THPVariable_Wrap(out);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// bump(tensors): count their versions up, as an in-place operation of torch does.
PyObject* bump(PyObject*, PyObject* list) {
    if (!PyList_Check(list)) {
        PyErr_SetString(PyExc_TypeError, "a list of tensors");
        return nullptr;
    }
    try {
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
            PyObject* item = PyList_GET_ITEM(list, i);
            if (!THPVariable_Check(item)) {
                PyErr_SetString(PyExc_TypeError, "a list of tensors");
                return nullptr;
            }
            const at::Tensor& t = THPVariable_Unpack(item);
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    Py_RETURN_NONE;
}

typedef int64_t (*GatedBytes)(int64_t, int64_t, int64_t);
typedef int (*GatedFwd)(const void*, const uint8_t*, const float*, void*, int64_t, int64_t, int64_t, int, int, void*,
                        int64_t, void*);
typedef int (*GatedBwd)(const void*, const void*, const uint8_t*, const float*, void*, int64_t, int64_t, int64_t, int,
                        int, void*, int64_t, void*);

// gated(function, workspace function, x, packed, absmax, N, K, blocksize, gradient or None, stream)
//   -> the output; None where the operands are not in the plain form (contiguous, aligned, on the
//   current GPU, sizes that fit: the Python layer copies or refuses them); a status if the call failed.
PyObject* gated(PyObject*, PyObject* args) {
    long long fn, ws_fn, N, K, bs, stream;
    PyObject *px, *pq, *pa, *pg;
    if (!PyArg_ParseTuple(args, "LLOOOLLLOL", &fn, &ws_fn, &px, &pq, &pa, &N, &K, &bs, &pg, &stream)) return nullptr;
    if (!THPVariable_Check(px) || !THPVariable_Check(pq) || !THPVariable_Check(pa)) Py_RETURN_NONE;
    if (pg != Py_None && !THPVariable_Check(pg)) Py_RETURN_NONE;
    try {
        const at::Tensor &x = THPVariable_Unpack(px), &q = THPVariable_Unpack(pq), &a = THPVariable_Unpack(pa);
        const int64_t inter = N / 2;
        if (!x.is_cuda() || !q.is_cuda() || !a.is_cuda() || x.dim() < 1 || N <= 0 || N % 16 || K <= 0 || K % 64 ||
            bs < 64 || bs > 4096 || (bs & (bs - 1)) || K % bs)
            Py_RETURN_NONE;
        const int tag = dtype_tag(x.scalar_type());
        const auto device = x.device();
        if ((tag != STM_BF16 && tag != STM_F16) || x.size(-1) != K || q.scalar_type() != at::kByte ||
            a.scalar_type() != at::kFloat || q.device() != device || a.device() != device || !x.is_contiguous() ||
            !q.is_contiguous() || !a.is_contiguous() || !aligned16(x) || !aligned16(q) ||
            q.numel() < inter * K || a.numel() * bs < N * K)
            Py_RETURN_NONE;
        if (!is_current(device)) Py_RETURN_NONE;
        const int64_t M = x.numel() / K;
        const void* grad = nullptr;
        if (pg != Py_None) {
            const at::Tensor& g = THPVariable_Unpack(pg);
            if (g.device() != device || g.scalar_type() != x.scalar_type() || !g.is_contiguous() || g.dim() < 1 ||
                g.size(-1) != inter || g.numel() != M * inter || !aligned16(g))
                Py_RETURN_NONE;
            grad = g.data_ptr();
        }
        at::DimVector shape(x.sizes().begin(), x.sizes().end());
        shape.back() = grad || pg != Py_None ? N : inter;
        at::Tensor out = at::empty(shape, x.options().requires_grad(false));
        const int64_t bytes = reinterpret_cast<GatedBytes>(ws_fn)(M, inter, K);
        if (bytes < 0) return PyLong_FromLongLong(bytes);
        at::Tensor ws;
        if (bytes) ws = at::empty({bytes}, a.options().dtype(at::kByte).requires_grad(false));
        void* wp = bytes ? ws.data_ptr() : nullptr;
        const auto* qp = static_cast<const uint8_t*>(q.data_ptr());
        const auto* ap = static_cast<const float*>(a.data_ptr());
        void* st = reinterpret_cast<void*>(stream);
        const int rc = pg == Py_None
                           ? reinterpret_cast<GatedFwd>(fn)(x.data_ptr(), qp, ap, out.data_ptr(), M, inter, K, (int)bs, tag, wp, bytes, st)
                           : reinterpret_cast<GatedBwd>(fn)(grad, x.data_ptr(), qp, ap, out.data_ptr(), M, inter, K, (int)bs, tag, wp, bytes, st);
        if (rc != STM_OK) return PyLong_FromLong(rc);
        return THPVariable_Wrap(out);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"collect", py_collect, METH_VARARGS, "addresses, sizes, type and device of a list of tensors"},
    {"bump", bump, METH_O, "count the versions of a list of tensors up"},
    {"grad_norm", grad_norm, METH_VARARGS, "the gradient norm of a list of tensors in its plain form"},
    {"gated", gated, METH_VARARGS, "a gated block's call in its plain form"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", "Host code of launch-bound calls.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast(void) { return PyModule_Create(&module); }
