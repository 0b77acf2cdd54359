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

#include <cstdint>
#include <exception>

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
PyObject* collect(PyObject*, PyObject* args) {
    PyObject* list;
    long long addresses, stride, sizes_in, sizes_out;
    if (!PyArg_ParseTuple(args, "O!LLLL", &PyList_Type, &list, &addresses, &stride, &sizes_in, &sizes_out)) return nullptr;
    auto* out = reinterpret_cast<int64_t*>(addresses);
    const auto* want = reinterpret_cast<const int64_t*>(sizes_in);
    auto* sizes = reinterpret_cast<int64_t*>(sizes_out);
    long long tag = -1, device = -1, count = 0, bad = -1;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    at::ScalarType type = at::kByte;
    try {
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* item = PyList_GET_ITEM(list, i);
            if (item == Py_None) {
                out[i * stride] = 0;
                if (sizes) sizes[i] = 0;
                continue;
            }
            if (!THPVariable_Check(item)) {
                bad = i;
                break;
            }
            const at::Tensor& t = THPVariable_Unpack(item);
            if (t.layout() != at::kStrided || !t.is_cuda()) {
                bad = i;
                break;
            }
            if (count == 0) {
                type = t.scalar_type();
                tag = dtype_tag(type);
                device = t.get_device();
            }
            if ((tag < 0 && type != at::kByte) || t.scalar_type() != type || t.get_device() != device || !t.is_contiguous() ||
                (want && t.numel() != want[i])) {
                bad = i;
                break;
            }
            out[i * stride] = reinterpret_cast<int64_t>(t.data_ptr());
            if (sizes) sizes[i] = t.numel();
            ++count;
        }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    return Py_BuildValue("LLLL", tag, device, count, bad);
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
        if (c10::impl::getDeviceGuardImpl(device.type())->getDevice() != device) Py_RETURN_NONE;
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
    {"collect", collect, METH_VARARGS, "addresses, sizes, type and device of a list of tensors"},
    {"bump", bump, METH_O, "count the versions of a list of tensors up"},
    {"gated", gated, METH_VARARGS, "a gated block's call in its plain form"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", "Host code of launch-bound calls.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast(void) { return PyModule_Create(&module); }
