// Host code of the calls whose time is the host's (CPython module stratum_amd._fast): reading
// a list of tensors into an address table, and the gated block's calls in their plain form.
// 448 tensors, us: dtype, device, size, layout and address of each read from Python
// 110, here 6; a forward of the gated block on one row 10.4, here 6.5; its forward and backward
// through autograd 118, here 42.
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
typedef int (*GatedKeep)(const void*, const uint8_t*, const float*, void*, float*, int64_t, int64_t, int64_t, int, int,
                         void*, int64_t, void*);
typedef int (*GatedBwd)(const void*, const void*, const uint8_t*, const float*, void*, int64_t, int64_t, int64_t, int,
                        int, void*, int64_t, void*);
typedef int (*GatedKept)(const void*, const float*, void*, int64_t, int64_t, int, void*);
typedef int64_t (*GemmBytes)(int64_t, int64_t, int64_t, int);
typedef int (*GemmDx)(const void*, const uint8_t*, const float*, const void*, const void*, int, void*, int64_t, int64_t,
                      int64_t, int, int, void*, int64_t, void*);

// Contiguous aligned rows of `width` on `device`.
bool rows_of(const at::Tensor& t, c10::Device device, int64_t width) {
    return t.device() == device && t.is_contiguous() && aligned16(t) && t.dim() >= 1 && t.size(-1) == width;
}

// A stacked NF4 weight [N, K] in the plain form, its payload on the current GPU.
struct Weight {
    const uint8_t* packed = nullptr;
    const float* absmax = nullptr;
    int64_t N, K;
    int bs;

    bool read(PyObject* pq, PyObject* pa, int64_t n, int64_t k, int64_t blocksize, c10::Device* device) {
        if (!THPVariable_Check(pq) || !THPVariable_Check(pa)) return false;
        const at::Tensor &q = THPVariable_Unpack(pq), &a = THPVariable_Unpack(pa);
        if (!q.is_cuda() || q.device() != a.device() || n <= 0 || n % 16 || k <= 0 || k % 64 || blocksize < 64 ||
            blocksize > 4096 || (blocksize & (blocksize - 1)) || k % blocksize || q.scalar_type() != at::kByte ||
            a.scalar_type() != at::kFloat || !q.is_contiguous() || !a.is_contiguous() || !aligned16(q) ||
            q.numel() < n / 2 * k || a.numel() * blocksize < n * k || !is_current(q.device()))
            return false;
        packed = static_cast<const uint8_t*>(q.data_ptr()), absmax = static_cast<const float*>(a.data_ptr());
        N = n, K = k, bs = (int)blocksize, *device = q.device();
        return true;
    }
};

at::Tensor bytes_on(int64_t bytes, const at::Tensor& like) {
    return at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false));
}

// Tensor of x's leading sizes and `width` columns.
at::Tensor shaped(const at::Tensor& x, int64_t width) {
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = width;
    return at::empty(shape, x.options().requires_grad(false));
}

// gated_fwd(function, workspace function, keeping function, sums function, keeping workspace function, x, packed, absmax,
//           N, K, blocksize, stream)
//   -> h, or with a sums function (not 0) (h, the kept sums or None); None where the operands are not in the
//   plain form (the Python layer copies or refuses them); a status if the call failed.
PyObject* gated_fwd(PyObject*, PyObject* args) {
    long long fn, ws_fn, keep_fn, sums_fn, keep_ws_fn, N, K, bs, stream;
    PyObject *px, *pq, *pa;
    if (!PyArg_ParseTuple(args, "LLLLLOOOLLLL", &fn, &ws_fn, &keep_fn, &sums_fn, &keep_ws_fn, &px, &pq, &pa, &N, &K, &bs,
                          &stream))
        return nullptr;
    try {
        Weight w;
        c10::Device device(c10::DeviceType::CPU);
        if (!THPVariable_Check(px) || !w.read(pq, pa, N, K, bs, &device)) Py_RETURN_NONE;
        const at::Tensor& x = THPVariable_Unpack(px);
        const int tag = dtype_tag(x.scalar_type());
        if ((tag != STM_BF16 && tag != STM_F16) || !rows_of(x, device, K)) Py_RETURN_NONE;
        const int64_t M = x.numel() / K, inter = N / 2;
        const int64_t kept = sums_fn ? reinterpret_cast<GatedBytes>(sums_fn)(M, inter, K) : 0;
        const int64_t bytes = reinterpret_cast<GatedBytes>(kept ? keep_ws_fn : ws_fn)(M, inter, K);
        if (bytes < 0 || kept < 0) return PyLong_FromLongLong(bytes < 0 ? bytes : kept);
        at::Tensor h = shaped(x, inter), ws, sums;
        if (bytes) ws = bytes_on(bytes, x);
        void* wp = bytes ? ws.data_ptr() : nullptr;
        void* st = reinterpret_cast<void*>(stream);
        int rc;
        if (kept) {
            sums = at::empty({M, N}, x.options().dtype(at::kFloat).requires_grad(false));
            rc = reinterpret_cast<GatedKeep>(keep_fn)(x.data_ptr(), w.packed, w.absmax, h.data_ptr(),
                                                      sums.data_ptr<float>(), M, inter, K, w.bs, tag, wp, bytes, st);
        } else {
            rc = reinterpret_cast<GatedFwd>(fn)(x.data_ptr(), w.packed, w.absmax, h.data_ptr(), M, inter, K, w.bs, tag,
                                                wp, bytes, st);
        }
        if (rc != STM_OK) return PyLong_FromLong(rc);
        if (!sums_fn) return THPVariable_Wrap(h);
        if (!kept) return Py_BuildValue("NO", THPVariable_Wrap(h), Py_None);
        return Py_BuildValue("NN", THPVariable_Wrap(h), THPVariable_Wrap(sums));
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// gated_bwd(function, workspace function, function on kept sums, gradient, x or the kept sums, packed, absmax,
//           N, K, blocksize, input gradient's function and workspace function or 0, stream)
//   -> the gradient of the projections' outputs, or of x with an input gradient's function; otherwise as gated_fwd.
PyObject* gated_bwd(PyObject*, PyObject* args) {
    long long fn, ws_fn, kept_fn, N, K, bs, dx_fn, dx_ws_fn, stream;
    PyObject *pg, *px, *pq, *pa;
    if (!PyArg_ParseTuple(args, "LLLOOOOLLLLLL", &fn, &ws_fn, &kept_fn, &pg, &px, &pq, &pa, &N, &K, &bs, &dx_fn,
                          &dx_ws_fn, &stream))
        return nullptr;
    try {
        Weight w;
        c10::Device device(c10::DeviceType::CPU);
        if (!THPVariable_Check(px) || !THPVariable_Check(pg) || !w.read(pq, pa, N, K, bs, &device)) Py_RETURN_NONE;
        const at::Tensor &x = THPVariable_Unpack(px), &g = THPVariable_Unpack(pg);
        const int64_t inter = N / 2;
        const bool kept = x.scalar_type() == at::kFloat;
        const int tag = dtype_tag(g.scalar_type());
        if ((tag != STM_BF16 && tag != STM_F16) || !rows_of(g, device, inter) || !rows_of(x, device, kept ? N : K) ||
            (!kept && x.scalar_type() != g.scalar_type()) || (dx_fn && N % 64))
            Py_RETURN_NONE;
        const int64_t M = g.numel() / inter;
        if (x.numel() != M * (kept ? N : K)) Py_RETURN_NONE;
        void* st = reinterpret_cast<void*>(stream);
        const at::Tensor& like = kept ? g : x;  // whose leading sizes the result has
        at::Tensor dgu = shaped(like, N);
        int rc;
        if (kept) {
            rc = reinterpret_cast<GatedKept>(kept_fn)(g.data_ptr(), x.data_ptr<float>(), dgu.data_ptr(), M, inter, tag, st);
        } else {
            const int64_t bytes = reinterpret_cast<GatedBytes>(ws_fn)(M, inter, K);
            if (bytes < 0) return PyLong_FromLongLong(bytes);
            at::Tensor ws;
            if (bytes) ws = bytes_on(bytes, g);
            rc = reinterpret_cast<GatedBwd>(fn)(g.data_ptr(), x.data_ptr(), w.packed, w.absmax, dgu.data_ptr(), M, inter,
                                                K, w.bs, tag, bytes ? ws.data_ptr() : nullptr, bytes, st);
        }
        if (rc != STM_OK) return PyLong_FromLong(rc);
        if (!dx_fn) return THPVariable_Wrap(dgu);
        const int64_t bytes = reinterpret_cast<GemmBytes>(dx_ws_fn)(M, N, K, 1);
        if (bytes < 0) return PyLong_FromLongLong(bytes);
        at::Tensor dx = shaped(like, K), ws;
        if (bytes) ws = bytes_on(bytes, g);
        rc = reinterpret_cast<GemmDx>(dx_fn)(dgu.data_ptr(), w.packed, w.absmax, nullptr, nullptr, 0, dx.data_ptr(), M, N,
                                             K, w.bs, tag, bytes ? ws.data_ptr() : nullptr, bytes, st);
        if (rc != STM_OK) return PyLong_FromLong(rc);
        return THPVariable_Wrap(dx);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef methods[] = {
    {"collect", py_collect, METH_VARARGS, "addresses, sizes, type and device of a list of tensors"},
    {"bump", bump, METH_O, "count the versions of a list of tensors up"},
    {"grad_norm", grad_norm, METH_VARARGS, "the gradient norm of a list of tensors in its plain form"},
    {"gated_fwd", gated_fwd, METH_VARARGS, "a gated block's forward in its plain form"},
    {"gated_bwd", gated_bwd, METH_VARARGS, "a gated block's backward in its plain form"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", "Host code of launch-bound calls.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern PyMethodDef stm_sparse_methods[];  // sparse_path.cpp

PyMODINIT_FUNC PyInit__fast(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddFunctions(m, stm_sparse_methods) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
