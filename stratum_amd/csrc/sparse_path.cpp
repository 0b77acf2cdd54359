// Host code of the sparse layer's operators (functions of the CPython module stratum_amd._fast): their
// calls and autograd nodes, whose time is the host's where a batch is small. One token through the norm, us a call:
// from Python 15, here 6; 8192 tokens routed with their gradient 102, here 48. A step of torch's own product with a number
// takes 42 to 48 beside it, one of a view 31 to 35: the engine wakes the device's thread. Of the norm's steps one of x takes
// 46, of x and the residual 62, of the weight too 73.
//
// Operands that are not as they have to be are handed back (None): the Python layer says what is wrong with them, or
// converts them (subclasses) or changes the device and calls again.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstdint>
#include <optional>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/stratum_nf4.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library's entry points, whose addresses sparse_setup receives (the library is loaded by ctypes).
struct Library {
    decltype(&stm_last_error) last_error = nullptr;
    decltype(&stm_rms_norm_fwd) norm_fwd = nullptr;
    decltype(&stm_rms_norm_workspace_bytes) norm_bytes = nullptr;
    decltype(&stm_rms_norm_bwd) norm_bwd = nullptr;
    decltype(&stm_moe_route) route = nullptr;
    decltype(&stm_moe_route_bwd) route_bwd = nullptr;
    decltype(&stm_moe_sort_workspace_bytes) sort_bytes = nullptr;
    decltype(&stm_moe_sort) sort = nullptr;
    decltype(&stm_moe_gather) gather = nullptr;
    decltype(&stm_moe_combine) combine = nullptr;
    decltype(&stm_moe_combine_bwd) combine_bwd = nullptr;
} lib;

void check(int64_t rc, const char* what) {
    if (rc < 0) throw std::runtime_error(std::string(what) + ": " + lib.last_error());
}

int tag_of(at::ScalarType t) {
    return t == at::kHalf ? STM_F16 : t == at::kBFloat16 ? STM_BF16 : t == at::kFloat ? STM_F32 : -1;
}

void* stream_on(const c10::Device& d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor like(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
    return at::empty(sizes, t.options().dtype(type).requires_grad(false).memory_format(c10::MemoryFormat::Contiguous));
}

// A tensor as torch's own classes make it (not a subclass with rules of its own), strided, no forward-mode dual.
bool ordinary(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return false;
    const Tensor& t = THPVariable_Unpack(o);
    return t.layout() == at::kStrided && !t._fw_grad(0).defined();
}

// The tensor of an argument, undefined for None.
Tensor tensor_of(PyObject* o) { return o == Py_None ? Tensor() : THPVariable_Unpack(o); }

bool given(PyObject* o) { return o == Py_None || ordinary(o); }

bool on_current(const Tensor& t) {
    return t.is_cuda() && c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice() == t.device();
}

bool beside(const Tensor& t, const Tensor& first) { return !t.defined() || t.device() == first.device(); }

bool recorded(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// The gradients of a node whose backward is not differentiable itself: asked for a graph of it, they are tensors that
// raise when they are differentiated.
variable_list once(variable_list grads, const char* name) {
    if (!at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads) {
        if (!g.defined()) continue;
        const auto error = std::make_shared<torch::autograd::DelayedError>(
            std::string("trying to differentiate twice ") + name + ", which is differentiable once", 1);
        g = (*error)({g.detach().requires_grad_(true)})[0];
    }
    return grads;
}

// The graph that a stream is being captured into (0: none; the null stream cannot be).
unsigned long long capture_of(hipStream_t stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (!stream) return 0;
    if (hipStreamGetCaptureInfo(stream, &status, &id) != hipSuccess) {
        (void)hipGetLastError();
        return 0;
    }
    return status == hipStreamCaptureStatusActive ? id : 0;
}

bool can_join(hipStream_t stream, unsigned long long capture) {
    const unsigned long long own = capture_of(stream);
    return stream && (own == 0 || own == capture);
}

// A gradient that is captured into a graph must end where the capture can follow: torch's engine makes the stream of each
// node wait for the one before, by which a stream becomes part of the capture; but not the null stream, to which a leaf
// is tied by an eager graph from there that still holds it, nor one of another capture. The engine then ends the process.
// So what follows a node in this backward pass is looked through first; what nobody asked for is not followed.
void check_capture(const char* name) {
    const unsigned long long now = capture_of(c10::hip::getCurrentHIPStream().stream());
    if (!now) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    std::vector<torch::autograd::Node*> left{node.get()};
    std::unordered_set<torch::autograd::Node*> seen;
    while (!left.empty()) {
        torch::autograd::Node* n = left.back();
        left.pop_back();
        for (uint32_t i = 0; i < n->num_outputs(); ++i) {
            if (!n->task_should_compute_output(i)) continue;
            torch::autograd::Node* next = n->next_edge(i).function.get();
            if (!seen.insert(next).second) continue;
            const auto stream = next->stream();
            if (stream && !can_join(c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *stream).stream(), now))
                throw std::runtime_error(std::string(name) +
                                         ": its gradient is captured into a graph, but goes on to a leaf of an eager graph, "
                                         "whose stream cannot take part in the capture; capture on leaves of its own "
                                         "(t.detach().requires_grad_()) or let go of the eager graph first");
            left.push_back(next);
        }
    }
}

std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// ------------------------------------------------------------ norm
struct Normed {
    Tensor y, h, rstd;
};

Normed norm_fwd(const Tensor& x, const Tensor& w, double eps, const Tensor& residual, bool keep) {
    const Tensor xc = x.contiguous(), wc = w.contiguous(), rc = residual.defined() ? residual.contiguous() : residual;
    const int64_t cols = x.size(-1), rows = cols ? x.numel() / cols : 0;
    Normed n;
    n.y = like(x, x.sizes(), x.scalar_type());
    if (residual.defined()) n.h = like(x, x.sizes(), residual.scalar_type());
    if (keep) n.rstd = like(x, {rows}, at::kFloat);
    check(lib.norm_fwd(data(xc), data(rc), tag_of((residual.defined() ? residual : x).scalar_type()), data(wc),
                       tag_of(w.scalar_type()), data(n.y), data(n.h), static_cast<float*>(data(n.rstd)), rows, cols, eps,
                       tag_of(x.scalar_type()), stream_on(x.device())),
          "stm_rms_norm_fwd");
    return n;
}

struct NormFn : torch::autograd::Function<NormFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& residual,
                                 double eps) {
        const Normed n = norm_fwd(x, w, eps, residual ? *residual : Tensor(), true);
        ctx->set_materialize_grads(false);
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        // the gradients take the sum's terms where h was rounded to 16 bits
        if (residual && n.h.scalar_type() != at::kFloat)
            ctx->save_for_backward({x, w, n.rstd, *residual});
        else
            ctx->save_for_backward({residual ? n.h : x, w, n.rstd});
        return residual ? variable_list{n.y, n.h} : variable_list{n.y};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_capture("rms_norm");
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &w = saved[1], &rstd = saved[2];
        const bool residual = grads.size() == 2;
        const at::ScalarType type = (at::ScalarType)ctx->saved_data["type"].toInt();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
                   need_r = residual && ctx->needs_input_grad(2);
        Tensor dx, dw, dr;
        if (!grads[0].defined()) {  // only the sum went on
            if (residual && grads[1].defined()) {
                if (need_x) dx = grads[1].to(type);
                if (need_r) dr = grads[1];
            }
        } else {
            const c10::DeviceGuard guard(h.device());
            const Tensor dy = grads[0].contiguous(), hc = h.contiguous(), wc = w.contiguous(),
                         rc = saved.size() == 4 ? saved[3].contiguous() : Tensor();
            const Tensor dh = residual && grads[1].defined() ? grads[1].contiguous() : Tensor();
            const int64_t cols = dy.size(-1), rows = cols ? dy.numel() / cols : 0;
            const bool apart = need_r && h.scalar_type() != type;
            if (need_x || (need_r && !apart)) dx = like(dy, dy.sizes(), type);
            if (apart) dr = like(dy, dy.sizes(), h.scalar_type());
            Tensor ws;
            int64_t bytes = 0;
            if (need_w) {
                check(bytes = lib.norm_bytes(rows, cols), "stm_rms_norm_workspace_bytes");
                dw = like(w, w.sizes(), w.scalar_type());
                ws = like(dy, {bytes / 4}, at::kFloat);
            }
            check(lib.norm_bwd(data(dy), data(dh), data(hc), data(rc), tag_of(h.scalar_type()), static_cast<float*>(data(rstd)),
                               data(wc), tag_of(w.scalar_type()), data(dx), data(dr), data(dw), rows, cols, tag_of(type),
                               data(ws), bytes, stream_on(h.device())),
                  "stm_rms_norm_bwd");
            if (need_r && !apart) dr = dx;
            if (!need_x) dx = Tensor();
        }
        // one gradient per argument of forward
        variable_list out = residual ? once({dx, dw, dr}, "rms_norm") : once({dx, dw}, "rms_norm");
        if (!residual) out.emplace_back();
        out.emplace_back();
        return out;
    }
};

// norm(x, weight, eps, residual or None) -> y, or (y, h); None where the Python layer refuses an operand or has a
// dual to refuse.
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 4 || !ordinary(args[0]) || !ordinary(args[1]) || !given(args[3])) Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(args[2]);
    if (eps == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    HANDLE_TH_ERRORS
    const Tensor x = THPVariable_Unpack(args[0]), w = THPVariable_Unpack(args[1]), r = tensor_of(args[3]);
    if (!on_current(x) || x.dim() < 1 || tag_of(x.scalar_type()) < 0 || !beside(w, x) || !beside(r, x) || w.dim() != 1 ||
        w.size(0) != x.size(-1) || (w.scalar_type() != x.scalar_type() && w.scalar_type() != at::kFloat) || !(eps >= 0.0))
        Py_RETURN_NONE;
    if (r.defined() &&
        (r.sizes() != x.sizes() || (r.scalar_type() != x.scalar_type() && r.scalar_type() != at::kFloat)))
        Py_RETURN_NONE;
    if (recorded({&x, &w, &r})) {
        const variable_list out = NormFn::apply(x, w, maybe(r), eps);
        return r.defined() ? Py_BuildValue("NN", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1])) :
                             THPVariable_Wrap(out[0]);
    }
    const at::NoGradGuard off;
    const Normed out = norm_fwd(x, w, eps, r, false);
    return r.defined() ? Py_BuildValue("NN", THPVariable_Wrap(out.y), THPVariable_Wrap(out.h)) : THPVariable_Wrap(out.y);
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ route
struct RouteArgs {
    Tensor bias, mask;
    int top_k, score, groups, top_groups, sums, renorm;
    double scale;
};

at::DimVector last(const Tensor& t, int64_t width) {
    at::DimVector s(t.sizes().begin(), t.sizes().end());
    s.back() = width;
    return s;
}

std::pair<Tensor, Tensor> route_fwd(const Tensor& logits, const RouteArgs& a) {
    const Tensor l = logits.contiguous(), b = a.bias.defined() ? a.bias.contiguous() : a.bias,
                 m = a.mask.defined() ? a.mask.contiguous() : a.mask;
    const int64_t E = logits.size(-1);
    const at::DimVector sizes = last(logits, a.top_k);
    Tensor weights = like(logits, sizes, at::kFloat), experts = like(logits, sizes, at::kInt);
    check(lib.route(data(l), static_cast<const float*>(data(b)), static_cast<const uint8_t*>(data(m)),
                    static_cast<float*>(data(weights)), static_cast<int32_t*>(data(experts)), logits.numel() / E, (int)E,
                    a.top_k, a.score, a.groups, a.top_groups, a.sums, a.renorm, a.scale, tag_of(logits.scalar_type()),
                    stream_on(logits.device())),
          "stm_moe_route");
    return {weights, experts};
}

struct RouteFn : torch::autograd::Function<RouteFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const RouteArgs* a) {
        const auto [weights, experts] = route_fwd(logits, *a);
        ctx->saved_data["args"] = c10::IValue(std::vector<double>{(double)a->top_k, (double)a->score, (double)a->renorm, a->scale});
        ctx->save_for_backward({logits, experts});
        ctx->mark_non_differentiable({experts});
        ctx->set_materialize_grads(false);
        return {weights, experts};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_capture("moe_route");
        const variable_list saved = ctx->get_saved_variables();
        const auto args = ctx->saved_data["args"].toDoubleVector();
        if (!grads[0].defined()) return {Tensor(), Tensor()};
        const c10::DeviceGuard guard(saved[0].device());
        const Tensor l = saved[0].contiguous(), e = saved[1], dw = grads[0].contiguous();
        const int64_t E = l.size(-1);
        Tensor dl = like(l, l.sizes(), l.scalar_type());
        check(lib.route_bwd(static_cast<const float*>(data(dw)), data(l), static_cast<const int32_t*>(data(e)), data(dl),
                            l.numel() / E, (int)E, (int)args[0], (int)args[1], (int)args[2], args[3],
                            tag_of(l.scalar_type()), stream_on(l.device())),
              "stm_moe_route_bwd");
        variable_list out = once({dl}, "moe_route");
        out.emplace_back();
        return out;
    }
};

// route(logits, bias, mask, top_k, score, groups, top_groups, sums, renormalize, scale) -> (weights, experts) or None
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 10 || !ordinary(args[0]) || !given(args[1]) || !given(args[2])) Py_RETURN_NONE;
    long v[6];
    for (int i = 0; i < 6; ++i) v[i] = PyLong_AsLong(args[3 + i]);
    RouteArgs a;
    a.scale = PyFloat_AsDouble(args[9]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    HANDLE_TH_ERRORS
    const Tensor x = THPVariable_Unpack(args[0]);
    a.bias = tensor_of(args[1]), a.mask = tensor_of(args[2]);
    if (!on_current(x) || x.dim() < 1 || tag_of(x.scalar_type()) < 0 || !beside(a.bias, x) || !beside(a.mask, x)) Py_RETURN_NONE;
    const int64_t E = x.size(-1);
    if (E < 1 || E > 1024 || v[0] < 1 || v[0] > 64 || v[0] > E || v[2] < 1 || v[2] > 64 || E % v[2] || v[3] < 1 ||
        v[3] > v[2] || v[0] > E / v[2] * v[3] || x.numel() / E >= (1ll << 31) / v[0])
        Py_RETURN_NONE;
    if (a.bias.defined() && (a.bias.scalar_type() != at::kFloat || a.bias.dim() != 1 || a.bias.size(0) != E)) Py_RETURN_NONE;
    if (a.mask.defined() &&
        (a.mask.scalar_type() != at::kBool || a.mask.sizes() != x.sizes().slice(0, x.dim() - 1)))
        Py_RETURN_NONE;
    a.top_k = (int)v[0], a.score = (int)v[1], a.groups = (int)v[2], a.top_groups = (int)v[3], a.sums = (int)v[4],
    a.renorm = (int)v[5];
    if (recorded({&x})) {
        const variable_list out = RouteFn::apply(x, &a);
        return Py_BuildValue("NN", THPVariable_Wrap(out[0]), THPVariable_Wrap(out[1]));
    }
    const at::NoGradGuard off;
    const auto out = route_fwd(x, a);
    return Py_BuildValue("NN", THPVariable_Wrap(out.first), THPVariable_Wrap(out.second));
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ sort, gather, combine
// sort(experts, num_experts) -> (offsets, slots, positions) or None
PyObject* sort(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2 || !THPVariable_CheckExact(args[0])) Py_RETURN_NONE;
    const long E = PyLong_AsLong(args[1]);
    if (E == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    HANDLE_TH_ERRORS
    const Tensor& e = THPVariable_Unpack(args[0]);
    if (e.layout() != at::kStrided || !on_current(e) || e.scalar_type() != at::kInt || e.dim() < 1 || E < 1 || E > 1024 ||
        e.numel() > INT_MAX)
        Py_RETURN_NONE;
    const Tensor ec = e.contiguous();
    const int64_t slots = e.numel(), bytes = lib.sort_bytes(slots, (int)E);
    check(bytes, "stm_moe_sort_workspace_bytes");
    Tensor offsets = like(e, {E + 1}, at::kInt), order = like(e, {slots}, at::kInt), positions = like(e, e.sizes(), at::kInt),
           ws;
    if (bytes) ws = like(e, {bytes / 4}, at::kInt);
    check(lib.sort(static_cast<const int32_t*>(data(ec)), slots, (int)E, static_cast<int32_t*>(data(offsets)),
                   static_cast<int32_t*>(data(order)), static_cast<int32_t*>(data(positions)), data(ws), bytes,
                   stream_on(e.device())),
          "stm_moe_sort");
    return Py_BuildValue("NNN", THPVariable_Wrap(offsets), THPVariable_Wrap(order), THPVariable_Wrap(positions));
    END_HANDLE_TH_ERRORS
}

struct Order {
    Tensor offsets, slots, positions;
    int64_t tokens = 0, top_k = 0;

    bool read(PyObject* o) {
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 3) return false;
        Tensor* t[3] = {&offsets, &slots, &positions};
        for (int i = 0; i < 3; ++i) {
            if (!THPVariable_CheckExact(PyTuple_GET_ITEM(o, i))) return false;
            *t[i] = THPVariable_Unpack(PyTuple_GET_ITEM(o, i));
            if (t[i]->layout() != at::kStrided || t[i]->scalar_type() != at::kInt || !t[i]->is_contiguous() ||
                t[i]->device() != offsets.device())
                return false;
        }
        if (positions.dim() < 1 || slots.numel() != positions.numel() || offsets.numel() < 2 || offsets.numel() > INT_MAX ||
            positions.size(-1) < 1 || positions.numel() > INT_MAX)
            return false;
        top_k = positions.size(-1), tokens = positions.numel() / top_k;
        return true;
    }
};

const int32_t* ints(const Tensor& t) { return static_cast<const int32_t*>(data(t)); }

Tensor gather_fwd(const Tensor& x, const Order& o) {
    const Tensor xc = x.contiguous();
    const int64_t hidden = x.size(-1);
    Tensor out = like(x, {o.tokens * o.top_k, hidden}, x.scalar_type());
    check(lib.gather(data(xc), ints(o.positions), ints(o.offsets), (int)o.offsets.numel() - 1, data(out), o.tokens,
                     (int)o.top_k, hidden, tag_of(x.scalar_type()), stream_on(x.device())),
          "stm_moe_gather");
    return out;
}

Tensor combine_fwd(const Tensor& y, const Tensor& weights, const Tensor& positions, const Tensor& residual,
                   at::IntArrayRef sizes) {
    const Tensor yc = y.contiguous(), w = weights.defined() ? weights.contiguous() : weights,
                 r = residual.defined() ? residual.contiguous() : residual;
    const int64_t top_k = positions.size(-1);
    Tensor out = like(y, sizes, (r.defined() ? r : y).scalar_type());
    check(lib.combine(data(yc), y.size(0), static_cast<const float*>(data(w)), ints(positions), data(r), data(out),
                      tag_of(out.scalar_type()), positions.numel() / top_k, (int)top_k, y.size(1), tag_of(y.scalar_type()),
                      stream_on(y.device())),
          "stm_moe_combine");
    return out;
}

struct GatherFn : torch::autograd::Function<GatherFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Order* o) {
        ctx->save_for_backward({o->positions});
        ctx->saved_data["sizes"] = x.sizes().vec();
        return gather_fwd(x, *o);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_capture("moe_gather");
        const c10::DeviceGuard guard(grads[0].device());
        const Tensor dx = combine_fwd(grads[0], Tensor(), ctx->get_saved_variables()[0], Tensor(),
                                      ctx->saved_data["sizes"].toIntVector());
        variable_list out = once({dx}, "moe_gather");
        out.emplace_back();
        return out;
    }
};

// gather(x, order) -> rows or None
PyObject* gather(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 2 || !ordinary(args[0])) Py_RETURN_NONE;
    HANDLE_TH_ERRORS
    const Tensor x = THPVariable_Unpack(args[0]);
    Order o;
    if (!o.read(args[1]) || !on_current(x) || !beside(o.offsets, x) || tag_of(x.scalar_type()) < 0 || x.dim() < 2 ||
        x.numel() != o.tokens * x.size(-1))
        Py_RETURN_NONE;
    if (recorded({&x})) return THPVariable_Wrap(GatherFn::apply(x, &o));
    const at::NoGradGuard off;
    return THPVariable_Wrap(gather_fwd(x, o));
    END_HANDLE_TH_ERRORS
}

struct CombineFn : torch::autograd::Function<CombineFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& weights, const std::optional<Tensor>& residual,
                          const Order* o, const at::DimVector* sizes) {
        // (what neither gradient needs is not kept)
        const bool need_y = y.requires_grad(), need_w = weights.requires_grad();
        ctx->save_for_backward({need_w ? y : Tensor(), need_y ? weights : Tensor(), o->offsets, o->positions});
        ctx->saved_data["y"] = std::vector<int64_t>{y.size(0), y.size(1), (int64_t)y.scalar_type(), residual.has_value()};
        return combine_fwd(y, weights, o->positions, residual ? *residual : Tensor(), *sizes);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_capture("moe_combine");
        const variable_list saved = ctx->get_saved_variables();
        const auto y_is = ctx->saved_data["y"].toIntVector();
        const Tensor &y = saved[0], &weights = saved[1], &offsets = saved[2], &positions = saved[3];
        const at::ScalarType type = (at::ScalarType)y_is[2];
        const bool need_y = ctx->needs_input_grad(0) && weights.defined(), need_w = ctx->needs_input_grad(1) && y.defined();
        Tensor dy, dw;
        if (need_y || need_w) {
            const c10::DeviceGuard guard(grads[0].device());
            const Tensor g = grads[0].contiguous(), yc = need_w ? y.contiguous() : Tensor(),
                         w = need_y ? weights.contiguous() : Tensor();
            if (need_y) dy = like(g, {y_is[0], y_is[1]}, type);
            if (need_w) dw = like(g, positions.sizes(), at::kFloat);
            const int64_t top_k = positions.size(-1);
            check(lib.combine_bwd(data(g), tag_of(g.scalar_type()), data(yc), y_is[0], static_cast<const float*>(data(w)),
                                  ints(positions), ints(offsets), (int)offsets.numel() - 1, data(dy),
                                  static_cast<float*>(data(dw)), positions.numel() / top_k, (int)top_k, y_is[1], tag_of(type),
                                  stream_on(g.device())),
                  "stm_moe_combine_bwd");
        }
        variable_list out = once({dy, dw}, "moe_combine");
        out.push_back(y_is[3] && ctx->needs_input_grad(2) ? grads[0] : Tensor());  // the residual's
        out.resize(5);
        return out;
    }
};

// combine(y, weights, order, residual or None) -> out or None
PyObject* combine(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 4 || !ordinary(args[0]) || !ordinary(args[1]) || !given(args[3])) Py_RETURN_NONE;
    HANDLE_TH_ERRORS
    const Tensor y = THPVariable_Unpack(args[0]), w = THPVariable_Unpack(args[1]), r = tensor_of(args[3]);
    Order o;
    if (!o.read(args[2]) || !on_current(y) || !beside(o.offsets, y) || !beside(w, y) || !beside(r, y) ||
        tag_of(y.scalar_type()) < 0 || y.dim() != 2 || y.size(0) > o.tokens * o.top_k ||
        w.scalar_type() != at::kFloat || w.sizes() != o.positions.sizes())
        Py_RETURN_NONE;
    if (r.defined() && ((r.scalar_type() != y.scalar_type() && r.scalar_type() != at::kFloat) || r.dim() < 1 ||
                        r.size(-1) != y.size(1) || r.numel() != o.tokens * y.size(1)))
        Py_RETURN_NONE;
    const at::DimVector sizes = r.defined() ? at::DimVector(r.sizes().begin(), r.sizes().end()) : last(w, y.size(1));
    if (recorded({&y, &w, &r})) return THPVariable_Wrap(CombineFn::apply(y, w, maybe(r), &o, &sizes));
    const at::NoGradGuard off;
    return THPVariable_Wrap(combine_fwd(y, w, o.positions, r, sizes));
    END_HANDLE_TH_ERRORS
}

// sparse_setup(addresses of Library's entries, in their order)
PyObject* sparse_setup(PyObject*, PyObject* list) {
    constexpr Py_ssize_t count = sizeof(Library) / sizeof(void*);
    if (!PyList_Check(list) || PyList_GET_SIZE(list) != count) {
        PyErr_SetString(PyExc_TypeError, "a list of the library's addresses");
        return nullptr;
    }
    void** entries = reinterpret_cast<void**>(&lib);
    for (Py_ssize_t i = 0; i < count; ++i) {
        entries[i] = PyLong_AsVoidPtr(PyList_GET_ITEM(list, i));
        if (!entries[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
            return nullptr;
        }
    }
    Py_RETURN_NONE;
}

}  // namespace

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f))
extern PyMethodDef stm_sparse_methods[];
PyMethodDef stm_sparse_methods[] = {
    {"sparse_setup", sparse_setup, METH_O, "the addresses of the library's entry points"},
    {"norm", FAST(norm), METH_FASTCALL, "the norm with its autograd node"},
    {"route", FAST(route), METH_FASTCALL, "a router's choice with its autograd node"},
    {"sort", FAST(sort), METH_FASTCALL, "the order of slots by expert"},
    {"gather", FAST(gather), METH_FASTCALL, "rows by expert with their autograd node"},
    {"combine", FAST(combine), METH_FASTCALL, "rows back to their tokens with their autograd node"},
    {nullptr, nullptr, 0, nullptr},
};
