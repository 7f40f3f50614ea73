// mtk_torch.cpp — torch's side of the small entry points: a CPython module that checks tensors, allocates results, calls the C ABI and, where
// autograd asks, is the node of the graph.
//
// A launch costs some microseconds; reading the shapes, types and addresses of a call's tensors in Python and converting twenty arguments costs
// several times that, a backward pass through a Python node more again (its thread waits for the interpreter), and a step over hundreds of
// tensors more than its kernels.  Each function here takes the ordinary case of a call and does it all at once.  Whatever it does not
// recognise (another device than the current one, strides it would have to copy, shapes that do not fit, a refusal by the library's
// checks) it leaves alone and returns None: the Python layer then makes the arguments ordinary and calls again, or raises.
// The library's functions come by address (bind), so there is one copy of it, wherever it was loaded from.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "mtk.h"

namespace {

struct Table {
    decltype(&mtk_last_error) last_error;
    decltype(&mtk_route_rows_work) route_rows_work;
    decltype(&mtk_route_rows) route_rows;
    decltype(&mtk_rows_dispatch) rows_dispatch;
    decltype(&mtk_rows_combine) rows_combine;
    decltype(&mtk_adapter_saved_bytes) saved_bytes;
    decltype(&mtk_adapter_streams) streams;
    decltype(&mtk_adapter_work_bytes) work_bytes;
    decltype(&mtk_adapter_forward) adapter_forward;
    decltype(&mtk_adapter_backward) adapter_backward;
    decltype(&mtk_adamw_step) adamw_step;
    decltype(&mtk_adamw_step_each) adamw_step_each;
};
constexpr int kEntries = sizeof(Table) / sizeof(void*);
union {
    Table fn;
    void* at[kEntries];
} lib = {};

struct Decline {};  // thrown to leave a call to the Python layer
thread_local std::string refusal;  // what the library said, where the last decline was its own

void need(bool ok) {
    if (!ok) throw Decline();
}
const at::Tensor& tensor(PyObject* o) {
    need(THPVariable_Check(o));
    return THPVariable_Unpack(o);
}
at::Tensor maybe(PyObject* o) { return o == Py_None ? at::Tensor() : tensor(o); }  // undefined for None
int code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MTK_DT_F32;
        case at::kBFloat16: return MTK_DT_BF16;
        case at::kHalf: return MTK_DT_F16;
        default: throw Decline();
    }
}
// on the current device, strided, an ordinary tensor
void here(const at::Tensor& t, int device) { need(t.is_cuda() && t.device().index() == device && t.layout() == at::kStrided && t.has_storage()); }
void dense(const at::Tensor& t, int device) {
    here(t, device);
    need(t.is_contiguous());
}
int current(const at::Tensor& t) {
    need(t.is_cuda());
    const int d = c10::hip::current_device();
    need(t.device().index() == d);
    return d;
}
mtk_stream stream_of(int device) { return (mtk_stream)c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }
// rows whose elements lie side by side, at any distance from each other
void rows(const at::Tensor& t, int device) {
    here(t, device);
    need(t.dim() == 2 && t.size(1) >= 1 && (t.stride(1) == 1 || t.size(1) == 1 || t.size(0) == 0) && t.stride(0) >= 0);
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
at::Tensor like(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type) { return at::empty(sizes, t.options().dtype(type).requires_grad(false)); }
int64_t integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Decline();
    }
    return v;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Decline();
    }
    return v;
}
template <typename F> void call(F f) {  // a library call without the interpreter's lock, where this thread has it
    int rc;
    {
        struct Unlocked {
            PyThreadState* s = PyGILState_Check() ? PyEval_SaveThread() : nullptr;
            ~Unlocked() {
                if (s) PyEval_RestoreThread(s);
            }
        } unlocked;
        rc = f();
    }
    if (rc == MTK_ERR_ARG || rc == MTK_ERR_UNSUPPORTED) {
        refusal = lib.fn.last_error();
        throw Decline();
    }
    if (rc != MTK_OK) throw std::runtime_error(std::string("libmtk_hip: ") + lib.fn.last_error());
}
PyObject* pack(std::initializer_list<at::Tensor> ts) {
    PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) PyTuple_SET_ITEM(out, i++, t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None));
    return out;
}
// the body of a module function: a decline is None; an error of torch's, or of a hook in Python, is the exception that torch's own functions raise
template <typename F> PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", n, want);
        return nullptr;
    }
    try {
        refusal.clear();
        return f();
    } catch (const Decline&) {
        Py_RETURN_NONE;
    } catch (const std::exception&) {
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "midst_toolkit_amd: unknown C++ exception");
        return nullptr;
    }
}
bool tracked(std::initializer_list<at::Tensor> ts) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const at::Tensor& t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
// The nodes go backward only, on tensors with memory: a tangent that the result would lose, or a functional transform's tensor, is left to the
// Python layer, which refuses it.
void plain(std::initializer_list<at::Tensor> ts) {
    for (const at::Tensor& t : ts) need(!t.defined() || (t.has_storage() && !t._fw_grad(0).defined()));
}
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
// The nodes differentiate once: a second time raises where it is tried.
variable_list once(const variable_list& grads, variable_list out, const char* what) {
    bool again = false;
    for (const at::Tensor& g : grads) again |= g.defined() && g.requires_grad();
    if (!again || !c10::GradMode::is_enabled()) return out;
    for (at::Tensor& t : out)
        if (t.defined()) t = t.detach().requires_grad_(true);
    return (*std::make_shared<torch::autograd::DelayedError>(std::string(what) + " differentiates once only", (int64_t)out.size()))(std::move(out));
}
// A node runs on the stream that was current when it was made, a leaf's accumulator on that of the first graph that needed it and still lives.  Where
// that is the default stream, a captured backward pass would make the default stream wait for the capture, which no stream outside of one
// may; the process did not survive it.
bool on_default_stream(torch::autograd::Node* node) {
    if (!node) return false;
    const auto s = node->stream();
    return s && s->id() == 0;
}
void may_capture(const char* what) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const auto* only = torch::autograd::get_current_graph_task_exec_info();  // torch.autograd.grad: the nodes on the way to what it asks for, and those
    for (const torch::autograd::Edge& e : node->next_edges()) {
        if (!on_default_stream(e.function.get())) continue;
        if (only && !only->empty()) {
            const auto it = only->find(e.function.get());
            if (it == only->end() || !it->second.should_execute()) continue;
        }
        throw std::runtime_error(std::string(what) + ": a captured backward pass, whose gradient an eager graph's node would take on the default stream: let go of the eager graphs of the same "
                                                     "parameters (their losses and outputs) before the capture");
    }
}
template <typename F> variable_list backward_of(const char* what, const at::Tensor& like_, F f) {
    const c10::DeviceGuard guard(like_.device());
    may_capture(what);
    try {
        return f();
    } catch (const Decline&) {
        throw std::runtime_error(std::string(what) + ": a gradient or saved tensor does not fit, or is no plain tensor (batched gradients are not offered)");
    }
}

// bind((address, ...)): the library's functions in Table's order
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, kEntries, [&]() -> PyObject* {
        for (int i = 0; i < kEntries; ++i) lib.at[i] = (void*)(intptr_t)integer(a[i]);
        Py_RETURN_TRUE;
    });
}

// declined() -> what the library said to this thread's last call that returned None; empty where its tensors were the reason
PyObject* declined(PyObject*, PyObject*) { return PyUnicode_FromString(refusal.c_str()); }

// accumulates_on_default(tensor) -> whether the tensor's gradient goes to a node of the default stream: what may_capture refuses
PyObject* accumulates_on_default(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 1, [&]() -> PyObject* {
        const at::Tensor& t = tensor(a[0]);
        const auto node = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
        return PyBool_FromLong(on_default_stream(node.get()));
    });
}

// route(index, n_groups) -> (order, slot, offsets)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 2, [&]() -> PyObject* {
        const at::Tensor& index = tensor(a[0]);
        const int64_t groups = integer(a[1]);
        const int d = current(index);
        dense(index, d);
        need(index.scalar_type() == at::kLong && (index.dim() == 1 || (index.dim() == 2 && index.size(1) >= 1)) && groups >= 1 && groups <= MTK_ROUTE_MAX_GROUPS);
        const int64_t P = index.numel();
        need(P <= 0x7fffffff);
        const int64_t w = lib.fn.route_rows_work(P, (int)groups);
        at::Tensor order = like(index, {P}, at::kInt), slot = like(index, index.sizes(), at::kInt), offsets = like(index, {groups + 1}, at::kInt), work;
        if (w) work = like(index, {w}, at::kInt);
        call([&] {
            return lib.fn.route_rows(P, index.const_data_ptr<int64_t>(), (int)groups, (int32_t*)ptr(order), (int32_t*)ptr(slot), (int32_t*)ptr(offsets), (int32_t*)ptr(work), w,
                                     stream_of(d));
        });
        return pack({order, slot, offsets});
    });
}

struct Pairs {  // of a plan
    at::Tensor slot;
    int64_t N, k;
    void check(int device) const {
        dense(slot, device);
        need(k >= 1 && N >= 0 && slot.numel() == N * k && slot.scalar_type() == at::kInt);
    }
    void weights(const at::Tensor& w, int device) const {
        if (!w.defined()) return;
        dense(w, device);
        need(w.scalar_type() == at::kFloat && w.dim() == 2 && w.size(0) == N && w.size(1) == k);
    }
};
// (xs if wanted, dw if y is given)
std::pair<at::Tensor, at::Tensor> rows_out(const at::Tensor& x, const Pairs& p, const at::Tensor& w, const at::Tensor& y, bool want) {
    const int d = current(x), dt = code(x);
    rows(x, d);
    p.check(d);
    p.weights(w, d);
    const int64_t D = x.size(1);
    need(x.size(0) == p.N);
    if (y.defined()) {
        dense(y, d);
        need(y.scalar_type() == x.scalar_type() && y.dim() == 2 && y.size(0) == p.N * p.k && y.size(1) == D);
    }
    at::Tensor xs, dw;
    if (want) xs = like(x, {p.N * p.k, D}, x.scalar_type());
    if (y.defined()) dw = like(x, {p.N, p.k}, at::kFloat);
    if (p.N && (want || y.defined()))
        call([&] {
            return lib.fn.rows_dispatch(p.N, (int)p.k, D, dt, ptr(x), x.stride(0), (const int32_t*)ptr(p.slot), (const float*)ptr(w), ptr(xs), ptr(y), (float*)ptr(dw), stream_of(d));
        });
    return {xs, dw};
}
at::Tensor rows_back(const at::Tensor& y, const Pairs& p, const at::Tensor& w) {
    const int d = current(y), dt = code(y);
    rows(y, d);
    p.check(d);
    p.weights(w, d);
    need(y.size(0) == p.N * p.k);
    at::Tensor out = like(y, {p.N, y.size(1)}, y.scalar_type());
    if (p.N)
        call([&] {
            return lib.fn.rows_combine(p.N, (int)p.k, y.size(1), dt, ptr(y), y.stride(0), (const int32_t*)ptr(p.slot), (const float*)ptr(w), ptr(out), stream_of(d));
        });
    return out;
}
at::Tensor as_rows(const at::Tensor& g) { return g.size(0) == 0 || ((g.stride(1) == 1 || g.size(1) == 1) && g.stride(0) >= 0) ? g : g.contiguous(); }

struct DispatchNode : torch::autograd::Function<DispatchNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& slot, int64_t N, int64_t k) {
        ctx->save_for_backward({slot});
        ctx->saved_data["N"] = N;
        ctx->saved_data["k"] = k;
        return rows_out(x, Pairs{slot, N, k}, {}, {}, true).first;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const Pairs p{ctx->get_saved_variables()[0], ctx->saved_data["N"].toInt(), ctx->saved_data["k"].toInt()};
        return backward_of("dispatch_rows", p.slot, [&] { return once(grads, {rows_back(as_rows(grads[0]), p, {}), {}, {}, {}}, "dispatch_rows"); });
    }
};
std::optional<at::Tensor> given(const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }
// (needs_input_grad counts the tensors that are given: what may be absent comes last)
struct CombineNode : torch::autograd::Function<CombineNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& slot, const std::optional<at::Tensor>& weights, int64_t N, int64_t k) {
        const at::Tensor w = weights.value_or(at::Tensor());
        at::Tensor keep;
        if (w.defined() && w.requires_grad()) keep = y;
        ctx->save_for_backward({keep, w, slot});
        ctx->saved_data["N"] = N;
        ctx->saved_data["k"] = k;
        return rows_back(y, Pairs{slot, N, k}, w);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Pairs p{saved[2], ctx->saved_data["N"].toInt(), ctx->saved_data["k"].toInt()};
        return backward_of("combine_rows", p.slot, [&] {
            const bool want_w = saved[1].defined() && saved[0].defined() && ctx->needs_input_grad(2);
            auto got = rows_out(as_rows(grads[0]), p, saved[1], want_w ? saved[0].contiguous() : at::Tensor(), ctx->needs_input_grad(0));
            return once(grads, {got.first, {}, got.second, {}, {}}, "combine_rows");
        });
    }
};

// dispatch(x, slot, n_rows, copies) -> xs
PyObject* dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 4, [&]() -> PyObject* {
        const at::Tensor& x = tensor(a[0]);
        const Pairs p{tensor(a[1]), integer(a[2]), integer(a[3])};
        plain({x});
        return THPVariable_Wrap(tracked({x}) ? DispatchNode::apply(x, p.slot, p.N, p.k) : rows_out(x, p, {}, {}, true).first);
    });
}
// combine(y, slot, n_rows, copies, weights | None) -> out
PyObject* combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 5, [&]() -> PyObject* {
        const at::Tensor& y = tensor(a[0]);
        const Pairs p{tensor(a[1]), integer(a[2]), integer(a[3])};
        const at::Tensor w = maybe(a[4]);
        plain({y, w});
        return THPVariable_Wrap(tracked({y, w}) ? CombineNode::apply(y, p.slot, given(w), p.N, p.k) : rows_back(y, p, w));
    });
}

struct Layer {  // an adapted layer's arguments, checked
    at::Tensor x, weight, down, up, offsets, bias, scales;
    double scale;
    int act, device, dt, din, dout, r, E;
    int64_t M;
    void check() {
        device = current(x);
        dt = code(x);
        rows(x, device);
        for (const at::Tensor* t : {&weight, &down, &up}) {
            dense(*t, device);
            need(t->scalar_type() == x.scalar_type());
        }
        dense(offsets, device);
        need(weight.dim() == 2 && down.dim() == 3 && up.dim() == 3 && offsets.dim() == 1 && offsets.scalar_type() == at::kInt);
        need(weight.size(0) <= MTK_ADAPTER_MAX_WIDTH && weight.size(1) <= MTK_ADAPTER_MAX_WIDTH && down.size(0) <= MTK_ROUTE_MAX_GROUPS && down.size(1) <= MTK_ADAPTER_MAX_RANK);
        M = x.size(0);
        din = (int)x.size(1), dout = (int)weight.size(0), E = (int)down.size(0), r = (int)down.size(1);
        need(dout >= 1 && E >= 1 && r >= 1 && weight.size(1) == din && down.size(2) == din && up.size(0) == E && up.size(1) == dout && up.size(2) == r && offsets.size(0) == E + 1);
        if (bias.defined()) {
            dense(bias, device);
            need(bias.scalar_type() == x.scalar_type() && bias.dim() == 1 && bias.size(0) == dout);
        }
        if (scales.defined()) {
            dense(scales, device);
            need(scales.scalar_type() == at::kFloat && scales.dim() == 1 && scales.size(0) == E);
        }
    }
    at::Tensor bytes(int64_t n) const { return n ? like(x, {n}, at::kByte) : at::Tensor(); }
    // y, and in `saved` what the backward reads
    at::Tensor forward(bool keep, at::Tensor& saved) {
        check();
        at::Tensor y = like(x, {M, dout}, x.scalar_type());
        const int64_t saved_bytes = lib.fn.saved_bytes(M, r, dt), work_bytes = lib.fn.work_bytes(M, din, dout, r, E, dt, act, 0, lib.fn.streams(ptr(x), x.stride(0), din, dt),
                                                                                                              lib.fn.streams(ptr(weight), din, din, dt));
        saved = like(x, {saved_bytes}, at::kByte);
        const at::Tensor work = bytes(work_bytes);
        if (M)
            call([&] {
                return lib.fn.adapter_forward(M, din, dout, r, E, dt, ptr(x), x.stride(0), ptr(weight), ptr(bias), ptr(down), ptr(up), (const int32_t*)ptr(offsets), (const float*)ptr(scales),
                                              scale, act, keep, ptr(y), ptr(saved), saved_bytes, ptr(work), work_bytes, stream_of(device));
            });
        return y;
    }
    variable_list backward(const at::Tensor& y, const at::Tensor& dy, const at::Tensor& saved, bool want_x, bool want_down, bool want_up) {
        check();
        dense(dy, device);
        need(dy.scalar_type() == x.scalar_type() && dy.dim() == 2 && dy.size(0) == M && dy.size(1) == dout);
        need(act == MTK_ACT_NONE || (y.defined() && y.is_contiguous() && y.sizes() == dy.sizes() && y.scalar_type() == x.scalar_type()));
        at::Tensor dx, ddown, dup;
        if (want_x) dx = like(x, {M, din}, x.scalar_type());
        if (want_down) ddown = M ? like(x, down.sizes(), x.scalar_type()) : at::zeros(down.sizes(), x.options().requires_grad(false));
        if (want_up) dup = M ? like(x, up.sizes(), x.scalar_type()) : at::zeros(up.sizes(), x.options().requires_grad(false));
        const int64_t work_bytes = lib.fn.work_bytes(M, din, dout, r, E, dt, act, 1, lib.fn.streams(act ? nullptr : ptr(dy), dout, dout, dt), 0);
        const at::Tensor work = bytes(work_bytes);
        if (M && (want_x || want_down || want_up))
            call([&] {
                return lib.fn.adapter_backward(M, din, dout, r, E, dt, ptr(x), x.stride(0), ptr(weight), ptr(down), ptr(up), (const int32_t*)ptr(offsets), (const float*)ptr(scales), scale, act,
                                               ptr(y), ptr(dy), ptr(saved), ptr(dx), ptr(ddown), ptr(dup), ptr(work), work_bytes, stream_of(device));
            });
        return {dx, ddown, dup};
    }
};

struct AdapterNode : torch::autograd::Function<AdapterNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& down, const at::Tensor& up, const at::Tensor& weight, const at::Tensor& offsets,
                              const std::optional<at::Tensor>& bias, const std::optional<at::Tensor>& scales_, double scale, int64_t act) {
        const at::Tensor scales = scales_.value_or(at::Tensor());
        Layer l{x, weight, down, up, offsets, bias.value_or(at::Tensor()), scales, scale, (int)act};
        at::Tensor saved;
        const at::Tensor y = l.forward(true, saved);
        ctx->save_for_backward({x, down, up, weight, offsets, scales, act ? y : at::Tensor(), saved});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const variable_list s = ctx->get_saved_variables();
        return backward_of("adapter_linear", s[0], [&] {
            Layer l{s[0], s[3], s[1], s[2], s[4], {}, s[5], ctx->saved_data["scale"].toDouble(), (int)ctx->saved_data["act"].toInt()};
            variable_list out = l.backward(s[6], grads[0].contiguous(), s[7], ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2));
            out.resize(9);
            return once(grads, std::move(out), "adapter_linear");
        });
    }
};

// adapter(x, weight, bias | None, down, up, offsets, scale, act) -> y.  A shared layer or scale that autograd tracks is declined.
PyObject* adapter(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        Layer l{tensor(a[0]), tensor(a[1]), tensor(a[3]), tensor(a[4]), tensor(a[5]), maybe(a[2]), {}, 1.0, (int)integer(a[7])};
        if (THPVariable_Check(a[6])) l.scales = tensor(a[6]);
        else l.scale = real(a[6]);
        need(!tracked({l.weight, l.bias, l.scales}));
        plain({l.x, l.weight, l.bias, l.down, l.up, l.scales});
        at::Tensor saved;
        if (!tracked({l.x, l.down, l.up})) return THPVariable_Wrap(l.forward(false, saved));
        return THPVariable_Wrap(AdapterNode::apply(l.x, l.down, l.up, l.weight, l.offsets, given(l.bias), given(l.scales), l.scale, (int64_t)l.act));
    });
}

struct Span {  // a tensor's memory
    uintptr_t at, end;
    bool operator<(const Span& o) const { return at < o.at; }
};
// What a step writes lies apart; a gradient is none of it but its own parameter's memory.  `written` becomes sorted: a list at a time, as lists
// often are in order, and merged (1,152 tensors: 8 us less than one sort).
bool apart(std::vector<Span>& written, const std::vector<size_t>& lists, const std::vector<Span>& params, const std::vector<Span>& grads) {
    const auto first = written.begin();
    for (size_t i = 0; i + 1 < lists.size(); ++i) {
        const auto from = first + lists[i], to = first + lists[i + 1];
        if (!std::is_sorted(from, to)) std::sort(from, to);
        if (i && from != first && from != to && *from < *(from - 1)) std::inplace_merge(first, from, to);
    }
    for (size_t i = 1; i < written.size(); ++i)
        if (written[i].at < written[i - 1].end) return false;
    auto next = first;  // the first that begins behind a gradient: near the last one's, where gradients are in order
    for (size_t j = 0; j < grads.size(); ++j) {
        const Span &g = grads[j], &p = params[j];
        if (g.at == g.end || (g.at == p.at && g.end == p.end)) continue;
        if ((next != written.end() && next->at < g.end) || (next != first && (next - 1)->at >= g.end)) next = std::lower_bound(written.begin(), written.end(), Span{g.end, 0});
        if (next != first && (next - 1)->end > g.at) return false;
    }
    return true;
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, scales | None, scales | None, step, lr, beta1, beta2, eps, weight_decay, hyper | None) -> True
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 13, [&]() -> PyObject* {
        const bool q8 = a[4] != Py_None;
        need(q8 == (a[5] != Py_None));
        const int lists = q8 ? 6 : 4;
        struct Held {
            PyObject* o[6] = {};
            ~Held() {
                for (PyObject* p : o) Py_XDECREF(p);
            }
        } held;
        for (int i = 0; i < lists; ++i) {
            held.o[i] = PySequence_Fast(a[i], "");
            if (!held.o[i]) {
                PyErr_Clear();
                throw Decline();
            }
        }
        const Py_ssize_t count = PySequence_Fast_GET_SIZE(held.o[0]);
        need(count >= 1);
        for (int i = 1; i < lists; ++i) need(PySequence_Fast_GET_SIZE(held.o[i]) == count);
        const at::Tensor& p0 = tensor(PySequence_Fast_GET_ITEM(held.o[0], 0));
        const int d = current(p0), dt = code(p0);
        const at::ScalarType type = p0.scalar_type();
        std::vector<void*> at[6];
        std::vector<int64_t> numel((size_t)count);
        std::vector<Span> written, spans[2];  // params, grads
        std::vector<size_t> starts;           // of the lists in `written`
        written.reserve((size_t)(count * lists));
        for (int i = 0; i < lists; ++i) {
            at[i].resize((size_t)count);
            if (i < 2) spans[i].reserve((size_t)count);
            if (i != 1) starts.push_back(written.size());
            for (Py_ssize_t j = 0; j < count; ++j) {
                const at::Tensor& t = tensor(PySequence_Fast_GET_ITEM(held.o[i], j));
                dense(t, d);
                if (i == 0) numel[(size_t)j] = t.numel();
                need(t.scalar_type() == (i < 2 ? type : i < 4 && q8 ? at::kFloat8_e4m3fn : at::kFloat));
                need(t.numel() == (i < 4 ? numel[(size_t)j] : (numel[(size_t)j] + 255) / 256));
                at[i][(size_t)j] = t.data_ptr();
                const uintptr_t from = (uintptr_t)at[i][(size_t)j];
                const Span span{from, from + t.nbytes()};
                if (i < 2) spans[i].push_back(span);
                if (i != 1 && span.at != span.end) written.push_back(span);
            }
        }
        starts.push_back(written.size());
        need(apart(written, starts, spans[0], spans[1]));
        const int64_t step = integer(a[6]);
        const double lr = real(a[7]), b1 = real(a[8]), b2 = real(a[9]), eps = real(a[10]), wd = real(a[11]);
        const at::Tensor hyper = maybe(a[12]);
        float *const *ms = q8 ? (float* const*)at[4].data() : nullptr, *const *vs = q8 ? (float* const*)at[5].data() : nullptr;
        call([&] {
            return hyper.defined() ? lib.fn.adamw_step_each((int)count, at[0].data(), at[1].data(), at[2].data(), at[3].data(), ms, vs, numel.data(), dt, q8 ? 8 : 32, ptr(hyper), stream_of(d))
                                   : lib.fn.adamw_step((int)count, at[0].data(), at[1].data(), at[2].data(), at[3].data(), ms, vs, numel.data(), dt, q8 ? 8 : 32, lr, b1, b2, eps, wd, step,
                                                       nullptr, stream_of(d));
        });
        // written through raw pointers: autograd and the modules' caches have to see it
        for (Py_ssize_t j = 0; j < count; ++j) {
            const at::Tensor& t = THPVariable_Unpack(PySequence_Fast_GET_ITEM(held.o[0], j));
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
        }
        Py_RETURN_TRUE;
    });
}

#define ENTRY(name) {#name, (PyCFunction)(void (*)())name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(bind), ENTRY(route), ENTRY(dispatch), ENTRY(combine), ENTRY(adapter), ENTRY(adamw), ENTRY(accumulates_on_default), {"declined", declined, METH_NOARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mtk_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mtk_torch(void) { return PyModule_Create(&module); }
