// mtk_torch.cpp — torch's side of the small entry points: a CPython module that checks tensors, allocates results and calls the C ABI.
//
// A launch costs some microseconds; reading the shapes, types and addresses of a call's tensors in Python and converting twenty arguments costs
// several times that, and a step over hundreds of tensors more than its kernels.  Each function here takes the ordinary case of a call and
// does it all at once.  Whatever it does not recognise (another device than the current one, strides it would have to copy, shapes that
// do not fit, a refusal by the library) it leaves alone and returns None: the Python layer then checks, copies or raises, in full.
// The library's functions come by address (bind), so there is one copy of it, wherever it was loaded from.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "mtk.h"

namespace {

struct Table {
    decltype(&mtk_route_rows_work) route_rows_work;
    decltype(&mtk_route_rows) route_rows;
    decltype(&mtk_rows_dispatch) rows_dispatch;
    decltype(&mtk_rows_combine) rows_combine;
    decltype(&mtk_adapter_saved_bytes) saved_bytes;
    decltype(&mtk_adapter_work_bytes) work_bytes;
    decltype(&mtk_adapter_forward) adapter_forward;
    decltype(&mtk_adapter_backward) adapter_backward;
    decltype(&mtk_adamw_step) adamw_step;
};
constexpr int kEntries = sizeof(Table) / sizeof(void*);
union {
    Table fn;
    void* at[kEntries];
} lib = {};

struct Decline {};  // thrown to leave a call to the Python layer

void need(bool ok) {
    if (!ok) throw Decline();
}
const at::Tensor& tensor(PyObject* o) {
    need(THPVariable_Check(o));
    return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o) { return o == Py_None ? nullptr : &tensor(o); }
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
    static const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
    const int d = guard.getDevice().index();
    need(t.device().index() == d);
    return d;
}
// rows whose elements lie side by side, at any distance from each other
void rows(const at::Tensor& t, int device) {
    here(t, device);
    need(t.dim() == 2 && t.size(1) >= 1 && (t.stride(1) == 1 || t.size(1) == 1 || t.size(0) == 0) && t.stride(0) >= 0);
}
void* ptr(const at::Tensor& t) { return t.data_ptr(); }
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
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
template <typename F> void call(F f) {  // a library call without the interpreter's lock
    int rc;
    Py_BEGIN_ALLOW_THREADS;
    rc = f();
    Py_END_ALLOW_THREADS;
    need(rc == MTK_OK);
}
PyObject* pack(std::initializer_list<at::Tensor> ts) {
    PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (const at::Tensor& t : ts) PyTuple_SET_ITEM(out, i++, t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None));
    return out;
}
// the body of a module function: a decline is None, an error of torch's (out of memory) a RuntimeError
template <typename F> PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F f) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", n, want);
        return nullptr;
    }
    try {
        return f();
    } catch (const Decline&) {
        Py_RETURN_NONE;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "midst_toolkit_amd: unknown C++ exception");
        return nullptr;
    }
}
bool tracked(std::initializer_list<const at::Tensor*> ts) {
    if (!c10::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : ts)
        if (t && t->requires_grad()) return true;
    return false;
}

// bind((address, ...)): the library's functions in Table's order
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, kEntries, [&]() -> PyObject* {
        for (int i = 0; i < kEntries; ++i) lib.at[i] = (void*)(intptr_t)integer(a[i]);
        Py_RETURN_TRUE;
    });
}

// route(index, n_groups, stream) -> (order, slot, offsets)
PyObject* route(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 3, [&]() -> PyObject* {
        const at::Tensor& index = tensor(a[0]);
        const int64_t groups = integer(a[1]);
        const mtk_stream s = (mtk_stream)(intptr_t)integer(a[2]);
        dense(index, current(index));
        need(index.scalar_type() == at::kLong && (index.dim() == 1 || (index.dim() == 2 && index.size(1) >= 1)) && groups >= 1 && groups <= MTK_ROUTE_MAX_GROUPS);
        const int64_t P = index.numel();
        need(P <= 0x7fffffff);
        const int64_t w = lib.fn.route_rows_work(P, (int)groups);
        at::Tensor order = like(index, {P}, at::kInt), slot = like(index, index.sizes(), at::kInt), offsets = like(index, {groups + 1}, at::kInt), work;
        if (w) work = like(index, {w}, at::kInt);
        call([&] {
            return lib.fn.route_rows(P, index.const_data_ptr<int64_t>(), (int)groups, (int32_t*)ptr(order), (int32_t*)ptr(slot), (int32_t*)ptr(offsets),
                                     w ? (int32_t*)work.data_ptr() : nullptr, w, s);
        });
        return pack({order, slot, offsets});
    });
}

// dispatch(x, slot, n_rows, copies, weights | None, y | None, want_rows, stream) -> (xs | None, dw | None)
PyObject* dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 8, [&]() -> PyObject* {
        const at::Tensor &x = tensor(a[0]), &slot = tensor(a[1]);
        const int64_t N = integer(a[2]), k = integer(a[3]);
        const at::Tensor *w = maybe(a[4]), *y = maybe(a[5]);
        const bool want = integer(a[6]) != 0;
        const mtk_stream s = (mtk_stream)(intptr_t)integer(a[7]);
        const int d = current(x), dt = code(x);
        rows(x, d);
        dense(slot, d);
        need(k >= 1 && x.size(0) == N && N >= 1 && slot.numel() == N * k && slot.scalar_type() == at::kInt);
        const int64_t D = x.size(1);
        if (w) {
            dense(*w, d);
            need(w->scalar_type() == at::kFloat && w->numel() == N * k);
        }
        if (y) {
            dense(*y, d);
            need(y->scalar_type() == x.scalar_type() && y->dim() == 2 && y->size(0) == N * k && y->size(1) == D);
        }
        at::Tensor xs, dw;
        if (want) xs = like(x, {N * k, D}, x.scalar_type());
        if (y) dw = like(x, {N, k}, at::kFloat);
        call([&] {
            return lib.fn.rows_dispatch(N, (int)k, D, dt, ptr(x), x.stride(0), (const int32_t*)ptr(slot), (const float*)ptr(w), want ? xs.data_ptr() : nullptr, ptr(y),
                                        y ? (float*)dw.data_ptr() : nullptr, s);
        });
        return pack({xs, dw});
    });
}

// combine(y, slot, n_rows, copies, weights | None, stream) -> out
PyObject* combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 6, [&]() -> PyObject* {
        const at::Tensor &y = tensor(a[0]), &slot = tensor(a[1]);
        const int64_t N = integer(a[2]), k = integer(a[3]);
        const at::Tensor* w = maybe(a[4]);
        const mtk_stream s = (mtk_stream)(intptr_t)integer(a[5]);
        const int d = current(y), dt = code(y);
        rows(y, d);
        dense(slot, d);
        need(k >= 1 && N >= 1 && y.size(0) == N * k && slot.numel() == N * k && slot.scalar_type() == at::kInt);
        if (w) {
            dense(*w, d);
            need(w->scalar_type() == at::kFloat && w->numel() == N * k);
        }
        at::Tensor out = like(y, {N, y.size(1)}, y.scalar_type());
        call([&] { return lib.fn.rows_combine(N, (int)k, y.size(1), dt, ptr(y), y.stride(0), (const int32_t*)ptr(slot), (const float*)ptr(w), out.data_ptr(), s); });
        return THPVariable_Wrap(out);
    });
}

struct Layer {  // the arguments that the two directions of an adapted layer share, checked
    int device, dt, din, dout, r, E;
    int64_t M, x_ld;
    const float* scales = nullptr;
    double scale = 1.0;
    Layer(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& down, const at::Tensor& up, const at::Tensor& offsets, PyObject* scale_) {
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
        x_ld = x.stride(0);
        din = (int)x.size(1), dout = (int)weight.size(0), E = (int)down.size(0), r = (int)down.size(1);
        need(M >= 1 && dout >= 1 && E >= 1 && r >= 1 && weight.size(1) == din && down.size(2) == din && up.size(0) == E && up.size(1) == dout && up.size(2) == r &&
             offsets.size(0) == E + 1);
        if (THPVariable_Check(scale_)) {
            const at::Tensor& s = THPVariable_Unpack(scale_);
            dense(s, device);
            need(s.scalar_type() == at::kFloat && s.dim() == 1 && s.size(0) == E);
            scales = s.const_data_ptr<float>();
        } else {
            scale = real(scale_);
        }
    }
    at::Tensor bytes(const at::Tensor& x, int64_t n) const { return n ? like(x, {n}, at::kByte) : at::Tensor(); }
};

// adapter_forward(x, weight, bias | None, down, up, offsets, scale, act, keep, stream) -> y, or (y, saved) with keep.  Without keep, inputs
// that autograd tracks are declined.
PyObject* adapter_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 10, [&]() -> PyObject* {
        const at::Tensor &x = tensor(a[0]), &weight = tensor(a[1]), &down = tensor(a[3]), &up = tensor(a[4]), &offsets = tensor(a[5]);
        const at::Tensor* bias = maybe(a[2]);
        const int act = (int)integer(a[7]);
        const bool keep = integer(a[8]) != 0;
        const mtk_stream s = (mtk_stream)(intptr_t)integer(a[9]);
        need(keep || !tracked({&x, &weight, bias, &down, &up}));
        const Layer l(x, weight, down, up, offsets, a[6]);
        if (bias) {
            dense(*bias, l.device);
            need(bias->scalar_type() == x.scalar_type() && bias->dim() == 1 && bias->size(0) == l.dout);
        }
        const int64_t saved_bytes = lib.fn.saved_bytes(l.M, l.r, l.dt), work_bytes = lib.fn.work_bytes(l.M, l.din, l.dout, l.r, l.E, l.dt, act, 0);
        at::Tensor y = like(x, {l.M, l.dout}, x.scalar_type()), saved = l.bytes(x, saved_bytes), work = l.bytes(x, work_bytes);
        call([&] {
            return lib.fn.adapter_forward(l.M, l.din, l.dout, l.r, l.E, l.dt, ptr(x), l.x_ld, ptr(weight), ptr(bias), ptr(down), ptr(up), (const int32_t*)ptr(offsets), l.scales,
                                          l.scale, act, keep, y.data_ptr(), saved.data_ptr(), saved_bytes, work.defined() ? work.data_ptr() : nullptr, work_bytes, s);
        });
        return keep ? pack({y, saved}) : THPVariable_Wrap(y);
    });
}

// adapter_backward(x, weight, down, up, offsets, scale, act, y | None, dy, saved, want (1: dx, 2: ddown, 4: dup), stream) -> (dx, ddown, dup)
PyObject* adapter_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 12, [&]() -> PyObject* {
        const at::Tensor &x = tensor(a[0]), &weight = tensor(a[1]), &down = tensor(a[2]), &up = tensor(a[3]), &offsets = tensor(a[4]), &dy = tensor(a[8]), &saved = tensor(a[9]);
        const int act = (int)integer(a[6]);
        const at::Tensor* y = maybe(a[7]);
        const int64_t want = integer(a[10]);
        const mtk_stream s = (mtk_stream)(intptr_t)integer(a[11]);
        const Layer l(x, weight, down, up, offsets, a[5]);
        dense(dy, l.device);
        dense(saved, l.device);
        need(dy.scalar_type() == x.scalar_type() && dy.dim() == 2 && dy.size(0) == l.M && dy.size(1) == l.dout && saved.numel() >= lib.fn.saved_bytes(l.M, l.r, l.dt));
        need(act == MTK_ACT_NONE || (y && y->is_contiguous() && y->sizes() == dy.sizes() && y->scalar_type() == x.scalar_type()));
        const int64_t work_bytes = lib.fn.work_bytes(l.M, l.din, l.dout, l.r, l.E, l.dt, act, 1);
        at::Tensor dx, ddown, dup, work = l.bytes(x, work_bytes);
        if (want & 1) dx = like(x, {l.M, l.din}, x.scalar_type());
        if (want & 2) ddown = like(x, down.sizes(), x.scalar_type());
        if (want & 4) dup = like(x, up.sizes(), x.scalar_type());
        call([&] {
            return lib.fn.adapter_backward(l.M, l.din, l.dout, l.r, l.E, l.dt, ptr(x), l.x_ld, ptr(weight), ptr(down), ptr(up), (const int32_t*)ptr(offsets), l.scales, l.scale, act,
                                           ptr(y), ptr(dy), ptr(saved), want & 1 ? dx.data_ptr() : nullptr, want & 2 ? ddown.data_ptr() : nullptr,
                                           want & 4 ? dup.data_ptr() : nullptr, work.data_ptr(), work_bytes, s);
        });
        return pack({dx, ddown, dup});
    });
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, scales | None, scales | None, step, lr, beta1, beta2, eps, weight_decay, hyper | None, stream) -> True
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded(n, 14, [&]() -> PyObject* {
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
        for (int i = 0; i < lists; ++i) {
            at[i].resize((size_t)count);
            for (Py_ssize_t j = 0; j < count; ++j) {
                const at::Tensor& t = tensor(PySequence_Fast_GET_ITEM(held.o[i], j));
                dense(t, d);
                if (i == 0) numel[(size_t)j] = t.numel();
                need(t.scalar_type() == (i < 2 ? type : i < 4 && q8 ? at::kFloat8_e4m3fn : at::kFloat));
                need(t.numel() == (i < 4 ? numel[(size_t)j] : (numel[(size_t)j] + 255) / 256));
                at[i][(size_t)j] = t.data_ptr();
            }
        }
        const int64_t step = integer(a[6]);
        const double lr = real(a[7]), b1 = real(a[8]), b2 = real(a[9]), eps = real(a[10]), wd = real(a[11]);
        const at::Tensor* hyper = maybe(a[12]);
        const mtk_stream s = (mtk_stream)(intptr_t)integer(a[13]);
        call([&] {
            return lib.fn.adamw_step((int)count, at[0].data(), at[1].data(), at[2].data(), at[3].data(), q8 ? (float* const*)at[4].data() : nullptr,
                                     q8 ? (float* const*)at[5].data() : nullptr, numel.data(), dt, q8 ? 8 : 32, lr, b1, b2, eps, wd, step, ptr(hyper), s);
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
PyMethodDef methods[] = {ENTRY(bind), ENTRY(route), ENTRY(dispatch), ENTRY(combine), ENTRY(adapter_forward), ENTRY(adapter_backward), ENTRY(adamw), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mtk_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mtk_torch(void) { return PyModule_Create(&module); }
