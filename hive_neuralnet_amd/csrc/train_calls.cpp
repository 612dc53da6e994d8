// train_calls.cpp -- the training operators' entry points, and the draw of a
// slot from each row of logits, from Python without Python's share of a call.
//
// A small norm, loss or step spends 2 to 6 us on the device and 4 in handing a
// launch over; checks of its arguments, the result tensors and the C call, taken
// one by one from Python, came to 6 to 10 more.  Each function here does for
// one entry point what training_ops.py or network_ops.py does for arguments that are plainly
// right -- the same conditions, results and C call -- and returns None, having
// done nothing, for any other: the Python module then finds what it serves
// besides (rows of more dimensions that are evenly spaced, gradients left out)
// or the words of the refusal.
//
// Measured (MI355X, a call's time on the host, Python alone / here): layer norm
// forward 10.3 / 5.9 us, backward 13.7 / 6.9, the loss of 16 positions 13.1 / 6.2,
// AdamW of 12 tensors 9.8 / 4.4, a draw from one row 9.8 / 5.5; 3.7 of each hand the launch over, 0.6 make a
// result tensor.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>

#include <algorithm>
#include <cstdint>
#include <limits>

#include "hive_gpu.h"

namespace {

using at::Tensor;

decltype(&hg_layer_norm_forward) norm_forward_;
decltype(&hg_layer_norm_backward) norm_backward_;
decltype(&hg_layer_norm_backward_workspace) norm_workspace_;
decltype(&hg_policy_value_loss) loss_;
decltype(&hg_policy_value_loss_workspace) loss_workspace_;
decltype(&hg_adamw_step) adamw_;
decltype(&hg_sample_actions) sample_;

// torch's: the current device, a device's current stream
PyObject *current_device_, *current_stream_;

// the current device, and its current stream
struct Place {
    int64_t device = -1;
    void* stream = nullptr;
    bool holds(const Tensor& t) const { return t.is_cuda() && t.get_device() == device; }
    // of a GPU tensor on the current device
    bool find(const Tensor* t) {
        if (!t || !t->is_cuda()) return false;
        PyObject* d = PyObject_CallNoArgs(current_device_);
        if (!d) return false;
        device = PyLong_AsLongLong(d);
        PyObject* s = t->get_device() == device ? PyObject_CallOneArg(current_stream_, d) : nullptr;
        Py_DECREF(d);
        if (!s) return false;
        stream = PyLong_AsVoidPtr(s);
        Py_DECREF(s);
        return true;
    }
};

const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return HG_F32;
        case at::kHalf: return HG_F16;
        case at::kBFloat16: return HG_BF16;
        default: return -1;
    }
}

// a contiguous [n] or [n, 1] of `type` there
bool is_vector(const Tensor* t, const Place& at, int64_t n, at::ScalarType type) {
    return t && at.holds(*t) && t->scalar_type() == type && t->is_contiguous() && t->numel() == n &&
           (t->dim() == 1 || (t->dim() == 2 && t->size(1) == 1));
}

// rows that are contiguous, or of two dimensions with contiguous rows
struct Rows {
    int64_t rows, cols, stride;
};
bool rows_of(const Tensor& t, Rows* r) {
    if (t.dim() == 0 || t.size(-1) == 0) return false;
    r->cols = t.size(-1);
    r->rows = t.numel() / r->cols;
    r->stride = r->cols;
    if (t.is_contiguous()) return true;
    if (t.dim() != 2 || t.stride(1) != 1) return false;
    r->stride = t.stride(0);
    return true;
}

// weight and bias: None, or vectors of one type
struct Params {
    const Tensor *w = nullptr, *b = nullptr;
    int type = HG_F32;
    const void* weight() const { return w ? w->const_data_ptr() : nullptr; }
    const void* bias() const { return b ? b->const_data_ptr() : nullptr; }
};
bool params_of(PyObject* weight, PyObject* bias, const Place& at, int64_t cols, Params* p) {
    for (int i = 0; i < 2; i++) {
        PyObject* o = i ? bias : weight;
        if (o == Py_None) continue;
        const Tensor* t = tensor(o);
        if (!t || type_of(*t) < 0 || (i && p->w && p->w->scalar_type() != t->scalar_type())) return false;
        if (!is_vector(t, at, cols, t->scalar_type())) return false;
        p->type = type_of(*t);
        (i ? p->b : p->w) = t;
    }
    return true;
}

Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
PyObject* wrap(Tensor t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(t));
}
PyObject* three(Tensor a, Tensor b, Tensor c) {
    PyObject* t = PyTuple_New(3);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(t, 0, wrap(std::move(a)));
    PyTuple_SET_ITEM(t, 1, wrap(std::move(b)));
    PyTuple_SET_ITEM(t, 2, wrap(std::move(c)));
    return t;
}

PyObject* failed(const char* what, int error) {
    return PyErr_Format(PyExc_RuntimeError, "%s: HIP error %d", what, error);
}

// None or "sigmoid"; -1 for anything else
int activation_of(PyObject* o) {
    if (o == Py_None) return 0;
    return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, "sigmoid") == 0 ? 1 : -1;
}

// A number among the arguments that is none, or a device that cannot be asked: errors for training_ops.py to raise.
bool bad_number() { return PyErr_Occurred() != nullptr; }
PyObject* not_here() {
    PyErr_Clear();
    Py_RETURN_NONE;
}

// (x, weight, bias, eps, activation) -> (y, mean, rstd)
PyObject* layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 5 || !norm_forward_) Py_RETURN_NONE;
    Place at;
    const double eps = PyFloat_AsDouble(a[3]);
    const int sigmoid = activation_of(a[4]);
    const Tensor* x = tensor(a[0]);
    Rows r;
    Params p;
    if (!at.find(x) || bad_number() || !(eps >= 0.0) || sigmoid < 0 || type_of(*x) < 0 || !rows_of(*x, &r) ||
        !params_of(a[1], a[2], at, r.cols, &p))
        return not_here();
    Tensor y = like(*x);
    const auto rest = x->sizes().slice(0, x->dim() - 1);
    const auto options = x->options().dtype(at::kFloat);
    Tensor mean = at::empty(rest, options), rstd = at::empty(rest, options);
    const int e = norm_forward_(x->const_data_ptr(), type_of(*x), r.rows, r.cols, r.stride, p.weight(), p.bias(),
                                p.type, (float)eps, sigmoid, y.mutable_data_ptr(), (float*)mean.mutable_data_ptr(),
                                (float*)rstd.mutable_data_ptr(), at.stream);
    if (e) return failed("layer_norm_forward", e);
    return three(std::move(y), std::move(mean), std::move(rstd));
    END_HANDLE_TH_ERRORS
}

// (dy, x, mean, rstd, weight, bias, activation, need_dx) -> (dx, dweight, dbias)
PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 8 || !norm_backward_) Py_RETURN_NONE;
    Place at;
    const int sigmoid = activation_of(a[6]), need_dx = PyObject_IsTrue(a[7]);
    const Tensor *dy = tensor(a[0]), *x = tensor(a[1]), *mean = tensor(a[2]), *rstd = tensor(a[3]);
    Rows r, q;
    Params p;
    if (!at.find(x) || bad_number() || sigmoid < 0 || !dy || !mean || !rstd || !at.holds(*dy) || type_of(*x) < 0 ||
        dy->scalar_type() != x->scalar_type() || dy->sizes() != x->sizes() || !rows_of(*x, &r) ||
        !rows_of(*dy, &q) || !params_of(a[4], a[5], at, r.cols, &p))
        return not_here();
    for (const Tensor* t : {mean, rstd})
        if (!at.holds(*t) || t->scalar_type() != at::kFloat || t->numel() != r.rows || !t->is_contiguous())
            Py_RETURN_NONE;
    Tensor dx, dw, db, workspace;
    if (need_dx) dx = like(*x);
    if (p.w) dw = like(*p.w);
    if (p.b) db = like(*p.b);
    if (p.w || p.b) workspace = at::empty({norm_workspace_(r.rows, r.cols)}, x->options().dtype(at::kByte));
    const int e = norm_backward_(
        dy->const_data_ptr(), q.stride, x->const_data_ptr(), type_of(*x), r.rows, r.cols, r.stride,
        (const float*)mean->const_data_ptr(), (const float*)rstd->const_data_ptr(), p.weight(), p.type, sigmoid,
        need_dx ? dx.mutable_data_ptr() : nullptr, p.w ? dw.mutable_data_ptr() : nullptr,
        p.b ? db.mutable_data_ptr() : nullptr, workspace.defined() ? workspace.mutable_data_ptr() : nullptr, at.stream);
    if (e) return failed("layer_norm_backward", e);
    return three(std::move(dx), std::move(dw), std::move(db));
    END_HANDLE_TH_ERRORS
}

// (logits, values, num_actions, policy_targets, policy_weights, value_targets, value_weights, value_coef, loss_scale)
// -> (losses, dlogits, dvalues)
PyObject* policy_value_loss(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 9 || !loss_) Py_RETURN_NONE;
    Place at;
    const double coef = PyFloat_AsDouble(a[7]), scale = PyFloat_AsDouble(a[8]);
    const Tensor *logits = tensor(a[0]), *values = tensor(a[1]), *counts = tensor(a[2]), *targets = tensor(a[3]),
                 *pw = tensor(a[4]), *vt = tensor(a[5]), *vw = tensor(a[6]);
    if (!at.find(logits) || bad_number() || !targets || !at.holds(*targets) || type_of(*logits) < 0 ||
        type_of(*targets) < 0 || logits->dim() != 1 || !logits->is_contiguous() || targets->dim() != 2 ||
        !targets->is_contiguous())
        return not_here();
    const int64_t B = targets->size(0), width = targets->size(1), N = logits->size(0);
    if ((B == 0 && N > 0) || !is_vector(values, at, B, logits->scalar_type()) ||
        !is_vector(counts, at, B, at::kLong) || !is_vector(pw, at, B, at::kFloat) ||
        !is_vector(vt, at, B, at::kFloat) || !is_vector(vw, at, B, at::kFloat))
        Py_RETURN_NONE;
    Tensor losses = at::empty({3}, logits->options().dtype(at::kFloat));
    Tensor dlogits = like(*logits), dvalues = like(*values);
    Tensor workspace = at::empty({loss_workspace_(B, width)}, logits->options().dtype(at::kByte));
    const int e = loss_(logits->const_data_ptr(), type_of(*logits), N, values->const_data_ptr(),
                        (const int64_t*)counts->const_data_ptr(), targets->const_data_ptr(), type_of(*targets), width,
                        (const float*)pw->const_data_ptr(), (const float*)vt->const_data_ptr(),
                        (const float*)vw->const_data_ptr(), B, (float)coef, (float)scale,
                        (float*)losses.mutable_data_ptr(), dlogits.mutable_data_ptr(), dvalues.mutable_data_ptr(),
                        workspace.mutable_data_ptr(), at.stream);
    if (e) return failed("policy_value_loss", e);
    return three(std::move(losses), std::move(dlogits), std::move(dvalues));
    END_HANDLE_TH_ERRORS
}

// What a step writes: the bounds of `count / 2` pieces of memory in order, each's first byte and one past its last.
struct Written {
    const uint64_t* bounds = nullptr;
    Py_ssize_t count = 0;
    bool apart(const Tensor& t) const {
        const uint64_t begin = (uint64_t)(uintptr_t)t.const_data_ptr(), end = begin + t.nbytes();
        const Py_ssize_t i = std::upper_bound(bounds, bounds + count, begin) - bounds;
        return begin == end || (i % 2 == 0 && (i == count || bounds[i] >= end));
    }
};

// (params, grads, table, param type, state bits, step, lr, beta1, beta2, eps, weight_decay, grad_scale, seed[, bounds,
// their number]) -> True.  `table` is the address of a plan's hg_adamw_tensor array, whose gradients are entered here;
// none may be left out.  `bounds`: the address of Written's; without them nothing is looked for in what the step writes.
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if ((count != 13 && count != 15) || !adamw_ || !PyList_Check(a[0]) ||
        !(PyList_Check(a[1]) || PyTuple_Check(a[1])))
        Py_RETURN_NONE;
    Place at;
    auto* table = (hg_adamw_tensor*)PyLong_AsVoidPtr(a[2]);
    const int param_type = (int)PyLong_AsLong(a[3]), bits = (int)PyLong_AsLong(a[4]);
    const int64_t step = PyLong_AsLongLong(a[5]);
    const double lr = PyFloat_AsDouble(a[6]), beta1 = PyFloat_AsDouble(a[7]), beta2 = PyFloat_AsDouble(a[8]),
                 eps = PyFloat_AsDouble(a[9]), decay = PyFloat_AsDouble(a[10]);
    const uint32_t seed = (uint32_t)PyLong_AsUnsignedLongMask(a[12]);
    Written written;
    if (count == 15) written = {(const uint64_t*)PyLong_AsVoidPtr(a[13]), PyLong_AsSsize_t(a[14])};
    const Py_ssize_t n = PyList_GET_SIZE(a[0]);
    if (bad_number() || n == 0 || PySequence_Fast_GET_SIZE(a[1]) != n || step < 1 ||
        !at.find(tensor(PyList_GET_ITEM(a[0], 0))) ||
        !(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0))
        return not_here();
    const float* scale = nullptr;
    if (a[11] != Py_None) {
        const Tensor* t = tensor(a[11]);
        if (!t || !at.holds(*t) || t->scalar_type() != at::kFloat || t->numel() != 1 || !written.apart(*t))
            Py_RETURN_NONE;
        scale = (const float*)t->const_data_ptr();
    }
    int grad_type = -1;
    for (Py_ssize_t i = 0; i < n; i++) {
        const Tensor *p = tensor(PyList_GET_ITEM(a[0], i)), *g = tensor(PySequence_Fast_GET_ITEM(a[1], i));
        if (!p || !g || !at.holds(*p) || !at.holds(*g) || g->sizes() != p->sizes() || !g->is_contiguous() ||
            p->const_data_ptr() != table[i].param || p->numel() != table[i].count)
            Py_RETURN_NONE;
        const int type = type_of(*g);
        if (type < 0 || (i && type != grad_type)) Py_RETURN_NONE;
        if (!written.apart(*g) && (g->const_data_ptr() != table[i].param || type != param_type)) Py_RETURN_NONE;
        grad_type = type;
    }
    for (Py_ssize_t i = 0; i < n; i++)  // once all of them are served: a call that is left changes nothing
        table[i].grad = tensor(PySequence_Fast_GET_ITEM(a[1], i))->const_data_ptr();
    const int e =
        adamw_(table, n, param_type, grad_type, bits, step, lr, beta1, beta2, eps, decay, scale, seed, at.stream);
    if (e) return failed("adamw_step", e);
    for (Py_ssize_t i = 0; i < n; i++) {  // autograd finds that a weight it saved has changed
        const Tensor* p = tensor(PyList_GET_ITEM(a[0], i));
        if (!p->is_inference()) p->unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// A setting of a draw: a tensor of a value a row, or a number for all.
struct Setting {
    const void* each = nullptr;
    double all = 0.0;
    // false: neither, or a number that is refused
    bool find(PyObject* o, const Place& at, int64_t rows, at::ScalarType type, double most) {
        if (const Tensor* t = tensor(o)) {
            if (!is_vector(t, at, rows, type)) return false;
            each = t->const_data_ptr();
            return true;
        }
        if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;  // other kinds of numbers, and what is none: network_ops.py
        all = PyFloat_AsDouble(o);
        return !bad_number() && all >= 0.0 && all <= most;
    }
};

// (logits, uniforms, num_actions, temperature, top_k, top_p, min_p) -> (actions, log_probs)
PyObject* sample_actions(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 7 || !sample_) Py_RETURN_NONE;
    Place at;
    const Tensor *logits = tensor(a[0]), *uniforms = tensor(a[1]), *counts = tensor(a[2]);
    if (!at.find(logits) || type_of(*logits) < 0 || logits->dim() != 2 || logits->size(1) == 0 ||
        logits->size(1) > 1 << 20 || (logits->stride(1) != 1 && logits->size(1) > 1) || logits->numel() == 0)
        return not_here();
    const int64_t rows = logits->size(0), width = logits->size(1);
    if (rows > (width <= 1024 ? 1 << 25 : 1 << 21)) return not_here();
    constexpr double any = std::numeric_limits<double>::infinity();
    Setting t, p, min_p, k;
    if (!is_vector(uniforms, at, rows, at::kFloat) || (a[2] != Py_None && !is_vector(counts, at, rows, at::kLong)) ||
        !t.find(a[3], at, rows, at::kFloat, any) || !p.find(a[5], at, rows, at::kFloat, any) ||
        !min_p.find(a[6], at, rows, at::kFloat, 1.0) || (!tensor(a[4]) && !PyLong_Check(a[4])) ||
        !k.find(a[4], at, rows, at::kLong, 0x1p62))
        return not_here();
    Tensor actions = at::empty({rows}, logits->options().dtype(at::kLong));
    Tensor log_probs = at::empty({rows}, logits->options().dtype(at::kFloat));
    const int e = sample_(logits->const_data_ptr(), type_of(*logits), rows, width, logits->stride(0),
                          a[2] == Py_None ? nullptr : (const int64_t*)counts->const_data_ptr(),
                          (const float*)uniforms->const_data_ptr(), (const float*)t.each, t.all, (const int64_t*)k.each,
                          (int64_t)k.all, (const float*)p.each, p.all, (const float*)min_p.each, min_p.all,
                          (int64_t*)actions.mutable_data_ptr(), (float*)log_probs.mutable_data_ptr(), at.stream);
    if (e) return failed("sample_actions", e);
    PyObject* both = PyTuple_New(2);
    if (!both) return nullptr;
    PyTuple_SET_ITEM(both, 0, wrap(std::move(actions)));
    PyTuple_SET_ITEM(both, 1, wrap(std::move(log_probs)));
    return both;
    END_HANDLE_TH_ERRORS
}

// (the address of libhive_gpu.so's hg_sample_actions), after bind
PyObject* bind_network(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 1) return PyErr_Format(PyExc_TypeError, "bind_network takes 1 address");
    void* f = PyLong_AsVoidPtr(a[0]);
    if (PyErr_Occurred()) return nullptr;
    sample_ = (decltype(sample_))f;
    Py_RETURN_NONE;
}

// (the addresses of libhive_gpu.so's functions, in the order below, torch's two)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t count) {
    if (count != 8) return PyErr_Format(PyExc_TypeError, "bind takes 6 addresses and 2 functions");
    void* f[6];
    for (int i = 0; i < 6; i++) f[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
    Py_INCREF(a[6]);
    Py_INCREF(a[7]);
    current_device_ = a[6];
    current_stream_ = a[7];
    norm_forward_ = (decltype(norm_forward_))f[0];
    norm_backward_ = (decltype(norm_backward_))f[1];
    norm_workspace_ = (decltype(norm_workspace_))f[2];
    loss_ = (decltype(loss_))f[3];
    loss_workspace_ = (decltype(loss_workspace_))f[4];
    adamw_ = (decltype(adamw_))f[5];
    Py_RETURN_NONE;
}

#define CALL(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CALL(layer_norm_forward), CALL(layer_norm_backward), CALL(policy_value_loss),
                         CALL(adamw_step),         CALL(bind),                CALL(sample_actions),
                         CALL(bind_network),       {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_train_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__train_calls(void) { return PyModule_Create(&module); }
