// b3x_train_py.cpp -- the Python side of the training operators: takes torch
// tensors, checks them and calls the C-ABI (b3x_train.h).  A module of its own
// (b3train_py) because a call's checks, made in Python, take as long as its
// launch; puffysics_b200/train.py has the signatures and the documentation.
//
// Every function takes its arguments in order and returns a cudaError_t code; an
// argument of a type, shape, stride or device that the operator does not take
// gives cudaErrorInvalidValue, and nothing is launched.  `device` and `stream`
// are the caller's current device and stream handle.
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "b3x_train.h"

// The torch and Python that this is compiled against (the build compares).
extern "C" __attribute__((visibility("default"))) const char b3train_py_built_for[] = B3X_BUILT_FOR;

namespace {

constexpr int kInvalid = 1;   // cudaErrorInvalidValue
struct Refused {};            // an argument that the operator does not take; never leaves call()

void require(bool ok) {
    if (!ok) throw Refused();
}

// A tensor, or null for None.
const at::Tensor* tensor(PyObject* o) {
    if (o == Py_None) return nullptr;
    require(THPVariable_Check(o));
    return &THPVariable_Unpack(o);
}

const at::Tensor& here(const at::Tensor* t, int64_t device) {
    require(t && t->is_cuda() && t->get_device() == device && t->layout() == at::kStrided && !t->is_neg());
    return *t;
}

int float_type(at::ScalarType t) {
    require(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf);
    return t == at::kFloat ? B3X_F32 : t == at::kBFloat16 ? B3X_BF16 : B3X_F16;
}

bool bytes(at::ScalarType t) { return t == at::kByte || t == at::kBool; }

// The memory of an optional dense tensor of this type and shape.
void* dense(PyObject* o, int64_t device, at::ScalarType type, at::IntArrayRef shape) {
    const at::Tensor* t = tensor(o);
    if (!t) return nullptr;
    here(t, device);
    require(t->scalar_type() == type && t->sizes() == shape && t->is_contiguous());
    return t->data_ptr();
}

int64_t whole(PyObject* o) {
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) throw Refused();
    return x;
}
double number(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw Refused();
    return x;
}
void* handle(PyObject* o) { return reinterpret_cast<void*>(whole(o)); }

// Runs f, and turns whatever it throws into a code: nothing crosses into Python.
template <class F>
PyObject* call(Py_ssize_t given, Py_ssize_t wanted, F f) {
    if (given != wanted) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    int rc = kInvalid;
    try {
        rc = f();
    } catch (const Refused&) {
        PyErr_Clear();
    } catch (...) {   // a tensor without memory
        PyErr_Clear();
    }
    return PyLong_FromLong(rc);
}

// (rows, width) logits with their actions and mask.
struct Rows {
    const void* logits;
    int type;
    at::ScalarType scalar;
    int64_t rows, width, stride;
    const unsigned char* mask = nullptr;
    int64_t mask_stride = 0;
    const void* actions = nullptr;
    int action_bytes = 0;

    Rows(PyObject* z, PyObject* a, PyObject* m, int64_t device) {
        const at::Tensor& t = here(tensor(z), device);
        scalar = t.scalar_type();
        type = float_type(scalar);
        require(t.dim() == 2);
        rows = t.size(0), width = t.size(1), stride = t.stride(0);
        require(width <= 1 || t.stride(1) == 1);
        logits = t.data_ptr();
        if (const at::Tensor* x = tensor(a)) {
            require(x->scalar_type() == at::kLong || x->scalar_type() == at::kInt);
            action_bytes = x->scalar_type() == at::kLong ? 8 : 4;
            actions = dense(a, device, x->scalar_type(), {rows});
        }
        if (const at::Tensor* x = tensor(m)) {
            here(x, device);
            require(bytes(x->scalar_type()) && x->sizes() == t.sizes() && (width <= 1 || x->stride(1) == 1));
            mask = static_cast<const unsigned char*>(x->data_ptr());
            mask_stride = x->stride(0);
        }
    }
};

// logits, actions, logp, entropy, stats, top_ids, top_logp, mask, scale, device, stream
PyObject* logprob(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 11, [&] {
        const int64_t device = whole(a[9]);
        const Rows r(a[0], a[1], a[7], device);
        int64_t top = 0;
        const at::Tensor *ids = tensor(a[5]), *best = tensor(a[6]);
        require(!ids == !best);
        if (ids) {
            require(ids->dim() == 2);
            top = ids->size(1);
        }
        return b3x_train_logprob_gpu(r.logits, r.type, r.rows, r.width, r.stride, r.mask, r.mask_stride, r.actions, r.action_bytes,
            (float)number(a[8]), (float*)dense(a[2], device, at::kFloat, {r.rows}), (float*)dense(a[3], device, at::kFloat, {r.rows}),
            (float*)dense(a[4], device, at::kFloat, {r.rows, 2}), (int)std::min<int64_t>(top, 1 << 20),
            (int*)dense(a[5], device, at::kInt, {r.rows, top}), (float*)dense(a[6], device, at::kFloat, {r.rows, top}), handle(a[10]));
    });
}

// logits, stats, grad, actions, d_logp, entropy, d_entropy, mask, scale, device, stream
PyObject* logprob_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 11, [&] {
        const int64_t device = whole(a[9]);
        const Rows r(a[0], a[3], a[7], device);
        const at::Tensor& g = here(tensor(a[2]), device);
        require(g.scalar_type() == r.scalar && g.dim() == 2 && g.size(0) == r.rows && g.size(1) == r.width &&
                (r.width <= 1 || g.stride(1) == 1) && a[1] != Py_None);
        return b3x_train_logprob_grad_gpu(r.logits, r.type, r.rows, r.width, r.stride, r.mask, r.mask_stride, r.actions,
            r.action_bytes, (float)number(a[8]), (float*)dense(a[1], device, at::kFloat, {r.rows, 2}),
            (float*)dense(a[5], device, at::kFloat, {r.rows}), (float*)dense(a[4], device, at::kFloat, {r.rows}),
            (float*)dense(a[6], device, at::kFloat, {r.rows}), g.data_ptr(), g.stride(0), handle(a[10]));
    });
}

// rewards, values, terminals, last_values, advantages, returns, gamma, lam, lengths, device, stream
PyObject* advantage(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 11, [&] {
        const int64_t device = whole(a[9]);
        const at::Tensor &r = here(tensor(a[0]), device), &v = here(tensor(a[1]), device), &d = here(tensor(a[2]), device),
                         &last = here(tensor(a[3]), device), &adv = here(tensor(a[4]), device);
        const at::Tensor* ret = tensor(a[5]);
        require(r.dim() == 2 && r.scalar_type() == at::kFloat && adv.scalar_type() == at::kFloat &&
                last.scalar_type() == v.scalar_type() && (d.scalar_type() == at::kFloat || bytes(d.scalar_type())) &&
                v.sizes() == r.sizes() && d.sizes() == r.sizes() && adv.sizes() == r.sizes() && last.dim() == 1 &&
                last.size(0) == r.size(1));
        if (ret) {
            here(ret, device);
            require(ret->scalar_type() == at::kFloat && ret->sizes() == r.sizes());
        }
        const long long strides[11] = {r.stride(0), r.stride(1), v.stride(0), v.stride(1), d.stride(0), d.stride(1), last.stride(0),
                                       adv.stride(0), adv.stride(1), ret ? ret->stride(0) : 0, ret ? ret->stride(1) : 0};
        return b3x_train_advantage_gpu(r.size(0), r.size(1), (const float*)r.data_ptr(), v.data_ptr(), float_type(v.scalar_type()),
            d.data_ptr(), d.scalar_type() == at::kFloat ? B3X_F32 : B3X_U8, last.data_ptr(),
            (const int*)dense(a[8], device, at::kInt, {r.size(1)}), (float*)adv.data_ptr(), ret ? (float*)ret->data_ptr() : nullptr,
            strides, (float)number(a[6]), (float)number(a[7]), handle(a[10]));
    });
}

// A list or tuple of dense tensors of one type with these element counts (or any, which it then notes).
struct List {
    std::vector<void*> at;
    at::ScalarType type = at::kFloat;

    List(PyObject* o, int64_t device, std::vector<long long>& sizes, bool note, long long block = 0) {
        require(PyList_Check(o) || PyTuple_Check(o));
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
        if (note) sizes.resize(n);
        require((size_t)n == sizes.size());
        at.resize(n);
        for (Py_ssize_t k = 0; k < n; k++) {
            const at::Tensor& t = here(tensor(PySequence_Fast_GET_ITEM(o, k)), device);
            if (k == 0) type = t.scalar_type();
            if (note) sizes[k] = t.numel();
            const long long want = block ? (sizes[k] + block - 1) / block * 2 : sizes[k];
            require(t.scalar_type() == type && t.numel() == want && t.is_contiguous());
            at[k] = t.data_ptr();
        }
    }
};

// grads, max_norm, out, workspace, device, stream
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 6, [&] {
        const int64_t device = whole(a[4]);
        std::vector<long long> sizes;
        const List g(a[0], device, sizes, true);
        const at::Tensor& ws = here(tensor(a[3]), device);
        require(a[2] != Py_None && ws.scalar_type() == at::kByte && ws.is_contiguous());
        return b3x_train_grad_norm_gpu((int)sizes.size(), g.at.data(), float_type(g.type), sizes.data(), number(a[1]),
            (float*)dense(a[2], device, at::kFloat, {2}), ws.data_ptr(), (size_t)ws.numel(), handle(a[5]));
    });
}

// params, grads, exp_avg, exp_avg_sq, step, lr, beta1, beta2, eps, weight_decay, scales, grad_scale, copies, seed, device, stream
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return call(n, 16, [&] {
        const int64_t device = whole(a[14]);
        std::vector<long long> sizes;
        const List p(a[0], device, sizes, true), g(a[1], device, sizes, false), m(a[2], device, sizes, false),
            v(a[3], device, sizes, false);
        const bool f8 = !sizes.empty() && m.type == at::kFloat8_e4m3fn;
        if (!sizes.empty())
            require((p.type == at::kFloat || p.type == at::kBFloat16) && (f8 || m.type == at::kFloat) && v.type == m.type &&
                    f8 == (a[10] != Py_None));
        std::vector<void*> scales, copies;
        if (a[10] != Py_None) {
            List s(a[10], device, sizes, false, B3X_TRAIN_BLOCK);
            require(s.type == at::kFloat);
            scales = std::move(s.at);
        }
        if (a[12] != Py_None) {
            List c(a[12], device, sizes, false);
            require(sizes.empty() || c.type == at::kBFloat16);
            copies = std::move(c.at);
        }
        std::vector<float> decays;
        double decay = 0.0;
        if (PyList_Check(a[9]) || PyTuple_Check(a[9])) {
            require((size_t)PySequence_Fast_GET_SIZE(a[9]) == sizes.size());
            for (size_t k = 0; k < sizes.size(); k++) decays.push_back((float)number(PySequence_Fast_GET_ITEM(a[9], k)));
        } else {
            decay = number(a[9]);
        }
        const float* factor = nullptr;
        if (const at::Tensor* t = tensor(a[11])) {
            here(t, device);
            require(t->scalar_type() == at::kFloat && t->numel() == 1);
            factor = (const float*)t->data_ptr();
        }
        const bool stochastic = a[13] != Py_None;
        unsigned seed = 0;
        if (stochastic) {
            seed = (unsigned)PyLong_AsUnsignedLongLongMask(a[13]);
            require(!PyErr_Occurred());
        }
        return b3x_train_adamw_gpu((int)sizes.size(), p.at.data(), p.type == at::kFloat ? B3X_F32 : B3X_BF16, g.at.data(),
            float_type(g.type), m.at.data(), v.at.data(), scales.empty() ? nullptr : (float* const*)scales.data(),
            f8 ? B3X_E4M3 : B3X_F32, copies.empty() ? nullptr : copies.data(), sizes.data(), decays.empty() ? nullptr : decays.data(),
            whole(a[4]), number(a[5]), number(a[6]), number(a[7]), number(a[8]), decay, factor, stochastic, seed, handle(a[15]));
    });
}

PyMethodDef methods[] = {
    {"logprob", (PyCFunction)(void (*)())logprob, METH_FASTCALL, nullptr},
    {"logprob_grad", (PyCFunction)(void (*)())logprob_grad, METH_FASTCALL, nullptr},
    {"advantage", (PyCFunction)(void (*)())advantage, METH_FASTCALL, nullptr},
    {"grad_norm", (PyCFunction)(void (*)())grad_norm, METH_FASTCALL, nullptr},
    {"adamw", (PyCFunction)(void (*)())adamw, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "b3train_py", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b3train_py(void) { return PyModule_Create(&module); }
