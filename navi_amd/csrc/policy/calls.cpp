// Calls of the policy's operators for a frame of every environment, from Python in one step: arguments looked
// over, output allocated, launched, autograd told of the writes. On the device such a call takes a few
// microseconds, a Python program's own reads of the tensors' shapes and strides three times that (a frame of one
// environment: 14.8 us a call through ctypes; each function below states what it takes).
//
// A function takes a call that is in order in every respect, and returns None for any other, with nothing done:
// navi_amd/policy.py then says by name what is wrong, or goes the way that keeps gradients. So nothing is
// refused here, and what is in order is what policy.py's `_fine_...` functions say.
#define __HIP_PLATFORM_AMD__ 1  // (the host compiler reads HIP's headers)
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "navi_policy.h"

namespace {

using at::Tensor;

using Step = int (*)(const navi_selective_scan_args*, void*);
using Conv = int (*)(const navi_causal_conv_args*, void*);
using Block = int (*)(const navi_block_norm_args*, void*);

Step step_entry = nullptr;
Conv conv_entry = nullptr;
Block block_entry = nullptr;

// A tensor of a call. `fine` falls to false at the first that is neither a plain tensor nor, where that is
// allowed, None.
struct Call {
    bool fine = true;
    bool grad = c10::GradMode::is_enabled();
    c10::Device device{c10::DeviceType::CPU};

    const Tensor* tensor(PyObject* o) {
        if (!THPVariable_CheckExact(o)) {  // (a tensor or a parameter, no class of a user's)
            fine = false;
            return nullptr;
        }
        const Tensor& t = THPVariable_Unpack(o);
        // (a conjugate or negative view's, a batch's of vmap, or a fake tensor's memory is not what it shows)
        if (t.layout() != at::kStrided || t.is_conj() || t.is_neg() || t.unsafeGetTensorImpl()->is_python_dispatch() ||
            t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::FuncTorchBatched) || (grad && t.requires_grad()))
            fine = false;
        return &t;
    }
    const Tensor* maybe(PyObject* o) { return o == Py_None ? nullptr : tensor(o); }
};

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return NAVI_POLICY_F32;
        case at::kBFloat16: return NAVI_POLICY_BF16;
        case at::kHalf: return NAVI_POLICY_F16;
        default: return -1;
    }
}

bool dense_last(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

bool vector(const Tensor* t, c10::Device device, int64_t length) {
    return !t || (t->scalar_type() == at::kFloat && t->device() == device && t->dim() == 1 && t->size(0) == length &&
                  t->is_contiguous());
}

bool mask(const Tensor* t, c10::Device device, int64_t length) {
    return !t || ((t->scalar_type() == at::kBool || t->scalar_type() == at::kByte) && t->device() == device &&
                  t->dim() == 1 && t->size(0) == length);
}

void* at_of(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

// (constant: data_ptr() of a lazily copied tensor would copy it)
template <typename T> const T* read_of(const Tensor* t) { return t ? static_cast<const T*>(t->const_data_ptr()) : nullptr; }

Tensor empty_like(const Tensor& t, at::ScalarType type) {
    return at::empty(t.sizes(), t.options().dtype(type).memory_format(at::MemoryFormat::Contiguous).requires_grad(false));
}

void wrote(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The device's current stream, if the device is the current one (entry points launch on that).
bool stream_of(c10::Device device, void** stream) {
    if (device.type() != c10::DeviceType::CUDA || device.index() != c10::hip::current_device()) return false;
    *stream = c10::hip::getCurrentHIPStream(device.index()).stream();
    return true;
}

template <typename Entry, typename Args> int launch(Entry entry, const Args& args, void* stream) {
    int code;
    Py_BEGIN_ALLOW_THREADS code = entry(&args, stream);
    Py_END_ALLOW_THREADS return code;
}

// (an entry point's refusal is told by policy.py, which asks for its words)
PyObject* refused(int code) { return PyLong_FromLong(code); }

// selective_step(x, dt, a, b, c, state, d, dt_bias, starts, out): the output, None or an entry point's code.
PyObject* selective_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || !step_entry) Py_RETURN_NONE;
    Call call;
    const Tensor *x = call.tensor(v[0]), *dt = call.tensor(v[1]), *a = call.tensor(v[2]), *b = call.tensor(v[3]),
                 *c = call.tensor(v[4]), *state = call.tensor(v[5]), *d = call.maybe(v[6]), *dt_bias = call.maybe(v[7]),
                 *starts = call.maybe(v[8]), *to = call.maybe(v[9]);
    if (!call.fine) Py_RETURN_NONE;
    const auto device = x->device();
    const int type = type_of(*x);
    void* stream;
    if (type < 0 || x->dim() != 3 || b->dim() != 3 || c->dim() != 3 || dt->dim() != 2 || state->dim() != 4 ||
        !stream_of(device, &stream))
        Py_RETURN_NONE;
    const int64_t envs = x->size(0), heads = x->size(1), width = x->size(2), groups = b->size(1), dim = b->size(2);
    const auto kind = x->scalar_type();
    if (b->scalar_type() != kind || c->scalar_type() != kind || dt->scalar_type() != at::kFloat ||
        state->scalar_type() != at::kFloat || b->device() != device || c->device() != device || dt->device() != device ||
        state->device() != device || b->size(0) != envs || c->sizes() != b->sizes() || dt->size(0) != envs ||
        dt->size(1) != heads || groups <= 0 || groups > heads || heads % groups || width <= 0 ||
        width > NAVI_POLICY_MAX_STATE_DIM || dim <= 0 || dim > NAVI_POLICY_MAX_STATE_DIM || heads > INT32_MAX ||
        !dense_last(*x) || !dense_last(*b) || !dense_last(*c) || state->size(0) != envs || state->size(1) != heads ||
        state->size(2) != dim || state->size(3) != width || !state->is_contiguous() || !vector(a, device, heads) ||
        !vector(d, device, heads) || !vector(dt_bias, device, heads) || !mask(starts, device, envs) ||
        (to && (to->scalar_type() != kind || to->device() != device || to->sizes() != x->sizes() || !to->is_contiguous())))
        Py_RETURN_NONE;
    Tensor out = to ? *to : empty_like(*x, kind);
    navi_selective_scan_args s{};
    s.dtype = type, s.heads = int32_t(heads), s.groups = int32_t(groups), s.state_dim = int32_t(dim), s.head_dim = int32_t(width);
    s.envs = envs, s.steps = 1;
    s.x = read_of<void>(x), s.b = read_of<void>(b), s.c = read_of<void>(c);
    s.x_stride[0] = x->stride(0), s.x_stride[2] = x->stride(1);
    s.b_stride[0] = b->stride(0), s.b_stride[2] = b->stride(1);
    s.c_stride[0] = c->stride(0), s.c_stride[2] = c->stride(1);
    s.dt = read_of<float>(dt), s.dt_stride[0] = dt->stride(0), s.dt_stride[2] = dt->stride(1);
    s.a = read_of<float>(a), s.d = read_of<float>(d), s.dt_bias = read_of<float>(dt_bias);
    s.starts = read_of<uint8_t>(starts), s.starts_stride[0] = starts ? starts->stride(0) : 0;
    s.final_state = static_cast<float*>(at_of(state)), s.initial_state = s.final_state;
    s.out = at_of(&out);
    if (const int code = launch(step_entry, s, stream)) return refused(code);
    wrote(*state);
    if (!to) return THPVariable_Wrap(std::move(out));
    wrote(out);
    Py_INCREF(v[9]);
    return v[9];
    END_HANDLE_TH_ERRORS
}

// conv_step(x, weight, window, bias, starts, activation's number, out): the output, None or an entry point's code.
PyObject* conv_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !conv_entry || !PyLong_CheckExact(v[5])) Py_RETURN_NONE;
    Call call;
    const Tensor *x = call.tensor(v[0]), *weight = call.tensor(v[1]), *window = call.tensor(v[2]), *bias = call.maybe(v[3]),
                 *starts = call.maybe(v[4]), *to = call.maybe(v[6]);
    if (!call.fine) Py_RETURN_NONE;
    const auto device = x->device();
    const int type = type_of(*x);
    void* stream;
    if (type < 0 || x->dim() != 2 || weight->dim() != 2 || window->dim() != 3 || !stream_of(device, &stream)) Py_RETURN_NONE;
    const int64_t envs = x->size(0), channels = x->size(1), taps = weight->size(1);
    const auto kind = x->scalar_type();
    if (channels <= 0 || channels > 65536 || taps < 2 || taps > NAVI_POLICY_MAX_TAPS || !dense_last(*x) ||
        weight->scalar_type() != at::kFloat || weight->device() != device || weight->size(0) != channels ||
        !weight->is_contiguous() || window->scalar_type() != kind || window->device() != device || window->size(0) != envs ||
        window->size(1) != taps - 1 || window->size(2) != channels || !window->is_contiguous() ||
        !vector(bias, device, channels) || !mask(starts, device, envs) ||
        (to && (to->scalar_type() != kind || to->device() != device || to->sizes() != x->sizes() || !to->is_contiguous())))
        Py_RETURN_NONE;
    Tensor out = to ? *to : empty_like(*x, kind);
    navi_causal_conv_args s{};
    s.dtype = type, s.channels = int32_t(channels), s.taps = int32_t(taps), s.activation = int32_t(PyLong_AsLong(v[5]));
    s.envs = envs, s.steps = 1;
    s.x = read_of<void>(x), s.x_stride[0] = x->stride(0);
    s.weight = read_of<float>(weight), s.bias = read_of<float>(bias);
    s.starts = read_of<uint8_t>(starts), s.starts_stride[0] = starts ? starts->stride(0) : 0;
    s.window_out = at_of(window), s.window = s.window_out;
    s.out = at_of(&out);
    if (const int code = launch(conv_entry, s, stream)) return refused(code);
    wrote(*window);
    if (!to) return THPVariable_Wrap(std::move(out));
    wrote(out);
    Py_INCREF(v[6]);
    return v[6];
    END_HANDLE_TH_ERRORS
}

// block_norm(y, residual, gate, scale, post_weight, pre_weight, eps): both outputs, None or an entry point's code.
PyObject* block_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !block_entry || !PyFloat_CheckExact(v[6])) Py_RETURN_NONE;
    Call call;
    const Tensor *y = call.tensor(v[0]), *residual = call.tensor(v[1]), *gate = call.maybe(v[2]), *scale = call.maybe(v[3]),
                 *post = call.maybe(v[4]), *pre = call.maybe(v[5]);
    if (!call.fine) Py_RETURN_NONE;
    const auto device = y->device();
    const int type = type_of(*y), stream_type = type_of(*residual);
    void* stream;
    if (type < 0 || y->dim() != 3 || !stream_of(device, &stream)) Py_RETURN_NONE;
    const int64_t width = y->size(2);
    if (residual->device() != device || (stream_type != type && stream_type != NAVI_POLICY_F32) ||
        residual->sizes() != y->sizes() || width <= 0 || width > NAVI_POLICY_MAX_BLOCK_WIDTH || !dense_last(*y) ||
        !dense_last(*residual) ||
        (gate && (gate->scalar_type() != y->scalar_type() || gate->device() != device || gate->sizes() != y->sizes() ||
                  !dense_last(*gate))) ||
        !vector(scale, device, width) || !vector(post, device, width) || !vector(pre, device, width))
        Py_RETURN_NONE;
    Tensor sum = empty_like(*y, residual->scalar_type()), normed = empty_like(*y, y->scalar_type());
    navi_block_norm_args s{};
    s.dtype = type, s.stream_dtype = stream_type, s.width = int32_t(width), s.eps = float(PyFloat_AS_DOUBLE(v[6]));
    s.envs = y->size(0), s.steps = y->size(1);
    s.y = read_of<void>(y), s.residual = read_of<void>(residual), s.gate = read_of<void>(gate);
    for (int i = 0; i < 2; i++) {
        s.y_stride[i] = y->stride(i), s.residual_stride[i] = residual->stride(i);
        s.gate_stride[i] = gate ? gate->stride(i) : 0;
    }
    s.scale = read_of<float>(scale), s.post_weight = read_of<float>(post), s.pre_weight = read_of<float>(pre);
    s.stream = at_of(&sum), s.normed = at_of(&normed);
    if (const int code = launch(block_entry, s, stream)) return refused(code);
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(sum)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(normed)));
    return pair;
    END_HANDLE_TH_ERRORS
}

// bind(selective_step's, causal_conv's, block_norm's address): the library's entry points.
PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "bind takes three addresses");
        return nullptr;
    }
    void* at[3];
    for (int i = 0; i < 3; i++)
        if (!(at[i] = PyLong_AsVoidPtr(v[i])) && PyErr_Occurred()) return nullptr;
    step_entry = reinterpret_cast<Step>(at[0]);
    conv_entry = reinterpret_cast<Conv>(at[1]);
    block_entry = reinterpret_cast<Block>(at[2]);
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(selective_step), METHOD(conv_step), METHOD(block_norm), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_policy_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__policy_calls() { return PyModule_Create(&module); }
