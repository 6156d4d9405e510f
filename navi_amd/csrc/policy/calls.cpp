// Calls of a block's operators (selective scan, convolution, norms) from Python, in one step: outputs and
// workspaces allocated, structures filled, launched, autograd told of writes. On the device a frame of every
// environment takes a few microseconds; a Python program's own reads of the tensors' shapes and strides, and its
// filling of structures, take more (a frame of one environment: 14.8 us a call through ctypes, 5.2 here; a training
// pass of a small scan, forward and backward: 201 us through ctypes and a function of Python's, 82 here).
//
// selective_step, conv_step, selective_scan, causal_conv and block_norm look their arguments over too. They take a
// call that is in order in every respect (and a frame's that asks for no gradients), and return None for any other,
// with nothing done: navi_amd/policy.py then says by name what is wrong, or takes tensors of a user's own class or
// of another device than the current one. What is in order is what policy.py's `_fine_...` functions say. scan, conv
// and block are the rollouts' calls of arguments that policy.py has looked over.
#define __HIP_PLATFORM_AMD__ 1  // (the host compiler reads HIP's headers)
#include <Python.h>

#include <cstring>
#include <initializer_list>
#include <optional>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "navi_policy.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library's entry points, in the order in which policy.py's binding gives their addresses.
struct Entries {
    int (*selective_step)(const navi_selective_scan_args*, void*);
    int (*selective_scan)(const navi_selective_scan_args*, void*);
    int (*selective_scan_backward)(const navi_selective_scan_args*, void*);
    int64_t (*selective_scan_scratch)(const navi_selective_scan_args*);
    int64_t (*selective_scan_workspace)(const navi_selective_scan_args*);
    int (*causal_conv)(const navi_causal_conv_args*, void*);
    int (*causal_conv_backward)(const navi_causal_conv_args*, void*);
    int64_t (*causal_conv_workspace)(const navi_causal_conv_args*);
    int (*block_norm)(const navi_block_norm_args*, void*);
    int (*block_norm_backward)(const navi_block_norm_args*, void*);
    int64_t (*block_norm_workspace)(const navi_block_norm_args*);
    const char* (*last_error)(void);
};
constexpr Py_ssize_t kEntries = sizeof(Entries) / sizeof(void*);

Entries entries{};

// A tensor of a call. `fine` falls to false at the first that is neither a plain tensor nor, where that is
// allowed, None.
struct Call {
    bool fine = true;
    const bool grad;  // gradients would be asked for and are not to be had

    explicit Call(bool differentiable) : grad(!differentiable && c10::GradMode::is_enabled()) {}

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

// Several of a call's arguments.
bool all_fine(Call& call, PyObject* const* v, int needed, int all) {
    for (int i = 0; i < all; i++) i < needed ? call.tensor(v[i]) : call.maybe(v[i]);
    return call.fine;
}

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

// (tensors that may be undefined)
bool vector(const Tensor& t, c10::Device device, int64_t length) { return vector(t.defined() ? &t : nullptr, device, length); }

bool mask(const Tensor& t, const Tensor& x) {
    return !t.defined() || ((t.scalar_type() == at::kBool || t.scalar_type() == at::kByte) && t.device() == x.device() &&
                            t.dim() == 2 && t.size(0) == x.size(0) && t.size(1) == x.size(1));
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

int64_t checked(int64_t code) {
    TORCH_CHECK(code >= 0, entries.last_error());
    return code;
}

// (a backward pass runs in a thread of autograd's, which does not hold Python's lock)
struct Unlocked {
    PyThreadState* kept = PyGILState_Check() ? PyEval_SaveThread() : nullptr;
    ~Unlocked() {
        if (kept) PyEval_RestoreThread(kept);
    }
};

template <typename Entry, typename Args> void launch(Entry entry, const Args& args, void* stream) {
    int code;
    {
        const Unlocked unlocked;
        code = entry(&args, stream);
    }
    checked(code);
}

// selective_step(x, dt, a, b, c, state, d, dt_bias, starts, out): the output, or None.
PyObject* selective_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || !entries.selective_step) Py_RETURN_NONE;
    Call call(false);
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
        width > NAVI_POLICY_MAX_STATE_DIM || dim <= 0 || dim > NAVI_POLICY_MAX_STATE_DIM || heads > NAVI_POLICY_MAX_HEADS ||
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
    launch(entries.selective_step, s, stream);
    wrote(*state);
    if (!to) return THPVariable_Wrap(std::move(out));
    wrote(out);
    Py_INCREF(v[9]);
    return v[9];
    END_HANDLE_TH_ERRORS
}

// conv_step(x, weight, window, bias, starts, activation's number, out): the output, or None.
PyObject* conv_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !entries.causal_conv || !PyLong_CheckExact(v[5])) Py_RETURN_NONE;
    Call call(false);
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
    launch(entries.causal_conv, s, stream);
    wrote(*window);
    if (!to) return THPVariable_Wrap(std::move(out));
    wrote(out);
    Py_INCREF(v[6]);
    return v[6];
    END_HANDLE_TH_ERRORS
}

// ---- whole rollouts and their gradients, of arguments that policy.py has looked over ----

// Memory that holds what a tensor shows: that of a lazily negated view holds its negative.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// Arguments: None is an undefined tensor.
variable_list given(PyObject* const* v, size_t n) {
    variable_list to(n);
    for (size_t i = 0; i < n; i++)
        if (v[i] != Py_None) {
            TORCH_CHECK(THPVariable_Check(v[i]), "a tensor is expected");
            to[i] = plain(THPVariable_Unpack(v[i]));
        }
    return to;
}

template <typename T> const T* read_of(const Tensor& t) { return read_of<T>(t.defined() ? &t : nullptr); }

template <typename T> T* write_of(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

template <size_t n> void strides_of(int64_t (&to)[n], const Tensor& t) {
    for (size_t i = 0; i < n; i++) to[i] = t.defined() ? t.stride(int64_t(i)) : 0;
}

Tensor like(const Tensor& t) { return t.defined() ? empty_like(t, t.scalar_type()) : Tensor(); }

// An input that may be left out, as autograd takes it.
using Maybe = std::optional<Tensor>;

Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }

// The gradient of saved input i, if one is asked for (autograd counts the inputs that are there).
Tensor like(const AutogradContext* ctx, const variable_list& saved, size_t i) {
    size_t edge = 0;
    for (size_t j = 0; j < i; j++) edge += saved[j].defined();
    return saved[i].defined() && ctx->needs_input_grad(edge) ? like(saved[i]) : Tensor();
}

Tensor floats(const Tensor& of, int64_t bytes) {
    return at::empty({bytes / 4}, of.options().dtype(at::kFloat).requires_grad(false));
}

// A gradient with its last axis dense; undefined stays so.
Tensor dense(const Tensor& given) {
    const Tensor t = plain(given);
    return !t.defined() || dense_last(t) ? t : t.contiguous();
}

// Steps that do not overlap and lie within the reach of the chunked kernels (policy.py's `_rows_apart`).
Tensor rows_apart(const Tensor& t) {
    constexpr int64_t farthest = INT32_MAX / NAVI_POLICY_CHUNK - (1 << 18);
    if (t.size(1) <= 1 || (t.size(3) <= t.stride(1) && t.stride(1) <= farthest / int64_t(t.element_size()))) return t;
    return t.contiguous();
}

// An env's steps within 2 GiB, which the convolution's offsets reach (rows of one element for masks).
Tensor steps_near(const Tensor& t) {
    if (!t.defined() || t.size(1) <= 1) return t;
    const int64_t row = t.dim() > 2 ? t.size(2) : 1;
    return t.stride(1) < ((int64_t{1} << 31) / int64_t(t.element_size()) - row) / t.size(1) ? t : t.contiguous();
}

// The device of a call is the current one during it: its stream.
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// The gradients of a backward pass that itself is differentiated (create_graph): there are none of them, which is
// an error where one is asked for, and no silence.
variable_list once(AutogradContext* ctx, const variable_list& given,
                   variable_list (*gradients)(AutogradContext*, const variable_list&)) {
    variable_list grads;
    {
        c10::AutoGradMode off(false);
        grads = gradients(ctx, given);
    }
    if (!c10::GradMode::is_enabled()) return grads;
    for (Tensor& t : grads)
        if (t.defined()) t.requires_grad_();
    const auto fail = std::make_shared<torch::autograd::DelayedError>(
        "the gradients of the policy's operators have no gradients of their own", int64_t(grads.size()));
    return (*fail)(std::move(grads));
}

bool records(std::initializer_list<const Tensor*> inputs) {
    if (c10::GradMode::is_enabled())
        for (const Tensor* t : inputs)
            if (t->defined() && t->requires_grad()) return true;
    return false;
}

// One output, or the outputs as a tuple.
PyObject* results(const variable_list& tensors) {
    if (tensors.size() == 1) return THPVariable_Wrap(tensors[0]);
    PyObject* tuple = PyTuple_New(Py_ssize_t(tensors.size()));
    if (!tuple) throw python_error();
    for (size_t i = 0; i < tensors.size(); i++) PyTuple_SET_ITEM(tuple, Py_ssize_t(i), THPVariable_Wrap(tensors[i]));
    return tuple;
}

void count(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK(n == want && entries.last_error, "wrong number of arguments"); }

struct Scan {
    Tensor x, dt, a, b, c, d, dt_bias, state, starts;
    explicit Scan(const variable_list& v)
        : x(v[0]), dt(v[1]), a(v[2]), b(v[3]), c(v[4]), d(v[5]), dt_bias(v[6]), state(v[7]), starts(v[8]) {}
    navi_selective_scan_args args() const {
        navi_selective_scan_args s{};
        s.dtype = type_of(x), s.heads = int32_t(x.size(2)), s.groups = int32_t(b.size(2)), s.state_dim = int32_t(b.size(3));
        s.head_dim = int32_t(x.size(3)), s.envs = x.size(0), s.steps = x.size(1);
        s.x = read_of<void>(x), s.b = read_of<void>(b), s.c = read_of<void>(c);
        strides_of(s.x_stride, x), strides_of(s.b_stride, b), strides_of(s.c_stride, c);
        s.dt = read_of<float>(dt), s.a = read_of<float>(a), s.d = read_of<float>(d), s.dt_bias = read_of<float>(dt_bias);
        strides_of(s.dt_stride, dt);
        s.starts = read_of<uint8_t>(starts), strides_of(s.starts_stride, starts);
        s.initial_state = read_of<float>(state);
        return s;
    }
    variable_list forward(bool return_state, bool stepwise) const {
        const On on(x);
        variable_list to{like(x)};
        if (return_state)
            to.push_back(at::empty({x.size(0), x.size(2), b.size(3), x.size(3)}, dt.options().requires_grad(false)));
        auto s = args();
        s.out = write_of<void>(to[0]), s.final_state = return_state ? write_of<float>(to[1]) : nullptr;
        if (stepwise) {
            launch(entries.selective_step, s, on.stream);
            return to;
        }
        Tensor scratch;
        if (const int64_t bytes = checked(entries.selective_scan_scratch(&s))) {
            scratch = floats(x, bytes);
            s.scratch = scratch.data_ptr();
        }
        launch(entries.selective_scan, s, on.stream);
        return to;
    }
};

struct ScanFunction : torch::autograd::Function<ScanFunction> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor dt, Tensor a, Tensor b, Tensor c, Maybe d,
                                 Maybe dt_bias, Maybe state, Maybe starts, bool return_state) {
        const variable_list inputs{x, dt, a, b, c, or_none(d), or_none(dt_bias), or_none(state), or_none(starts)};
        ctx->save_for_backward(inputs);
        ctx->set_materialize_grads(false);
        return Scan(inputs).forward(return_state, false);
    }

    static variable_list backward(AutogradContext* ctx, variable_list given) { return once(ctx, given, gradients); }

    static variable_list gradients(AutogradContext* ctx, const variable_list& given) {
        variable_list to(10);
        Tensor grad = given[0], grad_state = given.size() > 1 ? given[1] : Tensor();
        if (!grad.defined() && !grad_state.defined()) return to;
        const variable_list saved = ctx->get_saved_variables();
        const Scan g(saved);
        const On on(g.x);
        grad = grad.defined() ? rows_apart(dense(grad)) : like(g.x).zero_();
        if (grad_state.defined()) grad_state = plain(grad_state).contiguous();
        Tensor d_x = like(g.x), d_dt = like(g.dt), d_b = like(g.b), d_c = like(g.c), d_a = like(ctx, saved, 2),
               d_d = like(ctx, saved, 5), d_bias = like(ctx, saved, 6), d_state = like(ctx, saved, 7);
        if (g.x.numel() == 0) {
            for (Tensor t : {d_a, d_d, d_bias})
                if (t.defined()) t.zero_();
            if (d_state.defined()) grad_state.defined() ? d_state.copy_(grad_state) : d_state.zero_();
        } else {
            auto s = g.args();
            s.grad_out = read_of<void>(grad), s.grad_final_state = read_of<float>(grad_state);
            strides_of(s.grad_out_stride, grad);
            s.d_x = write_of<void>(d_x), s.d_b = write_of<void>(d_b), s.d_c = write_of<void>(d_c), s.d_dt = write_of<float>(d_dt);
            s.d_a = write_of<float>(d_a), s.d_d = write_of<float>(d_d), s.d_dt_bias = write_of<float>(d_bias);
            s.d_initial_state = write_of<float>(d_state);
            const Tensor workspace = floats(g.x, checked(entries.selective_scan_workspace(&s)));
            s.workspace = workspace.data_ptr();
            launch(entries.selective_scan_backward, s, on.stream);
        }
        return {d_x, d_dt, d_a, d_b, d_c, d_d, d_bias, d_state, Tensor(), Tensor()};
    }
};

PyObject* scan_of(const variable_list& in, bool return_state, int64_t stepwise) {
    if (records({&in[0], &in[1], &in[2], &in[3], &in[4], &in[5], &in[6], &in[7]}))
        return results(ScanFunction::apply(rows_apart(in[0]), in[1], in[2], rows_apart(in[3]), rows_apart(in[4]), maybe(in[5]),
                                           maybe(in[6]), maybe(in[7]), maybe(in[8]), return_state));
    if (in[0].size(1) <= stepwise) return results(Scan(in).forward(return_state, true));
    return results(Scan({rows_apart(in[0]), in[1], in[2], rows_apart(in[3]), rows_apart(in[4]), in[5], in[6], in[7], in[8]})
                       .forward(return_state, false));
}

// scan(x, dt, a, b, c, d, dt_bias, initial_state, starts, return_state, the most steps that go token by token): out, or
// (out, state).
PyObject* scan(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 11);
    return scan_of(given(v, 9), v[9] == Py_True, PyLong_AsLong(v[10]));
    END_HANDLE_TH_ERRORS
}

// selective_scan(the same): the same of a call that is in order, or None.
PyObject* selective_scan(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Call call(true);
    if (n != 11 || !entries.selective_scan || !all_fine(call, v, 5, 9)) Py_RETURN_NONE;
    const variable_list in = given(v, 9);
    const Tensor &x = in[0], &dt = in[1], &b = in[3], &c = in[4], &state = in[7];
    void* stream;
    if (type_of(x) < 0 || x.dim() != 4 || b.dim() != 4 || c.dim() != 4 || dt.dim() != 3 || !stream_of(x.device(), &stream))
        Py_RETURN_NONE;
    const auto device = x.device();
    const int64_t envs = x.size(0), steps = x.size(1), heads = x.size(2), width = x.size(3), groups = b.size(2), dim = b.size(3);
    if (b.scalar_type() != x.scalar_type() || c.scalar_type() != x.scalar_type() || dt.scalar_type() != at::kFloat ||
        b.device() != device || c.device() != device || dt.device() != device || b.size(0) != envs || b.size(1) != steps ||
        c.sizes() != b.sizes() || dt.size(0) != envs || dt.size(1) != steps || dt.size(2) != heads || groups <= 0 ||
        groups > heads || heads % groups || heads > NAVI_POLICY_MAX_HEADS || width <= 0 || width > NAVI_POLICY_MAX_STATE_DIM || dim <= 0 ||
        dim > NAVI_POLICY_MAX_STATE_DIM || !dense_last(x) || !dense_last(b) || !dense_last(c) || !vector(in[2], device, heads) ||
        !vector(in[5], device, heads) || !vector(in[6], device, heads) || !mask(in[8], x) ||
        (state.defined() && (state.scalar_type() != at::kFloat || state.device() != device || state.dim() != 4 ||
                             state.size(0) != envs || state.size(1) != heads || state.size(2) != dim || state.size(3) != width ||
                             !state.is_contiguous())))
        Py_RETURN_NONE;
    return scan_of(in, v[9] == Py_True, PyLong_AsLong(v[10]));
    END_HANDLE_TH_ERRORS
}

struct Convolution {
    Tensor x, weight, bias, window, starts;
    int64_t activation;
    Convolution(const variable_list& v, int64_t activation)
        : x(v[0]), weight(v[1]), bias(v[2]), window(v[3]), starts(v[4]), activation(activation) {}
    navi_causal_conv_args args() const {
        navi_causal_conv_args s{};
        s.dtype = type_of(x), s.channels = int32_t(x.size(2)), s.taps = int32_t(weight.size(1));
        s.activation = int32_t(activation), s.envs = x.size(0), s.steps = x.size(1);
        s.x = read_of<void>(x), s.weight = read_of<float>(weight), s.bias = read_of<float>(bias);
        strides_of(s.x_stride, x);
        s.starts = read_of<uint8_t>(starts), strides_of(s.starts_stride, starts);
        s.window = read_of<void>(window);
        return s;
    }
    variable_list forward(bool return_window) const {
        const On on(x);
        variable_list to{like(x)};
        if (return_window) to.push_back(at::empty({x.size(0), weight.size(1) - 1, x.size(2)}, x.options().requires_grad(false)));
        auto s = args();
        s.out = write_of<void>(to[0]), s.window_out = return_window ? write_of<void>(to[1]) : nullptr;
        launch(entries.causal_conv, s, on.stream);
        return to;
    }
};

struct ConvolutionFunction : torch::autograd::Function<ConvolutionFunction> {
    static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, Maybe bias, Maybe window, Maybe starts,
                                 int64_t activation, bool return_window) {
        const variable_list inputs{x, weight, or_none(bias), or_none(window), or_none(starts)};
        ctx->save_for_backward(inputs);
        ctx->saved_data["activation"] = activation;
        ctx->set_materialize_grads(false);
        return Convolution(inputs, activation).forward(return_window);
    }

    static variable_list backward(AutogradContext* ctx, variable_list given) { return once(ctx, given, gradients); }

    static variable_list gradients(AutogradContext* ctx, const variable_list& given) {
        variable_list to(7);
        Tensor grad = given[0], grad_window = given.size() > 1 ? given[1] : Tensor();
        if (!grad.defined() && !grad_window.defined()) return to;
        const variable_list saved = ctx->get_saved_variables();
        const Convolution g(saved, ctx->saved_data["activation"].toInt());
        const On on(g.x);
        grad = grad.defined() ? steps_near(dense(grad)) : like(g.x).zero_();
        if (grad_window.defined()) grad_window = plain(grad_window).contiguous();
        Tensor d_x = like(g.x), d_weight = like(ctx, saved, 1), d_bias = like(ctx, saved, 2),
               d_window = like(ctx, saved, 3);
        if (g.x.numel() == 0) {
            for (Tensor t : {d_weight, d_bias})
                if (t.defined()) t.zero_();
            if (d_window.defined()) grad_window.defined() ? d_window.copy_(grad_window) : d_window.zero_();
        } else {
            auto s = g.args();
            s.grad_out = read_of<void>(grad), s.grad_window = read_of<void>(grad_window);
            strides_of(s.grad_out_stride, grad);
            s.d_x = write_of<void>(d_x), s.d_weight = write_of<float>(d_weight), s.d_bias = write_of<float>(d_bias);
            s.d_window = write_of<void>(d_window);
            Tensor partial;
            if (d_weight.defined() || d_bias.defined()) {
                partial = floats(g.x, checked(entries.causal_conv_workspace(&s)));
                s.partial = write_of<float>(partial);
            }
            launch(entries.causal_conv_backward, s, on.stream);
        }
        return {d_x, d_weight, d_bias, d_window, Tensor(), Tensor(), Tensor()};
    }
};

PyObject* conv_of(const variable_list& in, int64_t activation, bool return_window) {
    const Tensor x = steps_near(in[0]), starts = steps_near(in[4]);
    if (records({&in[0], &in[1], &in[2], &in[3]}))
        return results(ConvolutionFunction::apply(x, in[1], maybe(in[2]), maybe(in[3]), maybe(starts), activation, return_window));
    return results(Convolution({x, in[1], in[2], in[3], starts}, activation).forward(return_window));
}

// conv(x, weight, bias, window, starts, activation's number, return_window): out, or (out, window after).
PyObject* conv(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 7);
    return conv_of(given(v, 5), PyLong_AsLong(v[5]), v[6] == Py_True);
    END_HANDLE_TH_ERRORS
}

// causal_conv(the same): the same of a call that is in order, or None.
PyObject* causal_conv(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Call call(true);
    if (n != 7 || !entries.causal_conv || !PyLong_CheckExact(v[5]) || !all_fine(call, v, 2, 5)) Py_RETURN_NONE;
    const variable_list in = given(v, 5);
    const Tensor &x = in[0], &weight = in[1], &window = in[3];
    void* stream;
    if (type_of(x) < 0 || x.dim() != 3 || weight.dim() != 2 || !stream_of(x.device(), &stream)) Py_RETURN_NONE;
    const auto device = x.device();
    const int64_t channels = x.size(2), taps = weight.size(1);
    if (channels <= 0 || channels > 65536 || taps < 2 || taps > NAVI_POLICY_MAX_TAPS || !dense_last(x) ||
        weight.scalar_type() != at::kFloat || weight.device() != device || weight.size(0) != channels || !weight.is_contiguous() ||
        !vector(in[2], device, channels) || !mask(in[4], x) ||
        (window.defined() && (window.scalar_type() != x.scalar_type() || window.device() != device || window.dim() != 3 ||
                              window.size(0) != x.size(0) || window.size(1) != taps - 1 || window.size(2) != channels ||
                              !window.is_contiguous())))
        Py_RETURN_NONE;
    return conv_of(in, PyLong_AsLong(v[5]), v[6] == Py_True);
    END_HANDLE_TH_ERRORS
}

struct Between {
    Tensor y, residual, gate, scale, post, pre;
    double eps;
    Between(const variable_list& v, double eps)
        : y(v[0]), residual(v[1]), gate(v[2]), scale(v[3]), post(v[4]), pre(v[5]), eps(eps) {}
    navi_block_norm_args args() const {
        navi_block_norm_args s{};
        s.dtype = type_of(y), s.stream_dtype = type_of(residual), s.width = int32_t(y.size(2)), s.eps = float(eps);
        s.envs = y.size(0), s.steps = y.size(1);
        s.y = read_of<void>(y), s.residual = read_of<void>(residual), s.gate = read_of<void>(gate);
        strides_of(s.y_stride, y), strides_of(s.residual_stride, residual), strides_of(s.gate_stride, gate);
        s.scale = read_of<float>(scale), s.post_weight = read_of<float>(post), s.pre_weight = read_of<float>(pre);
        return s;
    }
    variable_list forward() const {
        const On on(y);
        variable_list to{empty_like(y, residual.scalar_type()), like(y)};
        auto s = args();
        s.stream = write_of<void>(to[0]), s.normed = write_of<void>(to[1]);
        launch(entries.block_norm, s, on.stream);
        return to;
    }
};

struct BetweenFunction : torch::autograd::Function<BetweenFunction> {
    static variable_list forward(AutogradContext* ctx, Tensor y, Tensor residual, Maybe gate, Maybe scale, Maybe post,
                                 Maybe pre, double eps) {
        const variable_list inputs{y, residual, or_none(gate), or_none(scale), or_none(post), or_none(pre)};
        ctx->save_for_backward(inputs);
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        return Between(inputs, eps).forward();
    }

    static variable_list backward(AutogradContext* ctx, variable_list given) { return once(ctx, given, gradients); }

    static variable_list gradients(AutogradContext* ctx, const variable_list& given) {
        if (!given[0].defined() && !given[1].defined()) return variable_list(7);
        const variable_list saved = ctx->get_saved_variables();
        const Between g(saved, ctx->saved_data["eps"].toDouble());
        const On on(g.y);
        const Tensor grad_sum = dense(given[0]), grad_normed = dense(given[1]);
        Tensor d_y = like(g.y), d_residual = like(g.residual), d_gate = like(ctx, saved, 2), d_scale = like(ctx, saved, 3),
               d_post = like(ctx, saved, 4), d_pre = like(ctx, saved, 5);
        if (g.y.numel() == 0) {
            for (Tensor t : {d_scale, d_post, d_pre})
                if (t.defined()) t.zero_();
        } else {
            auto s = g.args();
            s.grad_stream = read_of<void>(grad_sum), s.grad_normed = read_of<void>(grad_normed);
            strides_of(s.grad_stream_stride, grad_sum), strides_of(s.grad_normed_stride, grad_normed);
            s.d_y = write_of<void>(d_y), s.d_residual = write_of<void>(d_residual), s.d_gate = write_of<void>(d_gate);
            s.d_scale = write_of<float>(d_scale), s.d_post_weight = write_of<float>(d_post);
            s.d_pre_weight = write_of<float>(d_pre);
            Tensor partial;
            if (d_scale.defined() || d_post.defined() || d_pre.defined()) {
                partial = floats(g.y, checked(entries.block_norm_workspace(&s)));
                s.partial = write_of<float>(partial);
            }
            launch(entries.block_norm_backward, s, on.stream);
        }
        return {d_y, d_residual, d_gate, d_scale, d_post, d_pre, Tensor()};
    }
};

PyObject* block_of(const variable_list& in, double eps) {
    if (records({&in[0], &in[1], &in[2], &in[3], &in[4], &in[5]}))
        return results(BetweenFunction::apply(in[0], in[1], maybe(in[2]), maybe(in[3]), maybe(in[4]), maybe(in[5]), eps));
    return results(Between(in, eps).forward());
}

// block(y, residual, gate, scale, post_weight, pre_weight, eps): (stream, normed).
PyObject* block(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    count(n, 7);
    return block_of(given(v, 6), PyFloat_AsDouble(v[6]));
    END_HANDLE_TH_ERRORS
}

// block_norm(the same): the same of a call that is in order, or None.
PyObject* block_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Call call(true);
    if (n != 7 || !entries.block_norm || !PyFloat_CheckExact(v[6]) || !all_fine(call, v, 2, 6)) Py_RETURN_NONE;
    const variable_list in = given(v, 6);
    const Tensor &y = in[0], &residual = in[1], &gate = in[2];
    const auto device = y.device();
    const int type = type_of(y), stream_type = type_of(residual);
    void* stream;
    if (type < 0 || y.dim() != 3 || !stream_of(device, &stream)) Py_RETURN_NONE;
    const int64_t width = y.size(2);
    if (residual.device() != device || (stream_type != type && stream_type != NAVI_POLICY_F32) || residual.sizes() != y.sizes() ||
        width <= 0 || width > NAVI_POLICY_MAX_BLOCK_WIDTH || !dense_last(y) || !dense_last(residual) ||
        (gate.defined() && (gate.scalar_type() != y.scalar_type() || gate.device() != device || gate.sizes() != y.sizes() ||
                            !dense_last(gate))) ||
        !vector(in[3], device, width) || !vector(in[4], device, width) || !vector(in[5], device, width))
        Py_RETURN_NONE;
    return block_of(in, PyFloat_AS_DOUBLE(v[6]));
    END_HANDLE_TH_ERRORS
}

// bind(the library's entry points): their addresses in the order above.
PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != kEntries) {
        PyErr_Format(PyExc_TypeError, "bind takes %zd addresses", kEntries);
        return nullptr;
    }
    void* at[kEntries];
    for (Py_ssize_t i = 0; i < n; i++)
        if (!(at[i] = PyLong_AsVoidPtr(v[i])) && PyErr_Occurred()) return nullptr;
    static_assert(sizeof(at) == sizeof(entries), "addresses alone");
    memcpy(&entries, at, sizeof(at));
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(selective_step), METHOD(conv_step), METHOD(block_norm),
                         METHOD(scan), METHOD(selective_scan), METHOD(conv), METHOD(causal_conv), METHOD(block),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_policy_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__policy_calls() { return PyModule_Create(&module); }
