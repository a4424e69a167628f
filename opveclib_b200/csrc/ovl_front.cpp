// The usual calls of the sequence operators (sequence.py) in one step from Python's arguments to the launch: everything on
// the current device and of the right types and shapes.  Any other call gets None back and takes the way through
// sequence.py, which says what is wrong with it, copies or changes the device; this file decides nothing that it does not,
// it only saves the time of its checks and, for what is differentiated, of autograd functions in Python (figures beside
// _load_front there).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <memory>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/ovl_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

using Launch = int (*)(const void*, void*);
enum Entry { kScan, kScanBackward, kScanStep, kConv, kConvBackward, kConvStep, kNorm, kNormBackward, kEntries };
Launch g_launch[kEntries] = {};
uint64_t (*g_scan_bytes)(const OvlSelectiveScan*, int) = nullptr;
uint64_t (*g_conv_bytes)(const OvlCausalConv*) = nullptr;
uint64_t (*g_norm_bytes)(const OvlRmsNorm*) = nullptr;
PyObject* g_parameter = nullptr;       // torch.nn.Parameter

constexpr int64_t kMaxStates = 128, kMaxTaps = 8, kMaxColumns = 32768;

// A call's tensors: one device, plain strided memory.
struct Tensors {
    c10::Device device = c10::kCPU;
    bool grad = c10::GradMode::is_enabled();
    bool differentiated = false;       // a gradient is wanted for one of them

    // the tensor behind an argument, or null if it is not one that is dealt with here
    const at::Tensor* get(PyObject* o) {
        if (Py_TYPE(o) != (PyTypeObject*)THPVariableClass && (PyObject*)Py_TYPE(o) != g_parameter) return nullptr;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.layout() != c10::kStrided || !t.unsafeGetTensorImpl()->has_storage()) return nullptr;
        if (device.is_cpu()) device = t.device();
        else if (t.device() != device) return nullptr;
        if (t.is_neg() || t._fw_grad(0).defined()) return nullptr;
        if (!t.const_data_ptr() && t.numel() > 0) return nullptr;        // (a null address would count as left out)
        differentiated |= grad && t.requires_grad();
        return &t;
    }
    // the same of a type and shape; None where allowed gives null and leaves `right`
    const at::Tensor* get(PyObject* o, c10::ScalarType type, c10::IntArrayRef shape, bool dense, bool optional, bool& right) {
        if (optional && o == Py_None) return nullptr;
        const at::Tensor* t = get(o);
        if (!t || t->scalar_type() != type || t->sizes() != shape) right = false;
        else if (!t->is_contiguous() && (dense || t->stride(-1) != 1)) right = false;
        return right ? t : nullptr;
    }
};

int64_t code_of(c10::ScalarType type) {
    return type == at::kFloat ? OVL_FLOAT32 : type == at::kHalf ? OVL_FLOAT16 : type == at::kBFloat16 ? OVL_BFLOAT16 : 0;
}
template <typename T = void>
T* data(const at::Tensor* t) { return t ? reinterpret_cast<T*>(t->data_ptr()) : nullptr; }
int64_t stride(const at::Tensor* t, int axis) { return t ? t->stride(axis) : 0; }

// The current device is the tensors', and nothing looks on or changes the calls: neither a dispatch mode nor a tracer,
// before dispatch either (sequence.py refuses those that would keep this call's answer).
bool plain(const Tensors& all) {
    return all.device.index() == c10::cuda::current_device() && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
           !torch::jit::tracer::isTracing() && !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
}

Maybe maybe(const at::Tensor* t) { return t ? Maybe(*t) : Maybe(); }
const at::Tensor* behind(const Maybe& t) { return t ? &*t : nullptr; }
const at::Tensor* behind(const Tensor& t) { return t.defined() ? &t : nullptr; }

// A launch that is refused: a call tries it again through sequence.py, which reports it; a backward pass raises this.
struct Failed : std::runtime_error {
    explicit Failed(int status) : std::runtime_error("a sequence operator could not be launched: status " + std::to_string(status)) {}
};

// Enqueues on torch's current stream of the device.
template <typename A>
void launch(Entry entry, const A& args, c10::Device device) {
    const int status = g_launch[entry](&args, c10::cuda::getCurrentCUDAStream(device.index()).stream());
    if (status != OVL_OK) throw Failed(status);
}
// Without Python's lock: a launch waits where the queue of launches is full.
template <typename F>
auto unlocked(F body) {
    pybind11::gil_scoped_release release;
    return body();
}

void changed(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* none() { Py_RETURN_NONE; }

PyObject* tuple_of(const variable_list& tensors) {
    PyObject* r = PyTuple_New(tensors.size());
    if (!r) return nullptr;
    for (size_t i = 0; i < tensors.size(); ++i) {
        PyObject* o = THPVariable_Wrap(tensors[i]);
        if (!o) {
            Py_DECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, i, o);
    }
    return r;
}

// Uninitialised memory from torch's allocator, without the way through its dispatcher (which nothing looks on here, see
// `plain`: 1 us of the 5 us of a small call).
Tensor fresh(c10::IntArrayRef shape, c10::ScalarType type, const Tensor& like) {
    return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

// Bytes that live until the launch is enqueued; torch's allocator keeps them for the stream.
template <typename A>
Tensor workspace(A& args, uint64_t size, const Tensor& like) {
    args.workspace_bytes = size;
    if (!size) return Tensor();
    Tensor w = fresh({(int64_t)size}, at::kByte, like);
    args.workspace = w.data_ptr();
    return w;
}

// A gradient from above may be a view of negated values, as an input (see Tensors::get): kernels read memory, so what they
// get goes through one of these two.  The gradient above an output that nothing used is zeros; a kernel reads any strides
// but the innermost axis's.
Tensor above(const Tensor& grad, const Tensor& like, int64_t columns) {
    if (!grad.defined()) return at::zeros({columns}, like.options()).expand(like.sizes());
    const Tensor g = grad.resolve_neg();
    return g.is_contiguous() || g.stride(-1) == 1 ? g : g.contiguous();
}
// the same of an output whose kernels read dense memory, or none for zeros
Tensor dense_above(const Tensor& grad) { return grad.defined() ? grad.resolve_neg().contiguous() : grad; }

// Gradients that are differentiated again (create_graph) say so instead of counting as constants.
variable_list once(variable_list grads, const char* what) {
    if (!c10::GradMode::is_enabled()) return grads;
    variable_list inputs(grads.size());
    for (size_t i = 0; i < grads.size(); ++i)
        if (grads[i].defined()) inputs[i] = grads[i].detach().requires_grad_();
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once", (int64_t)grads.size());
    return (*error)(std::move(inputs));
}

// 1 or 0 for Python's truth of a plain bool or None; -1 for anything else
int truth(PyObject* o) { return o == Py_True ? 1 : o == Py_False || o == Py_None ? 0 : -1; }
// 1 for 'silu', 0 for None; -1 for anything else
int silu_of(PyObject* o) {
    if (o == Py_None) return 0;
    return PyUnicode_CheckExact(o) && PyUnicode_CompareWithASCIIString(o, "silu") == 0 ? 1 : -1;
}

// No C++ exception leaves an entry: torch's become Python's (those of the hooks that pack saved tensors, by which
// checkpointing ends a repeated forward pass, among them).
template <typename F>
PyObject* guarded(F body) {
    HANDLE_TH_ERRORS
    try {
        return body();
    } catch (const Failed&) {
        return none();
    }
    END_HANDLE_TH_ERRORS
}

// state, u, delta, A, B, C, D, z, delta_bias, delta_softplus, slots
PyObject* selective_scan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Tensors all;
        const at::Tensor* u = n == 11 ? all.get(a[1]) : nullptr;
        const at::Tensor* state = u ? all.get(a[0]) : nullptr;
        const int softplus = u ? truth(a[9]) : -1;
        if (!state || softplus < 0 || u->dim() != 2 || state->dim() != 3 || state->scalar_type() != at::kFloat || !state->is_contiguous())
            return none();
        const c10::ScalarType t = u->scalar_type();
        const int64_t rows = u->size(0), channels = u->size(1), states = state->size(2);
        bool right = code_of(t) != 0 && channels >= 1 && states >= 1 && states <= kMaxStates && state->size(1) == channels &&
                     (u->is_contiguous() || u->stride(1) == 1);
        const at::Tensor* B = right ? all.get(a[4]) : nullptr;
        if (!B || B->dim() < 2 || B->dim() > 3) return none();
        const int64_t groups = B->dim() == 3 ? B->size(1) : 1;
        if (groups < 1 || channels % groups) return none();
        const int64_t full[3] = {rows, groups, states}, flat[2] = {rows, states};
        const c10::IntArrayRef shape = B->dim() == 3 ? c10::IntArrayRef(full, 3) : c10::IntArrayRef(flat, 2);
        B = all.get(a[4], t, shape, false, false, right);
        const at::Tensor* C = all.get(a[5], t, shape, false, false, right);
        const at::Tensor* delta = all.get(a[2], t, u->sizes(), false, false, right);
        const at::Tensor* z = all.get(a[7], t, u->sizes(), false, true, right);
        const at::Tensor* A = all.get(a[3], at::kFloat, {channels, states}, true, false, right);
        const at::Tensor* D = all.get(a[6], at::kFloat, {channels}, true, true, right);
        const at::Tensor* bias = all.get(a[8], at::kFloat, {channels}, true, true, right);
        const at::Tensor* slots = all.get(a[10], at::kInt, {rows}, true, true, right);
        if (!right || all.differentiated || (!slots && state->size(0) < rows) || !plain(all)) return none();
        const at::Tensor out = fresh({rows, channels}, u->scalar_type(), *u);
        const bool grouped = B->dim() == 3;
        OvlSelectiveScanStep s{};
        s.dtype = code_of(t), s.rows = rows, s.channels = channels, s.states = states, s.groups = groups, s.delta_softplus = softplus;
        s.slots = state->size(0);
        s.u = data(u), s.delta = data(delta), s.z = data(z), s.B = data(B), s.C = data(C);
        s.A = data<float>(A), s.D = data<float>(D), s.delta_bias = data<float>(bias), s.slot_of_row = data<int32_t>(slots);
        s.u_row = stride(u, 0), s.delta_row = stride(delta, 0), s.z_row = stride(z, 0);
        s.B_row = stride(B, 0), s.C_row = stride(C, 0);
        s.B_group = grouped ? stride(B, 1) : 0, s.C_group = grouped ? stride(C, 1) : 0;
        s.state = data<float>(state), s.out = out.data_ptr();
        unlocked([&] { launch(kScanStep, s, all.device); });
        changed(*state);
        return THPVariable_Wrap(out);
    });
}

// state, x, weight, bias, activation, slots
PyObject* causal_conv1d_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Tensors all;
        const at::Tensor* x = n == 6 ? all.get(a[1]) : nullptr;
        const at::Tensor* state = x ? all.get(a[0]) : nullptr;
        const at::Tensor* weight = state ? all.get(a[2]) : nullptr;
        const int silu = weight ? silu_of(a[4]) : -1;
        if (silu < 0 || x->dim() != 2 || state->dim() != 3 || weight->dim() != 2 || !state->is_contiguous()) return none();
        const c10::ScalarType t = x->scalar_type(), w = weight->scalar_type();
        const int64_t rows = x->size(0), channels = x->size(1), taps = weight->size(1);
        bool right = code_of(t) != 0 && (w == t || w == at::kFloat) && channels >= 1 && taps >= 1 && taps <= kMaxTaps &&
                     state->scalar_type() == t && state->size(1) == taps - 1 && state->size(2) == channels &&
                     weight->size(0) == channels && weight->is_contiguous() && (x->is_contiguous() || x->stride(1) == 1);
        const at::Tensor* bias = all.get(a[3], w, {channels}, true, true, right);
        const at::Tensor* slots = all.get(a[5], at::kInt, {rows}, true, true, right);
        if (!right || all.differentiated || (!slots && state->size(0) < rows) || !plain(all)) return none();
        const at::Tensor out = fresh({rows, channels}, x->scalar_type(), *x);
        OvlCausalConvStep s{};
        s.dtype = code_of(t), s.rows = rows, s.channels = channels, s.taps = taps, s.silu = silu, s.params_f32 = w == at::kFloat;
        s.slots = state->size(0);
        s.x = data(x), s.weight = data(weight), s.bias = data(bias), s.slot_of_row = data<int32_t>(slots);
        s.x_row = stride(x, 0), s.state = data(state), s.out = out.data_ptr();
        unlocked([&] { launch(kConvStep, s, all.device); });
        changed(*state);
        return THPVariable_Wrap(out);
    });
}

// ---- the scan over whole sequences

OvlSelectiveScan scan_args(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor* D,
                           const Tensor* z, const Tensor* bias, const Tensor* initial, const Tensor* lengths, int softplus) {
    OvlSelectiveScan s{};
    const bool grouped = B.dim() == 4;
    s.dtype = code_of(u.scalar_type()), s.batch = u.size(0), s.length = u.size(1), s.channels = u.size(2), s.states = A.size(1);
    s.groups = grouped ? B.size(2) : 1, s.delta_softplus = softplus;
    s.u = data(&u), s.delta = data(&delta), s.z = data(z), s.B = data(&B), s.C = data(&C);
    s.A = data<float>(&A), s.D = data<float>(D), s.delta_bias = data<float>(bias), s.initial_state = data<float>(initial);
    s.lengths = data<int32_t>(lengths);
    s.u_batch = u.stride(0), s.u_token = u.stride(1), s.delta_batch = delta.stride(0), s.delta_token = delta.stride(1);
    s.z_batch = stride(z, 0), s.z_token = stride(z, 1);
    s.B_batch = B.stride(0), s.B_token = B.stride(1), s.C_batch = C.stride(0), s.C_token = C.stride(1);
    s.B_group = grouped ? B.stride(2) : 0, s.C_group = grouped ? C.stride(2) : 0;
    return s;
}

// (out, final state); `saved` takes the states in front of every 16th token for the backward pass.
variable_list scan_forward(OvlSelectiveScan s, const Tensor& u, const Tensor& A, Tensor* saved) {
    Tensor out = fresh(u.sizes(), u.scalar_type(), u);
    Tensor final_state = fresh({s.batch, s.channels, s.states}, A.scalar_type(), A);
    if (saved) *saved = fresh({s.batch, (s.length + 15) / 16, s.channels, s.states}, A.scalar_type(), A);
    s.out = out.data_ptr(), s.final_state = data<float>(&final_state), s.checkpoints = saved ? data<float>(saved) : nullptr;
    const Tensor held = workspace(s, g_scan_bytes(&s, 0), u);
    launch(kScan, s, u.device());
    return {std::move(out), std::move(final_state)};
}

struct ScanFunction : torch::autograd::Function<ScanFunction> {
    static variable_list forward(AutogradContext* ctx, const OvlSelectiveScan* s, const Tensor& u, const Tensor& delta, const Tensor& A,
                                 const Tensor& B, const Tensor& C, const Maybe& D, const Maybe& z, const Maybe& bias,
                                 const Maybe& initial, const Maybe& lengths) {
        Tensor saved;
        variable_list out = scan_forward(*s, u, A, &saved);
        ctx->save_for_backward({u, delta, A, B, C, D.value_or(Tensor()), z.value_or(Tensor()), bias.value_or(Tensor()),
                                initial.value_or(Tensor()), lengths.value_or(Tensor()), saved});
        ctx->saved_data["softplus"] = (int64_t)s->delta_softplus;
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined() && !grads[1].defined()) return variable_list(11);
        const variable_list x = ctx->get_saved_variables();
        const Tensor &u = x[0], &delta = x[1], &A = x[2], &B = x[3], &C = x[4];
        const c10::cuda::CUDAGuard device(u.device());
        variable_list g(11);                                             // of the arguments of forward, the first of them ours
        {
            const c10::AutoGradMode off(false);
            OvlSelectiveScan s = scan_args(u, delta, A, B, C, behind(x[5]), behind(x[6]), behind(x[7]), behind(x[8]), behind(x[9]),
                                           ctx->saved_data["softplus"].toInt());
            const Tensor gout = above(grads[0], u, s.channels), gfinal = dense_above(grads[1]);
            for (int i = 0; i < 9; ++i)
                if (x[i].defined()) g[i + 1] = fresh(x[i].sizes(), x[i].scalar_type(), x[i]);
            s.checkpoints = data<float>(&x[10]);
            s.gout = gout.data_ptr(), s.gout_batch = gout.stride(0), s.gout_token = gout.stride(1);
            s.gfinal = data<float>(behind(gfinal));
            s.gu = data(&g[1]), s.gdelta = data(&g[2]), s.gA = data<float>(&g[3]), s.gB = data(&g[4]), s.gC = data(&g[5]);
            s.gD = data<float>(behind(g[6])), s.gz = data(behind(g[7])), s.gdelta_bias = data<float>(behind(g[8]));
            s.ginitial = data<float>(behind(g[9]));
            const Tensor held = workspace(s, g_scan_bytes(&s, 1), u);
            launch(kScanBackward, s, u.device());
        }
        return once(std::move(g), "selective_scan");
    }
};

// u, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state, lengths: (out, final state)
PyObject* selective_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Tensors all;
        const at::Tensor* u = n == 11 ? all.get(a[0]) : nullptr;
        const at::Tensor* A = u ? all.get(a[2]) : nullptr;
        const at::Tensor* B = A ? all.get(a[3]) : nullptr;
        const int softplus = B ? truth(a[8]) : -1;
        if (softplus < 0 || u->dim() != 3 || A->dim() != 2 || B->dim() < 3 || B->dim() > 4) return none();
        const c10::ScalarType t = u->scalar_type();
        const int64_t batch = u->size(0), length = u->size(1), channels = u->size(2), states = A->size(1);
        const int64_t groups = B->dim() == 4 ? B->size(2) : 1;
        bool right = code_of(t) != 0 && batch >= 1 && channels >= 1 && states >= 1 && states <= kMaxStates && groups >= 1 &&
                     channels % groups == 0 && (u->is_contiguous() || u->stride(2) == 1);
        if (!right) return none();
        const int64_t full[4] = {batch, length, groups, states}, flat[3] = {batch, length, states};
        const c10::IntArrayRef shape = B->dim() == 4 ? c10::IntArrayRef(full, 4) : c10::IntArrayRef(flat, 3);
        B = all.get(a[3], t, shape, false, false, right);
        const at::Tensor* C = all.get(a[4], t, shape, false, false, right);
        const at::Tensor* delta = all.get(a[1], t, u->sizes(), false, false, right);
        const at::Tensor* z = all.get(a[6], t, u->sizes(), false, true, right);
        A = all.get(a[2], at::kFloat, {channels, states}, true, false, right);
        const at::Tensor* D = all.get(a[5], at::kFloat, {channels}, true, true, right);
        const at::Tensor* bias = all.get(a[7], at::kFloat, {channels}, true, true, right);
        const at::Tensor* initial = all.get(a[9], at::kFloat, {batch, channels, states}, true, true, right);
        const at::Tensor* lengths = all.get(a[10], at::kInt, {batch}, true, true, right);
        if (!right || !plain(all)) return none();
        const OvlSelectiveScan s = scan_args(*u, *delta, *A, *B, *C, D, z, bias, initial, lengths, softplus);
        if (!all.differentiated) return tuple_of(unlocked([&] { return scan_forward(s, *u, *A, nullptr); }));
        return tuple_of(unlocked([&] {
            return ScanFunction::apply(&s, *u, *delta, *A, *B, *C, maybe(D), maybe(z), maybe(bias), maybe(initial), maybe(lengths));
        }));
    });
}

// ---- the convolution over whole sequences

OvlCausalConv conv_args(const Tensor& x, const Tensor& weight, const Tensor* bias, const Tensor* initial, const Tensor* lengths, int silu) {
    OvlCausalConv s{};
    s.dtype = code_of(x.scalar_type()), s.batch = x.size(0), s.length = x.size(1), s.channels = x.size(2), s.taps = weight.size(1);
    s.silu = silu, s.params_f32 = weight.scalar_type() == at::kFloat;
    s.x = data(&x), s.weight = data(&weight), s.bias = data(bias), s.initial_state = data(initial), s.lengths = data<int32_t>(lengths);
    s.x_batch = x.stride(0), s.x_token = x.stride(1);
    return s;
}

// (out,) or (out, state)
variable_list conv_forward(OvlCausalConv s, const Tensor& x, bool keep) {
    variable_list out{fresh(x.sizes(), x.scalar_type(), x)};
    if (keep) out.push_back(fresh({s.batch, s.taps - 1, s.channels}, x.scalar_type(), x));
    s.out = out[0].data_ptr(), s.final_state = keep ? out[1].data_ptr() : nullptr;
    launch(kConv, s, x.device());
    return out;
}

struct ConvFunction : torch::autograd::Function<ConvFunction> {
    static variable_list forward(AutogradContext* ctx, const OvlCausalConv* s, bool keep, const Tensor& x, const Tensor& weight,
                                 const Maybe& bias, const Maybe& initial, const Maybe& lengths) {
        ctx->save_for_backward({x, weight, bias.value_or(Tensor()), initial.value_or(Tensor()), lengths.value_or(Tensor())});
        ctx->saved_data["silu"] = (int64_t)s->silu;
        ctx->set_materialize_grads(false);
        return conv_forward(*s, x, keep);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor last = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !last.defined()) return variable_list(7);
        const variable_list x = ctx->get_saved_variables();
        const c10::cuda::CUDAGuard device(x[0].device());
        variable_list g(7);                                              // of the arguments of forward, the first two ours
        {
            const c10::AutoGradMode off(false);
            OvlCausalConv s = conv_args(x[0], x[1], behind(x[2]), behind(x[3]), behind(x[4]), ctx->saved_data["silu"].toInt());
            const Tensor gout = above(grads[0], x[0], s.channels), gfinal = dense_above(last);
            for (int i = 0; i < 4; ++i)
                if (x[i].defined()) g[i + 2] = fresh(x[i].sizes(), x[i].scalar_type(), x[i]);
            s.gout = gout.data_ptr(), s.gout_batch = gout.stride(0), s.gout_token = gout.stride(1);
            s.gfinal = data(behind(gfinal));
            s.gx = data(&g[2]), s.gweight = data(&g[3]), s.gbias = data(behind(g[4])), s.ginitial = data(behind(g[5]));
            const Tensor held = workspace(s, g_conv_bytes(&s), x[0]);
            launch(kConvBackward, s, x[0].device());
        }
        return once(std::move(g), "causal_conv1d");
    }
};

// x, weight, bias, activation, initial_state, lengths, return_state: (out,) or (out, state)
PyObject* causal_conv1d(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Tensors all;
        const at::Tensor* x = n == 7 ? all.get(a[0]) : nullptr;
        const at::Tensor* weight = x ? all.get(a[1]) : nullptr;
        const int silu = weight ? silu_of(a[3]) : -1, keep = weight ? truth(a[6]) : -1;
        if (silu < 0 || keep < 0 || x->dim() != 3 || weight->dim() != 2) return none();
        const c10::ScalarType t = x->scalar_type(), w = weight->scalar_type();
        const int64_t batch = x->size(0), length = x->size(1), channels = x->size(2), taps = weight->size(1);
        bool right = code_of(t) != 0 && (w == t || w == at::kFloat) && batch >= 1 && channels >= 1 && taps >= 1 && taps <= kMaxTaps &&
                     weight->size(0) == channels && weight->is_contiguous() && (x->is_contiguous() || x->stride(2) == 1);
        const at::Tensor* bias = all.get(a[2], w, {channels}, true, true, right);
        const at::Tensor* initial = all.get(a[4], t, {batch, taps - 1, channels}, true, true, right);
        const at::Tensor* lengths = all.get(a[5], at::kInt, {batch}, true, true, right);
        if (!right || !plain(all)) return none();
        const OvlCausalConv s = conv_args(*x, *weight, bias, initial, lengths, silu);
        if (!all.differentiated) return tuple_of(unlocked([&] { return conv_forward(s, *x, keep); }));
        return tuple_of(unlocked([&] { return ConvFunction::apply(&s, keep, *x, *weight, maybe(bias), maybe(initial), maybe(lengths)); }));
    });
}

// ---- the norm

int64_t row_stride(const Tensor& x) { return x.dim() == 2 ? x.stride(0) : x.size(-1); }

OvlRmsNorm norm_args(const Tensor& x, const Tensor& weight, const Tensor* residual, double eps) {
    OvlRmsNorm s{};
    s.dtype = code_of(x.scalar_type()), s.columns = x.size(-1), s.rows = x.numel() / s.columns;
    s.params_f32 = weight.scalar_type() == at::kFloat, s.eps = eps;
    s.x = data(&x), s.residual = data(residual), s.weight = data(&weight);
    s.x_row = row_stride(x), s.residual_row = residual ? row_stride(*residual) : 0;
    return s;
}

// (y,) or (y, sum)
variable_list norm_forward(OvlRmsNorm s, const Tensor& x, bool sum) {
    variable_list out{fresh(x.sizes(), x.scalar_type(), x)};
    if (sum) out.push_back(fresh(x.sizes(), x.scalar_type(), x));
    s.y = out[0].data_ptr(), s.residual_out = sum ? out[1].data_ptr() : nullptr;
    launch(kNorm, s, x.device());
    return out;
}

struct NormFunction : torch::autograd::Function<NormFunction> {
    static variable_list forward(AutogradContext* ctx, const OvlRmsNorm* s, const Tensor& x, const Tensor& weight, const Maybe& residual) {
        ctx->save_for_backward({x, weight, residual.value_or(Tensor())});
        ctx->saved_data["eps"] = s->eps;
        ctx->set_materialize_grads(false);
        return norm_forward(*s, x, residual.has_value());
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor last = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined() && !last.defined()) return variable_list(4);
        const variable_list v = ctx->get_saved_variables();
        const Tensor &x = v[0], &weight = v[1];
        const c10::cuda::CUDAGuard device(x.device());
        Tensor gx, gweight;
        {
            const c10::AutoGradMode off(false);
            OvlRmsNorm s = norm_args(x, weight, behind(v[2]), ctx->saved_data["eps"].toDouble());
            // (rows that follow each other, where there are other than two axes)
            const Tensor gy = x.dim() == 2 || !grads[0].defined() ? above(grads[0], x.dim() == 2 ? x : x.view({s.rows, s.columns}), s.columns)
                                                                  : dense_above(grads[0]);
            const Tensor gres = last.defined() && x.dim() == 2 ? above(last, x, s.columns) : dense_above(last);
            gx = fresh(x.sizes(), x.scalar_type(), x), gweight = fresh(weight.sizes(), weight.scalar_type(), weight);
            s.gy = gy.data_ptr(), s.gy_row = row_stride(gy);
            s.gresidual_out = data(behind(gres)), s.gresidual_out_row = gres.defined() ? row_stride(gres) : 0;
            s.gx = gx.data_ptr(), s.gweight = gweight.data_ptr();
            const Tensor held = workspace(s, g_norm_bytes(&s), x);
            launch(kNormBackward, s, x.device());
        }
        return once({Tensor(), gx, gweight, v[2].defined() ? gx : Tensor()}, "rms_norm");
    }
};

// x, weight, residual, eps: (y,) or (y, sum); with a fifth argument, the group's columns or None for the row: (q, scale[, sum])
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        Tensors all;
        const at::Tensor* x = n == 4 || n == 5 ? all.get(a[0]) : nullptr;
        const at::Tensor* weight = x ? all.get(a[1]) : nullptr;
        if (!weight || x->dim() < 1 || !PyFloat_CheckExact(a[3])) return none();
        const double eps = PyFloat_AS_DOUBLE(a[3]);
        const c10::ScalarType t = x->scalar_type(), w = weight->scalar_type();
        const int64_t columns = x->size(-1);
        if (columns < 1 || columns > kMaxColumns) return none();
        const bool dense = x->dim() != 2;                                // other ranks only where the rows follow each other
        int64_t group = 0;
        if (n == 5 && a[4] == Py_None) {
            group = columns;
        } else if (n == 5) {
            if (!PyLong_CheckExact(a[4])) return none();
            group = PyLong_AsLongLong(a[4]);
            if (group < 1) return PyErr_Clear(), none();
        }
        bool right = code_of(t) != 0 && (w == t || w == at::kFloat) && eps >= 0 && eps < 1e30 && weight->dim() == 1 &&
                     weight->size(0) == columns && weight->is_contiguous() &&
                     (x->is_contiguous() || (!dense && x->stride(1) == 1)) && (!group || columns % group == 0);
        const at::Tensor* residual = all.get(a[2], t, x->sizes(), dense, true, right);
        if (!right || !plain(all)) return none();
        OvlRmsNorm s = norm_args(*x, *weight, residual, eps);
        if (group) {
            if (all.differentiated) return none();
            at::DimVector scales(x->sizes());
            scales.back() = columns / group;
            variable_list out{fresh(x->sizes(), at::kFloat8_e4m3fn, *x),
                              fresh(scales, at::kFloat, *x)};
            if (residual) out.push_back(fresh(x->sizes(), x->scalar_type(), *x));
            s.group = group, s.q = out[0].data_ptr(), s.scale = data<float>(&out[1]);
            s.residual_out = residual ? out[2].data_ptr() : nullptr;
            unlocked([&] { launch(kNorm, s, all.device); });
            return tuple_of(out);
        }
        if (!all.differentiated) return tuple_of(unlocked([&] { return norm_forward(s, *x, residual != nullptr); }));
        return tuple_of(unlocked([&] { return NormFunction::apply(&s, *x, *weight, maybe(residual)); }));
    });
}

// bind(parameter class, addresses of the library's entries in the order of Entry, then of the three workspace queries)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    constexpr int count = kEntries + 3;
    if (n != count + 1) {
        PyErr_SetString(PyExc_TypeError, "bind takes the parameter class and the library's entries");
        return nullptr;
    }
    void* at[count];
    for (int i = 0; i < count; ++i) {
        at[i] = PyLong_AsVoidPtr(a[i + 1]);
        if (!at[i]) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an entry is missing");
            return nullptr;
        }
    }
    for (int i = 0; i < kEntries; ++i) g_launch[i] = reinterpret_cast<Launch>(at[i]);
    g_scan_bytes = reinterpret_cast<decltype(g_scan_bytes)>(at[kEntries]);
    g_conv_bytes = reinterpret_cast<decltype(g_conv_bytes)>(at[kEntries + 1]);
    g_norm_bytes = reinterpret_cast<decltype(g_norm_bytes)>(at[kEntries + 2]);
    Py_INCREF(a[0]);
    g_parameter = a[0];
    return none();
}

#define OVL_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {OVL_METHOD(bind),   OVL_METHOD(selective_scan), OVL_METHOD(selective_scan_step), OVL_METHOD(causal_conv1d),
                         OVL_METHOD(causal_conv1d_step), OVL_METHOD(rms_norm), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ovl_front", nullptr, -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_ovl_front(void) { return PyModule_Create(&module); }
