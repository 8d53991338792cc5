// The autograd node of a layer norm by itself (ops.layer_norm), and its call from Python.
//
// A small forward and backward pass is host time: autograd runs a node on a thread of its own, and a node written in Python pays
// there for the interpreter, four allocations through it and two launches.  This one keeps the arithmetic where it is - the entry
// points of libadvmix_hip.so, handed over by address (bind) - and only does the host's part in C++.  Launch groups keep the Python
// member (ops.LayerNorm); both call the same kernels.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

namespace {

using Fwd = int (*)(const void*, int64_t, const float*, const float*, void*, float*, float*, int64_t, int, int, float, void*);
using Bwd = int (*)(const void*, int64_t, const void*, int64_t, const float*, const float*, const float*, void*, float*, float*,
                    float*, int, int64_t, int, int, void*);
using Parts = int (*)(int64_t, int, int);
Fwd fwd_entry = nullptr;
Bwd bwd_entry = nullptr;
Parts parts_entry = nullptr;

at::MemoryFormat format_of(const at::Tensor& t) {
    return t.dim() == 4 ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous;
}
int64_t channels(const at::Tensor& t) { return t.dim() == 4 ? t.size(1) : t.size(-1); }

// Elements between the rows of t if its channels are neighbours and all its rows lie at one distance, else -1 (ops._row_stride).
int64_t row_stride(const at::Tensor& t) {
    const int64_t C = channels(t);
    if (t.is_contiguous(format_of(t))) return C;
    const int d = (int)t.dim();
    static const int map[3] = {3, 2, 0};                         // of an NCHW map: W, H, N outwards
    const int64_t last = d == 4 ? t.stride(1) : t.stride(-1);
    if (C > 1 && last != 1) return -1;
    int64_t step = -1, span = 0;
    for (int k = 0; k < d - 1; ++k) {
        const int dim = d == 4 ? map[k] : d - 2 - k;
        const int64_t n = t.size(dim), s = t.stride(dim);
        if (n == 1) continue;
        if (step < 0) {
            step = s;
            span = s * n;
        } else if (s != span) return -1;
        else span *= n;
    }
    return step < 0 ? C : step;
}

int kind_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

const float* floats(const at::Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }

// What records operations in order to run them again sees the output's allocation and nothing of the kernels that fill it.
void refuse_recording() {
    using Key = c10::impl::TorchDispatchModeKey;
    const auto mode = [](Key k) { return c10::impl::TorchDispatchModeTLS::get_mode(k).has_value(); };
    const auto included = [](c10::DispatchKey k) { return c10::impl::tls_is_dispatch_key_included(k); };
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !mode(Key::PROXY) && !mode(Key::FAKE) && !mode(Key::FUNCTIONAL) &&
                                    !included(c10::DispatchKey::PreDispatch) && !included(c10::DispatchKey::Functionalize) &&
                                    !included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode),
                                "layer_norm: its kernels cannot be recorded (torch.jit.trace, make_fx, fake tensors) or transformed (torch.func)");
}
// A tensor whose values are what its memory holds, by strides: no wrapper (subclasses with a dispatch of their own, torch.func's,
// batched gradients), no sparse or nested one.  ``values`` then makes memory of two views that hold none or other values.
bool plain(const at::Tensor& t) {
    static const c10::DispatchKeySet wrappers({c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::Batched,
                                               c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper});
    return t.layout() == at::kStrided && !t.is_nested() && !t.key_set().has_any(wrappers);
}
at::Tensor values(const at::Tensor& t) {
    if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
    return t.is_neg() ? t.resolve_neg() : t;
}
// Forward mode: a tangent would be dropped without a word, the result taken for a constant.
void refuse_tangent(const char* name, const at::Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "layer_norm: no forward-mode derivatives, and ", name, " has a tangent");
}

void done(const char* name, int rc) {
    TORCH_CHECK(rc == 0, name, " failed: ", rc == 1 ? "ADVMIX_EINVAL (bad argument / unsupported shape)" : "ADVMIX_ELAUNCH (HIP runtime error)");
}

struct Sizes {
    at::DimVector of_x;
    c10::Device device = c10::kCPU;
    int64_t rows;
    int C, kind;
};

// gamma and beta are no inputs of the node, so the engine does not order the passes that write their gradients.  A gradient that is
// made in a pass holds nothing until that pass's first write has run: it carries the stream of that write (with the tensor itself,
// as its backend meta), and whoever adds to it on another stream lets that one wait first.
struct FirstWrite : c10::BackendMeta {
    c10::hip::HIPStream stream = c10::hip::getCurrentHIPStream();
};
void first_written_here(const at::Tensor& grad) {
    grad.unsafeGetTensorImpl()->set_backend_meta(c10::make_intrusive<FirstWrite>());
}
// The graph capture that a stream takes part in, if any (the null stream takes part in none, and may not be asked during one).
struct Capture {
    bool active = false;
    unsigned long long id = 0;
    explicit Capture(hipStream_t s) {
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        if (s == nullptr) return;
        if (hipStreamGetCaptureInfo(s, &status, &id) == hipSuccess) active = status == hipStreamCaptureStatusActive;
        else (void)hipGetLastError();                            // (not the next launch's)
    }
};
void wait_for_first_write(const at::Tensor& grad) {
    const auto* first = dynamic_cast<const FirstWrite*>(grad.unsafeGetTensorImpl()->get_backend_meta());
    if (!first) return;
    const hipStream_t mine = c10::hip::getCurrentHIPStream().stream(), its = first->stream.stream();
    if (mine == its) return;
    const Capture a(mine), b(its);                               // (work of a capture and work outside it cannot wait for each other)
    if (a.active != b.active || (a.active && a.id != b.id)) return;
    hipEvent_t event;
    bool ok = hipEventCreateWithFlags(&event, hipEventDisableTiming) == hipSuccess;
    if (ok) {
        ok = hipEventRecord(event, its) == hipSuccess && hipStreamWaitEvent(mine, event, 0) == hipSuccess;
        ok = hipEventDestroy(event) == hipSuccess && ok;
    }
    TORCH_CHECK(ok, "layer_norm: could not order a parameter's gradient between streams (HIP runtime error)");
}

// One gradient of gamma or beta: where the kernel puts it, and whether it adds.
struct Slot {
    at::Tensor grad;
    bool add = false;
    float* at() const { return grad.defined() ? grad.mutable_data_ptr<float>() : nullptr; }
};
// p.grad, made if there is none: the optimizer's flat view (added to, as the kernels everywhere here do) or a fresh tensor, which
// the kernel may store to (``store``) or has to find zeroed.
Slot slot_of(const at::Tensor& p, const at::Tensor& flat, bool store) {
    Slot s;
    at::Tensor& g = p.mutable_grad();
    if (!g.defined() && flat.defined()) g = flat;
    if (!g.defined()) {
        g = store ? at::empty_like(p) : at::zeros_like(p);
        first_written_here(g);
        s.add = !store;
    } else {
        TORCH_CHECK(g.scalar_type() == at::kFloat && g.is_contiguous() && g.sizes() == p.sizes() && g.device() == p.device(),
                    "layer_norm: a parameter's .grad must be a contiguous fp32 tensor of its shape");
        wait_for_first_write(g);
        s.add = true;
    }
    s.grad = g;
    return s;
}

struct LayerNormNode : torch::autograd::Node {
    torch::autograd::SavedVariable x;
    at::Tensor gamma, beta, flat_gamma, flat_beta, stats;        // (leaves and buffers: gamma and beta are no inputs of the node)
    int64_t version = 0;
    bool want_x = false, want_gamma = false, want_beta = false;
    Sizes z{};

    std::string name() const override { return "LayerNorm"; }
    void release_variables() override {
        const std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data();
        stats.reset();
    }
    // t, read row by row: its layout is looked at here and now, since saved-tensor hooks may hand back x in another one (a copy
    // of rows that lay apart is dense), or something that is not x at all.
    struct Rows {
        at::Tensor t;
        int64_t ld;
    };
    Rows rows_of(const at::Tensor& t, const char* what) const {
        TORCH_CHECK(plain(t), "layer_norm: ", what, " is no plain tensor");
        TORCH_CHECK(t.sizes() == z.of_x && kind_of(t) == z.kind && t.device() == z.device, "layer_norm: ", what, " is ", t.scalar_type(), " ",
                    t.sizes(), " on ", t.device(), ", not ", z.of_x, " of x's type on ", z.device);
        const at::Tensor v = values(t);
        const int64_t ld = row_stride(v);
        return ld < 0 ? Rows{v.contiguous(format_of(v)), z.C} : Rows{v, ld};
    }
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        torch::autograd::variable_list out(num_outputs());
        if (!grads[0].defined()) return out;
        TORCH_CHECK(!at::GradMode::is_enabled(), "advmix_amd: layer_norm has no second derivative (backward with create_graph=True)");
        const std::lock_guard<std::mutex> lock(mutex_);
        const at::Tensor xs = x.unpack(shared_from_this());      // (refuses a second pass through a freed graph, and a changed x)
        TORCH_CHECK(!gamma.defined() || (int64_t)gamma._version() == version,
                    "layer_norm: gamma was modified in place between the forward and the backward pass");
        const c10::OptionalDeviceGuard guard(z.device);
        refuse_recording();
        refuse_tangent("the saved x", xs);
        refuse_tangent("the gradient of y", grads[0]);
        const Rows xr = rows_of(xs, "the saved x"), dr = rows_of(grads[0], "the gradient of y");
        at::Tensor dx = want_x ? at::empty_like(xr.t, xr.t.options(), format_of(xr.t)) : at::Tensor();
        const bool store = z.rows > 0 && !(want_gamma && want_beta && gamma.is_same(beta));      // (one parameter as both: two sums in one place)
        const Slot dg = want_gamma ? slot_of(gamma, flat_gamma, store) : Slot();
        const Slot db = want_beta ? slot_of(beta, flat_beta, store) : Slot();
        if (z.rows > 0) {
            at::Tensor part;                                     // (this call's own: two captured graphs must not share it)
            if (want_gamma || want_beta) part = at::empty({(int64_t)parts_entry(z.rows, z.C, z.kind) * 2 * z.C}, stats.options());
            const float* mean = stats.const_data_ptr<float>();
            done("advmix_layer_norm_bwd",
                 bwd_entry(dr.t.const_data_ptr(), dr.ld, xr.t.const_data_ptr(), xr.ld, floats(gamma), mean, mean + z.rows,
                           dx.defined() ? dx.mutable_data_ptr() : nullptr, dg.at(), db.at(),
                           part.defined() ? part.mutable_data_ptr<float>() : nullptr, (dg.add ? 1 : 0) + (db.add ? 2 : 0), z.rows, z.C,
                           z.kind, c10::hip::getCurrentHIPStream().stream()));
        }
        if (want_x) out[0] = dx;
        return out;
    }
};

void check_param(const char* name, const at::Tensor& p, const at::Tensor& x, int64_t C) {
    if (!p.defined()) return;
    TORCH_CHECK_TYPE(plain(p) && !p.is_neg() && !p._is_zerotensor(), "layer_norm: ", name, " must be a plain tensor");
    TORCH_CHECK_TYPE(p.scalar_type() == at::kFloat && p.device() == x.device(), "layer_norm: ", name, " must be fp32 on ", x.device(),
                     ", got ", p.scalar_type(), " on ", p.device());
    TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == C && p.is_contiguous(), "layer_norm: ", name, " must be a contiguous [", C, "], got ",
                      p.sizes());
    TORCH_CHECK_VALUE(!p.requires_grad() || p.is_leaf(), "layer_norm: ", name, " requires a gradient but is not a leaf (parameter)");
}

at::Tensor layer_norm(at::Tensor x, const at::Tensor& gamma, const at::Tensor& beta, double eps, const at::Tensor& flat_gamma,
                      const at::Tensor& flat_beta) {
    refuse_recording();
    refuse_tangent("x", x);
    refuse_tangent("gamma", gamma);
    refuse_tangent("beta", beta);
    Sizes z;
    z.kind = kind_of(x);
    TORCH_CHECK_TYPE(z.kind >= 0 && x.is_cuda(), "layer_norm needs fp32, bf16 or fp16 CUDA tensors (no CPU fallback), got ",
                     x.scalar_type(), " on ", x.device());
    TORCH_CHECK_TYPE(plain(x) && !x._is_zerotensor(), "layer_norm: x must be a plain tensor");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.dim() <= 4, "layer_norm: expected tokens [..., C] with up to 3 dimensions or a 4-D NCHW map, got ",
                      x.dim(), "-D");
    const int64_t C = channels(x);
    TORCH_CHECK_VALUE(C > 0, "layer_norm: no channels to normalise over");
    TORCH_CHECK_VALUE(C <= (1 << 30), "layer_norm: at most 2^30 channels, got ", C);
    TORCH_CHECK_VALUE(eps >= 0 && eps < std::numeric_limits<double>::infinity(), "layer_norm: eps must be finite and not negative, got ", eps);
    check_param("gamma", gamma, x, C);
    check_param("beta", beta, x, C);
    const c10::OptionalDeviceGuard guard(x.device());
    x = values(x);
    int64_t ldx = row_stride(x);
    if (ldx < 0) {                                               // (a torch op: its own backward brings dx back into x's layout)
        x = x.contiguous(format_of(x));
        ldx = C;
    }
    z.of_x = x.sizes();
    z.device = x.device();
    z.C = (int)C;
    z.rows = x.numel() / C;
    const bool on = at::GradMode::is_enabled(), wx = on && x.requires_grad(), wg = on && gamma.defined() && gamma.requires_grad(),
               wb = on && beta.defined() && beta.requires_grad(), keep = wx || wg || wb;
    at::Tensor y, stats;
    {
        const at::NoGradGuard off;
        y = at::empty_like(x, x.options(), format_of(x));
        if (keep) stats = at::empty({2 * z.rows}, x.options().dtype(at::kFloat));
    }
    if (z.rows > 0) {
        float* mean = keep ? stats.mutable_data_ptr<float>() : nullptr;
        done("advmix_layer_norm_fwd", fwd_entry(x.const_data_ptr(), ldx, floats(gamma), floats(beta), y.mutable_data_ptr(), mean,
                                                keep ? mean + z.rows : nullptr, z.rows, z.C, z.kind, (float)eps,
                                                c10::hip::getCurrentHIPStream().stream()));
    }
    if (keep) {
        auto node = std::shared_ptr<LayerNormNode>(new LayerNormNode(), torch::autograd::deleteNode);
        if (wx) node->set_next_edges(torch::autograd::collect_next_edges(x));
        node->x = torch::autograd::SavedVariable(x, false);
        node->gamma = gamma;
        node->beta = beta;
        node->flat_gamma = flat_gamma;
        node->flat_beta = flat_beta;
        node->stats = stats;
        node->version = gamma.defined() ? (int64_t)gamma._version() : 0;
        node->want_x = wx;
        node->want_gamma = wg;
        node->want_beta = wb;
        node->z = z;
        torch::autograd::set_history(y, node);
    }
    return y;
}

struct WithoutGil {
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

at::Tensor tensor_or_none(PyObject* o, const char* name) {
    if (o == Py_None) return at::Tensor();
    TORCH_CHECK_TYPE(THPVariable_Check(o), "layer_norm: ", name, " must be a tensor or None");
    return THPVariable_Unpack(o);
}

// layer_norm(x, gamma, beta, eps, gamma's and beta's flat gradient views or None)
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 6, "layer_norm takes 6 arguments");
    TORCH_CHECK_TYPE(fwd_entry != nullptr, "layer_norm: bind() comes first");
    TORCH_CHECK_TYPE(THPVariable_Check(a[0]), "layer_norm: x must be a tensor");
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    const at::Tensor gamma = tensor_or_none(a[1], "gamma"), beta = tensor_or_none(a[2], "beta"), fg = tensor_or_none(a[4], "gradient"),
                     fb = tensor_or_none(a[5], "gradient");
    at::Tensor x = THPVariable_Unpack(a[0]), y;
    {
        const WithoutGil free;                                   // (a launch may wait for room in a queue)
        y = layer_norm(std::move(x), gamma, beta, eps, fg, fb);
    }
    return THPVariable_Wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

// first_written_here(t), wait_for_first_write(t): for gradients that the launch groups' member makes and adds to
template <void (*F)(const at::Tensor&)> PyObject* py_grad(PyObject*, PyObject* t) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(THPVariable_Check(t), "expected a tensor");
    const at::Tensor& grad = THPVariable_Unpack(t);
    const c10::OptionalDeviceGuard guard(grad.device());
    F(grad);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// bind(address of advmix_layer_norm_fwd, of _bwd, of _parts)
PyObject* py_bind(PyObject*, PyObject* args) {
    unsigned long long f = 0, b = 0, p = 0;
    if (!PyArg_ParseTuple(args, "KKK", &f, &b, &p)) return nullptr;
    fwd_entry = reinterpret_cast<Fwd>(f);
    bwd_entry = reinterpret_cast<Bwd>(b);
    parts_entry = reinterpret_cast<Parts>(p);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_layer_norm)), METH_FASTCALL, nullptr},
                         {"first_written_here", py_grad<first_written_here>, METH_O, nullptr},
                         {"wait_for_first_write", py_grad<wait_for_first_write>, METH_O, nullptr},
                         {"bind", py_bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_node", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__node(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", ADVMIX_TORCH) != 0) Py_CLEAR(m);      // (torch's C++ types are not the same from one to the next)
    return m;
}
