// The torch side of trainer.py's calls: takes the tensors' addresses, strides and types, allocates
// results and scratch, and calls the C ABI (include/crukx_b200.h), which has no torch types.  In C++
// because a call waits for it: 112 gradients took 80 us of Python, a loss and its backward pass 90.
//
// Arguments that do not fit make a function return None (or False) before anything is launched;
// trainer.py then says which one it is.
#include <c10/core/AutogradState.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "../../../include/crukx_b200.h"

namespace {

constexpr int kBf16 = 1, kFp16 = 2, kFp32 = 4;   // sets of element types

int type_bit(at::ScalarType t) {
    return t == at::kBFloat16 ? kBf16 : t == at::kHalf ? kFp16 : t == at::kFloat ? kFp32 : 0;
}
int32_t type_code(at::ScalarType t) { return t == at::kBFloat16 ? CRX_BF16 : t == at::kHalf ? CRX_FP16 : CRX_FP32; }

[[noreturn]] void fail(int status, const char* err) {
    if (status == CRX_VALUE_ERROR) throw py::value_error(err);
    if (status == CRX_NO_MEMORY) throw std::bad_alloc();
    throw std::runtime_error("crukx_sync_b200: status " + std::to_string(status) + ": " + err);
}

bool same_name(PyObject* a, PyObject* b) {
    return a == b || (PyUnicode_CheckExact(a) && PyUnicode_CheckExact(b) && PyUnicode_GET_LENGTH(a) == PyUnicode_GET_LENGTH(b) &&
                      PyUnicode_Compare(a, b) == 0);
}

// Tensors of one dict (which keeps them alive through the call).
struct Set {
    std::vector<c10::TensorImpl*> t;
    std::vector<void*> ptr;
    std::vector<int64_t> numel;
    std::vector<int32_t> code;
    int dev = -1;

    bool add(PyObject* v, int types) {
        if (!THPVariable_Check(v)) return false;
        c10::TensorImpl* x = THPVariable_Unpack(v).unsafeGetTensorImpl();
        const at::ScalarType type = c10::typeMetaToScalarType(x->dtype());
        if (!(type_bit(type) & types) || !x->is_cuda() || x->layout() != at::kStrided || !x->is_contiguous()) return false;
        const int d = x->device().index();
        if (dev < 0) dev = d;
        if (d != dev) return false;
        t.push_back(x);
        ptr.push_back(x->mutable_data());
        numel.push_back(x->numel());
        code.push_back(type_code(type));
        return true;
    }
    void room(size_t n) {
        t.reserve(n);
        ptr.reserve(n);
        numel.reserve(n);
        code.reserve(n);
    }
    bool take(const py::dict& d, int types) {
        room(d.size());
        PyObject *k, *v;
        Py_ssize_t at = 0;
        while (PyDict_Next(d.ptr(), &at, &k, &v))
            if (!add(v, types)) return false;
        return true;
    }
    // the tensors of d under `like`'s names, in that order, with the sizes that `of` has
    bool match(const py::dict& d, const py::dict& like, const Set& of, int types) {
        if (d.size() != like.size()) return false;
        room(d.size());
        dev = of.dev;
        PyObject *k, *v, *k2, *x;
        Py_ssize_t at = 0, at2 = 0;
        bool alike = true;   // so far d has its names in the same order: no lookups
        while (PyDict_Next(like.ptr(), &at, &k, &v)) {
            alike = alike && PyDict_Next(d.ptr(), &at2, &k2, &x) && same_name(k, k2);
            if (!alike) {
                x = PyDict_GetItemWithError(d.ptr(), k);
                if (!x) {
                    if (PyErr_Occurred()) throw py::error_already_set();
                    return false;
                }
            }
            if (!add(x, types)) return false;
        }
        return numel == of.numel;
    }
    bool writable() const {
        return c10::InferenceMode::is_enabled() || std::none_of(t.begin(), t.end(), [](c10::TensorImpl* x) { return x->is_inference(); });
    }
    // written through raw pointers: the version moves as for any in-place write
    void written() const {
        for (c10::TensorImpl* x : t)
            if (!x->is_inference()) x->bump_version();
    }
};

float narrow(double x) { return static_cast<float>(std::min(x, 3.0e38)); }   // of a limit: what fp32 holds of it

at::TensorOptions on(int dev, at::ScalarType t) { return at::TensorOptions().device(at::kCUDA, static_cast<c10::DeviceIndex>(dev)).dtype(t); }
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

// One value of type t on the device, or none.
template <class T>
bool scalar(const c10::optional<at::Tensor>& x, at::ScalarType t, int dev, const T** p) {
    *p = nullptr;
    if (!x) return true;
    if (x->scalar_type() != t || x->numel() != 1 || !x->is_cuda() || x->get_device() != dev) return false;
    *p = static_cast<const T*>(x->data_ptr());
    return true;
}

py::object grad_norm(const py::dict& grads, int dev_if_empty) {
    Set g;
    if (!g.take(grads, kBf16 | kFp16 | kFp32)) return py::none();
    if (g.dev < 0) g.dev = dev_if_empty;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(g.dev));
    const int32_t n = static_cast<int32_t>(g.t.size());
    const at::Tensor norm = at::empty({}, on(g.dev, at::kFloat));
    const int64_t bytes = crx_grads_workspace(n);
    const at::Tensor ws = at::empty({bytes}, on(g.dev, at::kByte));
    char err[512] = "";
    const int st = crx_grad_norm(n, g.ptr.data(), g.code.data(), g.numel.data(), ws.data_ptr(), bytes, norm.data_ptr<float>(),
                                 stream_of(g.dev), err, sizeof err);
    if (st != CRX_OK) fail(st, err);
    return py::cast(norm);
}

py::object clip_grads(const py::dict& grads, double max_norm, const c10::optional<py::dict>& out, const c10::optional<at::Tensor>& norm,
                      int dev_if_empty) {
    Set g, o;
    if (!g.take(grads, kBf16 | kFp16 | kFp32)) return py::none();
    if (out && (!o.match(*out, grads, g, kBf16 | kFp16 | kFp32) || o.code != g.code)) return py::none();
    const Set& to = out ? o : g;
    if (!to.writable()) return py::none();
    if (g.dev < 0) g.dev = dev_if_empty;
    const float* norm_in;
    if (!scalar(norm, at::kFloat, g.dev, &norm_in)) return py::none();
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(g.dev));
    const int32_t n = static_cast<int32_t>(g.t.size());
    at::Tensor result, ws;
    int64_t bytes = 0;
    if (!norm) {
        result = at::empty({}, on(g.dev, at::kFloat));
        bytes = crx_grads_workspace(n);
        ws = at::empty({bytes}, on(g.dev, at::kByte));
    }
    char err[512] = "";
    const int st = crx_clip_grads(n, g.ptr.data(), to.ptr.data(), g.code.data(), g.numel.data(), narrow(max_norm), norm_in,
                                  norm ? nullptr : ws.data_ptr(), bytes, norm ? nullptr : result.data_ptr<float>(), stream_of(g.dev), err,
                                  sizeof err);
    if (st != CRX_OK) fail(st, err);
    to.written();
    return py::cast(norm ? *norm : result);
}

bool adamw_step(const py::dict& masters, const py::dict& grads, const py::dict& exp_avg, const py::dict& exp_avg_sq,
                const c10::optional<py::dict>& weights, double lr, const c10::optional<at::Tensor>& lr_t, int64_t step,
                const c10::optional<at::Tensor>& step_t, double beta1, double beta2, double eps, double weight_decay,
                const c10::optional<at::Tensor>& norm, double max_norm) {
    Set g, p, m, v, w;
    if (!g.take(grads, kBf16 | kFp16 | kFp32) || !p.match(masters, grads, g, kFp32) || !m.match(exp_avg, grads, g, kFp32) ||
        !v.match(exp_avg_sq, grads, g, kFp32) || (weights && !w.match(*weights, grads, g, kBf16)))
        return false;
    if (!p.writable() || !m.writable() || !v.writable() || !w.writable()) return false;
    if (g.t.empty()) return true;
    crx_adamw_args a = {};
    if (!scalar(lr_t, at::kFloat, g.dev, &a.lr_p) || !scalar(step_t, at::kLong, g.dev, &a.step_p) || !scalar(norm, at::kFloat, g.dev, &a.norm))
        return false;
    a.lr = lr;
    a.beta1 = beta1;
    a.beta2 = beta2;
    a.eps = eps;
    a.weight_decay = weight_decay;
    a.step = step;
    a.max_norm = narrow(max_norm);
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(g.dev));
    char err[512] = "";
    const int st = crx_adamw_step(static_cast<int32_t>(g.t.size()), reinterpret_cast<float* const*>(p.ptr.data()), g.ptr.data(), g.code.data(),
                                  reinterpret_cast<float* const*>(m.ptr.data()), reinterpret_cast<float* const*>(v.ptr.data()),
                                  weights ? w.ptr.data() : nullptr, g.numel.data(), &a, stream_of(g.dev), err, sizeof err);
    if (st != CRX_OK) fail(st, err);
    for (const Set* s : {&p, &m, &v, &w}) s->written();
    return true;
}

// Memory for the gradient: laid out as the logits are, with rows starting at the same places between
// 16-byte boundaries (a row is then written in the vectors it was read in), unless that would waste or
// share memory; then rows padded to 16 bytes.
at::Tensor grad_like(const at::Tensor& logits) {
    const auto size = logits.sizes(), stride = logits.strides();
    const int64_t V = size.back(), es = logits.element_size(), d = logits.dim();
    const int64_t phase = static_cast<int64_t>(reinterpret_cast<uintptr_t>(logits.data_ptr()) % 16) / es;
    const at::TensorOptions opt = at::TensorOptions().device(logits.device()).dtype(logits.scalar_type());
    if (phase == 0 && logits.is_contiguous()) return at::empty(size, opt);
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t i = 0; i + 1 < d; ++i)
        if (size[i] > 1) dims.emplace_back(stride[i], size[i]);
    std::sort(dims.begin(), dims.end());
    int64_t end = V;   // elements up to the end of what the dims so far span
    bool fits = true;
    for (const auto& [s, n] : dims) {
        fits = fits && s >= end;
        end += s * (n - 1);
    }
    if (fits && end <= 2 * logits.numel() + 64) return at::empty({end + phase}, opt).as_strided(size, stride, phase);
    const int64_t vec = 16 / es;
    auto padded = size.vec();
    padded.back() = (V + vec - 1) / vec * vec;
    return at::empty(padded, opt).narrow(d - 1, 0, V);
}

struct Call {
    crx_policy_args a;
    at::Tensor tokens;
    int dev;
};

// Per-token values: at least one stride per dimension of the tokens, 0 along one of size 1.
bool rows(const at::Tensor& x, const at::Tensor& tokens, bool broadcast, crx_rows* r) {
    const auto size = x.sizes(), want = tokens.sizes(), stride = x.strides();
    if (x.layout() != at::kStrided || size.size() != want.size() || !x.is_cuda() || x.get_device() != tokens.get_device()) return false;
    int64_t s[2] = {0, 0};
    const size_t d = size.size();
    for (size_t i = 0; i < d; ++i) {
        if (size[i] != want[i] && !(broadcast && size[i] == 1)) return false;
        s[2 - d + i] = size[i] == 1 ? 0 : stride[i];
    }
    *r = crx_rows{x.data_ptr(), s[0], s[1]};
    return true;
}
// Whether tensors that were saved came back as what they were.  Hooks may have moved them meanwhile
// (offloading to the host), so addresses and strides are taken anew.
bool same_again(const at::Tensor& logits, const at::Tensor& tokens, int dev, const crx_policy_args& a) {
    const int64_t d = tokens.dim();
    if ((d != 1 && d != 2) || logits.dim() != d + 1 || tokens.size(d - 1) != a.steps || (d == 2 ? tokens.size(0) : 1) != a.batch) return false;
    if (!std::equal(tokens.sizes().begin(), tokens.sizes().end(), logits.sizes().begin()) || logits.size(d) != a.vocab) return false;
    if (tokens.scalar_type() != (a.tokens64 ? at::kLong : at::kInt) || !type_bit(logits.scalar_type()) || type_code(logits.scalar_type()) != a.dtype) return false;
    return logits.layout() == at::kStrided && (a.vocab == 1 || logits.stride(d) == 1) && logits.is_cuda() && logits.get_device() == dev &&
           tokens.is_cuda() && tokens.get_device() == dev;
}
crx_rows wide_rows(const at::Tensor& x) {
    const int64_t d = x.dim();
    return crx_rows{x.data_ptr(), d == 3 ? x.stride(0) : 0, x.stride(d - 2)};
}

struct Results {
    at::Tensor loss, logp, stats, rows, grad;
};

Results run(Call& c, const at::Tensor& logits, bool want_grad) {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.dev));
    crx_policy_args& a = c.a;
    Results r;
    a.logits = wide_rows(logits);
    a.grad = crx_rows{nullptr, 0, 0};
    if (want_grad) {
        r.grad = grad_like(logits);
        a.grad = wide_rows(r.grad);
    }
    r.loss = at::empty({}, on(c.dev, at::kFloat));
    r.logp = at::empty(c.tokens.sizes(), on(c.dev, at::kFloat));
    r.stats = at::empty({2}, on(c.dev, at::kFloat));
    r.rows = at::empty({crx_policy_workspace(a.batch, a.steps)}, on(c.dev, at::kByte));
    a.logp = r.logp.data_ptr<float>();
    a.loss = r.loss.data_ptr<float>();
    a.stats = r.stats.data_ptr<float>();
    a.rows = static_cast<float*>(r.rows.data_ptr());
    char err[512] = "";
    const int st = crx_policy_loss(&a, stream_of(c.dev), err, sizeof err);
    if (st != CRX_OK) fail(st, err);
    return r;
}

// What the backward pass needs beside the saved tensors.
struct Kept : torch::CustomClassHolder {
    crx_policy_args a;
    int64_t capture;        // the graph that the forward pass was captured into
    at::Tensor rows, grad;   // grad: until it is handed out
};

// The graph that the device's current stream is being captured into, 0 for none.
int64_t capture_of(int dev) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    C10_CUDA_CHECK(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream_of(dev)), &status, &id));
    return status == cudaStreamCaptureStatusActive ? static_cast<int64_t>(id) : 0;
}

// The forward pass leaves the gradient for an incoming gradient of 1.  The backward pass hands it
// out; for another one (and the second time) it is computed again from the logits, so that it is
// rounded once whatever its scale.  Also where only one of the passes runs again: a replayed backward
// pass finds what it left the time before, and a replayed loss would write into what was handed out.
struct PolicyLossFn : public torch::autograd::Function<PolicyLossFn> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, Call* c) {
        Results r = run(*c, logits, true);
        const auto stats = r.stats.unbind(0);
        ctx->save_for_backward({logits, c->tokens});
        auto keep = c10::make_intrusive<Kept>();
        keep->a = c->a;
        keep->capture = capture_of(c->dev);
        keep->rows = std::move(r.rows);
        keep->grad = std::move(r.grad);
        ctx->saved_data["kept"] = c10::IValue::make_capsule(std::move(keep));
        ctx->mark_non_differentiable({r.logp, stats[0], stats[1]});
        ctx->set_materialize_grads(false);
        return {r.loss, r.logp, stats[0], stats[1]};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& scales) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "policy_loss: its gradient is not differentiable (create_graph=True)");
        const at::Tensor& scale = scales[0];
        if (!scale.defined()) return {at::Tensor(), at::Tensor()};
        const auto saved = ctx->get_saved_variables();   // refuses tensors modified since
        const at::Tensor &logits = saved[0], &tokens = saved[1];
        const auto capsule = ctx->saved_data["kept"].toCapsule();
        Kept& kept = static_cast<Kept&>(*capsule);
        crx_policy_args a = kept.a;
        const int dev = kept.rows.get_device();
        TORCH_CHECK(same_again(logits, tokens, dev, a) && rows(tokens, tokens, false, &a.tokens),
                    "policy_loss: saved logits or tokens came back with another shape, type or device");
        const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
        const bool first = kept.grad.defined() && kept.capture == capture_of(dev);
        const at::Tensor grad = first ? std::exchange(kept.grad, at::Tensor()) : grad_like(logits);
        a.logits = wide_rows(logits);
        a.grad = wide_rows(grad);
        a.rows = static_cast<float*>(kept.rows.data_ptr());
        a.logp = a.loss = a.stats = a.rows;   // results that this pass does not touch
        char err[512] = "";
        const int st = crx_policy_backward(&a, scale.data_ptr<float>(), first, stream_of(dev), err, sizeof err);
        if (st != CRX_OK) fail(st, err);
        return {grad, at::Tensor()};
    }
};

py::object policy_loss(const at::Tensor& logits, const at::Tensor& tokens, const at::Tensor& advantages,
                       const c10::optional<at::Tensor>& old_logp, const c10::optional<at::Tensor>& ref_logp,
                       const c10::optional<at::Tensor>& mask, double clip_low, double clip_high, double kl_coef, double temperature,
                       double denom) {
    const int64_t d = tokens.dim();
    if (!type_bit(logits.scalar_type()) || logits.layout() != at::kStrided || !logits.is_cuda() || (d != 1 && d != 2) || logits.dim() != d + 1)
        return py::none();
    const int64_t V = logits.size(d);
    if (V < 1 || (V > 1 && logits.stride(d) != 1) || !std::equal(tokens.sizes().begin(), tokens.sizes().end(), logits.sizes().begin())) return py::none();
    if (!tokens.is_cuda() || tokens.get_device() != logits.get_device() || advantages.scalar_type() != at::kFloat ||
        (tokens.scalar_type() != at::kLong && tokens.scalar_type() != at::kInt))
        return py::none();
    if (logits._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode()) return py::none();
    Call c = {};
    crx_policy_args& a = c.a;
    c.tokens = tokens;
    c.dev = logits.get_device();
    a.batch = d == 2 ? tokens.size(0) : 1;
    a.steps = tokens.size(d - 1);
    a.vocab = V;
    if (!rows(tokens, tokens, false, &a.tokens) || !rows(advantages, tokens, true, &a.advantages)) return py::none();
    if (old_logp && (old_logp->scalar_type() != at::kFloat || !rows(*old_logp, tokens, false, &a.old_logp))) return py::none();
    if (ref_logp && (ref_logp->scalar_type() != at::kFloat || !rows(*ref_logp, tokens, false, &a.ref_logp))) return py::none();
    if (mask && ((mask->scalar_type() != at::kFloat && mask->scalar_type() != at::kBool) || !rows(*mask, tokens, true, &a.mask))) return py::none();
    a.denom = denom;
    a.clip_low = narrow(clip_low);
    a.clip_high = narrow(clip_high);
    a.kl_coef = static_cast<float>(kl_coef);
    a.temperature = static_cast<float>(temperature);
    a.dtype = type_code(logits.scalar_type());
    a.tokens64 = tokens.scalar_type() == at::kLong;
    a.mask_f32 = mask && mask->scalar_type() == at::kFloat;
    if (logits.requires_grad() && at::GradMode::is_enabled()) {
        const auto out = PolicyLossFn::apply(logits, &c);
        return py::make_tuple(out[0], out[1], out[2], out[3]);
    }
    const Results r = run(c, logits, false);
    const auto stats = r.stats.unbind(0);
    return py::make_tuple(r.loss, r.logp, stats[0], stats[1]);
}

}  // namespace

PYBIND11_MODULE(_glue, m) {
    m.def("grad_norm", &grad_norm);
    m.def("clip_grads", &clip_grads);
    m.def("adamw_step", &adamw_step);
    m.def("policy_loss", &policy_loss);
    m.def("grad_like", &grad_like);
}
