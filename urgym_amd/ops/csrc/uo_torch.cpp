// The policy operators for torch: argument checks, outputs and workspaces from torch's allocator, torch's current stream, and
// autograd nodes, around the C-ABI of include/urgym_ops.h.  In C++ because a call's own time matters: a rollout step enqueues
// several of these on a few thousand envs, whose kernels take less time than the same calls from Python do.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <initializer_list>
#include <optional>

#include "../../../include/urgym_ops.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

static void done(int rc) { TORCH_CHECK(rc == 0, urgym_ops_last_error()); }

static int code(at::ScalarType t) { return t == at::kFloat ? URGYM_OPS_F32 : t == at::kBFloat16 ? URGYM_OPS_BF16 : URGYM_OPS_F16; }

static bool known(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }

static void need_known(const char* name, const Tensor& x) {
    TORCH_CHECK_TYPE(known(x.scalar_type()), name, " must be float32, bfloat16 or float16, not ", x.scalar_type());
}

static void need_type(const char* name, const Tensor& x, at::ScalarType t) {
    TORCH_CHECK_TYPE(x.scalar_type() == t, name, " must be ", t, ", not ", x.scalar_type());
}

static void need_device(const char* name, const Tensor& x, const Tensor& with) {
    TORCH_CHECK_VALUE(x.device() == with.device(), name, " is on ", x.device(), ", not on ", with.device());
}

static void need_gpu(const Tensor& x) {
    TORCH_CHECK_VALUE(x.is_cuda(), "the operators run on the GPU, the tensors are on ", x.device(), "; no CPU fallback exists");
}

// Refuses what would be lost without a word: the kernels answer no forward-mode tangent, and a trace sees only the outputs' allocation.
static void need_eager(const char* what, std::initializer_list<const Tensor*> inputs) {
    for (const Tensor* x : inputs)
        TORCH_CHECK_VALUE(!x->defined() || !x->_fw_grad(0).defined(), what, ": forward-mode gradients are not offered");
    TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced (torch.jit.trace would record its outputs' allocation only)");
}

static void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream(); }

static const void* ptr(const Tensor& x) { return x.defined() ? x.const_data_ptr() : nullptr; }

static Tensor given(const Maybe& x) { return x.has_value() ? *x : Tensor(); }

static Maybe maybe(const Tensor& x) { return x.defined() ? Maybe(x) : Maybe(); }

// x with its last axis contiguous (a copy only if it is not)
static Tensor rows(const Tensor& x) { return x.stride(-1) == 1 || x.size(-1) == 1 ? x : x.contiguous(); }

// ---- layer norm ----

// x as [rows, width] with contiguous rows: a view where its leading axes allow one
static Tensor matrix(const Tensor& x) {
    if (x.dim() == 2 && x.stride(1) == 1) return x;
    Tensor m = x.is_contiguous() ? x.view({-1, x.size(-1)}) : rows(x).reshape({-1, x.size(-1)});
    return m.stride(1) == 1 || m.size(1) == 1 ? m : m.contiguous();
}

static int64_t row_stride(const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : m.size(1); }

static Tensor norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats) {
    at::DeviceGuard guard(x.device());
    Tensor m = matrix(x), y = at::empty(x.sizes(), x.options());
    int64_t n = m.size(0), width = m.size(1);
    float *mean = nullptr, *rstd = nullptr;
    if (stats) {
        *stats = at::empty({2, n}, x.options().dtype(at::kFloat));
        mean = stats->mutable_data_ptr<float>(), rstd = mean + n;
    }
    at::ScalarType param = weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
    done(urgym_ops_layer_norm(code(x.scalar_type()), code(param), n, width, m.const_data_ptr(), row_stride(m), ptr(weight), ptr(bias),
                              (float)eps, y.mutable_data_ptr(), mean, rstd, stream_of(x)));
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight_, const Maybe& bias_, double eps) {
        Tensor weight = given(weight_), bias = given(bias_);
        Tensor stats, y = norm_forward(x, weight, bias, eps, &stats);
        ctx->save_for_backward({x, weight, stats});
        ctx->saved_data["x"] = x.requires_grad();
        ctx->saved_data["w"] = weight.defined() && weight.requires_grad();
        ctx->saved_data["b"] = bias.defined() && bias.requires_grad();
        ctx->saved_data["param"] = (int64_t)(weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type());
        ctx->set_materialize_grads(false);
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm: gradients of gradients are not offered");
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        at::DeviceGuard guard(x.device());
        Tensor m = matrix(x), d = matrix(grads[0]), dx, dw, db, ws;
        int64_t n = m.size(0), width = m.size(1);
        auto param = (at::ScalarType)ctx->saved_data["param"].toInt();
        bool want_w = ctx->saved_data["w"].toBool(), want_b = ctx->saved_data["b"].toBool();
        if (ctx->saved_data["x"].toBool()) dx = at::empty(x.sizes(), x.options());
        if (want_w) dw = at::empty({width}, x.options().dtype(param));
        if (want_b) db = at::empty({width}, x.options().dtype(param));
        if (want_w || want_b) ws = at::empty({urgym_ops_layer_norm_workspace(n, width)}, x.options().dtype(at::kFloat));
        const float* mean = stats.const_data_ptr<float>();
        done(urgym_ops_layer_norm_backward(code(x.scalar_type()), code(param), n, width, d.const_data_ptr(), row_stride(d), m.const_data_ptr(),
                                           row_stride(m), ptr(weight), mean, mean + n, (void*)ptr(dx), (void*)ptr(dw), (void*)ptr(db),
                                           (float*)ptr(ws), stream_of(x)));
        return {dx, dw, db, Tensor()};
    }
};

static Tensor layer_norm(const Tensor& x, const Maybe& weight_, const Maybe& bias_, double eps) {
    need_known("x", x);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x of shape ", x.sizes(), " has no last axis to normalise");
    TORCH_CHECK_VALUE(eps > 0, "eps must be positive, not ", eps);
    Tensor weight = given(weight_), bias = given(bias_);
    auto param = [&](const char* name, Tensor& p) {
        if (!p.defined()) return;
        need_known(name, p);
        need_device(name, p, x);
        TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == x.size(-1), name, " has shape ", p.sizes(), ", x's last axis is ", x.size(-1));
        TORCH_CHECK_TYPE(p.scalar_type() == x.scalar_type() || p.scalar_type() == at::kFloat, name, " is ", p.scalar_type(),
                         ": x's dtype (", x.scalar_type(), ") or float32 is needed");
        p = p.contiguous();
    };
    param("weight", weight);
    param("bias", bias);
    TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "weight is ",
                     weight.scalar_type(), ", bias ", bias.scalar_type(), ": one dtype is needed");
    need_eager("layer_norm", {&x, &weight, &bias});
    need_gpu(x);
    if (at::GradMode::is_enabled() && (x.requires_grad() || (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad())))
        return LayerNorm::apply(x, maybe(weight), maybe(bias), eps);
    return norm_forward(x, weight, bias, eps, nullptr);
}

// ---- attention with a decay ----

static void need_heads(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, int64_t dims, const char* what) {
    need_known("q", q);
    need_type("k", k, q.scalar_type());
    need_type("v", v, q.scalar_type());
    need_device("k", k, q);
    need_device("v", v, q);
    bool fit = q.dim() == dims && k.sizes() == q.sizes() && v.dim() == dims;
    for (int64_t i = 0; fit && i + 1 < dims; i++) fit = v.size(i) == q.size(i);
    TORCH_CHECK_VALUE(fit, "q, k and v must be ", what, ", not ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
    for (const Tensor* x : {&q, &v})
        TORCH_CHECK_VALUE(x->size(-1) >= 1 && x->size(-1) <= URGYM_OPS_MAX_HEAD_DIM, x == &q ? "dk" : "dv", " = ", x->size(-1), " must be 1 .. ",
                          URGYM_OPS_MAX_HEAD_DIM);
    TORCH_CHECK_VALUE(q.size(-2) >= 1, "at least one head is needed");
    need_type("log_decay", log_decay, at::kFloat);
    need_device("log_decay", log_decay, q);
    TORCH_CHECK_VALUE(log_decay.dim() == 1 && log_decay.size(0) == q.size(-2), "log_decay has shape ", log_decay.sizes(), ", not [", q.size(-2),
                      "]: one value for each head");
    TORCH_CHECK_VALUE(!log_decay.requires_grad(), "log_decay is a constant of the policy: no gradient is computed for it (detach it)");
}

static void need_start(const Tensor& start, at::IntArrayRef shape, const Tensor& q) {
    if (!start.defined()) return;
    TORCH_CHECK_TYPE(start.scalar_type() == at::kBool || start.scalar_type() == at::kByte, "start must be bool or uint8, not ", start.scalar_type());
    need_device("start", start, q);
    TORCH_CHECK_VALUE(start.sizes() == shape, "start has shape ", start.sizes(), ", not ", shape);
}

static void need_state(const char* name, const Tensor& state, at::IntArrayRef shape, const Tensor& q) {
    need_type(name, state, at::kFloat);
    need_device(name, state, q);
    TORCH_CHECK_VALUE(state.sizes() == shape, name, " has shape ", state.sizes(), ", not ", shape);
}

static urgym_ops_seq sequence(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state, const Tensor& start,
                              double scale) {
    urgym_ops_seq s = {};
    s.dtype = code(q.scalar_type()), s.heads = (int32_t)q.size(2), s.dk = (int32_t)q.size(3), s.dv = (int32_t)v.size(3);
    s.steps = q.size(0), s.envs = q.size(1);
    s.q = q.const_data_ptr(), s.k = k.const_data_ptr(), s.v = v.const_data_ptr();
    for (int i = 0; i < 3; i++) s.q_stride[i] = q.stride(i), s.k_stride[i] = k.stride(i), s.v_stride[i] = v.stride(i);
    s.log_decay = log_decay.const_data_ptr<float>(), s.state = (const float*)ptr(state), s.scale = (float)scale;
    if (start.defined()) s.start = (const uint8_t*)start.const_data_ptr(), s.start_stride[0] = start.stride(0), s.start_stride[1] = start.stride(1);
    return s;
}

static Tensor workspace(int64_t floats, const Tensor& q) {
    TORCH_CHECK(floats >= 0, urgym_ops_last_error());
    return floats ? at::empty({floats}, q.options().dtype(at::kFloat)) : Tensor();
}

static std::tuple<Tensor, Tensor> decay_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                                                const Tensor& start, double scale) {
    at::DeviceGuard guard(q.device());
    Tensor o = at::empty(v.sizes(), q.options());
    const int64_t shape[4] = {q.size(1), q.size(2), q.size(3), v.size(3)};
    if (q.size(0) == 0)  // no step: nothing is answered and nothing forgotten
        return {o, state.defined() ? state.clone() : at::zeros(shape, q.options().dtype(at::kFloat))};
    Tensor final = at::empty(shape, q.options().dtype(at::kFloat));
    if (q.size(1)) {
        urgym_ops_seq s = sequence(q, k, v, log_decay, state, start, scale);
        Tensor ws = workspace(urgym_ops_decay_workspace(&s), q);
        done(urgym_ops_decay(&s, o.mutable_data_ptr(), final.mutable_data_ptr<float>(), (float*)ptr(ws), stream_of(q)));
    }
    return {o, final};
}

struct DecayAttention : torch::autograd::Function<DecayAttention> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& state_,
                                 const Maybe& start_, double scale) {
        Tensor state = given(state_), start = given(start_);
        auto [o, final] = decay_forward(q, k, v, log_decay, state, start, scale);
        ctx->save_for_backward({q, k, v, log_decay, state, start});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["state"] = state.defined() && state.requires_grad();
        ctx->set_materialize_grads(false);
        return {o, final};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "decay_attention: gradients of gradients are not offered");
        variable_list saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &log_decay = saved[3], &state = saved[4], &start = saved[5];
        at::DeviceGuard guard(q.device());
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options()), dstate;
        if (ctx->saved_data["state"].toBool() && q.size(0) == 0)
            dstate = grads[1].defined() ? grads[1].clone(at::MemoryFormat::Contiguous) : at::zeros(state.sizes(), state.options());
        else if (ctx->saved_data["state"].toBool())
            dstate = at::empty(state.sizes(), state.options());
        if (q.size(0) && q.size(1)) {
            Tensor d_out = grads[0].defined() ? rows(grads[0]) : at::zeros(v.sizes(), v.options());
            Tensor d_final = grads[1].defined() ? grads[1].contiguous() : Tensor();
            urgym_ops_seq s = sequence(q, k, v, log_decay, state, start, ctx->saved_data["scale"].toDouble());
            int64_t stride[3] = {d_out.stride(0), d_out.stride(1), d_out.stride(2)};
            Tensor ws = workspace(urgym_ops_decay_backward_workspace(&s, d_out.const_data_ptr(), stride), q);
            done(urgym_ops_decay_backward(&s, d_out.const_data_ptr(), stride, (const float*)ptr(d_final), dq.mutable_data_ptr(), dk.mutable_data_ptr(),
                                          dv.mutable_data_ptr(), (float*)ptr(dstate), (float*)ptr(ws), stream_of(q)));
        }
        return {dq, dk, dv, Tensor(), dstate, Tensor(), Tensor()};
    }
};

static std::tuple<Tensor, Tensor> decay_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Maybe& state_,
                                                  const Maybe& start_, std::optional<double> scale_) {
    Tensor state = given(state_), start = given(start_);
    need_heads(q, k, v, log_decay, 4, "[steps, envs, heads, dk], the same and [steps, envs, heads, dv]");
    const int64_t shape[4] = {q.size(1), q.size(2), q.size(3), v.size(3)};
    if (state.defined()) need_state("state", state, shape, q);
    need_start(start, q.sizes().slice(0, 2), q);
    need_eager("decay_attention", {&q, &k, &v, &log_decay, &state});
    need_gpu(q);
    double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)q.size(3));
    Tensor a = rows(q), b = rows(k), c = rows(v), g = log_decay.contiguous();
    if (state.defined()) state = state.contiguous();
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || (state.defined() && state.requires_grad()))) {
        variable_list r = DecayAttention::apply(a, b, c, g, maybe(state), maybe(start), scale);
        return {r[0], r[1]};
    }
    return decay_forward(a, b, c, g, state, start, scale);
}

static std::tuple<Tensor, Tensor> decay_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                                                       const Maybe& start_, std::optional<double> scale, const Maybe& out_) {
    Tensor start = given(start_), out = given(out_);
    need_heads(q, k, v, log_decay, 3, "[envs, heads, dk], the same and [envs, heads, dv]");
    const int64_t shape[4] = {q.size(0), q.size(1), q.size(2), v.size(2)};
    need_state("state", state, shape, q);
    need_start(start, q.sizes().slice(0, 1), q);
    TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous");
    if (out.defined() && !out.is_same(state)) {
        need_state("state_out", out, shape, q);
        TORCH_CHECK_VALUE(out.is_contiguous(), "state_out must be contiguous");
        int64_t apart = (const char*)out.const_data_ptr() - (const char*)state.const_data_ptr();
        TORCH_CHECK_VALUE(apart == 0 || std::abs(apart) >= 4 * state.numel(), "state_out overlaps state without being it");
    }
    TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad() || state.requires_grad() ||
                                                        (out.defined() && out.requires_grad())),
                      "decay_attention_step has no gradient: call it under torch.no_grad(), or decay_attention for training");
    need_eager("decay_attention_step", {&q, &k, &v, &log_decay, &state, &out});
    need_gpu(q);
    at::DeviceGuard guard(q.device());
    if (out.defined()) out.unsafeGetTensorImpl()->bump_version();  // a graph that has saved it must not use what it becomes
    else out = at::empty_like(state);
    Tensor o = at::empty(v.sizes(), q.options()), a = rows(q), b = rows(k), c = rows(v), g = log_decay.contiguous();
    if (shape[0])
        done(urgym_ops_decay_step(code(q.scalar_type()), shape[0], (int)shape[1], (int)shape[2], (int)shape[3], a.const_data_ptr(), a.stride(0), a.stride(1),
                                  b.const_data_ptr(), b.stride(0), b.stride(1), c.const_data_ptr(), c.stride(0), c.stride(1), g.const_data_ptr<float>(),
                                  (const uint8_t*)ptr(start), start.defined() ? start.stride(0) : 0,
                                  (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)shape[2])), state.const_data_ptr<float>(),
                                  out.mutable_data_ptr<float>(), o.mutable_data_ptr(), stream_of(q)));
    return {o, out};
}

PYBIND11_MODULE(urgym_ops_torch, m) {
    namespace py = pybind11;
    m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
    m.def("decay_attention", &decay_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("state"), py::arg("start"),
          py::arg("scale"));
    m.def("decay_attention_step", &decay_attention_step, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("state"),
          py::arg("start"), py::arg("scale"), py::arg("state_out"));
}
