// policy_torch.cpp — module drone_amd/policy_torch: the policy operators of include/drone_vec.h for torch tensors, with their
// autograd nodes. Host code only (g++, libtorch): it checks tensors, fills the call structs and calls the C-ABI on torch's
// current stream. Compiled rather than ctypes because what it saves is what small policies wait for: a forward call costs
// about 5 us of host time instead of 12, forward + gradient 40 to 60 (33 of them autograd's own two threads) instead of 130.
// The library's entry points come from drone_amd.binding (bind()), so that DRONE_HIP_LIB and its load errors hold here too.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cstring>
#include <string>
#include <vector>

#include "../include/drone_vec.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
    decltype(&drone_linear_forward) linear_forward = nullptr;
    decltype(&drone_linear_backward) linear_backward = nullptr;
    decltype(&drone_linear_workspace) linear_workspace = nullptr;
    decltype(&drone_norm_forward) norm_forward = nullptr;
    decltype(&drone_norm_backward) norm_backward = nullptr;
    decltype(&drone_norm_workspace) norm_workspace = nullptr;
    decltype(&drone_adamw_step) adamw_step = nullptr;
    decltype(&drone_adamw_workspace) adamw_workspace = nullptr;
    decltype(&drone_last_error) last_error = nullptr;
} lib;

void bind(const std::map<std::string, uintptr_t>& at) {
    auto take = [&](const char* name, auto& fn) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at.at(name)); };
    take("drone_linear_forward", lib.linear_forward);
    take("drone_linear_backward", lib.linear_backward);
    take("drone_linear_workspace", lib.linear_workspace);
    take("drone_norm_forward", lib.norm_forward);
    take("drone_norm_backward", lib.norm_backward);
    take("drone_norm_workspace", lib.norm_workspace);
    take("drone_adamw_step", lib.adamw_step);
    take("drone_adamw_workspace", lib.adamw_workspace);
    take("drone_last_error", lib.last_error);
}

void run(int rc) { TORCH_CHECK(rc == 0, "libdrone_hip: ", lib.last_error()); }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int dtype_of(const Tensor& t, const char* name) {
    const auto s = t.scalar_type();
    TORCH_CHECK_TYPE(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, name, " is ", s, ": float32, bfloat16 or float16");
    TORCH_CHECK_VALUE(t.is_cuda(), name, " is on ", t.device(), ": the policy operators run on a GPU only");
    return s == at::kFloat ? DRONE_F32 : s == at::kBFloat16 ? DRONE_BF16 : DRONE_F16;
}

// A tensor argument: its shape, and the type and device of x.
void check(const char* name, const Tensor& t, at::IntArrayRef shape, const Tensor& x) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " has shape ", t.sizes(), ", expected ", shape);
    TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " is ", t.scalar_type(), ", x is ", x.scalar_type());
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", x on ", x.device());
}

// What would vanish without a word: a call that torch.jit traces (it would record the empty output), a dual tensor's tangent.
void not_traced(const char* what) { TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced"); }
void no_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors) TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}
const Tensor* there(const OptTensor& t) { return t.has_value() && t->defined() ? &*t : nullptr; }

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }  // autograd takes absent tensors, not undefined ones
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool good_rows(const Tensor& t) { return t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)); }

// A tensor [..., n] as [rows][n] with contiguous rows and a leading dimension of at least n: a view where there is one,
// else a copy. Overlapping rows (an expanded tensor) are copied, and so is a view whose sign is still to be taken.
Tensor rows_of(const Tensor& t) {
    if (t.defined() && t.is_neg()) return rows_of(t.resolve_neg());
    if (!t.defined() || good_rows(t)) return t;
    const Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / std::max<int64_t>(1, t.size(-1)), t.size(-1)});
    return good_rows(r) ? r : r.contiguous();
}

Tensor dense(const Tensor& t) { return t.resolve_neg().contiguous(); }

int64_t ld(const Tensor& t) { return !t.defined() ? 0 : t.size(0) > 1 ? std::max(t.stride(0), t.size(1)) : t.size(1); }

int activation_of(const std::string& name) {
    static const char* names[] = {"none", "relu", "tanh", "silu", "gelu"};
    for (int i = 0; i < 5; i++) if (name == names[i]) return i;
    TORCH_CHECK_VALUE(false, "unknown activation '", name, "'; one of none, relu, tanh, silu, gelu");
}

Tensor workspace(uint64_t bytes, const Tensor& x) { return at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)); }

// What a call has written in place, by address: autograd's version counter has to move, so that a backward pass through a
// graph that saved the tensor fails as it does behind torch's own in-place operators.
void written(const Tensor& t) { if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }

// Which of an operator's tensors (bit i: the i-th, if it is there) this backward pass wants the gradient of. torch counts those
// that are there.
int64_t wanted(const AutogradContext* ctx, int64_t there) {
    int64_t wants = 0;
    size_t edge = 0;
    for (int64_t bit = 1; bit <= there; bit <<= 1)
        if (there & bit) wants |= ctx->needs_input_grad(edge++) ? bit : 0;
    return wants;
}

// In a backward pass: a captured one may hand nothing to a leaf's accumulator that an eager graph of the default stream still
// holds. It would run on that stream, where a capture cannot follow, and torch ends the process over it.
void capturable(const Tensor& x, const char* what) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(c10::hip::getCurrentHIPStream(x.get_device()), &status) != hipSuccess) {
        (void)hipGetLastError();  // (the null stream beside someone else's capture: not this pass's error, and not the next call's)
        return;
    }
    if (status == hipStreamCaptureStatusNone) return;
    const auto node = torch::autograd::get_current_node();
    for (size_t i = 0; i < node->num_outputs(); i++) {
        const auto& leaf = node->next_edge(i).function;
        if (!dynamic_cast<const torch::autograd::AccumulateGrad*>(leaf.get()) || !node->task_should_compute_output(i)) continue;
        const auto stream = leaf->stream();
        TORCH_CHECK(!stream || stream->id() != 0, what, ": a graph built on the default stream still holds a leaf of this captured backward pass; let go of it (del loss) before the capture");
    }
}

// The gradients as a second differentiation has to see them: there is none.
variable_list once(variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once", 1);
    for (auto& g : grads)
        if (g.defined()) g = (*error)({g.detach().requires_grad_(true)})[0];
    return grads;
}

// ------------------------------------------------------------------------------------------------------------------ linear

DroneLinear linear_call(const Tensor& x, const Tensor& w, int activation) {
    DroneLinear c;
    std::memset(&c, 0, sizeof(c));
    c.struct_size = sizeof(c);
    c.device = x.get_device();
    c.dtype = x.scalar_type() == at::kFloat ? DRONE_F32 : x.scalar_type() == at::kBFloat16 ? DRONE_BF16 : DRONE_F16;
    c.activation = activation;
    c.rows = x.size(0);
    c.in_features = w.size(1);
    c.out_features = w.size(0);
    c.x = ptr(x);
    c.weight = ptr(w);
    c.x_ld = ld(x);
    c.weight_ld = ld(w);
    return c;
}

void linear_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& res, int activation, const Tensor& y, const Tensor& slope) {
    DroneLinear c = linear_call(x, w, activation);
    c.bias = ptr(b);
    c.residual = ptr(res);
    c.residual_ld = ld(res);
    c.y = ptr(y);
    c.y_ld = ld(y);
    c.slope = ptr(slope);
    run(lib.linear_forward(&c, stream_of(x)));
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, int64_t activation) {
        const Tensor b = bias.value_or(Tensor()), res = residual.value_or(Tensor());
        const Tensor y = at::empty({x.size(0), w.size(0)}, x.options());
        Tensor slope;
        if (activation) slope = at::empty({x.size(0), w.size(0)}, x.options().dtype(x.scalar_type() == at::kBFloat16 ? at::kHalf : at::kFloat));
        linear_forward(x, w, b, res, (int)activation, y, slope);
        ctx->save_for_backward({x, w, slope});
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["there"] = (int64_t)(3 | (b.defined() ? 4 : 0) | (res.defined() ? 8 : 0));
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dys) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &slope = saved[2];
        capturable(x, "linear");
        const int64_t wants = wanted(ctx, ctx->saved_data["there"].toInt());
        const Tensor dy = rows_of(dys[0]);
        Tensor dx, dw, db, work;
        if (wants & 7) {
            DroneLinear c = linear_call(x, w, (int)ctx->saved_data["activation"].toInt());
            c.dy = ptr(dy);
            c.dy_ld = ld(dy);
            c.slope = ptr(slope);
            if (wants & 1) { dx = at::empty({x.size(0), x.size(1)}, x.options()); c.dx = ptr(dx); c.dx_ld = x.size(1); }
            if (wants & 2) { dw = at::empty({w.size(0), w.size(1)}, x.options()); c.dweight = ptr(dw); }
            if (wants & 4) { db = at::empty({w.size(0)}, x.options()); c.dbias = ptr(db); }
            // (dx alone needs none, but streams through one where the layer is wide and whole 16-byte pieces)
            const auto whole = [&](int64_t n) { return n * (int64_t)x.element_size() % 16 == 0; };
            if ((wants & 6) || (w.numel() > 128 * 128 && whole(w.size(0)) && whole(w.size(1)))) { work = workspace(lib.linear_workspace(&c), x); c.workspace = ptr(work); c.workspace_bytes = work.numel(); }
            run(lib.linear_backward(&c, stream_of(x)));
        }
        return once({dx, dw, db, wants & 8 ? dys[0] : Tensor(), Tensor()}, "linear");
    }
};

// Whether two row matrices of one allocation share an element (exact for equal leading dimensions, by address range else).
bool overlap(const Tensor& a, const Tensor& b) {
    if (!a.defined() || !b.defined() || !a.numel() || !b.numel() || !a.is_alias_of(b)) return false;
    const int64_t d = (int64_t)((const char*)b.data_ptr() - (const char*)a.data_ptr()) / (int64_t)a.element_size(), la = ld(a), lb = ld(b);
    const int64_t end_a = (a.size(0) - 1) * la + a.size(1), end_b = (b.size(0) - 1) * lb + b.size(1);
    if (d >= end_a || -d >= end_b) return false;
    if (la != lb) return true;
    const int64_t c = ((d % la) + la) % la;  // b's first column as a counts them
    return c < a.size(1) || c + b.size(1) > la;
}

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const std::string& activation, const OptTensor& residual, const OptTensor& out) {
    dtype_of(x, "x");
    not_traced("linear");
    no_tangents("linear", {&x, &weight, there(bias), there(residual), there(out)});
    const int act = activation_of(activation);
    TORCH_CHECK_VALUE(weight.dim() == 2 && x.dim() >= 1, "weight must be [out, in] and x [..., in], got ", weight.sizes(), " and ", x.sizes());
    const int64_t n = weight.size(0), k = weight.size(1);
    TORCH_CHECK_VALUE(x.size(-1) == k, "x has ", x.size(-1), " features, the weight takes ", k);
    check("weight", weight, weight.sizes(), x);
    const bool flat = x.dim() == 2;
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    if (has(bias)) check("bias", *bias, {n}, x);
    if (has(residual)) check("residual", *residual, shape, x);
    const bool learn = at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (has(bias) && bias->requires_grad()) || (has(residual) && residual->requires_grad()));
    const Tensor x2 = rows_of(x), w2 = rows_of(weight), b2 = has(bias) ? dense(*bias) : Tensor(), r2 = has(residual) ? rows_of(*residual) : Tensor();
    if (has(out)) {
        check("out", *out, shape, x);
        TORCH_CHECK_VALUE(!learn && !(at::GradMode::is_enabled() && out->requires_grad()), "out= cannot be differentiated: call under torch.no_grad()");
        const Tensor o = flat ? *out : out->view({x2.size(0), n});
        TORCH_CHECK_VALUE(good_rows(o) && !o.is_neg(), "out must have contiguous rows that do not overlap");
        const bool in_place = r2.defined() && r2.data_ptr() == o.data_ptr() && ld(r2) == ld(o);
        TORCH_CHECK_VALUE(!overlap(x2, o) && !overlap(w2, o) && !(b2.defined() && overlap(b2.unsqueeze(0), o)) && (in_place || !overlap(r2, o)),
                          "out overlaps an input (only the residual may be updated in place)");
        linear_forward(x2, w2, b2, r2, act, o, Tensor());
        written(*out);
        return *out;
    }
    Tensor y;
    if (learn) {
        y = LinearFunction::apply(x2, w2, opt(b2), opt(r2), (int64_t)act);
    } else {
        y = at::empty({x2.size(0), n}, x.options());
        linear_forward(x2, w2, b2, r2, act, y, Tensor());
    }
    return flat ? y : y.view(shape);
}

// ----------------------------------------------------------------------------------------------------------- norm_residual

DroneNorm norm_call(const Tensor& x, const Tensor& block, const Tensor& gate, const Tensor& post, const Tensor& pre, double scale, double eps) {
    DroneNorm c;
    std::memset(&c, 0, sizeof(c));
    c.struct_size = sizeof(c);
    c.device = x.get_device();
    c.dtype = x.scalar_type() == at::kFloat ? DRONE_F32 : x.scalar_type() == at::kBFloat16 ? DRONE_BF16 : DRONE_F16;
    c.gate_kind = gate.defined() ? (int)gate.dim() : 0;
    c.rows = x.size(0);
    c.width = x.size(1);
    c.x = ptr(x);
    c.block = ptr(block);
    c.gate = ptr(gate);
    c.post_weight = ptr(post);
    c.pre_weight = ptr(pre);
    c.x_ld = ld(x);
    c.block_ld = ld(block);
    c.gate_ld = c.gate_kind == 2 ? ld(gate) : 0;
    c.scale = (float)scale;
    c.eps = (float)eps;
    return c;
}

void norm_forward(const Tensor& x, const Tensor& block, const Tensor& gate, const Tensor& post, const Tensor& pre, double scale, double eps, const Tensor& r, const Tensor& h) {
    DroneNorm c = norm_call(x, block, gate, post, pre, scale, eps);
    c.r = ptr(r);
    c.h = ptr(h);
    run(lib.norm_forward(&c, stream_of(x)));
}

struct NormFunction : torch::autograd::Function<NormFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& block_, const OptTensor& gate_, const OptTensor& post_, const OptTensor& pre_, double scale, double eps) {
        const Tensor block = block_.value_or(Tensor()), gate = gate_.value_or(Tensor()), post = post_.value_or(Tensor()), pre = pre_.value_or(Tensor());
        const Tensor r = at::empty({x.size(0), x.size(1)}, x.options()), h = at::empty({x.size(0), x.size(1)}, x.options());
        norm_forward(x, block, gate, post, pre, scale, eps, r, h);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, block, gate, post, pre});
        int64_t there = 0, bit = 1;
        for (const Tensor* t : {&x, &block, &gate, &post, &pre}) { there |= t->defined() ? bit : 0; bit <<= 1; }
        ctx->saved_data["there"] = there;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["eps"] = eps;
        return {r, h};
    }
    static variable_list backward(AutogradContext* ctx, variable_list ds) {
        variable_list grads(7);
        if (!ds[0].defined() && !ds[1].defined()) return grads;
        const variable_list in = ctx->get_saved_variables();
        const Tensor &x = in[0];
        capturable(x, "norm_residual");
        const int64_t wants = wanted(ctx, ctx->saved_data["there"].toInt());
        const Tensor dr = ds[0].defined() ? dense(ds[0]) : Tensor(), dh = ds[1].defined() ? dense(ds[1]) : Tensor();
        DroneNorm c = norm_call(x, in[1], in[2], in[3], in[4], ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble());
        c.dr = ptr(dr);
        c.dh = ptr(dh);
        for (int i = 0; i < 5; i++)
            if (wants >> i & 1) grads[i] = at::empty(in[i].sizes(), x.options());
        c.dx = ptr(grads[0]);
        c.dblock = ptr(grads[1]);
        c.dgate = ptr(grads[2]);
        c.dpost_weight = ptr(grads[3]);
        c.dpre_weight = ptr(grads[4]);
        const Tensor work = workspace(lib.norm_workspace(&c), x);
        c.workspace = ptr(work);
        c.workspace_bytes = work.numel();
        run(lib.norm_backward(&c, stream_of(x)));
        return once(std::move(grads), "norm_residual");
    }
};

std::tuple<Tensor, Tensor> norm_residual(const Tensor& x, const OptTensor& block, const OptTensor& gate, double scale, const OptTensor& post_weight, const OptTensor& pre_weight, double eps) {
    dtype_of(x, "x");
    not_traced("norm_residual");
    no_tangents("norm_residual", {&x, there(block), there(gate), there(post_weight), there(pre_weight)});
    TORCH_CHECK_VALUE(x.dim() >= 1, "x must be [..., width]");
    const int64_t width = x.size(-1);
    TORCH_CHECK_VALUE(width >= 1 && width <= 4096, "width must be 1 ... 4096, got ", width);
    if (has(block)) check("block", *block, x.sizes(), x);
    if (has(post_weight)) check("post_weight", *post_weight, {width}, x);
    if (has(pre_weight)) check("pre_weight", *pre_weight, {width}, x);
    TORCH_CHECK_VALUE(has(block) || !(has(gate) || has(post_weight)), "gate and post_weight belong to a block");
    const bool channel = has(gate) && gate->dim() == 1 && x.dim() > 1;
    if (has(gate)) check("gate", *gate, channel ? at::IntArrayRef({width}) : x.sizes(), x);
    TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative");
    auto learns = [](const OptTensor& t) { return has(t) && t->requires_grad(); };
    const bool learn = at::GradMode::is_enabled() && (x.requires_grad() || learns(block) || learns(gate) || learns(post_weight) || learns(pre_weight)), flat = x.dim() == 2;
    auto weight = [](const OptTensor& t) { return has(t) ? dense(*t) : Tensor(); };
    const auto two = [](const Tensor& t) { return t.dim() == 1 ? t.unsqueeze(0) : t; };
    const Tensor x2 = rows_of(two(x)), block2 = has(block) ? rows_of(two(*block)) : Tensor(), gate2 = channel ? dense(*gate) : has(gate) ? rows_of(two(*gate)) : Tensor();
    Tensor r, h;
    if (learn) {
        const variable_list out = NormFunction::apply(x2, opt(block2), opt(gate2), opt(weight(post_weight)), opt(weight(pre_weight)), scale, eps);
        r = out[0];
        h = out[1];
    } else {
        r = at::empty({x2.size(0), width}, x.options());
        h = at::empty({x2.size(0), width}, x.options());
        norm_forward(x2, block2, gate2, weight(post_weight), weight(pre_weight), scale, eps, r, h);
    }
    return flat ? std::make_tuple(r, h) : std::make_tuple(r.view(x.sizes()), h.view(x.sizes()));
}

// -------------------------------------------------------------------------------------------------------------- adamw_step

Tensor adamw_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& exp_avgs, const std::vector<Tensor>& exp_avg_sqs, const Tensor& step, double lr,
                  std::pair<double, double> betas, double eps, double weight_decay, std::optional<double> max_grad_norm, const std::optional<std::vector<Tensor>>& masters) {
    TORCH_CHECK_VALUE(!params.empty(), "no parameters");
    not_traced("adamw_step");
    TORCH_CHECK_VALUE(!max_grad_norm || *max_grad_norm > 0, "max_grad_norm must be positive (None: no clipping), got ", *max_grad_norm);
    const Tensor& first = params[0];
    const int dtype = dtype_of(first, "params[0]");
    TORCH_CHECK_VALUE(masters.has_value() == (dtype != DRONE_F32), "16-bit params need float32 masters, float32 params have none");
    const size_t count = params.size();
    std::vector<std::pair<const char*, const char*>> seen;  // first byte, one past the last
    seen.reserve(5 * count);
    auto check_list = [&](const char* name, const std::vector<Tensor>& list, at::ScalarType type) {
        TORCH_CHECK_VALUE(list.size() == count, list.size(), " ", name, " for ", count, " params");
        for (size_t i = 0; i < count; i++) {
            const Tensor& t = list[i];
            TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == first.device() && t.sizes() == params[i].sizes() && t.is_contiguous() && !t.is_neg(), name, ": expected a contiguous ", type,
                              " tensor of shape ", params[i].sizes(), " on ", first.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
            if (t.numel()) seen.emplace_back((const char*)t.data_ptr(), (const char*)t.data_ptr() + t.numel() * t.element_size());
        }
    };
    check_list("params", params, first.scalar_type());
    check_list("grads", grads, first.scalar_type());
    check_list("exp_avgs", exp_avgs, at::kFloat);
    check_list("exp_avg_sqs", exp_avg_sqs, at::kFloat);
    if (masters) check_list("masters", *masters, at::kFloat);
    std::sort(seen.begin(), seen.end());
    for (size_t i = 1; i < seen.size(); i++) {
        TORCH_CHECK_VALUE(seen[i].first != seen[i - 1].first, "a tensor is there twice");
        TORCH_CHECK_VALUE(seen[i].first >= seen[i - 1].second, "two tensors overlap");
    }
    TORCH_CHECK_VALUE(step.scalar_type() == at::kInt && step.numel() == 1 && step.device() == first.device(), "step must be an int32 tensor of one element on the params' device");
    std::vector<DroneAdamWTensor> table(count);
    for (size_t i = 0; i < count; i++)
        table[i] = {ptr(params[i]), ptr(grads[i]), (float*)ptr(exp_avgs[i]), (float*)ptr(exp_avg_sqs[i]), masters ? (float*)ptr((*masters)[i]) : nullptr, params[i].numel()};
    const Tensor norm = at::empty({1}, first.options().dtype(at::kFloat));
    DroneAdamW c;
    std::memset(&c, 0, sizeof(c));
    c.struct_size = sizeof(c);
    c.device = first.get_device();
    c.dtype = dtype;
    c.count = (int)count;
    c.tensors = table.data();
    c.step = (int32_t*)ptr(step);
    c.grad_norm = (float*)ptr(norm);
    c.lr = lr;
    c.beta1 = betas.first;
    c.beta2 = betas.second;
    c.eps = eps;
    c.weight_decay = weight_decay;
    c.max_grad_norm = max_grad_norm.value_or(0.0);
    const Tensor work = workspace(lib.adamw_workspace(&c), first);
    c.workspace = ptr(work);
    c.workspace_bytes = work.numel();
    run(lib.adamw_step(&c, stream_of(first)));
    for (const auto* list : {&params, &exp_avgs, &exp_avg_sqs}) for (const Tensor& t : *list) written(t);
    if (masters) for (const Tensor& t : *masters) written(t);
    written(step);
    return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    m.def("bind", &bind);
    m.def("linear", &linear, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("activation"), py::arg("residual"), py::arg("out"));
    m.def("norm_residual", &norm_residual);
    m.def("adamw_step", &adamw_step);
}
