// drone_policy.cpp — the C-ABI of the policy operators (include/drone_vec.h: drone_linear_*, drone_norm_*, drone_adamw_*):
// argument checks, device and stream, then the launchers of drone_linear.hip / drone_norm.hip / drone_adamw.hip.
#include "drone_policy.hpp"

#include <cfloat>
#include <cmath>

#include "drone_vec_impl.hpp"

using namespace drone_impl;

namespace {

// The device of a call: made current for its launches, the caller's put back behind them.
struct OnDevice {
    DeviceRestore restore;
    bool ok;
    explicit OnDevice(int device) {
        (void)hipGetLastError();  // an error an earlier call of someone else left is not this call's
        const hipError_t e = hipSetDevice(device);
        ok = e == hipSuccess;
        if (!ok) { set_err("hipSetDevice(%d) failed: %s", device, hipGetErrorString(e)); (void)hipGetLastError(); }
    }
};

int launched(int rc, const char* what) {
    if (rc) set_err("%s: launch failed: %s", what, hipGetErrorString((hipError_t)rc));
    return rc ? -1 : 0;
}

bool fail(const char* what, const char* why) {
    set_err("%s: %s", what, why);
    return false;
}

bool known(int dtype) { return dtype == DRONE_F32 || dtype == DRONE_BF16 || dtype == DRONE_F16; }
uintptr_t elem_mask(int dtype) { return dtype == DRONE_F32 ? 3 : 1; }
bool odd(const void* p, uintptr_t mask) { return ((uintptr_t)p & mask) != 0; }

bool check_linear(const DroneLinear* c, const char* what) {
    err_text()[0] = 0;
    if (!c) return fail(what, "call is NULL");
    if (c->struct_size != sizeof(DroneLinear)) return fail(what, "struct_size is not sizeof(DroneLinear)");
    if (!known(c->dtype)) return fail(what, "unknown dtype");
    if (c->activation < DRONE_ACTIVATION_NONE || c->activation > DRONE_ACTIVATION_GELU) return fail(what, "unknown activation");
    if (c->rows < 0 || c->rows > (1LL << 30)) return fail(what, "rows must be 0 ... 2^30");
    if (c->in_features < 1 || c->in_features > 65536 || c->out_features < 1 || c->out_features > 65536) return fail(what, "in_features and out_features must be 1 ... 65536");
    return true;
}

LinearArgs linear_args(const DroneLinear* c) {
    LinearArgs a = {};
    a.rows = c->rows; a.in = (int)c->in_features; a.out = (int)c->out_features;
    a.x = c->x; a.w = c->weight; a.b = c->bias; a.res = c->residual; a.dy = c->dy;
    a.y = c->y; a.slope = c->slope; a.dx = c->dx; a.dw = c->dweight; a.db = c->dbias;
    a.work = (float*)c->workspace;
    a.x_ld = c->x_ld; a.w_ld = c->weight_ld; a.res_ld = c->residual_ld; a.y_ld = c->y_ld; a.dy_ld = c->dy_ld; a.dx_ld = c->dx_ld;
    a.act = c->activation;
    return a;
}

bool check_norm(const DroneNorm* c, const char* what) {
    err_text()[0] = 0;
    if (!c) return fail(what, "call is NULL");
    if (c->struct_size != sizeof(DroneNorm)) return fail(what, "struct_size is not sizeof(DroneNorm)");
    if (!known(c->dtype)) return fail(what, "unknown dtype");
    if (c->gate_kind < 0 || c->gate_kind > 2) return fail(what, "gate_kind must be 0, 1 or 2");
    if (c->rows < 0 || c->rows > (1LL << 30)) return fail(what, "rows must be 0 ... 2^30");
    if (c->width < 1 || c->width > 4096) return fail(what, "width must be 1 ... 4096");
    if (!(c->eps >= 0.f)) return fail(what, "eps must not be negative");
    if (c->gate_kind && !c->gate) { if (c->rows || c->gate_kind == 1) return fail(what, "gate is NULL"); }
    if (c->gate_kind && !c->block && c->rows) return fail(what, "a gate needs a block");
    if (c->rows && !c->x) return fail(what, "x is NULL");
    if (c->x_ld < c->width || (c->block && c->block_ld < c->width) || (c->gate_kind == 2 && c->gate_ld < c->width)) return fail(what, "a leading dimension is smaller than width");
    const uintptr_t m = elem_mask(c->dtype);
    if (odd(c->x, m) || odd(c->block, m) || odd(c->gate, m) || odd(c->post_weight, m) || odd(c->pre_weight, m) || odd(c->dr, m) || odd(c->dh, m) || odd(c->r, m) || odd(c->h, m) ||
        odd(c->dx, m) || odd(c->dblock, m) || odd(c->dgate, m) || odd(c->dpost_weight, m) || odd(c->dpre_weight, m)) return fail(what, "a pointer is not aligned to its elements");
    return true;
}

NormArgs norm_args(const DroneNorm* c) {
    NormArgs a = {};
    a.rows = c->rows; a.width = (int)c->width;
    a.x = c->x; a.block = c->block; a.gate = c->gate; a.post = c->post_weight; a.pre = c->pre_weight; a.dr = c->dr; a.dh = c->dh;
    a.r = c->r; a.h = c->h; a.dx = c->dx; a.dblock = c->dblock; a.dgate = c->dgate; a.dpost = c->dpost_weight; a.dpre = c->dpre_weight;
    a.x_ld = c->x_ld; a.block_ld = c->block_ld; a.gate_ld = c->gate_ld;
    a.work = (float*)c->workspace;
    a.gate_rows = c->gate_kind; a.scale = c->scale; a.eps = c->eps;
    return a;
}

long long chunks_of(int64_t n) { return (n + kAdamwChunk - 1) / kAdamwChunk; }

bool check_adamw(const DroneAdamW* c, const char* what) {
    err_text()[0] = 0;
    if (!c) return fail(what, "call is NULL");
    if (c->struct_size != sizeof(DroneAdamW)) return fail(what, "struct_size is not sizeof(DroneAdamW)");
    if (!known(c->dtype)) return fail(what, "unknown dtype");
    if (c->count < 0 || (c->count && !c->tensors)) return fail(what, "tensors is NULL");
    for (int i = 0; i < c->count; i++)
        if (c->tensors[i].elements < 0 || c->tensors[i].elements > (1LL << 34)) return fail(what, "a tensor's elements must be 0 ... 2^34");
    return true;
}

// One launch's share of the tensors: up to kAdamwTensors of them, at most 2^23 chunks (one tensor may be as many). Returns how many it took.
int fill_adamw(const DroneAdamW* c, int from, AdamwArgs* a) {
    const uintptr_t align = 15;
    long long chunks = 0;
    int i = from;
    a->count = 0;
    for (; i < c->count && a->count < kAdamwTensors; i++) {
        const DroneAdamWTensor& s = c->tensors[i];
        if (!s.elements) continue;
        const long long more = chunks_of(s.elements);
        if (a->count && chunks + more > (1LL << 23)) break;
        AdamwTensor& t = a->t[a->count++];
        t.p = s.param; t.g = s.grad; t.m = s.exp_avg; t.v = s.exp_avg_sq; t.master = s.master;
        t.n = s.elements;
        t.first_chunk = (int)chunks;
        t.vec = !(odd(s.param, align) || odd(s.grad, align) || odd(s.exp_avg, align) || odd(s.exp_avg_sq, align) || odd(s.master, align));
        chunks += more;
    }
    a->chunks = (int)chunks;
    return i - from;
}

int adamw_parts(const AdamwArgs& a) { return a.chunks < kAdamwParts ? a.chunks : kAdamwParts; }

}  // namespace

extern "C" {

uint64_t drone_linear_workspace(const DroneLinear* c) {
    if (!check_linear(c, "drone_linear_workspace")) return 0;
    return linear_work_bytes(c->dtype, c->rows, (int)c->in_features, (int)c->out_features);
}

int drone_linear_forward(const DroneLinear* c, void* stream) {
    const char* what = "drone_linear_forward";
    if (!check_linear(c, what)) return -1;
    if (c->rows == 0) return 0;
    if (!c->x || !c->weight || !c->y) return fail(what, "x, weight and y must not be NULL"), -1;
    if (c->x_ld < c->in_features || c->weight_ld < c->in_features || c->y_ld < c->out_features || (c->residual && c->residual_ld < c->out_features))
        return fail(what, "a leading dimension is smaller than its rows"), -1;
    const uintptr_t m = elem_mask(c->dtype);
    if (odd(c->x, m) || odd(c->weight, m) || odd(c->y, m) || odd(c->bias, m) || odd(c->residual, m) || odd(c->slope, m)) return fail(what, "a pointer is not aligned to its elements"), -1;
    OnDevice dev(c->device);
    return dev.ok ? launched(linear_forward_launch(c->dtype, linear_args(c), (hipStream_t)stream), what) : -1;
}

int drone_linear_backward(const DroneLinear* c, void* stream) {
    const char* what = "drone_linear_backward";
    if (!check_linear(c, what)) return -1;
    if (!c->dx && !c->dweight && !c->dbias) return 0;
    if (c->rows && !c->dy) return fail(what, "dy is NULL"), -1;
    if (c->rows && c->activation != DRONE_ACTIVATION_NONE && !c->slope) return fail(what, "the slope that the forward call wrote is needed"), -1;
    if (c->dx && !c->weight) return fail(what, "dx needs the weight"), -1;
    if ((c->dweight || c->dbias) && c->rows && !c->x) return fail(what, "dweight and dbias need x"), -1;
    if (c->dy_ld < c->out_features || (c->dx && (c->dx_ld < c->in_features || c->weight_ld < c->in_features)) || ((c->dweight || c->dbias) && c->x_ld < c->in_features))
        return fail(what, "a leading dimension is smaller than its rows"), -1;
    const uintptr_t m = elem_mask(c->dtype);
    if (odd(c->x, m) || odd(c->weight, m) || odd(c->dy, m) || odd(c->slope, m) || odd(c->dx, m) || odd(c->dweight, m) || odd(c->dbias, m)) return fail(what, "a pointer is not aligned to its elements"), -1;
    LinearArgs a = linear_args(c);
    if (c->activation == DRONE_ACTIVATION_NONE) a.slope = nullptr;
    if (!c->workspace || odd(c->workspace, 15) || c->workspace_bytes < linear_work_bytes(c->dtype, c->rows, a.in, a.out)) {
        if (c->dweight || c->dbias) return fail(what, "dweight and dbias need drone_linear_workspace bytes, 16-byte aligned"), -1;
        a.work = nullptr;
    }
    OnDevice dev(c->device);
    return dev.ok ? launched(linear_backward_launch(c->dtype, a, (hipStream_t)stream), what) : -1;
}

uint64_t drone_norm_workspace(const DroneNorm* c) {
    if (!check_norm(c, "drone_norm_workspace")) return 0;
    return norm_work_bytes(c->dtype, c->rows, (int)c->width);
}

int drone_norm_forward(const DroneNorm* c, void* stream) {
    const char* what = "drone_norm_forward";
    if (!check_norm(c, what)) return -1;
    if (c->rows == 0) return 0;
    if (!c->h) return fail(what, "h is NULL"), -1;
    OnDevice dev(c->device);
    return dev.ok ? launched(norm_forward_launch(c->dtype, norm_args(c), (hipStream_t)stream), what) : -1;
}

int drone_norm_backward(const DroneNorm* c, void* stream) {
    const char* what = "drone_norm_backward";
    if (!check_norm(c, what)) return -1;
    if (!c->block && c->rows && (c->dblock || c->dgate || c->dpost_weight)) return fail(what, "there is no block to differentiate"), -1;
    if (c->dgate && !c->gate_kind) return fail(what, "there is no gate to differentiate"), -1;
    const bool sums = c->dpost_weight || c->dpre_weight || (c->dgate && c->gate_kind == 1);
    if (sums && (!c->workspace || odd(c->workspace, 15) || c->workspace_bytes < norm_work_bytes(c->dtype, c->rows, (int)c->width)))
        return fail(what, "the gradients over the rows need drone_norm_workspace bytes, 16-byte aligned"), -1;
    if (!sums && !c->dx && !c->dblock && !c->dgate) return 0;
    OnDevice dev(c->device);
    return dev.ok ? launched(norm_backward_launch(c->dtype, norm_args(c), (hipStream_t)stream), what) : -1;
}

uint64_t drone_adamw_workspace(const DroneAdamW* c) {
    if (!check_adamw(c, "drone_adamw_workspace")) return 0;
    uint64_t parts = 2;
    AdamwArgs a;
    for (int from = 0; from < c->count;) {
        from += fill_adamw(c, from, &a);
        parts += adamw_parts(a);
    }
    return parts * sizeof(float);
}

int drone_adamw_step(const DroneAdamW* c, void* stream) {
    const char* what = "drone_adamw_step";
    if (!check_adamw(c, what)) return -1;
    if (!c->step || odd(c->step, 3)) return fail(what, "step is NULL or misaligned"), -1;
    if (!(c->beta1 >= 0 && c->beta1 < 1 && c->beta2 >= 0 && c->beta2 < 1)) return fail(what, "beta1 and beta2 must be in [0, 1)"), -1;
    if (!(c->lr >= 0) || !(c->weight_decay >= 0)) return fail(what, "lr and weight_decay must not be negative"), -1;
    // the update multiplies m by rcp(sqrt(v) + eps) of the hardware, which take denormals for 0: without eps that is infinite
    if (!((float)c->eps >= FLT_MIN)) return fail(what, "eps must be positive (a normal 32-bit number)"), -1;
    if (c->max_grad_norm != c->max_grad_norm) return fail(what, "max_grad_norm is not a number"), -1;
    if (c->max_grad_norm > 0 && (float)c->max_grad_norm < FLT_MIN) return fail(what, "max_grad_norm must be a normal 32-bit number (or not positive: no clipping)"), -1;
    const uintptr_t m = elem_mask(c->dtype);
    for (int i = 0; i < c->count; i++) {
        const DroneAdamWTensor& t = c->tensors[i];
        if (!t.elements) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return fail(what, "a tensor's pointer is NULL"), -1;
        if ((c->dtype != DRONE_F32) != (t.master != nullptr)) return fail(what, "16-bit tensors need a 32-bit master, DRONE_F32 ones have none"), -1;
        if (odd(t.param, m) || odd(t.grad, m) || odd(t.exp_avg, 3) || odd(t.exp_avg_sq, 3) || odd(t.master, 3)) return fail(what, "a pointer is not aligned to its elements"), -1;
    }
    if (!c->workspace || odd(c->workspace, 15) || c->workspace_bytes < drone_adamw_workspace(c)) return fail(what, "drone_adamw_workspace bytes are needed, 16-byte aligned"), -1;
    OnDevice dev(c->device);
    if (!dev.ok) return -1;
    const hipStream_t s = (hipStream_t)stream;
    const bool clip = c->max_grad_norm > 0;
    AdamwArgs a = {};
    a.partial = (float*)c->workspace;
    a.norm = c->grad_norm;
    a.step = c->step;
    a.lr = (float)c->lr; a.decay = (float)(1.0 - c->lr * c->weight_decay);
    a.b1 = (float)c->beta1; a.b2 = (float)c->beta2; a.rest1 = (float)(1.0 - c->beta1); a.rest2 = (float)(1.0 - c->beta2);
    a.log_b1 = (float)std::log(c->beta1); a.log_b2 = (float)std::log(c->beta2);  // (beta 0: -inf, and the correction is 1)
    a.eps = (float)c->eps; a.max_norm = clip ? (float)c->max_grad_norm : 0.f;
    const bool norm = clip || c->grad_norm;  // the norm is also reported without a clip
    if (fill_adamw(c, 0, &a) == c->count && a.chunks <= kAdamwSmall) return launched(adamw_small_launch(c->dtype, a, s), what);
    int parts = 0, rc = 0;
    for (int from = 0; from < c->count || from == 0;) {
        from += from < c->count ? fill_adamw(c, from, &a) : 0;
        const int blocks = norm ? adamw_parts(a) : 0;
        a.part0 = parts;
        a.parts = blocks;
        a.advance = parts == 0;
        if (blocks || a.advance) rc = adamw_norm_launch(c->dtype, a, blocks ? blocks : 1, s);
        if (rc) return launched(rc, what);
        parts += blocks;
        if (!norm || from >= c->count) break;
    }
    a.parts = parts;
    for (int from = 0; from < c->count;) {
        a.advance = from == 0;
        from += fill_adamw(c, from, &a);
        rc = adamw_update_launch(c->dtype, a, s);
        if (rc) return launched(rc, what);
    }
    return 0;
}

}  // extern "C"
