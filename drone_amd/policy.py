"""A policy beside the env, on the GPU it lives on: its layers, their gradients, the optimizer step.

The env's observations, rewards and flags stay in HBM (``DroneVec`` with a device); what a learner runs between two env
steps are many-row, narrow layers and an update of a dozen small tensors, where launches and passes over memory are the
cost. Three operators over the C-ABI of ``include/drone_vec.h``, each one or two launches on torch's current stream:

* ``linear``: ``y = act(x W^T + b) + residual`` (``drone_linear_forward`` / ``_backward``)
* ``norm_residual``: the norms after and before a block, its gate and residual scale (``drone_norm_forward`` / ``_backward``)
* ``adamw_step``: clip by the global gradient norm and the AdamW update of all tensors (``drone_adamw_step``)

and over them ``Linear``, ``Policy`` and ``AdamW`` for torch programs. Tensors are float32, bfloat16 or float16 on one GPU;
sums, statistics and moments are held in 32 bits. There is no CPU path. The reference snapshot holds no policy or trainer
source to cite (``/root/reference/.gitmodules:1-3``).
"""
import ctypes as C

import torch

from . import abi, binding

_DTYPES = {torch.float32: abi.F32, torch.bfloat16: abi.BF16, torch.float16: abi.F16}


def _fail(what):
    raise RuntimeError(f"libdrone_hip: {binding.last_error() or what}")


def _call(name, blob, device):
    """One C-ABI call on torch's current stream of the device."""
    if binding.functions()[name](blob, torch.cuda.current_stream(device).cuda_stream):
        _fail(name)


def _workspace(name, blob, device):
    return torch.empty(binding.functions()[name](blob), dtype=torch.uint8, device=device)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _check(name, t, shape, like):
    """A tensor argument: its shape, and the type and device of ``like``."""
    if t is None:
        return
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != like.dtype:
        raise TypeError(f"{name} is {t.dtype}, x is {like.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, x on {like.device}")


def _check_x(x, name="x"):
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} is {x.dtype}: float32, bfloat16 or float16")
    if x.device.type != "cuda":
        raise ValueError(f"{name} is on {x.device}: the policy operators run on a GPU only")


def _rows(t):
    """A tensor [..., n] as [rows][n] with contiguous rows and a leading dimension of at least n: a view where there is
    one, else a copy. Overlapping rows (an expanded tensor) are copied."""
    if t is None:
        return None
    n = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, n)
    if (n > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < n):
        t = t.contiguous()
    return t


def _ld(t):
    return 0 if t is None else max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _slope_type(dtype):
    return torch.float16 if dtype == torch.bfloat16 else torch.float32


_LINEAR_SIZE, _NORM_SIZE, _ADAMW_SIZE = abi.LINEAR_CALL.size, abi.NORM_CALL.size, abi.ADAMW_CALL.size


def _linear_forward(x, weight, bias, residual, activation, slope, y=None):
    n, k = weight.shape
    rows = x.shape[0]
    if y is None:
        y = x.new_empty((rows, n))
    _call("drone_linear_forward", abi.LINEAR_CALL.pack(
        _LINEAR_SIZE, x.get_device(), _DTYPES[x.dtype], activation, rows, k, n,
        x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(residual), 0, y.data_ptr(), _ptr(slope), 0, 0, 0,
        _ld(x), _ld(weight), _ld(residual), 0, _ld(y), 0, 0, 0), x.device)
    return y


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        slope = torch.empty((x.shape[0], weight.shape[0]), dtype=_slope_type(x.dtype), device=x.device) if activation else None
        y = _linear_forward(x, weight, bias, residual, activation, slope)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, slope)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, slope = ctx.saved_tensors
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dx = dw = db = work = None
        if want_x or want_w or want_b:
            d = _rows(dy)
            n, k = weight.shape
            if want_x:
                dx = x.new_empty((x.shape[0], k))
            if want_w:
                dw = x.new_empty((n, k))
            if want_b:
                db = x.new_empty(n)

            def blob(work):
                return abi.LINEAR_CALL.pack(
                    _LINEAR_SIZE, x.get_device(), _DTYPES[x.dtype], ctx.activation, x.shape[0], k, n,
                    x.data_ptr(), weight.data_ptr(), 0, 0, d.data_ptr(), 0, _ptr(slope), _ptr(dx), _ptr(dw), _ptr(db),
                    _ld(x), _ld(weight), 0, _ld(d), 0, k, _ptr(work), 0 if work is None else work.numel())

            if want_w or want_b:
                work = _workspace("drone_linear_workspace", blob(None), x.device)
            _call("drone_linear_backward", blob(work), x.device)
        return dx, dw, db, dy if want_r else None, None


def linear(x, weight, bias=None, activation="none", residual=None, out=None):
    """``act(x @ weight.T + bias) + residual`` in one launch, differentiable (once) in all four.

    x ``[..., in]``, weight ``[out, in]``, bias ``[out]``, residual ``[..., out]``, one type (float32, bfloat16, float16)
    and one GPU; activation: none, relu, tanh, silu, gelu (the erf form). Sums are 32-bit, the result is rounded once.
    ``out``: a tensor to write instead of a new one (the env's action buffer), ``[..., out]`` with contiguous rows; only
    where nothing is differentiated. Rows may be a strided view; anything else is copied first."""
    _check_x(x)
    if activation not in abi.ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; one of {', '.join(abi.ACTIVATIONS)}")
    if weight.dim() != 2 or x.dim() < 1:
        raise ValueError(f"weight must be [out, in] and x [..., in], got {tuple(weight.shape)} and {tuple(x.shape)}")
    n, k = weight.shape
    lead = x.shape[:-1]
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} features, the weight takes {k}")
    _check("weight", weight, (n, k), x)
    _check("bias", bias, (n,), x)
    _check("residual", residual, (*lead, n), x)
    _check("out", out, (*lead, n), x)
    act = abi.ACTIVATIONS[activation]
    learn = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))
    if out is not None:
        if learn:
            raise ValueError("out= cannot be differentiated: call under torch.no_grad()")
        o = out if out.dim() == 2 else out.view(-1, n)
        if (n > 1 and o.stride(1) != 1) or (o.shape[0] > 1 and o.stride(0) < n):
            raise ValueError("out must have contiguous rows that do not overlap")
    args = _rows(x), _rows(weight), None if bias is None else bias.contiguous(), _rows(residual), act
    if learn:
        return _LinearFunction.apply(*args).view(*lead, n)
    if out is not None:
        _linear_forward(*args, None, o)
        return out
    return _linear_forward(*args, None).view(*lead, n)


def _norm_blob(x, block, gate, post, pre, scale, eps, dr=None, dh=None, r=None, h=None, grads=(None,) * 5, work=None):
    kind = 0 if gate is None else gate.dim()
    dx, dblock, dgate, dpost, dpre = grads
    return abi.NORM_CALL.pack(
        _NORM_SIZE, x.get_device(), _DTYPES[x.dtype], kind, x.shape[0], x.shape[1],
        x.data_ptr(), _ptr(block), _ptr(gate), _ptr(post), _ptr(pre), _ptr(dr), _ptr(dh),
        _ptr(r), _ptr(h), _ptr(dx), _ptr(dblock), _ptr(dgate), _ptr(dpost), _ptr(dpre),
        _ld(x), _ld(block), _ld(gate) if kind == 2 else 0, scale, eps, _ptr(work), 0 if work is None else work.numel())


def _norm_forward(x, block, gate, post, pre, scale, eps):
    r, h = x.new_empty((x.shape[0], x.shape[1])), x.new_empty((x.shape[0], x.shape[1]))
    _call("drone_norm_forward", _norm_blob(x, block, gate, post, pre, scale, eps, r=r, h=h), x.device)
    return r, h


class _NormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, gate, post, pre, scale, eps):
        ctx.set_materialize_grads(False)
        ctx.numbers = scale, eps
        ctx.save_for_backward(x, block, gate, post, pre)
        return _norm_forward(x, block, gate, post, pre, scale, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dr, dh):
        x, block, gate, post, pre = ctx.saved_tensors
        if dr is None and dh is None:
            return (None,) * 7
        dr, dh = (None if d is None else d.contiguous() for d in (dr, dh))
        grads = [t.new_empty(t.shape) if want else None for t, want in zip((x, block, gate, post, pre), ctx.needs_input_grad)]
        args = (x, block, gate, post, pre, *ctx.numbers, dr, dh, None, None, grads)
        work = _workspace("drone_norm_workspace", _norm_blob(*args), x.device)
        _call("drone_norm_backward", _norm_blob(*args, work), x.device)
        return (*grads, None, None)


def norm_residual(x, block=None, *, gate=None, scale=1.0, post_weight=None, pre_weight=None, eps=1e-6):
    """The norms around a residual block in one pass: ``(r, h)`` with

        r = x + scale * sigmoid(gate) * (n(block) * post_weight)        n(a) = a / sqrt(mean(a^2) + eps)
        h = n(r) * pre_weight

    ``r`` is the residual stream behind the block, ``h`` what the next block reads. x, block ``[..., width]``; gate
    ``[width]`` or ``[..., width]`` or None (1); weights ``[width]`` or None (1); width 1 ... 4096. Without a block
    ``r = x``. Differentiable (once) in all five tensors; scale and eps are numbers."""
    _check_x(x)
    if x.dim() < 1:
        raise ValueError("x must be [..., width]")
    lead, width = x.shape[:-1], x.shape[-1]
    if not 1 <= width <= 4096:
        raise ValueError(f"width must be 1 ... 4096, got {width}")
    _check("block", block, x.shape, x)
    _check("post_weight", post_weight, (width,), x)
    _check("pre_weight", pre_weight, (width,), x)
    if block is None and (gate is not None or post_weight is not None):
        raise ValueError("gate and post_weight belong to a block")
    if gate is not None:
        _check("gate", gate, (width,) if gate.dim() == 1 and x.dim() > 1 else x.shape, x)
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    flat = None if gate is None else gate.contiguous() if gate.dim() == 1 and x.dim() > 1 else _rows(gate)
    args = (_rows(x), _rows(block), flat, None if post_weight is None else post_weight.contiguous(),
            None if pre_weight is None else pre_weight.contiguous(), float(scale), float(eps))
    learn = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, block, gate, post_weight, pre_weight))
    r, h = _NormFunction.apply(*args) if learn else _norm_forward(*args)
    return r.view(*lead, width), h.view(*lead, width)


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_grad_norm=None, masters=None):
    """One AdamW step over all tensors, in place, two launches; returns the gradients' global norm before clipping
    (``[1]`` float32 on the device). ``max_grad_norm``: scale the gradients by ``min(1, max_grad_norm / (norm + 1e-6))``.

    params and grads of one type; exp_avgs, exp_avg_sqs float32; 16-bit params need float32 ``masters`` (the params are
    their rounded copies). ``step``: int32 tensor ``[1]`` on the device, the steps done so far; the call adds 1, so a step
    captured into a graph replays with an advancing count. All tensors contiguous, on one GPU, none twice."""
    params = list(params)
    if not params:
        raise ValueError("no parameters")
    first = params[0]
    _check_x(first, "params[0]")
    lists = [("grads", grads, first.dtype), ("exp_avgs", exp_avgs, torch.float32), ("exp_avg_sqs", exp_avg_sqs, torch.float32)]
    if (masters is None) == (first.dtype != torch.float32):
        raise ValueError("16-bit params need float32 masters, float32 params have none")
    if masters is not None:
        lists.append(("masters", masters, torch.float32))
    seen = set()
    for name, tensors, dtype in [("params", params, first.dtype), *lists]:
        if len(tensors) != len(params):
            raise ValueError(f"{len(tensors)} {name} for {len(params)} params")
        for t, p in zip(tensors, params):
            if t.dtype != dtype or t.device != first.device or t.shape != p.shape or not t.is_contiguous():
                raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {tuple(p.shape)} on {first.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
            if t.numel() and t.data_ptr() in seen:
                raise ValueError(f"{name}: a tensor is there twice")
            seen.add(t.data_ptr())
    if step.dtype != torch.int32 or step.numel() != 1 or step.device != first.device:
        raise ValueError("step must be an int32 tensor of one element on the params' device")
    pack = abi.ADAMW_TENSOR.pack
    table = b"".join([
        pack(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), _ptr(w), p.numel())
        for p, g, m, v, w in zip(params, grads, exp_avgs, exp_avg_sqs, masters or [None] * len(params))])
    at = C.cast(table, C.c_void_p).value  # the table is read during the call
    norm = torch.empty(1, dtype=torch.float32, device=first.device)

    def blob(work):
        return abi.ADAMW_CALL.pack(
            _ADAMW_SIZE, first.get_device(), _DTYPES[first.dtype], len(params), at, step.data_ptr(), norm.data_ptr(),
            lr, betas[0], betas[1], eps, weight_decay, 0.0 if max_grad_norm is None else max_grad_norm, _ptr(work), 0 if work is None else work.numel())

    work = _workspace("drone_adamw_workspace", blob(None), first.device)
    _call("drone_adamw_step", blob(work), first.device)
    return norm


class AdamW(torch.optim.Optimizer):
    """``adamw_step`` as a torch optimizer: one parameter group's tensors of one type per step call, moments and (for 16-bit
    parameters) masters in float32. ``max_grad_norm`` clips by the norm over a whole group; ``grad_norm`` holds the last
    step's norms, one ``[1]`` tensor per group. Parameters without a gradient are left alone; the step count is the
    group's. ``lr`` and the rest are read at every call (a captured step keeps those of its capture)."""

    def __init__(self, params, lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_grad_norm=None):
        if lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr, eps and weight_decay must not be negative, betas must be in [0, 1)")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError("max_grad_norm must be positive (None: no clipping)")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_grad_norm=max_grad_norm))
        self.grad_norm = []
        for group in self.param_groups:
            if len({p.dtype for p in group["params"]}) != 1 or len({p.device for p in group["params"]}) != 1:
                raise ValueError("the parameters of a group must have one type and one device")
            _check_x(group["params"][0], "a parameter")
            group["step"] = torch.zeros(1, dtype=torch.int32, device=group["params"][0].device)
            for p in group["params"]:
                if not p.is_contiguous():
                    raise ValueError("parameters must be contiguous")
                self.state[p] = {"exp_avg": torch.zeros(p.shape, dtype=torch.float32, device=p.device), "exp_avg_sq": torch.zeros(p.shape, dtype=torch.float32, device=p.device)}
                if p.dtype != torch.float32:
                    self.state[p]["master"] = p.detach().float()

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch's, but moments and masters stay float32 (torch would cast them to a 16-bit parameter's type) and keep
        their addresses, so that a captured step goes on from the loaded state."""
        mine = {p: self.state[p] for g in self.param_groups for p in g["params"]}
        steps = [g["step"] for g in self.param_groups]
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        for (p, state), i in zip(mine.items(), saved):
            for k, v in state.items():
                v.copy_(state_dict["state"][i][k])
            self.state[p] = state
        for g, step in zip(self.param_groups, steps):
            step.copy_(g["step"])
            g["step"] = step

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.grad_norm = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            states = [self.state[p] for p in params]
            masters = [s["master"] for s in states] if params[0].dtype != torch.float32 else None
            self.grad_norm.append(adamw_step(
                params, [p.grad.contiguous() for p in params], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], group["step"],
                lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], max_grad_norm=group["max_grad_norm"], masters=masters))
        return loss


class Linear(torch.nn.Module):
    """``linear`` with its weights: ``act(x W^T + b) (+ residual)``."""

    def __init__(self, in_features, out_features, activation="none", bias=True, device=None, dtype=None):
        super().__init__()
        if activation not in abi.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}; one of {', '.join(abi.ACTIVATIONS)}")
        self.activation = activation
        self.weight = torch.nn.Parameter(torch.empty((out_features, in_features), device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) if bias else None
        torch.nn.init.normal_(self.weight, std=in_features ** -0.5)

    def forward(self, x, residual=None, out=None):
        return linear(x, self.weight, self.bias, self.activation, residual, out)


class Policy(torch.nn.Module):
    """Observations to actions in [-1, 1]: ``obs_dim -> width`` with an activation, ``blocks`` residual blocks, a tanh head
    of four. A block reads the normed stream and adds ``scale * sigmoid(gate) * n(act(W h + b))`` to it, with
    ``norm_residual`` doing both norms; with ``blocks = 0`` hidden layers are plain (``hidden`` of them)."""

    def __init__(self, obs_dim=abi.OBS_DIM, width=64, hidden=1, blocks=0, activation="tanh", scale=0.5, device=None, dtype=None):
        super().__init__()
        kw = dict(device=device, dtype=dtype)
        self.first = Linear(obs_dim, width, activation, **kw)
        self.hidden = torch.nn.ModuleList(Linear(width, width, activation, **kw) for _ in range(0 if blocks else hidden))
        self.blocks = torch.nn.ModuleList(Linear(width, width, activation, **kw) for _ in range(blocks))
        self.head = Linear(width, abi.ACT_DIM, "tanh", **kw)
        self.scale = scale
        ones = lambda n: torch.nn.ParameterList(torch.nn.Parameter(torch.ones(width, **kw)) for _ in range(n))  # noqa: E731
        self.post, self.pre = ones(blocks), ones(blocks + 1 if blocks else 0)
        self.gates = torch.nn.ParameterList(torch.nn.Parameter(torch.zeros(width, **kw)) for _ in range(blocks))

    def forward(self, obs, out=None):
        """``out``: the action tensor to write (float32 policies; under ``torch.no_grad``)."""
        dtype = self.head.weight.dtype
        h = self.first(obs if obs.dtype == dtype else obs.to(dtype))
        for layer in self.hidden:
            h = layer(h)
        if len(self.blocks):
            r, h = norm_residual(h, pre_weight=self.pre[0])
            for layer, post, gate, pre in zip(self.blocks, self.post, self.gates, list(self.pre)[1:]):
                r, h = norm_residual(r, layer(h), gate=gate, scale=self.scale, post_weight=post, pre_weight=pre)
        if out is not None and out.dtype != dtype:
            return out.copy_(self.head(h))
        return self.head(h, out=out)
