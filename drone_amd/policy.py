"""A policy beside the env, on the GPU it lives on: its layers, their gradients, the optimizer step.

The env's observations, rewards and flags stay in HBM (``DroneVec`` with a device); what a learner runs between two env
steps are many-row, narrow layers and an update of a dozen small tensors, where launches and passes over memory are the
cost. Three operators over the C-ABI of ``include/drone_vec.h``, on torch's current stream; a forward call is one launch, the
gradient of norms one or two, that of a layer two (narrow) to six (odd widths), the optimizer step one or two:

* ``linear``: ``y = act(x W^T + b) + residual`` (``drone_linear_forward`` / ``_backward``)
* ``norm_residual``: the norms after and before a block, its gate and residual scale (``drone_norm_forward`` / ``_backward``)
* ``adamw_step``: clip by the global gradient norm and the AdamW update of all tensors (``drone_adamw_step``)

and over them ``Linear``, ``Policy`` and ``AdamW`` for torch programs. Tensors are float32, bfloat16 or float16 on one GPU;
sums, statistics and moments are held in 32 bits. There is no CPU path. Every call can be captured into a graph; a captured
backward pass is refused where a graph built on the default stream still holds one of its leaves (an eager loss: let go of
it). The reference snapshot holds no policy or trainer source to cite (``/root/reference/.gitmodules:1-3``).
"""
import ctypes as C

import torch

from . import abi, binding

_native_module = None


def _native():
    """The compiled module over the C-ABI (bindings/policy_torch.cpp), given the loaded library's entry points on first use."""
    global _native_module
    if _native_module is None:
        lib = binding.load()
        try:
            from . import policy_torch
        except ImportError as e:
            raise RuntimeError("drone_amd/policy_torch is missing or does not load: build it first "
                               f"(python -c 'import __graft_entry__ as g; g.build()' or make -C bindings policy): {e}") from e
        names = [n for n in abi.SYMBOLS if n.startswith(("drone_linear", "drone_norm", "drone_adamw"))] + ["drone_last_error"]
        policy_torch.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in names})
        _native_module = policy_torch
    return _native_module


def linear(x, weight, bias=None, activation="none", residual=None, out=None):
    """``act(x @ weight.T + bias) + residual`` in one launch, differentiable (once, backward) in all four.

    x ``[..., in]``, weight ``[out, in]``, bias ``[out]``, residual ``[..., out]``, one type (float32, bfloat16, float16)
    and one GPU; activation: none, relu, tanh, silu, gelu (the erf form). Sums are 32-bit, the result is rounded once; calls of
    one shape give the same bits, another number of rows may sum in another order. The gradient rounds dy act'(z) to the type
    once more for its products: 16-bit dx and dweight are 1.4 times as far off as their own rounding.
    ``out``: a tensor to write instead of a new one (the env's action buffer), ``[..., out]`` with contiguous rows; only
    where nothing is differentiated; it may be the residual. Rows may be a strided view; anything else is copied first."""
    return _native().linear(x, weight, bias, activation, residual, out)


def norm_residual(x, block=None, *, gate=None, scale=1.0, post_weight=None, pre_weight=None, eps=1e-6):
    """The norms around a residual block in one pass: ``(r, h)`` with

        r = x + scale * sigmoid(gate) * (n(block) * post_weight)        n(a) = a / sqrt(mean(a^2) + eps)
        h = n(r) * pre_weight

    ``r`` is the residual stream behind the block, ``h`` what the next block reads. x, block ``[..., width]``; gate
    ``[width]`` or ``[..., width]`` or None (1); weights ``[width]`` or None (1); width 1 ... 4096. Without a block
    ``r = x``. Differentiable (once, backward) in all five tensors; scale and eps are numbers."""
    return _native().norm_residual(x, block, gate, scale, post_weight, pre_weight, eps)


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_grad_norm=None, masters=None):
    """One AdamW step over all tensors, in place, two launches (one where all tensors together are a few thousand values);
    returns the gradients' global norm before clipping (``[1]`` float32 on the device). ``max_grad_norm`` (positive): scale
    the gradients by ``min(1, max_grad_norm / (norm + 1e-6))``.

    params and grads of one type; exp_avgs, exp_avg_sqs float32; 16-bit params need float32 ``masters`` (the params are
    their rounded copies; a value that is not has been written since, and the step starts from it). ``step``: int32 tensor
    ``[1]`` on the device, the steps done so far; the call adds 1, so a step captured into a graph replays with an advancing
    count. All tensors contiguous, on one GPU, none twice or over another."""
    return _native().adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay, max_grad_norm, masters)


def _check_parameter(p):
    if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"a parameter is {p.dtype}: float32, bfloat16 or float16")
    if p.device.type != "cuda":
        raise ValueError(f"a parameter is on {p.device}: the policy operators run on a GPU only")
    if not p.is_contiguous():
        raise ValueError("parameters must be contiguous")


class AdamW(torch.optim.Optimizer):
    """``adamw_step`` as a torch optimizer: one parameter group's tensors of one type per step call, moments and (for 16-bit
    parameters) masters in float32. Weights may be written between steps (a loaded state, a target network's copy): the next
    step starts from what is there. ``max_grad_norm`` clips by the norm over a whole group; ``grad_norm`` holds the last
    step's norms, one ``[1]`` tensor per group (None where no parameter had a gradient). Parameters without a gradient are
    left alone; the step count is the group's. ``lr`` and the rest are read at every call (a captured step keeps those of
    its capture)."""

    def __init__(self, params, lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_grad_norm=None):
        if lr < 0 or weight_decay < 0 or not eps > 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr and weight_decay must not be negative, eps must be positive, betas in [0, 1)")
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError("max_grad_norm must be positive (None: no clipping)")
        self.grad_norm = []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_grad_norm=max_grad_norm))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            for p in group["params"]:
                _check_parameter(p)
            if len({p.dtype for p in group["params"]}) != 1 or len({p.device for p in group["params"]}) != 1:
                raise ValueError("the parameters of a group must have one type and one device")
        except Exception:
            self.param_groups.pop()
            raise
        group["step"] = torch.zeros(1, dtype=torch.int32, device=group["params"][0].device)
        for p in group["params"]:
            self.state[p] = {"exp_avg": torch.zeros(p.shape, dtype=torch.float32, device=p.device), "exp_avg_sq": torch.zeros(p.shape, dtype=torch.float32, device=p.device)}
            if p.dtype != torch.float32:
                self.state[p]["master"] = p.detach().float()

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch's, but moments and masters stay float32 (torch would cast them to a 16-bit parameter's type) and keep
        their addresses, so that a captured step goes on from the loaded state."""
        mine = {p: self.state[p] for g in self.param_groups for p in g["params"]}
        steps = [g["step"] for g in self.param_groups]
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        if len(saved) != len(mine) or not all("step" in g for g in state_dict["param_groups"]):
            raise ValueError("the state is not one of these parameter groups")
        for (p, state), i in zip(mine.items(), saved):
            theirs = state_dict["state"].get(i, {})
            if any(k not in theirs or theirs[k].shape != p.shape for k in state):
                raise ValueError(f"the state of parameter {i} is not {', '.join(state)} of shape {tuple(p.shape)}")
        super().load_state_dict(state_dict)
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
                self.grad_norm.append(None)
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
