"""The policy operators on real work: what a device-resident learner of the env runs between two env steps.

Three operators of ``drone_amd.policy``: ``linear`` (matrix product with bias, activation and residual; its gradient),
``norm_residual`` (the norms after and before a block with its gate and residual scale; its gradient) and ``adamw_step``
(clip by the global norm and the AdamW update of many tensors). M is the number of envs a batch holds, the widths are a
policy's. Where ``own`` is false the same is computed by elementary torch operations in 32 bits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-6
_ADAM = {"lr": 3e-4, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01, "max_grad_norm": 0.5}


def listed():
    return [
        # one drone flown by a wide policy: a hidden layer for a single row, all latency
        {"name": "act_single", "op": "linear", "m": 1, "k": 512, "n": 512, "type": "bf16", "act": "silu", "res": True, "learn": False, "dx": False},
        # the first layer on the observations of 1 024 envs, the smallest vectorised run
        {"name": "act_obs", "op": "linear", "m": 1024, "k": 20, "n": 64, "type": "f32", "act": "tanh", "res": False, "learn": False, "dx": False},
        # the action head of the 20-64-64-4 policy at 65 536 envs: four outputs a row
        {"name": "act_head", "op": "linear", "m": 65536, "k": 64, "n": 4, "type": "f32", "act": "tanh", "res": False, "learn": False, "dx": False},
        # a residual layer of a middling policy at 262 144 envs: bound by memory
        {"name": "act_torso", "op": "linear", "m": 262144, "k": 256, "n": 256, "type": "bf16", "act": "gelu", "res": True, "learn": False, "dx": False},
        # a layer of a wide policy at 65 536 envs: bound by the matrix cores
        {"name": "act_wide", "op": "linear", "m": 65536, "k": 1024, "n": 1024, "type": "bf16", "act": "relu", "res": False, "learn": False, "dx": False},
        # the hidden layer of the 20-64-64-4 policy, forward and gradient: weight gradients summed over 65 536 rows
        {"name": "learn_small", "op": "linear", "m": 65536, "k": 64, "n": 64, "type": "f32", "act": "tanh", "res": False, "learn": True, "dx": True},
        # a wide residual layer over the batch of one GPU's shard, forward and gradient
        {"name": "learn_wide", "op": "linear", "m": 131072, "k": 512, "n": 512, "type": "bf16", "act": "silu", "res": True, "learn": True, "dx": True},
        # the first layer on a ragged minibatch of 24-float observations: no gradient of the observations
        {"name": "learn_ragged", "op": "linear", "m": 5003, "k": 24, "n": 200, "type": "f16", "act": "gelu", "res": False, "learn": True, "dx": False},
        # the norms around a block while acting with 1 024 envs, one gate for every channel
        {"name": "norm_act", "op": "norm", "m": 1024, "c": 256, "type": "bf16", "gate": "channel", "learn": False},
        # the same while learning from 65 536 rows, a gate for every row and channel
        {"name": "norm_learn", "op": "norm", "m": 65536, "c": 512, "type": "bf16", "gate": "full", "learn": True},
        # the optimizer step of the 20-64-64-4 policy: six tensors, 5 764 weights, all latency
        {"name": "adamw_small", "op": "adamw", "width": 64, "hidden": 1, "obs": 20, "type": "f32"},
        # the optimizer step of a wide policy with 16-bit weights and 32-bit masters, 21 million weights
        {"name": "adamw_wide", "op": "adamw", "width": 2048, "hidden": 5, "obs": 24, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "norm", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind == "linear":
        learn = rng.random() < 0.5
        k, n = _log(rng, 4, 1024), _log(rng, 4, 1024)
        most = 131072 * 512 * 512 if learn else 65536 * 1024 * 1024
        most = most // 4 if dtype == "f32" else most  # 32-bit products cost more than the listed 16-bit ones
        m = _log(rng, 1, max(2, min(262144, most // (k * n))))
        return {"op": "linear", "m": m, "k": k, "n": n, "type": dtype, "act": rng.choice(["none", "relu", "tanh", "silu", "gelu"]),
                "res": rng.random() < 0.5, "learn": learn, "dx": learn and rng.random() < 0.7}
    if kind == "norm":
        c = _log(rng, 8, 2048)
        return {"op": "norm", "m": _log(rng, 1, min(131072, 65536 * 512 // c)), "c": c, "type": dtype,
                "gate": rng.choice(["none", "channel", "full"]), "learn": rng.random() < 0.6}
    return {"op": "adamw", "width": _log(rng, 16, 1500), "hidden": rng.randint(1, 5), "obs": rng.choice([20, 24]), "type": dtype}


def _shapes(case):
    w, shapes = case["width"], [(case["width"], case["obs"]), (case["width"],)]
    for _ in range(case["hidden"]):
        shapes += [(w, w), (w,)]
    return shapes + [(4, w), (4,)]


def prepare(case, seed):
    t = _TYPES[case["type"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, of=1.0, to=t):
        return (torch.randn(shape, device="cuda", generator=gen) * of).to(to)

    s = dict(case)
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = normal(m, k)
        s["w"] = normal(n, k, of=k ** -0.5)
        s["b"] = normal(n, of=0.1)
        s["residual"] = normal(m, n) if case["res"] else None
        if case["learn"]:
            s["dy"] = normal(m, n, of=m ** -0.5)
            s["leaves"] = [s["w"], s["b"]] + ([s["x"]] if case["dx"] else []) + ([s["residual"]] if case["res"] else [])
            for a in s["leaves"]:
                a.requires_grad_(True)
    elif case["op"] == "norm":
        m, c = case["m"], case["c"]
        s["x"], s["block"] = normal(m, c), normal(m, c, of=3.0)
        s["gate"] = None if case["gate"] == "none" else normal(m, c) if case["gate"] == "full" else normal(c)
        s["post"], s["pre"] = (1 + 0.1 * normal(c, to=torch.float32)).to(t), (1 + 0.1 * normal(c, to=torch.float32)).to(t)
        s["scale"] = 0.5
        if case["learn"]:
            s["dr"], s["dh"] = normal(m, c, of=m ** -0.5), normal(m, c, of=m ** -0.5)
            s["leaves"] = [s["x"], s["block"], s["post"], s["pre"]] + ([s["gate"]] if s["gate"] is not None else [])
            for a in s["leaves"]:
                a.requires_grad_(True)
    else:  # a run in its 100th update: moments that earlier gradients left
        shapes = _shapes(case)
        s["masters"] = [normal(*d, of=d[-1] ** -0.5, to=torch.float32) for d in shapes]
        s["params"] = [p.to(t) for p in s["masters"]] if t != torch.float32 else s["masters"]
        s["grads"] = [normal(*d, of=1e-2) for d in shapes]
        s["exp_avgs"] = [normal(*d, of=1e-3, to=torch.float32) for d in shapes]
        s["exp_avg_sqs"] = [normal(*d, of=1e-3, to=torch.float32).square() + 1e-8 for d in shapes]
        s["step"] = torch.full((1,), 100, dtype=torch.int32, device="cuda")
    return s


def _slope_and_value(z, act):
    """act(z) and its derivative, in 32 bits."""
    if act == "relu":
        on = (z > 0).float()
        return z * on, on
    if act == "tanh":
        a = torch.tanh(z)
        return a, 1 - a * a
    if act == "silu":
        g = 1 / (1 + torch.exp(-z))
        return z * g, g * (1 + z * (1 - g))
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    return z, torch.ones_like(z)


def _linear(s):
    if own:
        from drone_amd import policy

        y = policy.linear(s["x"], s["w"], s["b"], activation=s["act"], residual=s["residual"])
        return [y, *torch.autograd.grad(y, s["leaves"], s["dy"])] if s["learn"] else y
    t = s["x"].dtype
    with torch.no_grad():
        x, w = s["x"].float(), s["w"].float()
        z = x @ w.t() + s["b"].float()
        a, slope = _slope_and_value(z, s["act"])
        y = (a + s["residual"].float() if s["res"] else a).to(t)
        if not s["learn"]:
            return y
        dz = s["dy"].float() * slope
        grads = [dz.t() @ x, dz.sum(0)] + ([dz @ w] if s["dx"] else []) + ([s["dy"]] if s["res"] else [])
        return [y, *(g.to(t) for g in grads)]


def _norm_grad(a, rms, g):
    """The gradient of a / rms with respect to a, for the gradient g of the quotient."""
    n = a / rms
    return (g - n * (g * n).mean(1, keepdim=True)) / rms


def _norm(s):
    if own:
        from drone_amd import policy

        r, h = policy.norm_residual(s["x"], s["block"], gate=s["gate"], scale=s["scale"], post_weight=s["post"], pre_weight=s["pre"], eps=_EPS)
        return [r, h, *torch.autograd.grad([r, h], s["leaves"], [s["dr"], s["dh"]])] if s["learn"] else [r, h]
    t, scale = s["x"].dtype, s["scale"]
    with torch.no_grad():
        x, block, post, pre = s["x"].float(), s["block"].float(), s["post"].float(), s["pre"].float()
        gate = torch.ones_like(post) if s["gate"] is None else 1 / (1 + torch.exp(-s["gate"].float()))
        rms_b = torch.sqrt((block * block).mean(1, keepdim=True) + _EPS)
        nb = block / rms_b
        r = x + scale * gate * (nb * post)
        rms_r = torch.sqrt((r * r).mean(1, keepdim=True) + _EPS)
        nr = r / rms_r
        out = [r.to(t), (nr * pre).to(t)]
        if not s["learn"]:
            return out
        dh = s["dh"].float()
        d = s["dr"].float() + _norm_grad(r, rms_r, dh * pre)
        u = d * scale * gate
        grads = [d, _norm_grad(block, rms_b, u * post), (u * nb).sum(0), (dh * nr).sum(0)]
        if s["gate"] is not None:
            dgate = d * scale * (nb * post) * gate * (1 - gate)
            grads.append(dgate.sum(0) if s["gate"].dim() == 1 else dgate)
        return out + [g.to(t) for g in grads]


def _adamw(s):
    half = s["params"][0].dtype != torch.float32
    (b1, b2), lr = _ADAM["betas"], _ADAM["lr"]
    if own:
        from drone_amd import policy

        norm = policy.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["step"], masters=s["masters"] if half else None, **_ADAM)
    else:
        s["step"] += 1
        t = s["step"].double()
        c1, c2 = (1 - b1 ** t).float(), (1 - b2 ** t).float()
        norm = torch.sqrt(torch.stack([g.float().square().sum() for g in s["grads"]]).sum()).reshape(1)
        clip = torch.clamp(_ADAM["max_grad_norm"] / (norm + 1e-6), max=1.0)
        for p, master, g, m, v in zip(s["params"], s["masters"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"]):
            g = g.float() * clip
            m.mul_(b1).add_(g * (1 - b1))
            v.mul_(b2).add_(g * g * (1 - b2))
            master.mul_(1 - lr * _ADAM["weight_decay"]).sub_(lr * (m / c1) / (torch.sqrt(v / c2) + _ADAM["eps"]))
            if half:
                p.copy_(master)
    return [norm, s["params"], s["exp_avgs"], s["exp_avg_sqs"], s["masters"] if half else []]


def run(s):
    return {"linear": _linear, "norm": _norm, "adamw": _adamw}[s["op"]](s)


def work(case):
    e = _BYTES[case["type"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        values = m * k + n * k + n + m * n * (2 if case["res"] else 1)  # x, w, b, the residual; y
        if case["learn"]:
            values += m * n + n * k + n + (m * k if case["dx"] else 0)  # dy; dw, db, dx (the residual's gradient is dy itself)
        return {"bytes": e * values, "flops": 2 * m * k * n * (1 + (1 + case["dx"] if case["learn"] else 0))}
    if case["op"] == "norm":
        m, c = case["m"], case["c"]
        gate = {"none": 0, "channel": c, "full": m * c}[case["gate"]]
        values = 4 * m * c + gate + 2 * c  # x, block, the gate; r, h; the weights
        if case["learn"]:
            values += 4 * m * c + gate + 2 * c  # dr, dh; dx, dblock, the gate's and the weights' gradients
        return {"bytes": e * values, "flops": m * c * (60 if case["learn"] else 20)}
    count = sum(math.prod(d) for d in _shapes(case))
    return {"bytes": count * (6 * 4 + e + (e if e < 4 else 0)), "flops": 16 * count}  # 32-bit weight and moments in and out; the gradient; the 16-bit weight


def exact(case, seed):
    """The same from the definitions in 64 bits: torch's own layers, differentiated by autograd, and its optimizer."""
    s = prepare(case, seed)

    def wide(a):
        return None if a is None else a.detach().double().requires_grad_(True)

    if case["op"] == "linear":
        x, w, b, residual = (wide(s[a]) for a in ("x", "w", "b", "residual"))
        f = torch.nn.functional
        act = {"none": lambda z: z, "relu": f.relu, "tanh": torch.tanh, "silu": f.silu, "gelu": f.gelu}[case["act"]]
        y = act(f.linear(x, w, b))
        y = y if residual is None else y + residual
        if not case["learn"]:
            return y.detach()
        leaves = [w, b] + ([x] if case["dx"] else []) + ([residual] if case["res"] else [])
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"].double())]
    if case["op"] == "norm":
        x, block, gate, post, pre = (wide(s[a]) for a in ("x", "block", "gate", "post", "pre"))
        norm = lambda a, w: torch.nn.functional.rms_norm(a, (case["c"],), w, _EPS)  # noqa: E731
        after = norm(block, post) if gate is None else torch.sigmoid(gate) * norm(block, post)
        r = x + s["scale"] * after
        h = norm(r, pre)
        if not case["learn"]:
            return [r.detach(), h.detach()]
        leaves = [x, block, post, pre] + ([gate] if gate is not None else [])
        return [r.detach(), h.detach(), *torch.autograd.grad([r, h], leaves, [s["dr"].double(), s["dh"].double()])]
    params = [wide(p) for p in s["masters"]]
    opt = torch.optim.AdamW(params, lr=_ADAM["lr"], betas=_ADAM["betas"], eps=_ADAM["eps"], weight_decay=_ADAM["weight_decay"], foreach=False)
    for p, g, m, v in zip(params, s["grads"], s["exp_avgs"], s["exp_avg_sqs"]):
        p.grad = g.double()
        opt.state[p] = {"step": torch.tensor(100.0), "exp_avg": m.double(), "exp_avg_sq": v.double()}
    norm = torch.nn.utils.clip_grad_norm_(params, _ADAM["max_grad_norm"], foreach=False)
    opt.step()
    params = [p.detach() for p in params]
    half = case["type"] != "f32"
    return [norm.reshape(1), params, [opt.state[p]["exp_avg"] for p in opt.state], [opt.state[p]["exp_avg_sq"] for p in opt.state], params if half else []]
