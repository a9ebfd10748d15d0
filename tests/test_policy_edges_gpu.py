"""The policy operators at the edges of what they allow: calls that the other tests do not make, each against 64-bit
formulas, against the same work done another way, or refused."""
import math
import os
import subprocess
import sys

import pytest
import torch

from drone_amd import policy
from test_policy_gpu import HYPER, MLP, TINY, TYPES, U32, adamw_case, check_linear, check_norm, close, half_step, linear_case, norm_case, rand, step

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("m", [1, 3, 33, 65])
@pytest.mark.parametrize("c", [24, 200, 1500])
def test_norm_without_eps(t, gate, eps, m, c):
    """eps = 0 (and one that 32 bits round to 0) for rows that are not zero: threads behind the last row, of which every
    width class has some at these row counts, add nothing to the sums over the rows."""
    check_norm(*norm_case(m, c, t, gate), 0.5, eps, f"{m}x{c} {gate} eps={eps}")


@pytest.mark.parametrize("t", TYPES)
def test_a_graph_from_before_the_step_is_refused(t):
    """adamw_step writes in place: a backward pass through a graph that saved the old weights has to fail, as it does with
    torch's own optimizers, and not to take the new ones."""
    x, w, b, _, dy = linear_case(50, 24, 32, t, "tanh", res=False)
    y = policy.linear(x, w, b, "tanh")
    r, h = policy.norm_residual(y, pre_weight=b)
    opt = policy.AdamW([w, b], lr=1e-2)
    w.grad, b.grad = torch.ones_like(w), torch.ones_like(b)
    written = [w, b, opt.param_groups[0]["step"]] + [v for p in (w, b) for v in opt.state[p].values()]
    before = [v._version for v in written]
    read = (w.grad._version, b.grad._version)
    opt.step()
    assert all(v._version > n for v, n in zip(written, before)) and (w.grad._version, b.grad._version) == read
    for out in (y, h):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward(torch.ones_like(out), retain_graph=True)
    again = policy.linear(x, w, b, "tanh")  # a graph built after it goes through
    torch.autograd.grad(again, [x, w, b], dy)


@pytest.mark.parametrize("t", TYPES)
def test_out_into_a_saved_tensor_is_refused(t):
    x, w, b, _, dy = linear_case(50, 24, 32, t, "none", res=False)
    saved = x.detach().clone()
    y = policy.linear(saved, w, b)
    with torch.no_grad():
        policy.linear(saved.new_ones(50, 8), saved.new_ones(24, 8), out=saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    with torch.inference_mode():  # tensors that keep no version are written all the same
        free = torch.zeros(50, 32, dtype=t, device="cuda")
        assert torch.equal(policy.linear(x, w, b, out=free), policy.linear(x, w, b))


def test_collected_blocks_are_written_again(hip):
    """collect reuses its blocks and writes the env's buffers: graphs that saved either are refused after the next call."""
    from drone_amd.env import Drone

    env = Drone(num_envs=300, device="cuda:0", seed=3, log_interval=0)
    env.reset(3)
    net = policy.Policy(width=32, device="cuda:0")
    blocks = env.collect(net, 3)
    versions = [b._version for b in blocks[:5]] + [v._version for v in (env.observations, env.actions, env.rewards, env.terminals, env.truncations)]
    of_block, of_now = net(blocks[0]), net(env.observations)
    env.collect(net, 3)
    after = [b._version for b in blocks[:5]] + [v._version for v in (env.observations, env.actions, env.rewards, env.terminals, env.truncations)]
    assert all(n > v for n, v in zip(after, versions))
    for y in (of_block, of_now):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    env.close()


def test_out_that_autograd_knows_is_refused():
    x, w = rand(6, 8, seed=1), rand(5, 8, seed=2)
    leaf = torch.zeros(6, 5, device="cuda", requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="out= cannot be differentiated"):
            policy.linear(x, w, out=out)
    with torch.no_grad():
        policy.linear(x, w, out=leaf)
    assert torch.equal(leaf, policy.linear(x, w))


def test_forward_mode_and_tracing_are_refused():
    """Neither has a formula here: a dual tensor's tangent, or a traced call, would vanish without a word."""
    import torch.autograd.forward_ad as fwd

    x, w, b, r, _ = (v.detach() for v in linear_case(6, 8, 5, torch.float32, "tanh"))
    n = r.shape[1]
    with fwd.dual_level():
        for at in range(4):
            for grad in (False, True):
                a = [v.clone().requires_grad_(grad) for v in (x, w, b, r)]
                a[at] = fwd.make_dual(a[at], torch.ones_like(a[at]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    policy.linear(a[0], a[1], a[2], "tanh", a[3])
        for at in range(5):
            for grad in (False, True):
                a = [v.clone().requires_grad_(grad) for v in (r, r, r, b, b)]
                a[at] = fwd.make_dual(a[at], torch.ones_like(a[at]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    policy.norm_residual(a[0], a[1], gate=a[2], post_weight=a[3], pre_weight=a[4])
    assert n == 5
    for f in (lambda v: policy.linear(v, w, b), lambda v: policy.norm_residual(v)[0], lambda v: policy.linear(v, w, b, out=torch.empty(6, 5, device="cuda"))):
        with pytest.raises(RuntimeError, match="trac"):
            torch.jit.trace(f, (x,), check_trace=False)
    s = adamw_case([(4,)], torch.float32)

    def traced(v):
        policy.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], lr=1e-3)
        return v + 1

    with pytest.raises(RuntimeError, match="trac"):
        torch.jit.trace(traced, (x,), check_trace=False)
    for transform in (lambda: torch.func.jvp(lambda v: policy.linear(v, w, b), (x,), (x,)), lambda: torch.func.vmap(lambda v: policy.linear(v, w, b))(x.view(2, 3, 8)),
                      lambda: torch.func.grad(lambda v: policy.linear(v, w, b).sum())(x)):
        with pytest.raises(RuntimeError):
            transform()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shapes", [MLP, [(300, 257), (129, 513), (5,)]])
def test_weights_written_between_steps_are_kept(t, shapes):
    """A weight written after the optimizer was built (a loaded state, a re-initialised layer, a target network's copy) is
    what the next step starts from, one element or all of them; the untouched ones keep their 32-bit masters."""
    ps = [torch.nn.Parameter(rand(*d, to=t, seed=i)) for i, d in enumerate(shapes)]
    opt = policy.AdamW(ps, lr=1e-2, weight_decay=0.0)
    for k, p in enumerate(ps):
        p.grad = rand(*p.shape, to=t, of=0.1, seed=50 + k)
    opt.step()
    masters = [(opt.state[p]["master"] if t != torch.float32 else p.detach()).clone() for p in ps]
    with torch.no_grad():
        ps[0].copy_(rand(*ps[0].shape, to=t, seed=90))
        ps[1][1] = -3.0
    # (a written value that the master rounds to cannot be told from the old one: the master is it, to the type's precision)
    starts = [torch.where(masters[0].to(t) == ps[0], masters[0], ps[0].float()).detach(), masters[1].clone(), *masters[2:]]
    starts[1][1] = -3.0
    twins = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = policy.AdamW(twins, lr=1e-2, weight_decay=0.0)
    other.load_state_dict(opt.state_dict())
    for p, q, s in zip(ps, twins, starts):
        q.grad = p.grad
        if t != torch.float32:
            other.state[q]["master"].copy_(s)
    opt.step()
    other.step()
    for p, q in zip(ps, twins):
        assert torch.equal(p, q)
        if t != torch.float32:
            assert torch.equal(opt.state[p]["master"], other.state[q]["master"]) and torch.equal(p, opt.state[p]["master"].to(t))
    assert (ps[0].detach().float() - starts[0]).abs().max().item() <= 1.1e-2 + half_step(t) * 5  # a step of lr, and its rounding


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_weights_written_between_replays_are_kept(t):
    """The same for a captured step, which no Python runs before."""
    p = torch.nn.Parameter(rand(40, 30, to=t, seed=1))
    p.grad = rand(40, 30, to=t, seed=2)
    opt = policy.AdamW([p], lr=1e-3, weight_decay=0.0)
    opt.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    for k in range(3):
        loaded = rand(40, 30, to=t, seed=10 + k)
        with torch.no_grad():
            p.copy_(loaded)
        g.replay()
        torch.cuda.synchronize()
        # a step of lr, from a start that is the loaded value or rounds to it: within half a step of the type of it
        over = (opt.state[p]["master"].double() - loaded.double()).abs() - 1.1e-3 - half_step(t) * loaded.double().abs()
        assert over.max().item() <= 0 and torch.equal(p, opt.state[p]["master"].to(t))
        assert not torch.equal(opt.state[p]["master"], loaded.float())
    assert opt.param_groups[0]["step"].item() == 4


def diagonal(m, n, t, z):
    """A layer whose z is its x: the unit weight, no bias; the rows hold the values of z in turn."""
    x = z[torch.arange(m * n, device="cuda") % z.numel()].view(m, n).to(t)
    return x.requires_grad_(True), torch.eye(n, device="cuda").to(t).requires_grad_(True)


FORMS = [(5, 64), (333, 65), (5000, 64), (9001, 100), (66001, 256), (20001, 333)]  # few rows, tiled, one pass, odd widths, streamed


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m, n", FORMS + [(270001, 64)])
def test_linear_tanh_near_zero(t, m, n):
    """tanh of small z, relative to itself: the rounding to the type and 2e-6 (a dozen 32-bit operations)."""
    z = torch.logspace(-8, -0.5, 41, device="cuda")
    x, w = diagonal(m, n, t, torch.cat([z, -z]))
    with torch.no_grad():
        y = policy.linear(x, w, None, "tanh")
    want = torch.tanh(x.detach().double())
    close(y, want, want.abs() * (half_step(t) + 2e-6) + TINY[t], f"{m}x{n}")


@pytest.mark.parametrize("shapes", [MLP, [(300, 257), (129, 513)]])
def test_adamw_of_denormal_moments(shapes):
    """Gradients of 1e-20 and an eps below them: v is a denormal number and counts all the same. Against the formula on the
    moments as they were stored: a few 2^-24 of the step, and half a step of a denormal v / (1 - b2^t) around 1e-40 (2e-5)."""
    s = adamw_case(shapes, torch.float32, zero=True)
    for g in s["grads"]:
        g.copy_(torch.where(g >= 0, 1e-20, -1e-20))
    before = [p.double() for p in s["masters"]]
    step(s, eps=1e-30, weight_decay=0.0)
    (b1, b2), lr = HYPER["betas"], HYPER["lr"]
    for p, q, m, v in zip(s["masters"], before, s["m"], s["v"]):
        assert 0 < v.max().item() < 2.0 ** -126
        move = lr * (m.double() / (1 - b1)) / (torch.sqrt(v.double() / (1 - b2)) + 1e-30)
        close(p, q - move, 1e-4 * move.abs() + 2 * U32 * q.abs(), "p")


@pytest.mark.parametrize("t", [torch.bfloat16])
def test_linear_weight_gradient_of_a_very_wide_layer(t):
    """2^29 weights: more joins than one launch has threads for."""
    n, k = 32768, 16384
    x, dy = rand(2, k, to=t, seed=1), rand(2, n, to=t, seed=2)
    w = torch.zeros(n, k, dtype=t, device="cuda").requires_grad_(True)
    b = torch.zeros(n, dtype=t, device="cuda").requires_grad_(True)
    dw, db = torch.autograd.grad(policy.linear(x, w, b), [w, b], dy)
    close(db, dy.double().sum(0), dy.double().abs().sum(0) * (half_step(t) + 2 * U32) + TINY[t], "db")
    for at in range(0, n, 4096):
        d = dy[:, at:at + 4096].double()
        close(dw[at:at + 4096], d.t() @ x.double(), d.abs().t() @ x.double().abs() * (half_step(t) + 4 * U32) + TINY[t], f"dw {at}")


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m, k, n", [(66001, 520, 264), (66001, 1032, 520), (66001, 264, 520), (66001, 261, 523)])
def test_linear_wide_streaming_form(t, m, k, n):
    """Sizes at which 256 x 256 tiles stream, forward (reductions over 1 KiB a row) and input gradient (264 and 261 by 520
    and more), with a last row tile, feature tile and reduction step that are not whole; the last pair is laid out first."""
    check_linear(*linear_case(m, k, n, t, "silu"), "silu", f"{m}x{k}x{n}")


def test_linear_computes_only_what_a_backward_pass_asks_for():
    """autograd.grad for some of the leaves: the others' gradients are neither allocated nor computed."""
    m, k, n = 20000, 512, 64
    x, w, b, _, dy = linear_case(m, k, n, torch.float32, "tanh", res=False)
    full = torch.autograd.grad(policy.linear(x, w, b, "tanh"), [x, w, b], dy)
    for asked in ((1,), (2,), (1, 2), (0, 1)):
        y = policy.linear(x, w, b, "tanh")
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        had = torch.cuda.memory_allocated()
        got = torch.autograd.grad(y, [(x, w, b)[i] for i in asked], dy)
        peak = torch.cuda.max_memory_allocated() - had
        assert all(torch.equal(g, full[i]) for g, i in zip(got, asked)), asked
        if 0 not in asked:
            c = policy.linear(x.detach(), w, b, "tanh")  # x needs no gradient at all: the same work
            torch.cuda.reset_peak_memory_stats()
            had = torch.cuda.memory_allocated()
            torch.autograd.grad(c, [(x, w, b)[i] for i in asked], dy)
            assert peak <= torch.cuda.max_memory_allocated() - had + (2 << 20), asked  # (blocks of the allocator; dx is 41 MB)


def test_norm_computes_only_what_a_backward_pass_asks_for():
    (x, block, gate, post, pre), dr, dh = norm_case(20000, 512, torch.float32, "full")
    run = lambda *a: policy.norm_residual(a[0], a[1], gate=a[2], scale=0.5, post_weight=post, pre_weight=pre)  # noqa: E731
    full = torch.autograd.grad(run(x, block, gate), [x, block, gate, post, pre], [dr, dh])
    r, h = run(x, block, gate)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    had = torch.cuda.memory_allocated()
    got = torch.autograd.grad([r, h], [post, pre], [dr, dh])
    peak = torch.cuda.max_memory_allocated() - had
    assert torch.equal(got[0], full[3]) and torch.equal(got[1], full[4])
    assert peak < x.numel() * 4  # not one of the three large ones


def test_adamw_refuses_tensors_that_overlap():
    flat = torch.zeros(300, device="cuda")
    s = adamw_case([(100,), (100,)], torch.float32)
    call = lambda **o: policy.adamw_step(**{**dict(params=s["params"], grads=s["grads"], exp_avgs=s["m"], exp_avg_sqs=s["v"], step=s["step"], lr=1e-3), **o})  # noqa: E731
    with pytest.raises(ValueError, match="overlap"):
        call(params=[flat[:100], flat[99:199]])
    with pytest.raises(ValueError, match="overlap"):
        call(exp_avgs=[flat[:100], flat[100:200]], exp_avg_sqs=[flat[199:299], s["v"][1]])
    assert not flat.any()
    call(params=[flat[:100], flat[100:200]])  # neighbours are not the same
    assert flat[:200].all() and not flat[200:].any()


def test_negated_views_count_as_what_they_are():
    """A conjugate's imaginary part is a view whose sign waits to be taken: by address it is the other sign."""
    x, w, b, r, dy = linear_case(9, 16, 8, torch.float32, "tanh")
    flip = lambda v: torch._neg_view(v.detach().neg())  # noqa: E731
    assert flip(x).is_neg() and torch.equal(flip(x), x)
    want = policy.linear(x, w, b, "tanh", r)
    for at in range(4):
        a = [v.detach() for v in (x, w, b, r)]
        a[at] = flip(a[at])
        assert torch.equal(policy.linear(a[0], a[1], a[2], "tanh", a[3]), want), at
    leaf = x.detach().neg().requires_grad_(True)
    dx, = torch.autograd.grad(policy.linear(torch._neg_view(leaf), w, b, "tanh", r), leaf, flip(dy))
    assert torch.equal(dx, torch.autograd.grad(want, x, dy)[0].neg())
    ts, dr, dh = norm_case(9, 16, torch.float32, "full", leaf=False)
    keep = policy.norm_residual(ts[0], ts[1], gate=ts[2], post_weight=ts[3], pre_weight=ts[4])
    for at in range(5):
        a = list(ts)
        a[at] = flip(a[at])
        got = policy.norm_residual(a[0], a[1], gate=a[2], post_weight=a[3], pre_weight=a[4])
        assert torch.equal(got[0], keep[0]) and torch.equal(got[1], keep[1]), at
    s = adamw_case([(7,)], torch.float32)
    with pytest.raises(ValueError, match="contiguous"):
        policy.adamw_step(s["params"], [flip(s["grads"][0])], s["m"], s["v"], s["step"], lr=1e-3)
    with torch.no_grad(), pytest.raises(ValueError, match="out"):
        policy.linear(x, w, b, out=torch._neg_view(torch.zeros(9, 8, device="cuda")))


def test_collect_stopped_by_its_policy(hip):
    """A policy that raises in the middle: the env and its buffers are where as many step calls leave them."""
    from drone_amd.env import Drone

    net = policy.Policy(width=32, device="cuda:0")
    a, b = (Drone(num_envs=501, task="waypoint", device="cuda:0", seed=4, log_interval=0, horizon=9) for _ in range(2))
    for e in (a, b):
        e.reset(4)
    calls = []

    def stops(obs, out):
        calls.append(1)
        if len(calls) == 5:
            raise KeyboardInterrupt
        return net(obs, out=out)

    a.collect(net, 6)
    with pytest.raises(KeyboardInterrupt):
        a.collect(stops, 6)
    for _ in range(6 + 4):
        with torch.no_grad():
            net(b.observations, out=b.actions)
        b.step(b.actions)
    for name in ("observations", "actions", "rewards", "terminals", "truncations"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert a.tick == b.tick and a.vec.gstep == b.vec.gstep
    a.collect(net, 2)
    for _ in range(2):
        with torch.no_grad():
            net(b.observations, out=b.actions)
        b.step(b.actions)
    assert torch.equal(a.observations, b.observations) and torch.equal(a.rewards, b.rewards)
    for e in (a, b):
        e.close()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", ["channel", "full"])
@pytest.mark.parametrize("m, c", [(33, 32), (50, 200), (9, 1500)])
def test_norm_gate_gradient_of_open_and_shut_gates(t, gate, m, c):
    """dgate carries s (1 - s): at a gate of 5 ... 14 both factors keep their own precision, 1e-5 for an exponential of an
    argument up to 14 and the operations around it. dr alone, so that the other factors are one product each."""
    (x, block, _, post, pre), dr, _ = norm_case(m, c, t, "none", leaf=False)
    g = (torch.arange(m * c, device="cuda") % 10 + 5.0).view(m, c) * torch.where(torch.arange(c, device="cuda") % 2 == 0, 1.0, -1.0)
    g = (g if gate == "full" else g[0]).to(t).requires_grad_(True)
    dr = dr * 256
    r, _ = policy.norm_residual(x, block, gate=g, scale=0.5, post_weight=post, pre_weight=pre)
    got, = torch.autograd.grad(r, g, dr)
    B, G = block.double(), g.detach().double()
    each = dr.double() * 0.5 * (B / torch.sqrt(B.square().mean(1, keepdim=True) + 1e-6)) * post.double() * torch.sigmoid(G) * torch.sigmoid(-G)
    want, size = (each, each.abs()) if gate == "full" else (each.sum(0), each.abs().sum(0))
    close(got, want, size * (1e-5 + 200 * U32) + want.abs() * half_step(t) + TINY[t], f"{m}x{c}")


def test_adamw_norm_of_many_equal_gradients():
    """2^28 equal values, whose squares a running 32-bit sum takes in with the same rounding again and again."""
    n = 1 << 28
    s = {k: torch.full((n,), v, device="cuda") for k, v in (("p", 0.5), ("g", 0.1), ("m", 0.0), ("v", 0.0))}
    norm = policy.adamw_step([s["p"]], [s["g"]], [s["m"]], [s["v"]], torch.zeros(1, dtype=torch.int32, device="cuda"), lr=1e-3, max_grad_norm=1.0)
    want = s["g"][0].double().item() * math.sqrt(n)
    assert abs(norm.item() - want) <= 64 * U32 * want


def test_optimizer_reports_a_norm_for_every_group():
    ps = [torch.nn.Parameter(rand(9, seed=i)) for i in range(3)]
    opt = policy.AdamW([{"params": [p]} for p in ps])
    ps[0].grad, ps[2].grad = torch.ones(9, device="cuda"), torch.full((9,), 2.0, device="cuda")
    opt.step()
    assert opt.grad_norm[1] is None  # no gradient in the group: no step, no norm
    assert [opt.grad_norm[i].item() for i in (0, 2)] == [3.0, 6.0]
    assert [g["step"].item() for g in opt.param_groups] == [1, 0, 1]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ["tanh", "silu"])
@pytest.mark.parametrize("m, n", FORMS)
def test_linear_gradient_of_saturated_units(t, act, m, n):
    """The slopes of far z, relative to themselves: 2^-11 for the 16 bits a bf16 layer keeps them in, 1e-5 for the exponential
    of an argument up to 20 (rounded to 2^-24 of itself) and a handful of operations on it, and the roundings of dz and dx to
    the type. (dx is dz times one.) dy is a power of two large enough that dz is a normal number of the type."""
    z = torch.arange(-20, 21, device="cuda") / 2.0
    z = z[z.abs() >= 2.5]
    z = z[z < 0] if act == "silu" else z  # (silu's slope is near 1 on the other side)
    if t == torch.float16:
        z = z[z.abs() <= 8]
    x, w = diagonal(m, n, t, z)
    dy = torch.full((m, n), 2.0 ** 12, device="cuda").to(t)
    dx, _ = torch.autograd.grad(policy.linear(x, w, None, act), [x, w], dy)
    Z = x.detach().double()
    s = 1 / torch.cosh(Z).square() if act == "tanh" else torch.sigmoid(Z) * (1 + Z * torch.sigmoid(-Z))
    want = 2.0 ** 12 * s
    tol = want.abs() * (2 * half_step(t) + (2.0 ** -11 if t == torch.bfloat16 else 0) + 1e-5)
    close(dx, want, tol, f"{act} {m}x{n}")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m, k, n", [(66001, 264, 520), (20001, 520, 384), (9001, 1024, 520)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_linear_input_gradient_alone_of_a_wide_layer(t, m, k, n, act):
    """Asked for alone it takes the same form as beside the weights', so it has the same bits."""
    x, w, b, _, dy = linear_case(m, k, n, t, act, res=False)
    y = policy.linear(x, w, b, act)
    full = torch.autograd.grad(y, [x, w, b], dy, retain_graph=True)
    alone, = torch.autograd.grad(y, [x], dy)
    assert torch.equal(alone, full[0])


def test_captured_collect_replays(hip):
    """collect in one graph, replayed with the program's own work in between, against the same calls made eagerly. The log's
    interval passes inside the captured call: it cannot be read there, and is read by the next eager one."""
    from drone_amd.env import Drone

    net = policy.Policy(width=32, device="cuda:0")
    a, b = (Drone(num_envs=777, task="waypoint", device="cuda:0", seed=6, log_interval=4, horizon=9) for _ in range(2))
    for e in (a, b):
        e.reset(6)
    a.vec.enable_graph_capture(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.collect(net, 4)
    torch.cuda.synchronize()
    b.collect(net, 4)
    g = torch.cuda.CUDAGraph()
    tick = a.tick
    with torch.cuda.graph(g, stream=side):
        blocks = a.collect(net, 4)
    assert blocks[5] == [] and a.tick == tick  # nothing has run yet
    for k in range(5):
        g.replay()
        torch.cuda.synchronize()
        want = b.collect(net, 4)
        torch.cuda.synchronize()
        for x, y in zip(blocks[:5], want[:5]):
            assert torch.equal(x, y), k
        assert torch.equal(a.observations, b.observations) and torch.equal(a.actions, b.actions) and torch.equal(a.truncations, b.truncations), k
        assert a.vec.gstep == b.vec.gstep
    infos = a.collect(net, 4)[5]
    assert len(infos) == 1 and infos[0]["n"] > 0
    # another K: the captured blocks stay the graph's own, whoever else has let go of them
    shape = blocks[0].shape
    del blocks, x, y
    a.collect(net, 2)
    others = [torch.full(shape, 7.0, device="cuda") for _ in range(8)]
    g.replay()
    torch.cuda.synchronize()
    assert all((o == 7).all() for o in others)
    for e in (a, b):
        e.close()


@pytest.mark.parametrize("op", ["linear", "norm"])
def test_a_backward_pass_is_not_captured_beside_an_eager_graph_of_its_leaves(op):
    """Leaves' gradients go to accumulators that live as long as a graph holds them. One that an eager graph on the default
    stream holds runs there, where a captured pass cannot follow: refused before it gets there, and the capture ends whole.
    Without that graph the same capture goes through."""
    if op == "linear":
        x, w, b, _, dy = linear_case(700, 24, 32, torch.float32, "tanh", res=False)
        leaves, run, ds = [w, b], (lambda: [policy.linear(x, w, b, "tanh")]), [dy]
    else:
        (x, block, gate, post, pre), dr, dh = norm_case(700, 32, torch.float32, "channel")
        leaves, run, ds = [gate, post, pre], (lambda: list(policy.norm_residual(x, block, gate=gate, post_weight=post, pre_weight=pre))), [dr, dh]
    held = run()
    want = torch.autograd.grad(held, leaves, ds, retain_graph=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(g):
            torch.autograd.grad(run(), leaves, ds)
    if op == "linear":  # a captured pass that asks for another leaf only has nothing to hand to those
        other = x.detach().clone().requires_grad_(True)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            dx, = torch.autograd.grad(policy.linear(other, w, b, "tanh"), other, dy)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, torch.autograd.grad(policy.linear(other, w, b, "tanh"), other, dy)[0])
    assert torch.equal(torch.autograd.grad(held, leaves, ds)[0], want[0])  # nothing else is the worse for it
    del held
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(run(), leaves, ds)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_policy_loop_runs_with_residual_blocks():
    """The command's own network with norm_residual in it: acting in a graph, collecting, learning."""
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "torch_policy_loop.py"), "--envs", "2048", "--steps", "40", "--blocks", "2"], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "act, learn, update" in r.stdout and "nan" not in r.stdout, r.stdout


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_optimizer_refuses_a_state_that_is_not_its_own(t):
    """A state of other shapes, of torch's AdamW or without its masters is refused before anything is written."""
    def make():
        ps = [torch.nn.Parameter(rand(6, 5, to=t, seed=1)), torch.nn.Parameter(rand(5, to=t, seed=2))]
        for p in ps:
            p.grad = torch.ones_like(p)
        opt = policy.AdamW(ps, lr=1e-2)
        opt.step()
        return ps, opt

    ps, opt = make()
    good = opt.state_dict()
    other = [torch.nn.Parameter(rand(6, 5, seed=1)), torch.nn.Parameter(rand(1, seed=2))]
    theirs = torch.optim.AdamW(ps)
    theirs.step()
    bad = [theirs.state_dict()]
    for key, value in (("exp_avg", torch.zeros(1, device="cuda")), ("exp_avg_sq", None)):
        broken = {"param_groups": good["param_groups"], "state": {i: dict(s) for i, s in good["state"].items()}}
        if value is None:
            del broken["state"][1][key]
        else:
            broken["state"][1][key] = value
        bad.append(broken)
    bad.append(policy.AdamW(other).state_dict())
    for state in bad:
        with pytest.raises(ValueError, match="state"):
            opt.load_state_dict(state)
    twins, twin = make()
    theirs_undone = [p.detach().clone() for p in twins]
    with torch.no_grad():
        for p, q in zip(ps, theirs_undone):
            p.copy_(q)
    opt.step()
    twin.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, twins)) and opt.param_groups[0]["lr"] == 1e-2
    opt.load_state_dict(good)
    assert opt.param_groups[0]["step"].item() == 2
