"""The policy operators (drone_amd.policy) on the GPU against plain 64-bit implementations of their formulas.

Tolerances are sums of what the arithmetic may lose, element by element: half a step of the type (U) for every rounding to
it, 2^-24 for every 32-bit operation on the magnitudes that are added up, and the stated error of the 16-bit types' fast
activations (2e-6 of 1 + |z|: exp2 and rcp to one unit in 2^-23, erf to 1.5e-7)."""
import math

import pytest
import torch
import torch.nn.functional as F

from drone_amd import policy

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0 ** -24
ACTS = {"none": lambda z: z, "relu": F.relu, "tanh": torch.tanh, "silu": F.silu, "gelu": F.gelu}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # smallest step of the type


def half_step(t):
    return torch.finfo(t).eps / 2


def rand(*shape, to=torch.float32, of=1.0, seed=None):
    g = torch.Generator(device="cuda").manual_seed(seed if seed is not None else sum((i + 3) * (s + 1) for i, s in enumerate(shape)))
    return (torch.randn(shape, device="cuda", generator=g) * of).to(to)


def close(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got).all() and (off.numel() == 0 or off.max().item() <= 0), f"{what}: {off.max().item():.3e} over its tolerance"


def slope_of(z, act):
    z = z.detach().requires_grad_(True)
    return torch.autograd.grad(ACTS[act](z).sum(), z)[0]


def linear_reference(x, w, b, res, dy, act):
    """Outputs and gradients in 64 bits, and how far 32-bit sums with the roundings of type x.dtype may be from them."""
    t, X, W = x.dtype, x.double(), w.double()
    u, us = half_step(t), (half_step(torch.float16) if t == torch.bfloat16 else U32)
    tiny = TINY[t] + (2.0 ** -24 if t == torch.bfloat16 else 0)  # the slope of a bf16 layer is kept in fp16
    B = 0.0 if b is None else b.double()
    z = X @ W.t() + B
    size = X.abs() @ W.abs().t() + (0.0 if b is None else b.double().abs())
    ez = (x.shape[1] + 2) * U32 * size
    y = ACTS[act](z)
    ey = 1.13 * ez + 2e-6 * (1 + z.abs())
    if res is not None:
        y = y + res.double()
        ey = ey + U32 * y.abs()
    out = {"y": (y, ey * (1 + u) + u * y.abs() + TINY[t])}
    if dy is None:
        return out
    D, s = dy.double(), slope_of(z, act) if act != "none" else torch.ones_like(z)
    es = 0 * z if act == "none" else (z.abs() <= ez).double() if act == "relu" else ez + us * s.abs() + 2e-6 * (1 + z.abs()) + tiny
    dz = D * s
    e_sum = D.abs() * es + U32 * dz.abs()                    # the 32-bit dz the bias gradient adds up
    e = e_sum * (1 + u) + u * dz.abs() + TINY[t]             # rounded for the matrix product
    m = x.shape[0]
    big = dz.abs() + e

    def done(v, err):
        return v, err * (1 + u) + u * v.abs() + TINY[t]

    out["dx"] = done(dz @ W, e @ W.abs() + (w.shape[0] + 2) * U32 * (big @ W.abs()))
    out["dw"] = done(dz.t() @ X, e.t() @ X.abs() + (m + 2) * U32 * (big.t() @ X.abs()))
    out["db"] = done(dz.sum(0), e_sum.sum(0) + (m + 2) * U32 * big.sum(0))
    return out


def linear_case(m, k, n, t, act, bias=True, res=True, seed=1):
    leaf = lambda *s, **kw: rand(*s, to=t, **kw).requires_grad_(True)  # noqa: E731
    return (leaf(m, k, seed=seed), leaf(n, k, of=k ** -0.5, seed=seed + 1), leaf(n, seed=seed + 2) if bias else None, leaf(m, n, seed=seed + 3) if res else None, rand(m, n, to=t, seed=seed + 4))


def check_linear(x, w, b, res, dy, act, what):
    y = policy.linear(x, w, b, act, res)
    leaves = [v for v in (x, w, b, res) if v is not None]
    grads = dict(zip([n for n, v in zip(("dx", "dw", "db", "dres"), (x, w, b, res)) if v is not None], torch.autograd.grad(y, leaves, dy)))
    ref = linear_reference(*(None if v is None else v.detach() for v in (x, w, b, res)), dy, act)
    close(y.detach(), *ref["y"], f"{what} y")
    for g in ("dx", "dw", "db"):
        if g in grads:
            close(grads[g], *ref[g], f"{what} {g}")
    if res is not None:
        assert torch.equal(grads["dres"], dy)
    with torch.no_grad():
        assert torch.equal(policy.linear(x, w, b, act, res), y), f"{what}: the same numbers without a gradient"
    return y, grads


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m, k, n", [(1, 1, 1), (1, 512, 512), (2, 20, 64), (3, 5, 7), (8, 1024, 96), (9, 130, 33), (31, 64, 4), (64, 64, 64), (65, 63, 65), (127, 129, 128), (130, 20, 64),
                                     (257, 24, 200), (300, 256, 256), (513, 333, 129), (1000, 512, 40), (2048, 130, 66), (4099, 24, 31), (5000, 64, 64), (700, 1024, 260)])
def test_linear_shapes(t, m, k, n):
    check_linear(*linear_case(m, k, n, t, "tanh"), "tanh", f"{m}x{k}x{n}")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m, k, n", [(66001, 256, 256), (66001, 512, 264), (66001, 136, 200), (66001, 40, 136), (140001, 128, 100), (140001, 64, 128), (270001, 72, 64), (530001, 24, 8), (530001, 32, 48),
                                     (9001, 1024, 520), (20001, 520, 384), (9001, 333, 259), (70001, 20, 7)])
@pytest.mark.parametrize("act, res", [("silu", True), ("gelu", False)])
def test_linear_many_rows(t, m, k, n, act, res):
    """Row counts at which the streaming forms run (weights in registers, tiles from memory to LDS, dz in a pass of its own),
    with a last tile that is not whole, for reductions and feature counts of every class; unaligned widths keep theirs."""
    check_linear(*linear_case(m, k, n, t, act, True, res), act, f"{m}x{k}x{n}")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("bias, res", [(True, False), (False, True), (False, False)])
def test_linear_activations(t, act, bias, res):
    check_linear(*linear_case(333, 40, 72, t, act, bias, res), act, f"{act} bias={bias} res={res}")
    check_linear(*linear_case(5, 40, 72, t, act, bias, res), act, f"{act} few rows bias={bias} res={res}")


@pytest.mark.parametrize("t", TYPES)
def test_linear_strides_offsets_and_orders(t):
    """Row views of wider tensors, addresses that are not 16-byte aligned, a transposed weight, leading dimensions."""
    for m, k, n, shift in ((70, 24, 32, 0), (70, 24, 32, 3), (129, 64, 68, 1), (6, 64, 68, 5)):
        x = rand(m, k + 8, to=t, seed=3)[:, shift:shift + k].detach().requires_grad_(True)
        w = rand(k, n, to=t, of=k ** -0.5, seed=4).t().detach().requires_grad_(True)
        b = rand(n + 8, to=t, seed=5)[shift:shift + n].detach().requires_grad_(True)
        r = rand(m, n + 9, to=t, seed=6)[:, shift:shift + n].detach().requires_grad_(True)
        dy = rand(m, n + 5, to=t, seed=7)[:, shift % 5:shift % 5 + n]
        check_linear(x, w, b, r, dy, "silu", f"{m}x{k}x{n}+{shift}")
    x, w, b, _, dy = linear_case(24, 16, 8, t, "tanh", res=False)
    y = policy.linear(x.view(2, 3, 4, 16), w, b, "tanh")
    assert y.shape == (2, 3, 4, 8) and torch.equal(y.reshape(24, 8), policy.linear(x, w, b, "tanh"))
    row = policy.linear(x[0], w, b, "tanh")  # one row without a batch axis
    assert row.shape == (8,)
    wide = rand(1, 16, to=t, seed=9).expand(24, 16)  # the same row again and again
    assert torch.equal(policy.linear(wide, w, b), policy.linear(wide.contiguous(), w, b))


@pytest.mark.parametrize("t", TYPES)
def test_linear_writes_out_and_nothing_else(t):
    x, w, b, r, _ = (None if v is None else v.detach() for v in linear_case(37, 20, 6, t, "tanh"))
    want = policy.linear(x, w, b, "tanh", r)
    block = torch.full((41, 11), 7.0, dtype=t, device="cuda")
    got = policy.linear(x, w, b, "tanh", r, out=block[2:39, 3:9])
    assert got.data_ptr() == block[2:39, 3:9].data_ptr() and torch.equal(got, want)
    block[2:39, 3:9] = 7.0
    assert (block == 7.0).all()
    stream = r.clone()  # the residual stream updated in place
    assert torch.equal(policy.linear(x, w, b, "tanh", stream, out=stream), want) and torch.equal(stream, want)


@pytest.mark.parametrize("t", TYPES)
def test_linear_without_rows(t):
    x, w, b, r, dy = linear_case(0, 20, 64, t, "silu")
    y = policy.linear(x, w, b, "silu", r)
    dx, dw, db, dr = torch.autograd.grad(y, [x, w, b, r], dy)
    assert y.shape == (0, 64) and dx.shape == (0, 20) and dr.shape == (0, 64)
    assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [6, 150])
def test_linear_keeps_bad_values_in_their_rows(t, rows):
    """A NaN or infinity in one row (a diverged env) shows in that row's outputs and in no other's; the limits of the
    activations at the infinities are finite where they should be."""
    x, w, b, r, _ = (v.detach() for v in linear_case(rows, 44, 52, t, "silu"))
    want = {a: policy.linear(x, w, b, a, r) for a in ACTS}
    bad = x.clone()
    bad[2, 5], bad[4, 43] = float("nan"), float("inf")
    for a in ACTS:
        y = policy.linear(bad, w, b, a, r)
        keep = [i for i in range(rows) if i not in (2, 4)]
        assert torch.equal(y[keep], want[a][keep]), a
        assert torch.isnan(y[2]).all(), a
        assert not torch.isnan(y[4]).any(), a
    x1 = torch.tensor([[float("inf")], [-float("inf")], [200.0], [-200.0]], device="cuda").to(t).requires_grad_(True)
    one = torch.ones(1, 1, device="cuda").to(t)
    for a, (hi, lo, s_hi, s_lo) in {"relu": (math.inf, 0, 1, 0), "tanh": (1, -1, 0, 0), "silu": (math.inf, 0, 1, 0), "gelu": (math.inf, 0, 1, 0)}.items():
        y = policy.linear(x1, one, None, a)
        assert y[0].item() == hi and y[1].item() == lo, a
        dx, = torch.autograd.grad(y, x1, torch.ones_like(y))
        assert dx[0].item() == s_hi and dx[1].item() == s_lo and dx[2].item() == s_hi and dx[3].item() == s_lo, a


def test_linear_offsets_beyond_32_bits():
    """Rows whose element offsets pass 2^31 (a narrow view of a wide history): first and last rows against the same rows
    on their own, forward and input gradient."""
    m, ld, k, n = 70001, 32768, 24, 20
    wide = torch.zeros((m, ld), dtype=torch.bfloat16, device="cuda")
    x = wide[:, 8:8 + k]
    x.copy_(rand(m, k, to=torch.bfloat16, seed=1))
    w, b = rand(n, k, to=torch.bfloat16, seed=2), rand(n, to=torch.bfloat16, seed=3)
    out = policy.linear(x, w, b, "tanh")
    assert torch.equal(out[-500:], policy.linear(x[-500:].contiguous(), w, b, "tanh"))
    assert torch.equal(out[:500], policy.linear(x[:500].contiguous(), w, b, "tanh"))
    far = wide[:, 100:100 + n]
    policy.linear(x, w, b, "tanh", out=far)
    assert torch.equal(far, out)
    leaf = w.detach().requires_grad_(True)
    y = policy.linear(x, leaf, b, "tanh")
    dw, = torch.autograd.grad(y, leaf, far)
    leaf2 = w.detach().requires_grad_(True)
    want, = torch.autograd.grad(policy.linear(x.contiguous(), leaf2, b, "tanh"), leaf2, far.contiguous())
    assert torch.equal(dw, want)


@pytest.mark.parametrize("t", TYPES)
def test_linear_is_the_same_every_time(t):
    case = linear_case(20000, 64, 68, t, "gelu")
    first = check_linear(*case, "gelu", "first")
    again = check_linear(*case, "gelu", "again")
    assert torch.equal(first[0], again[0]) and all(torch.equal(first[1][g], again[1][g]) for g in first[1])


@pytest.mark.parametrize("m, k, n", [(300, 33, 65), (5000, 64, 64), (9001, 30, 100), (20001, 264, 136), (20001, 333, 129)])
@pytest.mark.parametrize("act", ["relu", "none"])
def test_linear_only_the_gradients_asked_for(m, k, n, act):
    """Every subset of the three, in each of the gradient's forms (tiled, one pass, streamed; laid out or as it is). The
    input gradient alone takes the tiled form: the same sums in another order, held to the tolerance."""
    for t in TYPES:
        x, w, b, _, dy = linear_case(m, k, n, t, act, res=False)
        full = torch.autograd.grad(policy.linear(x, w, b, act), [x, w, b], dy)
        for needs in range(1, 8):
            vs = [v.detach().requires_grad_(bool(needs >> i & 1)) for i, v in enumerate((x, w, b))]
            got = torch.autograd.grad(policy.linear(*vs, act), [v for v in vs if v.requires_grad], dy)
            want = [f for f, v in zip(full, vs) if v.requires_grad]
            if needs == 1:
                ref = linear_reference(x.detach(), w.detach(), b.detach(), None, dy, act)["dx"]
                close(got[0], *ref, "dx alone")
            else:
                assert all(torch.equal(a, c) for a, c in zip(got, want)), (t, needs)


def test_linear_refuses_overlapping_out():
    x, w = rand(40, 32, seed=1), rand(32, 32, seed=2)
    block = torch.zeros(40, 80, device="cuda")
    with torch.no_grad():
        for kw in (dict(out=x), dict(residual=block[:, :32], out=block[:, 8:40])):
            with pytest.raises(ValueError, match="overlaps"):
                policy.linear(x, w, **kw)
        inside = block[:, :32].copy_(x)
        with pytest.raises(ValueError, match="overlaps"):
            policy.linear(inside, w, out=block[:, 31:63])
        assert torch.equal(policy.linear(inside, w, out=block[:, 32:64]), policy.linear(x, w))
        with pytest.raises(ValueError, match="overlaps"):
            policy.linear(x[:32], w, out=w)


@pytest.mark.parametrize("act", ["none", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("m", [4, 200])
def test_linear_gradient_against_differences(act, m):
    """g . v against the symmetric difference of f = sum(y dy) along v. What the difference itself is off by is taken from
    the same difference in 64 bits; the rest is 32-bit noise of f over the step."""
    x, w, b, r, dy = linear_case(m, 40, 48, torch.float32, act)
    vs = [rand(*t.shape, seed=90 + i) for i, t in enumerate((x, w, b, r))]
    g = torch.autograd.grad(policy.linear(x, w, b, act, r), [x, w, b, r], dy)
    h = 2.0 ** -5

    def f(sign, wide):
        a = [(p.detach() + sign * h * v) for p, v in zip((x, w, b, r), vs)]
        if not wide:
            return (policy.linear(*a[:3], act, a[3]).double() * dy).sum().item()
        a = [p.double() for p in a]
        return ((ACTS[act](a[0] @ a[1].t() + a[2]) + a[3]) * dy).sum().item()

    X = [p.detach().double().requires_grad_(True) for p in (x, w, b, r)]
    G = torch.autograd.grad(ACTS[act](X[0] @ X[1].t() + X[2]) + X[3], X, dy.double())
    slope64 = sum((a * v).sum().item() for a, v in zip(G, vs))
    diff64 = (f(1, True) - f(-1, True)) / (2 * h)
    diff = (f(1, False) - f(-1, False)) / (2 * h)
    slope = sum((a.double() * v).sum().item() for a, v in zip(g, vs))
    ref = linear_reference(x.detach(), w.detach(), b.detach(), r.detach(), dy, act)
    noise = 1.5 * (ref["y"][1] * dy.double().abs()).sum().item() / h  # both values of f, inputs up to half again as large
    off = sum((ref[n][1] * v.abs()).sum().item() for n, v in zip(("dx", "dw", "db"), vs)) + U32 * (dy.abs() * vs[3].abs()).sum().item()
    assert abs(diff - diff64) <= noise
    assert abs(slope - diff) <= abs(slope64 - diff64) + noise + off


# ---------------------------------------------------------------------------------------------------------- norm_residual


def norm_reference(x, block, gate, post, pre, scale, eps, dr, dh):
    """64-bit outputs and gradients with their tolerances. Statistics are sums over at most 64 steps of 32-bit additions
    (columns of a thread, then a tree) and a square root and reciprocal; sigmoid is off by 2e-7 of itself or so: K units."""
    t = x.dtype
    u, K = half_step(t), 200 * U32
    c = x.shape[-1]
    v = [None if a is None else a.detach().double().requires_grad_(True) for a in (x, block, gate, post, pre)]
    X, Bk, Ga, Po, Pr = v
    s = torch.sigmoid(Ga) if Ga is not None else torch.ones((), dtype=torch.float64, device="cuda")
    po = Po if Po is not None else torch.ones(c, dtype=torch.float64, device="cuda")
    pr = Pr if Pr is not None else torch.ones(c, dtype=torch.float64, device="cuda")
    R = X
    if Bk is not None:
        rb = torch.sqrt(Bk.square().mean(-1, keepdim=True) + eps)
        nb = Bk / rb
        add = scale * s * (nb * po)
        R = X + add
    rr = torch.sqrt(R.square().mean(-1, keepdim=True) + eps)
    nr = R / rr
    H = nr * pr
    size = X.detach().abs() + (add.detach().abs() if Bk is not None else 0)  # what r adds up
    er = K * size
    en = (er + nr.detach().abs() * (er * nr.detach().abs()).mean(-1, keepdim=True)) / rr.detach() + K * nr.detach().abs()  # of n(r)
    done = lambda w, e: (w.detach(), e * (1 + u) + u * w.detach().abs() + TINY[t])  # noqa: E731
    out = {"r": done(R, er), "h": done(H, en * pr.detach().abs())}
    leaves = [a for a in v if a is not None]
    G = torch.autograd.grad([R, H], leaves, [dr.double(), dh.double()])
    G = dict(zip([n for n, a in zip(("dx", "dblock", "dgate", "dpost", "dpre"), v) if a is not None], G))
    with torch.no_grad():
        g = (dh.double() * pr).abs()
        dn = (g + nr.abs() * (g * nr.abs()).mean(-1, keepdim=True)) / rr      # magnitudes that dn(r)[g] adds up
        er_rel = (er / rr).square().mean(-1, keepdim=True).sqrt() + K         # relative error of rms(r)
        e_t = K * (dr.double().abs() + dn) + er_rel * 4 * dn + (en * (g * nr.abs()).mean(-1, keepdim=True) + nr.abs() * (g * en).mean(-1, keepdim=True)) / rr
        td = dr.double() + 0
        td = G["dx"] if "dx" in G else td
        out["dx"] = done(td, e_t)
        m = max(1, x.shape[0])
        if Pr is not None:
            out["dpre"] = done(G["dpre"], (dh.double().abs() * en).sum(0) + (m + 200) * U32 * (dh.double().abs() * nr.abs()).sum(0))
        if Bk is not None:
            a_t = (td.abs() + e_t) * abs(scale)
            ut, et = a_t * s, (e_t * abs(scale) + K * a_t) * s
            if Po is not None:
                out["dpost"] = done(G["dpost"], (et * nb.abs() + K * ut * nb.abs()).sum(0) + m * U32 * (ut * nb.abs()).sum(0))
            q = ut * po.abs()
            eq = et * po.abs()
            out["dblock"] = done(G["dblock"], (eq + nb.abs() * (eq * nb.abs()).mean(-1, keepdim=True) + 4 * K * (q + nb.abs() * (q * nb.abs()).mean(-1, keepdim=True))) / rb)
            if Ga is not None:
                one = et * (nb * po).abs() + 2 * K * ut * (nb * po).abs()     # (1 - s cancels to K of 1)
                if Ga.dim() == 1 and x.dim() > 1:
                    out["dgate"] = done(G["dgate"], one.sum(0) + m * U32 * (ut * (nb * po).abs()).sum(0))
                else:
                    out["dgate"] = done(G["dgate"], one)
    return out


def norm_case(m, c, t, gate, seed=1, leaf=True):
    ts = [rand(m, c, to=t, seed=seed), rand(m, c, to=t, of=3.0, seed=seed + 1), None if gate == "none" else rand(*((c,) if gate == "channel" else (m, c)), to=t, seed=seed + 2),
          rand(c, to=t, seed=seed + 3), rand(c, to=t, seed=seed + 4)]
    return [None if a is None else a.requires_grad_(leaf) for a in ts], rand(m, c, to=t, seed=seed + 5), rand(m, c, to=t, seed=seed + 6)


def check_norm(ts, dr, dh, scale, eps, what):
    x, block, gate, post, pre = ts
    r, h = policy.norm_residual(x, block, gate=gate, scale=scale, post_weight=post, pre_weight=pre, eps=eps)
    ref = norm_reference(*ts, scale, eps, dr, dh)
    close(r.detach(), *ref["r"], f"{what} r")
    close(h.detach(), *ref["h"], f"{what} h")
    names = [n for n, a in zip(("dx", "dblock", "dgate", "dpost", "dpre"), ts) if a is not None]
    grads = dict(zip(names, torch.autograd.grad([r, h], [a for a in ts if a is not None], [dr, dh])))
    for n in names:
        close(grads[n], *ref[n], f"{what} {n}")
    with torch.no_grad():
        r2, h2 = policy.norm_residual(x, block, gate=gate, scale=scale, post_weight=post, pre_weight=pre, eps=eps)
        assert torch.equal(r, r2) and torch.equal(h, h2), what
    return r.detach(), h.detach(), grads


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
@pytest.mark.parametrize("m, c", [(1, 1), (1, 256), (3, 7), (33, 32), (100, 64), (65, 333), (50, 512), (7, 513), (40, 1024), (21, 1500), (9, 2048), (5, 4096), (3, 4095), (4099, 24), (2500, 264)])
def test_norm_shapes(t, gate, m, c):
    check_norm(*norm_case(m, c, t, gate), 0.5, 1e-6, f"{m}x{c} {gate}")


@pytest.mark.parametrize("t", TYPES)
def test_norm_optional_parts_and_one_sided_gradients(t):
    (x, block, gate, post, pre), dr, dh = norm_case(77, 72, t, "full")
    for ts in ([x, block, None, None, None], [x, block, gate, None, pre], [x, block, None, post, None], [x, None, None, None, pre], [x, None, None, None, None]):
        check_norm(ts, dr, dh, -1.25, 1e-3, "parts")
    zero = torch.zeros_like(dr)
    for a, b in ((dr, None), (None, dh)):
        r, h = policy.norm_residual(x, block, gate=gate, scale=0.5, post_weight=post, pre_weight=pre)
        out, d = ([r], [a]) if b is None else ([h], [b])
        leaves = [x, block, gate, post] + ([pre] if b is not None else [])
        got = torch.autograd.grad(out, leaves, d)
        ref = norm_reference(x, block, gate, post, pre, 0.5, 1e-6, zero if a is None else a, zero if b is None else b)
        for n, g in zip(("dx", "dblock", "dgate", "dpost", "dpre"), got):
            close(g, *ref[n], n)


@pytest.mark.parametrize("t", TYPES)
def test_norm_strides_and_leading_axes(t):
    (x, block, gate, post, pre), dr, dh = norm_case(60, 40, t, "full")
    want = policy.norm_residual(x, block, gate=gate, scale=0.5, post_weight=post, pre_weight=pre)
    wide = [torch.zeros(60, 55, dtype=t, device="cuda") for _ in range(3)]
    views = [w[:, 3 + i:43 + i] for i, w in enumerate(wide)]
    for v, a in zip(views, (x, block, gate)):
        v.copy_(a.detach())
    got = policy.norm_residual(views[0], views[1], gate=views[2], scale=0.5, post_weight=post, pre_weight=pre)
    # (unaligned rows take the element-wise loads: the same sums in the same order)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    three = policy.norm_residual(x.view(5, 12, 40), block.view(5, 12, 40), gate=gate.view(5, 12, 40), scale=0.5, post_weight=post, pre_weight=pre)
    assert three[0].shape == (5, 12, 40) and torch.equal(three[0].view(60, 40), want[0]) and torch.equal(three[1].view(60, 40), want[1])
    row = policy.norm_residual(x[0], block[0], gate=gate[0], scale=0.5, post_weight=post, pre_weight=pre)
    assert row[0].shape == (40,) and torch.equal(row[1], want[1][0])


@pytest.mark.parametrize("t", TYPES)
def test_norm_rows_of_zeros_and_bad_values(t):
    (x, block, gate, post, pre), dr, dh = norm_case(40, 96, t, "channel", leaf=False)
    x[3], block[3], block[5] = 0, 0, 0
    want = policy.norm_residual(x, block, gate=gate, scale=0.5, post_weight=post, pre_weight=pre)
    assert not want[0][3].any() and not want[1][3].any() and torch.equal(want[0][5], x[5])
    bad = block.clone()
    bad[8, 2], bad[9, 2] = float("nan"), float("inf")
    got = policy.norm_residual(x, bad, gate=gate, scale=0.5, post_weight=post, pre_weight=pre)
    keep = [i for i in range(40) if i not in (8, 9)]
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])
    assert torch.isnan(got[0][8]).all() and torch.isnan(got[1][8]).all()
    shut = torch.full_like(gate, -math.inf)  # a closed gate: the block adds nothing
    r, _ = policy.norm_residual(x, block, gate=shut, scale=0.5, post_weight=post, pre_weight=pre)
    assert torch.equal(r, x)
    e = torch.empty(0, 96, dtype=t, device="cuda").requires_grad_(True)
    w = pre.clone().requires_grad_(True)
    r, h = policy.norm_residual(e, pre_weight=w)
    assert r.shape == h.shape == (0, 96) and not torch.autograd.grad(h, w, h.detach())[0].any()


@pytest.mark.parametrize("gate", ["channel", "full"])
def test_norm_gradient_against_differences(gate):
    ts, dr, dh = norm_case(30, 48, torch.float32, gate)
    vs = [rand(*a.shape, seed=70 + i) for i, a in enumerate(ts)]
    scale, eps, step = 0.75, 1e-6, 2.0 ** -7
    g = torch.autograd.grad(policy.norm_residual(ts[0], ts[1], gate=ts[2], scale=scale, post_weight=ts[3], pre_weight=ts[4], eps=eps), ts, [dr, dh])

    def wide(x, block, ga, post, pre):
        norm = lambda a: a / torch.sqrt(a.square().mean(-1, keepdim=True) + eps)  # noqa: E731
        r = x + scale * torch.sigmoid(ga) * (norm(block) * post)
        return r, norm(r) * pre

    def f(sign, is_wide):
        a = [p.detach() + sign * step * v for p, v in zip(ts, vs)]
        r, h = wide(*(p.double() for p in a)) if is_wide else policy.norm_residual(a[0], a[1], gate=a[2], scale=scale, post_weight=a[3], pre_weight=a[4], eps=eps)
        return ((r.double() * dr).sum() + (h.double() * dh).sum()).item()

    X = [p.detach().double().requires_grad_(True) for p in ts]
    slope64 = sum((a * v).sum().item() for a, v in zip(torch.autograd.grad(wide(*X), X, [dr.double(), dh.double()]), vs))
    diff64 = (f(1, True) - f(-1, True)) / (2 * step)
    diff = (f(1, False) - f(-1, False)) / (2 * step)
    slope = sum((a.double() * v).sum().item() for a, v in zip(g, vs))
    ref = norm_reference(*ts, scale, eps, dr, dh)
    noise = 1.5 * ((ref["r"][1] * dr.abs()).sum() + (ref["h"][1] * dh.abs()).sum()).item() / step
    off = sum((ref[n][1] * v.abs()).sum().item() for n, v in zip(("dx", "dblock", "dgate", "dpost", "dpre"), vs))
    assert abs(diff - diff64) <= noise
    assert abs(slope - diff) <= abs(slope64 - diff64) + noise + off


# -------------------------------------------------------------------------------------------------------------- adamw_step

HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)


def adamw_case(shapes, t, seed=1, zero=False):
    s = {"masters": [rand(*d, seed=seed + i) for i, d in enumerate(shapes)], "grads": [rand(*d, to=t, of=0.1, seed=seed + 100 + i) for i, d in enumerate(shapes)]}
    s["params"] = [m.to(t) for m in s["masters"]] if t != torch.float32 else s["masters"]
    s["m"] = [torch.zeros_like(w) if zero else 1e-2 * rand(*w.shape, seed=seed + 200 + i) for i, w in enumerate(s["masters"])]
    s["v"] = [torch.zeros_like(w) if zero else (1e-2 * rand(*w.shape, seed=seed + 300 + i)).square() for i, w in enumerate(s["masters"])]
    s["step"] = torch.full((1,), 0 if zero else 17, dtype=torch.int32, device="cuda")
    return s


def step(s, max_grad_norm=None, **over):
    half = s["params"][0].dtype != torch.float32
    return policy.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], max_grad_norm=max_grad_norm, masters=s["masters"] if half else None, **{**HYPER, **over})


def check_adamw(s, max_grad_norm, what, **over):
    """One step against the formulas in 64 bits. 32-bit roundings: two products and a sum for each moment (the clip factor
    behind a sum over the gradients adds a few dozen), a dozen more in the update."""
    hyper = {**HYPER, **over}
    before = {k: [a.double() for a in s[k]] for k in ("masters", "grads", "m", "v")}
    t = int(s["step"].item()) + 1
    norm = step(s, max_grad_norm, **over)
    want_norm = math.sqrt(sum(g.square().sum().item() for g in before["grads"]))
    K = 64 * U32
    assert abs(norm.item() - want_norm) <= K * want_norm
    clip = min(1.0, max_grad_norm / (want_norm + 1e-6)) if max_grad_norm else 1.0
    (b1, b2), lr = hyper["betas"], hyper["lr"]
    for i, (p, g, m, v) in enumerate(zip(before["masters"], before["grads"], before["m"], before["v"])):
        g = g * clip
        want_m, size_m = b1 * m + (1 - b1) * g, (b1 * m).abs() + ((1 - b1) * g).abs()
        want_v = b2 * v + (1 - b2) * g * g
        close(s["m"][i], want_m, K * size_m + 2.0 ** -149, f"{what} m[{i}]")
        close(s["v"][i], want_v, 2 * K * want_v + 2.0 ** -149, f"{what} v[{i}]")
        den = torch.sqrt(want_v / (1 - b2 ** t)) + hyper["eps"]
        want_p = p * (1 - lr * hyper["weight_decay"]) - lr * (want_m / (1 - b1 ** t)) / den
        close(s["masters"][i], want_p, 3 * U32 * p.abs() + lr * 4 * K * (size_m / (1 - b1 ** t)) / den + 2.0 ** -149, f"{what} p[{i}]")
        if s["params"][i].dtype != torch.float32:
            assert torch.equal(s["params"][i], s["masters"][i].to(s["params"][i].dtype))
    assert s["step"].item() == t


MLP = [(64, 20), (64,), (64, 64), (64,), (4, 64), (4,)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("clip", [None, 0.5, 1e6])
def test_adamw_steps(t, clip):
    s = adamw_case(MLP, t, zero=True)
    for k in range(3):
        check_adamw(s, clip, f"step {k}")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shapes", [[(1,)], [(3, 5), (0,), (7,), (0, 4)], [(2048,), (2049,), (2047,)], [(300, 257), (1,), (129, 513), (1000003,)], [(5 + i,) for i in range(95)]])
def test_adamw_sizes(t, shapes):
    """One value, empty tensors, around a workgroup's share, long ones, more tensors than one launch takes."""
    s = adamw_case(shapes, t)
    check_adamw(s, 0.5, "first")
    check_adamw(s, None, "second", lr=0.0)


def test_adamw_extreme_settings():
    """Moments that forget at once, no decay, a large eps, a count far along: the bias corrections' two ends."""
    for t, over in ((torch.float32, dict(betas=(0.0, 0.5), eps=1e-3)), (torch.bfloat16, dict(betas=(0.0, 0.0), weight_decay=0.0)), (torch.float32, dict(betas=(0.99, 0.9999)))):
        s = adamw_case([(70, 33), (5,)], t)
        check_adamw(s, 0.5, str(over), **over)
        s["step"].fill_(2_000_000)
        check_adamw(s, None, f"late {over}", **over)


def test_adamw_large_total():
    """Enough values that the norm's partial sums are spread over all its workgroups, many chunks each."""
    check_adamw(adamw_case([(1024, 1024), (1024,), (3000, 999)], torch.bfloat16), 1.0, "large")


@pytest.mark.parametrize("t", TYPES)
def test_adamw_unaligned_and_repeatable(t):
    def case():
        s = adamw_case([(513,), (70, 33)], t)
        for k in ("masters", "grads", "m", "v"):  # one element into their allocations
            s[k] = [torch.cat([a.new_zeros(1), a.reshape(-1)])[1:].view(a.shape) for a in s[k]]
        s["params"] = [m.to(t) for m in s["masters"]] if t != torch.float32 else s["masters"]
        return s

    a, b, plain = case(), case(), adamw_case([(513,), (70, 33)], t)
    check_adamw(a, 0.5, "unaligned")
    step(b, 0.5)
    step(plain, 0.5)
    for k in ("masters", "params", "m", "v"):
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a[k], b[k], plain[k])), k


def test_adamw_nothing_outside_and_nan():
    base = torch.full((1000,), 3.0, device="cuda")
    s = adamw_case([(100,)], torch.float32)
    s["params"] = s["masters"] = [base[450:550]]
    check_adamw(s, 0.5, "inside")
    assert (base[:450] == 3).all() and (base[550:] == 3).all()
    s["grads"][0][7] = float("nan")  # the norm is a NaN: with clipping every value shows it
    assert math.isnan(step(s, 0.5).item()) and torch.isnan(s["params"][0]).all()


def test_adamw_refusals():
    s = adamw_case(MLP, torch.float32)
    call = lambda **o: policy.adamw_step(**{**dict(params=s["params"], grads=s["grads"], exp_avgs=s["m"], exp_avg_sqs=s["v"], step=s["step"], lr=1e-3), **o})  # noqa: E731
    for over, why in ((dict(masters=s["masters"]), "masters"), (dict(grads=s["grads"][:-1]), "5 grads"), (dict(grads=[g.half() for g in s["grads"]]), "grads: expected"),
                      (dict(exp_avgs=s["v"]), "twice"), (dict(params=s["params"][:1] * 6), "expected|twice"), (dict(step=s["step"].long()), "int32"),
                      (dict(grads=[s["grads"][0].t().contiguous().t(), *s["grads"][1:]]), "contiguous")):
        with pytest.raises(ValueError, match=why):
            call(**over)
    with pytest.raises(RuntimeError, match="beta"):
        call(betas=(1.0, 0.9))
    h = adamw_case(MLP, torch.bfloat16)
    with pytest.raises(ValueError, match="masters"):
        policy.adamw_step(h["params"], h["grads"], h["m"], h["v"], h["step"], lr=1e-3)


def test_operator_refusals():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(3, 8, device="cuda")
    for args, kw, err in (((x, w.half()), {}, TypeError), ((x, w[:, :7]), {}, ValueError), ((x, w, torch.zeros(4, device="cuda")), {}, ValueError), ((x, w, torch.zeros(3)), {}, ValueError),
                          ((x, w), dict(activation="swish"), ValueError), ((x, w), dict(residual=torch.zeros(4, 4, device="cuda")), ValueError),
                          ((x, w), dict(out=torch.zeros(3, 4, device="cuda").t()), ValueError), ((x, w), dict(out=torch.zeros(4, 3, device="cuda", dtype=torch.half)), TypeError),
                          ((x, w.requires_grad_(True)), dict(out=torch.zeros(4, 3, device="cuda")), ValueError)):
        with pytest.raises(err):
            policy.linear(*args, **kw)
    for kw, err in ((dict(block=x[:2]), ValueError), (dict(gate=x), ValueError), (dict(post_weight=x[0]), ValueError), (dict(block=x, gate=x[:2]), ValueError), (dict(block=x, gate=x.half()), TypeError),
                    (dict(pre_weight=x[0][:4]), ValueError), (dict(eps=-1.0), ValueError)):
        with pytest.raises(err):
            policy.norm_residual(x, **kw)
    with pytest.raises(ValueError, match="width"):
        policy.norm_residual(torch.zeros(2, 4097, device="cuda"))
    y = policy.linear(x, w)
    g, = torch.autograd.grad(y, w, torch.ones_like(y).requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---------------------------------------------------------------------------------------------------------------- together


def reference_policy(p, obs):
    """drone_amd.policy.Policy in 64 bits with torch's own layers, on the given parameters by name."""
    act = torch.tanh
    h = act(obs @ p["first.weight"].t() + p["first.bias"])
    k = 0
    while f"hidden.{k}.weight" in p:
        h = act(h @ p[f"hidden.{k}.weight"].t() + p[f"hidden.{k}.bias"])
        k += 1
    if "pre.0" in p:
        norm = lambda a: a / torch.sqrt(a.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
        r, h, k = h, norm(h) * p["pre.0"], 0
        while f"blocks.{k}.weight" in p:
            y = act(h @ p[f"blocks.{k}.weight"].t() + p[f"blocks.{k}.bias"])
            r = r + 0.5 * torch.sigmoid(p[f"gates.{k}"]) * (norm(y) * p[f"post.{k}"])
            h = norm(r) * p[f"pre.{k + 1}"]
            k += 1
    return torch.tanh(h @ p["head.weight"].t() + p["head.bias"])


@pytest.mark.parametrize("blocks", [0, 2])
def test_act_learn_update_together(hip, blocks):
    """The whole loop on one env: collect, loss, gradient, clipped step - and the step's result against the same loop's
    64-bit form. float32, a dozen operators deep: each keeps its relative error around 1e-6 (the tests above), so outputs
    and gradients stay within 1e-4 of their own size, and Adam's first step (m / sqrt(v) = the gradient's sign) is compared
    through the moments."""
    from drone_amd.env import Drone

    torch.manual_seed(0)
    n, K = 1500, 5
    env = Drone(num_envs=n, task="waypoint", device="cuda:0", seed=2, log_interval=0, horizon=30)
    env.reset(2)
    net = policy.Policy(width=64, hidden=1, blocks=blocks, device="cuda:0")
    opt = policy.AdamW(net.parameters(), lr=1e-3, max_grad_norm=0.05)
    obs, act, rew, term, trunc, _ = env.collect(net, K)
    p64 = {k: v.detach().double().requires_grad_(True) for k, v in net.named_parameters()}
    want = reference_policy(p64, obs.double())
    assert (act.double() - want).norm() <= 1e-5 * want.norm()
    target = (rew - rew.mean()).unsqueeze(-1) * 0.1
    loss = (net(obs) - act - target).square().mean()
    opt.zero_grad()
    loss.backward()
    ((reference_policy(p64, obs.double()) - act.double() - target.double()).square().mean()).backward()
    total = math.sqrt(sum(v.grad.square().sum().item() for v in p64.values()))
    for k, v in net.named_parameters():
        assert (v.grad.double() - p64[k].grad).norm().item() <= 1e-4 * total, k
    opt.step()
    assert abs(opt.grad_norm[0].item() - total) <= 1e-4 * total
    clip = min(1.0, 0.05 / (total + 1e-6))
    for k, v in net.named_parameters():
        m = opt.state[v]["exp_avg"].double()
        assert (m - 0.1 * clip * p64[k].grad).norm().item() <= 1e-4 * 0.1 * clip * total, k
        assert (v.detach().double() - p64[k].detach()).abs().max().item() <= 1.1e-3, k  # one step of lr 1e-3 (and its decay)
        assert not torch.equal(v.detach().double(), p64[k].detach()), k
    env.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_collect_is_the_step_loop(oracle, hip, dtype):
    """Drone.collect against the loop it stands for, bit for bit, on a twin env (which itself is held to the oracle), for
    an odd number of envs; the env goes on from where step calls would leave it."""
    from drone_amd.env import Drone

    torch.manual_seed(1)
    n, K, seed = 1001, 6, 5
    net = policy.Policy(width=32, hidden=2, device="cuda:0", dtype=dtype)
    a, b = (Drone(num_envs=n, task="waypoint", device="cuda:0", seed=seed, log_interval=0, horizon=9) for _ in range(2))
    o = oracle.OracleVec(n, seed=seed, cfg=oracle.default_config(1, horizon=9))
    for e in (a, b, o):
        e.reset(seed)
    for _ in range(3):
        obs, act, rew, term, trunc, infos = a.collect(net, K)
        assert infos == []
        for k in range(K):
            assert torch.equal(obs[k], b.observations)
            with torch.no_grad():
                net(b.observations, out=b.actions)
            assert torch.equal(act[k], b.actions)
            b.step(b.actions)
            o.actions[:] = b.actions.cpu().numpy()
            o.step()
            assert torch.equal(rew[k], b.rewards) and torch.equal(term[k], b.terminals) and torch.equal(trunc[k], b.truncations)
            assert (o.rewards == rew[k].cpu().numpy()).all() and (o.observations == b.observations.cpu().numpy()).all()
        for name in ("observations", "actions", "rewards", "terminals", "truncations"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name
        assert a.vec.gstep == b.vec.gstep and a.tick == b.tick
    assert trunc.any()
    with pytest.raises(ValueError, match="at least 1"):
        a.collect(net, 0)
    host = Drone(num_envs=8)
    with pytest.raises(ValueError, match="device buffers"):
        host.collect(net, 2)
    for e in (a, b, host):
        e.close()


def test_other_stream_and_two_calls_at_once():
    """Two streams, each with its own chain of operators and workspaces, give what each gives alone."""
    cases = [linear_case(30000, 64, 64, torch.bfloat16, "silu", seed=10 * k) for k in range(2)]
    alone = [torch.autograd.grad(policy.linear(*c[:3], "silu", c[3]), c[:4], c[4]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(4):
        for k, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[k].append(torch.autograd.grad(policy.linear(*c[:3], "silu", c[3]), c[:4], c[4]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(g, alone[k]))


def test_captured_learning_step_replays():
    """Forward, gradient and optimizer step in one hipGraph, replayed five times with eager work in between, against the
    same five steps run eagerly: the same bits, the step count advancing."""
    def make():
        torch.manual_seed(3)
        net = policy.Policy(width=48, blocks=1, device="cuda:0")
        return net, policy.AdamW(net.parameters(), lr=1e-2, max_grad_norm=0.5)

    obs, goal = rand(2000, 20, seed=1), rand(2000, 4, seed=2).tanh()

    def learn(net, opt, x):
        for p in net.parameters():
            p.grad = None
        y = net(x)
        d = (y.detach() - goal) * (2.0 / y.numel())
        grads = torch.autograd.grad(y, list(net.parameters()), d)
        for p, g in zip(net.parameters(), grads):
            p.grad = g
        opt.step()

    eager, opt_e = make()
    net, opt = make()
    warm, opt_w = make()
    x = obs.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        learn(warm, opt_w, x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        learn(net, opt, x)
    for k in range(5):
        x.copy_(obs + 0.01 * k)
        g.replay()
        torch.cuda.synchronize()
        learn(eager, opt_e, obs + 0.01 * k)
        torch.cuda.synchronize()
        for (name, p), q in zip(net.named_parameters(), eager.parameters()):
            assert torch.equal(p, q), (k, name)
        assert opt.param_groups[0]["step"].item() == opt_e.param_groups[0]["step"].item() == k + 1


def test_optimizer_groups_state_and_skipped_parameters():
    ps = [torch.nn.Parameter(rand(40, 30, to=torch.bfloat16, seed=1)), torch.nn.Parameter(rand(30, to=torch.bfloat16, seed=2)), torch.nn.Parameter(rand(9, seed=3))]
    opt = policy.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 1e-2}], lr=1e-3)
    before = [p.detach().clone() for p in ps]
    ps[0].grad, ps[2].grad = torch.ones_like(ps[0]), torch.ones_like(ps[2])
    opt.step()
    assert torch.equal(ps[1], before[1]) and not torch.equal(ps[0], before[0])
    # (first step on a gradient of ones: lr, and the decay lr 0.01 |p|)
    want = before[2].double() * (1 - 1e-2 * 0.01) - 1e-2
    assert (ps[2].detach().double() - want).abs().max().item() <= 4 * U32 * (before[2].abs().max().item() + 1)
    state = opt.state_dict()
    fresh = policy.AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 1e-2}], lr=1e-3)
    fresh.load_state_dict(state)
    a = [p.detach().clone() for p in ps]
    masters = opt.state[ps[0]]["master"].clone()
    opt.step()
    after = [p.detach().clone() for p in ps]
    with torch.no_grad():
        for p, q in zip(ps, a):
            p.copy_(q)
    assert torch.equal(fresh.state[ps[0]]["master"], masters) and fresh.state[ps[0]]["exp_avg"].dtype == torch.float32
    fresh.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, after))
    with pytest.raises(ValueError, match="one type"):
        policy.AdamW([ps[0], ps[2]])
    late = torch.nn.Parameter(rand(5, seed=8))
    opt.add_param_group({"params": [late]})  # a group added later has its state too
    late.grad = torch.ones_like(late)
    was = late.detach().clone()
    opt.step()
    assert not torch.equal(late, was) and opt.param_groups[2]["step"].item() == 1
