"""The policy operators' boundary without a GPU: struct layouts, refusals, what Python checks before a call."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from drone_amd import abi, policy

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = (("DroneLinear", abi.DroneLinear), ("DroneNorm", abi.DroneNorm), ("DroneAdamWTensor", abi.DroneAdamWTensor), ("DroneAdamW", abi.DroneAdamW))


def test_call_structs_match_the_header(tmp_path):
    lines = []
    for name, cls in STRUCTS:
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _t in cls._fields_]
    lines += [f'printf("{n} %d\\n", {n});' for n in ("DRONE_F32", "DRONE_BF16", "DRONE_F16")]
    lines += [f'printf("DRONE_ACTIVATION_{n} %d\\n", DRONE_ACTIVATION_{n});' for n in ("NONE", "RELU", "TANH", "SILU", "GELU")]
    (tmp_path / "l.c").write_text('#include <stdio.h>\n#include "drone_vec.h"\nint main(void){' + "".join(lines) + "return 0;}")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = {k: int(v) for k, v in (l.split() for l in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines())}
    for name, cls in STRUCTS:
        assert got[name] == C.sizeof(cls), name
        for f, _t in cls._fields_:
            assert got[f"{name}.{f}"] == getattr(cls, f).offset, f"{name}.{f}"
    assert (got["DRONE_F32"], got["DRONE_BF16"], got["DRONE_F16"]) == (abi.F32, abi.BF16, abi.F16)
    assert {n.lower(): got[f"DRONE_ACTIVATION_{n}"] for n in ("NONE", "RELU", "TANH", "SILU", "GELU")} == abi.ACTIVATIONS


P = 1 << 20  # a made-up, aligned address: every call below is refused before anything reads it


def linear_call(**over):
    c = abi.DroneLinear(struct_size=C.sizeof(abi.DroneLinear), rows=8, in_features=16, out_features=32, x=P, weight=P, y=P, dy=P, slope=P, dx=P, dweight=P, dbias=P,
                        x_ld=16, weight_ld=16, y_ld=32, dy_ld=32, dx_ld=16, activation=1)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def refused(hip, name, call, why):
    rc = hip.functions()[name](C.byref(call) if call is not None else None, None)
    assert rc == -1 and why in hip.last_error(), (rc, hip.last_error())


@pytest.mark.parametrize("over, why", [
    (dict(struct_size=8), "struct_size"), (dict(dtype=3), "unknown dtype"), (dict(activation=5), "unknown activation"), (dict(activation=-1), "unknown activation"),
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(in_features=0), "in_features"), (dict(out_features=65537), "out_features"),
    (dict(x=None), "must not be NULL"), (dict(weight=None), "must not be NULL"), (dict(y=None), "must not be NULL"),
    (dict(x_ld=15), "leading dimension"), (dict(weight_ld=15), "leading dimension"), (dict(y_ld=31), "leading dimension"), (dict(residual=P, residual_ld=31), "leading dimension"),
    (dict(x=P + 2), "not aligned"), (dict(bias=P + 1), "not aligned"), (dict(slope=P + 2), "not aligned")])
def test_linear_forward_refuses(hip, over, why):
    refused(hip, "drone_linear_forward", linear_call(**over), why)


@pytest.mark.parametrize("over, why", [
    (dict(dy=None), "dy is NULL"), (dict(slope=None), "slope"), (dict(weight=None), "needs the weight"), (dict(x=None), "need x"),
    (dict(dy_ld=31), "leading dimension"), (dict(dx_ld=15), "leading dimension"), (dict(dx=P + 2), "not aligned"),
    (dict(workspace=None), "drone_linear_workspace"), (dict(workspace=P, workspace_bytes=16), "drone_linear_workspace"), (dict(workspace=P + 4, workspace_bytes=1 << 30), "drone_linear_workspace")])
def test_linear_backward_refuses(hip, over, why):
    refused(hip, "drone_linear_backward", linear_call(**over), why)


def norm_call(**over):
    c = abi.DroneNorm(struct_size=C.sizeof(abi.DroneNorm), gate_kind=1, rows=8, width=32, x=P, block=P, gate=P, h=P, r=P, x_ld=32, block_ld=32, scale=1.0, eps=1e-6)
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("over, why", [
    (dict(struct_size=8), "struct_size"), (dict(dtype=7), "unknown dtype"), (dict(gate_kind=3), "gate_kind"), (dict(rows=-1), "rows"), (dict(width=0), "width"), (dict(width=4097), "width"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(gate=None), "gate is NULL"), (dict(block=None), "needs a block"), (dict(x=None), "x is NULL"), (dict(h=None), "h is NULL"),
    (dict(x_ld=31), "leading dimension"), (dict(block_ld=31), "leading dimension"), (dict(gate_kind=2, gate_ld=31), "leading dimension"), (dict(pre_weight=P + 2), "not aligned")])
def test_norm_forward_refuses(hip, over, why):
    refused(hip, "drone_norm_forward", norm_call(**over), why)


@pytest.mark.parametrize("over, why", [
    (dict(block=None, gate=None, gate_kind=0, dblock=P), "no block"), (dict(gate_kind=0, dgate=P), "no gate"), (dict(dpre_weight=P), "drone_norm_workspace"),
    (dict(dgate=P, workspace=P, workspace_bytes=4), "drone_norm_workspace"), (dict(dh=P + 1), "not aligned")])
def test_norm_backward_refuses(hip, over, why):
    refused(hip, "drone_norm_backward", norm_call(**over), why)


@pytest.mark.parametrize("over, tensor, why", [
    (dict(struct_size=8), {}, "struct_size"), (dict(dtype=9), {}, "unknown dtype"), (dict(count=-1), {}, "tensors"), (dict(tensors=None), {}, "tensors"),
    (dict(step=None), {}, "step"), (dict(step=P + 1), {}, "step"), (dict(beta1=1.0), {}, "beta"), (dict(beta2=-0.1), {}, "beta"), (dict(beta2=float("nan")), {}, "beta"),
    (dict(lr=-1.0), {}, "lr"), (dict(eps=float("nan")), {}, "eps"), (dict(eps=0.0), {}, "eps"), (dict(eps=1e-46), {}, "eps"), (dict(weight_decay=-1.0), {}, "weight_decay"), (dict(max_grad_norm=float("nan")), {}, "max_grad_norm"),
    ({}, dict(elements=-1), "elements"), ({}, dict(elements=1 << 41), "elements"), ({}, dict(grad=None), "NULL"), ({}, dict(master=P), "master"), (dict(dtype=1), {}, "master"),
    ({}, dict(exp_avg=P + 2), "not aligned"), (dict(workspace=None), {}, "drone_adamw_workspace"), (dict(workspace_bytes=8), {}, "drone_adamw_workspace")])
def test_adamw_refuses(hip, over, tensor, why):
    t = (abi.DroneAdamWTensor * 1)(abi.DroneAdamWTensor(P, P, P, P, None, 100))
    for k, v in tensor.items():
        setattr(t[0], k, v)
    c = abi.DroneAdamW(struct_size=C.sizeof(abi.DroneAdamW), count=1, tensors=t, step=P, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, workspace=P, workspace_bytes=1 << 20)
    for k, v in over.items():
        setattr(c, k, v)
    refused(hip, "drone_adamw_step", c, why)


def test_null_calls_are_refused(hip):
    for name in ("drone_linear_forward", "drone_linear_backward", "drone_norm_forward", "drone_norm_backward", "drone_adamw_step"):
        refused(hip, name, None, "call is NULL")
    for name in ("drone_linear_workspace", "drone_norm_workspace", "drone_adamw_workspace"):
        assert hip.functions()[name](None) == 0 and "call is NULL" in hip.last_error()


def test_empty_calls_do_nothing(hip):
    """No rows: nothing to write, so no pointer is needed and no device touched."""
    f = hip.functions()
    assert f["drone_linear_forward"](C.byref(linear_call(rows=0, x=None, y=None)), None) == 0
    assert f["drone_norm_forward"](C.byref(norm_call(rows=0, x=None, h=None)), None) == 0
    assert f["drone_linear_backward"](C.byref(linear_call(dx=None, dweight=None, dbias=None)), None) == 0


@pytest.fixture(scope="module")
def native(hip):
    """The compiled module (bindings/policy_torch.cpp): git-ignored like the library, built where it is missing."""
    if not any(f.startswith("policy_torch") for f in os.listdir(os.path.join(ROOT, "drone_amd"))):
        subprocess.run(["make", "-C", os.path.join(ROOT, "bindings")], check=True, capture_output=True)
    return policy._native()


def test_cpu_tensors_are_refused(native):
    x, w = torch.zeros(4, 8), torch.zeros(3, 8)
    with pytest.raises(ValueError, match="GPU only"):
        policy.linear(x, w)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        policy.linear(x.double(), w.double())
    with pytest.raises(ValueError, match="GPU only"):
        policy.norm_residual(x)
    with pytest.raises(ValueError, match="GPU only"):
        policy.adamw_step([w], [w], [w], [w], torch.zeros(1, dtype=torch.int32), lr=1e-3)
    with pytest.raises(ValueError, match="no parameters"):
        policy.adamw_step([], [], [], [], torch.zeros(1, dtype=torch.int32), lr=1e-3)
    with pytest.raises(ValueError, match="unknown activation"):
        policy.Linear(4, 4, "swish")
    with pytest.raises(ValueError, match="must not be negative"):
        policy.AdamW([torch.nn.Parameter(w)], lr=-1.0)
    with pytest.raises(ValueError, match="must be positive"):
        policy.AdamW([torch.nn.Parameter(w)], max_grad_norm=0.0)
    for eps in (0.0, -1e-8, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            policy.AdamW([torch.nn.Parameter(w)], eps=eps)
