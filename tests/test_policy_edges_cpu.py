"""The policy operators at the edges of what they allow, without a GPU: refusals that no device is needed for."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from drone_amd import abi, policy
from test_policy_cpu import P, ROOT, native, refused  # noqa: F401


def adamw_call(**over):
    t = (abi.DroneAdamWTensor * 1)(abi.DroneAdamWTensor(P, P, P, P, None, 100))
    c = abi.DroneAdamW(struct_size=C.sizeof(abi.DroneAdamW), count=1, tensors=t, step=P, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, workspace=P, workspace_bytes=1 << 20)
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("bound", [1e-50, 1e-40])
def test_adamw_refuses_a_clip_that_32_bits_cannot_hold(hip, bound):
    """It would become 0, and 0 is no clipping at all."""
    refused(hip, "drone_adamw_step", adamw_call(max_grad_norm=bound), "max_grad_norm")


@pytest.mark.parametrize("bound", [0.0, -1.0, float("nan")])
def test_adamw_step_refuses_a_bound_that_is_not_positive(native, bound):  # noqa: F811
    w = torch.zeros(3)
    with pytest.raises(ValueError, match="max_grad_norm must be positive"):
        policy.adamw_step([w], [w], [w], [w], torch.zeros(1, dtype=torch.int32), lr=1e-3, max_grad_norm=bound)


def test_the_cpython_binding_builds_without_torch():
    """bindings/Makefile: the CPython binding needs gcc alone; the policy operators' module is a target of its own, and part of
    `all` where torch is there."""
    def planned(*args):
        r = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "bindings"), *args], capture_output=True, text=True)
        return r.returncode, "drone_binding.c" in r.stdout, "policy_torch.cpp" in r.stdout

    assert planned() == (0, True, True)
    assert planned("TORCH=") == (0, True, False)
    assert planned("binding") == (0, True, False)
    assert planned("policy") == (0, False, True)
    assert subprocess.run(["make", "-B", "-C", os.path.join(ROOT, "bindings"), "policy", "TORCH="], capture_output=True).returncode != 0
