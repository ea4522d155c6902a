"""The adapter operators as operators of torch's: what others register for them is what runs, eagerly too, and the profiler shows them."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from _lora import make
from triton_grouped_gemm_amd import _native, ops

NAMES = ("lora_linear", "lora_linear_hidden", "lora_linear_backward")


def test_an_implementation_for_all_devices_takes_the_native_path_out():
    """In a process of its own: registrations last."""
    code = f"""
import torch
from triton_grouped_gemm_amd import _native, lora, ops
for name in {NAMES}:
    op = torch._library.custom_ops._maybe_get_opdef('moe::' + name)
    assert isinstance(op, _native.EagerOp) and not op.replaced, name
    torch.library.register_kernel('moe::' + name, None, lambda x, *rest: x + 3)
    assert op.replaced, name
class Host:  # the native path must not be asked
    def __getattr__(self, name):
        raise AssertionError(name)
_native._host = Host()
lora.require_gpu = lambda *tensors: None
z = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16)
assert ops.lora_linear(z(4, 8), z(8, 8), z(2, 8, 8), z(2, 8, 8), torch.zeros(4, dtype=torch.int32)).eq(3).all()
print("checked")
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=Path(_native.__file__).parents[1], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "checked" in run.stdout, run.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("key", ["CUDA", "AutocastCUDA", "AutogradCUDA"])
def test_what_others_register_is_what_runs(dev, key):
    x, w, a, b, _, adapters, s = make(20, 64, 64, 8, 3, torch.bfloat16, 0, dev)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=key == "AutocastCUDA"), torch.library._scoped_library("moe", "IMPL") as moe:
        moe.impl("lora_linear", lambda x, *rest: x.new_full((2,), 7.0), key)
        assert ops.lora_linear(x, w, a, b, adapters, s).tolist() == [7.0] * 2
    assert ops.lora_linear(x, w, a, b, adapters, s).shape == (20, 64)


@pytest.mark.gpu
def test_profiles_show_the_operators(dev):
    x, w, a, b, g, adapters, s = make(20, 64, 64, 8, 3, torch.bfloat16, 1, dev)
    leaf = a.clone().requires_grad_(True)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as profile:
        ops.lora_linear(x, w, a, b, adapters, s)
        ops.lora_linear(x, w, leaf, b, adapters, s).backward(g)
    seen = {event.key for event in profile.key_averages()}
    assert {"moe::" + name for name in NAMES} <= seen, sorted(seen)
