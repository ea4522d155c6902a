"""The router, gated and 4-bit operators as operators of torch's: what others register for them is what runs, eagerly too, and the
profiler shows them."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from triton_grouped_gemm_amd import _native, ops
from triton_grouped_gemm_amd.gemm.gated import gated_backward, m_grouped_gated_gemm, m_grouped_gated_gemm_projections
from triton_grouped_gemm_amd.gemm.INT4.m_grouped_gemm_int4 import m_grouped_gemm_int4
from triton_grouped_gemm_amd.quant.int4_cast import per_group_cast_to_int4


def test_an_implementation_for_all_devices_takes_the_native_path_out():
    """In a process of its own: registrations last."""
    code = """
import torch
from triton_grouped_gemm_amd import _native, ops
from triton_grouped_gemm_amd.gemm.gated import gated_backward, m_grouped_gated_gemm, m_grouped_gated_gemm_projections
from triton_grouped_gemm_amd.gemm.INT4.m_grouped_gemm_int4 import m_grouped_gemm_int4
names = ('topk_router', 'topk_router_backward', 'm_grouped_gated_gemm', 'm_grouped_gated_gemm_projections', 'gated_backward', 'm_grouped_gemm_int4')
for name in names:
    op = torch._library.custom_ops._maybe_get_opdef('moe::' + name)
    assert isinstance(op, _native.EagerOp) and not op.replaced, name
    op.register_kernel('cpu')(lambda x, *rest: (x + 1, x + 2))
    assert not op.replaced, name
    torch.library.register_kernel('moe::' + name, None, lambda x, *rest: x + 3)
    assert op.replaced, name
class Host:  # the native path must not be asked
    def __getattr__(self, name):
        raise AssertionError(name)
_native._host = Host()
ops.require_gpu = lambda *tensors: None
assert ops.topk_router(torch.zeros(4, 8), 2)[1].eq(2).all()
print("checked")
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=Path(_native.__file__).parents[1], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "checked" in run.stdout, run.stderr[-2000:]


def _operands(dev):
    a, b = torch.randn(20, 64, device=dev).to(torch.bfloat16), torch.randn(4, 64, 64, device=dev).to(torch.bfloat16)
    codes, scales, _ = per_group_cast_to_int4(b, 32)
    return a, b, torch.tensor([5, 0, 9, 6], device=dev), codes, scales, torch.randn(20, 32, device=dev).to(torch.bfloat16), torch.randn(20, 64, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("key", ["CUDA", "AutocastCUDA", "AutogradCUDA"])
def test_what_others_register_is_what_runs(dev, key):
    a, b, sizes, codes, scales, grad, h = _operands(dev)
    logits = torch.randn(20, 16, device=dev)
    calls = {"m_grouped_gated_gemm": lambda: m_grouped_gated_gemm(a, b, sizes, True),
             "m_grouped_gated_gemm_projections": lambda: m_grouped_gated_gemm_projections(a, b, sizes, True),
             "gated_backward": lambda: gated_backward(grad, h),
             "m_grouped_gemm_int4": lambda: m_grouped_gemm_int4(a, codes, scales, sizes, 32),
             "topk_router": lambda: ops.topk_router(logits, 3)}
    two = lambda x, *rest: (x.new_full((2,), 7.0), x.new_full((3,), 8.0))
    one = lambda x, *rest: x.new_full((2,), 7.0)
    several = lambda out: out if isinstance(out, (tuple, list)) else (out,)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=key == "AutocastCUDA"):
        plain = {name: several(call()) for name, call in calls.items()}
        with torch.library._scoped_library("moe", "IMPL") as moe:
            for name in calls:
                moe.impl(name, two if len(plain[name]) == 2 else one, key)
            for name, call in calls.items():
                assert several(call())[0].tolist() == [7.0] * 2, name
            assert ops.gated_gmm(a, b, sizes, trans_b=True).tolist() == [7.0] * 2
        for name, call in calls.items():
            assert all(torch.equal(x[:5], y[:5]) for x, y in zip(several(call()), plain[name])), name


@pytest.mark.gpu
def test_what_others_register_for_the_router_s_gradient_is_what_runs(dev):
    logits = torch.randn(6, 16, device=dev, requires_grad=True)
    grad = torch.randn(6, 3, device=dev)
    gradient = lambda: torch.autograd.grad(ops.topk_router(logits, 3)[0], logits, grad)[0]
    plain = gradient()
    with torch.library._scoped_library("moe", "IMPL") as moe:
        moe.impl("topk_router_backward", lambda x, *rest: torch.full_like(x, 5.0), "CUDA")
        assert torch.equal(gradient(), torch.full_like(logits, 5.0))
    assert torch.equal(gradient(), plain)


@pytest.mark.gpu
def test_the_profiler_shows_the_operators(dev):
    a, b, sizes, codes, scales, grad, h = _operands(dev)
    logits = torch.randn(20, 16, device=dev)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU], record_shapes=True) as seen:
        m_grouped_gated_gemm(a, b, sizes, True)
        m_grouped_gated_gemm_projections(a, b, sizes, True)
        gated_backward(grad, h)
        m_grouped_gemm_int4(a, codes, scales, sizes, 32)
        ops.topk_router(logits, 3)
        probs, _ = ops.topk_router(logits[:9].requires_grad_(True), 3)
        probs.sum().backward()
    shapes = {}
    for e in seen.events():
        shapes.setdefault(e.name, []).append(e.input_shapes)
    assert shapes["moe::m_grouped_gated_gemm"][0][:2] == [[20, 64], [4, 64, 64]]
    assert shapes["moe::m_grouped_gated_gemm_projections"][0][:2] == [[20, 64], [4, 64, 64]]
    assert shapes["moe::gated_backward"][0][:2] == [[20, 32], [20, 64]]
    assert shapes["moe::m_grouped_gemm_int4"][0][:2] == [[20, 64], list(codes.shape)]
    assert [s[0] for s in shapes["moe::topk_router"]] == [[20, 16], [9, 16]]
    assert shapes["moe::topk_router_backward"][0][:3] == [[9, 16], [9, 3], [9, 3]]


@pytest.mark.gpu
def test_the_router_s_gradient_with_saved_tensors_elsewhere(dev):
    """Hooks of saved tensors are Python; the native record runs without the interpreter lock."""
    logits, grad = torch.randn(300, 64, device=dev, requires_grad=True), torch.randn(300, 6, device=dev)
    want = torch.autograd.grad(ops.topk_router(logits, 6)[0], logits, grad)[0]
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t.cpu(), lambda t: t.to(dev)):
        probs, _ = ops.topk_router(logits, 6)
    assert len(packed) == 3
    assert torch.equal(torch.autograd.grad(probs, logits, grad)[0], want)
    got = torch.utils.checkpoint.checkpoint(lambda t: ops.topk_router(t, 6)[0], logits, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(got, logits, grad)[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True)])
def test_what_hooks_of_saved_tensors_give_back(dev, scoring, renormalize):
    """Other strides are the same values; another device, type or shape is refused, before the launch where the kernel could read out of range."""
    logits, grad = torch.randn(40, 24, device=dev, requires_grad=True), torch.randn(40, 3, device=dev)

    def gradient(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
            probs, _ = ops.topk_router(logits, 3, scoring=scoring, renormalize=renormalize)
        return torch.autograd.grad(probs, logits, grad)[0]

    want = gradient(lambda t: t)
    assert torch.equal(gradient(lambda t: t.t().contiguous().t()), want)
    wide = lambda t: torch.cat([t, t], 1)[:, :t.shape[1]]
    assert torch.equal(gradient(wide), want)
    for unpack in (lambda t: t.cpu(), lambda t: t.cpu() if t.dtype is torch.int32 else t):
        with pytest.raises(RuntimeError, match="must be on cuda"):
            gradient(unpack)
    for unpack in (lambda t: t.double(), lambda t: t[:39], lambda t: t[:, :2] if t.shape[1] == 3 else t, lambda t: t.long() if t.dtype is torch.int32 else t,
                   lambda t: t.reshape(-1)):
        with pytest.raises(RuntimeError, match="changed in shape or type"):
            gradient(unpack)
    with pytest.raises(RuntimeError, match="invalid gradient"):
        gradient(lambda t: t[:, :20] if t.shape[1] == 24 else t)
