"""CPU: what the Newton-Schulz entry points refuse before anything touches a GPU, at the C ABI and in Python."""
import ctypes

import pytest
import torch

from triton_grouped_gemm_amd import _native, ops


@pytest.fixture
def p():
    buf = ctypes.create_string_buffer(4096)
    at = ctypes.addressof(buf)
    yield at + (-at) % 256
    del buf


def refused(word, name, *args):
    assert getattr(_native.load(), name)(*args) == 1
    assert word in _native.last_error(), _native.last_error()


def workspace(batch, rows, cols):
    need = ctypes.c_int64(-1)
    _native.call("tgg_newton_schulz_workspace_bytes", batch, rows, cols, ctypes.addressof(need))
    return need.value


def test_workspace_holds_the_planes():
    assert workspace(0, 5, 5) == 0
    for batch, rows, cols in ((1, 1, 1), (3, 100, 64), (2, 64, 100), (64, 1536, 2048)):
        few, many = min(rows, cols), max(rows, cols)
        pad = lambda v: -(-v // 8) * 8
        assert workspace(batch, rows, cols) >= batch * few * 2 * 4 * (pad(many) + pad(few))
    need = ctypes.c_int64()
    refused("null", "tgg_newton_schulz_workspace_bytes", 1, 5, 5, None)
    for shape in ((-1, 5, 5), (1, 0, 5), (1, 5, 0)):
        refused("bad stack", "tgg_newton_schulz_workspace_bytes", *shape, ctypes.addressof(need))
    refused("at most 65536", "tgg_newton_schulz_workspace_bytes", 1, 65537, 5, ctypes.addressof(need))
    refused("too large", "tgg_newton_schulz_workspace_bytes", 1 << 31, 8, 8, ctypes.addressof(need))
    # launches of fewer than 2^32 threads, 256 for a block of 64 x 64 values; nothing of a call may run where a later launch of it cannot
    refused("too large", "tgg_newton_schulz_workspace_bytes", 1 << 62, 65536, 65536, ctypes.addressof(need))
    refused("too large", "tgg_newton_schulz_workspace_bytes", 1 << 24, 1, 1, ctypes.addressof(need))
    refused("too large", "tgg_newton_schulz_workspace_bytes", 1 << 14, 65536, 1, ctypes.addressof(need))
    assert workspace((1 << 24) - 1, 1, 1) > 0 and workspace(15, 65536, 65536) > 0


def test_newton_schulz_c_abi(p):
    good = dict(x=p, out=p, batch=2, rows=8, cols=16, steps=5, a=3.0, b=-4.0, c=2.0, eps=0.0, dt=0, ws=p, bytes=1 << 40, s=None)
    call = lambda word, **change: refused(word, "tgg_newton_schulz", *{**good, **change}.values())
    call("null", x=None)
    call("null", out=None)
    call("null", ws=None)
    call("not supported", dt=3)
    call("not supported", dt=-1)
    call("steps=-1", steps=-1)
    call("steps=101", steps=101)
    call("bad stack", rows=0)
    call("at most", cols=1 << 20)
    call("aligned to their type", x=p + 1)
    call("aligned to their type", dt=2, out=p + 2)
    call("256-byte", ws=p + 128)
    call("too small", bytes=workspace(2, 8, 16) - 1)
    good["batch"] = 0
    assert _native.load().tgg_newton_schulz(*good.values()) == 0


def test_muon_c_abi(p):
    good = dict(w=p, wdt=0, g=p, gdt=2, m=p, batch=2, rows=8, cols=16, keep=1.0, step=0.1, beta=0.9, nesterov=1, steps=5, a=3.0, b=-4.0, c=2.0, eps=0.0, ws=p, bytes=1 << 40, s=None)
    call = lambda word, **change: refused(word, "tgg_muon_update", *{**good, **change}.values())
    call("null", w=None)
    call("null", g=None)
    call("null", m=None)
    call("aligned to their type", m=p + 2)
    call("aligned to their type", g=p + 2)
    call("not supported", wdt=4)
    call("not supported", gdt=3)
    call("too small", bytes=0)
    good["batch"] = 0
    assert _native.load().tgg_muon_update(*good.values()) == 0


def test_python_refusals():
    x = torch.zeros(2, 8, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="tensor in bf16"):
        ops.orthogonalize(x.double())
    with pytest.raises(ValueError, match="tensor in bf16"):
        ops.orthogonalize(x[0, 0])
    with pytest.raises(ValueError, match="between 1 and"):
        ops.orthogonalize(x[:, :0])
    with pytest.raises(ValueError, match="steps"):
        ops.orthogonalize(x, steps=-1)
    with pytest.raises(ValueError, match="coefficients"):
        ops.orthogonalize(x, coefficients=(1.0, 2.0))
    with pytest.raises(ValueError, match="coefficients"):
        ops.orthogonalize(x, coefficients=(1.0, float("nan"), 2.0))
    with pytest.raises(ValueError, match="eps"):
        ops.orthogonalize(x, eps=-1.0)
    with pytest.raises(AssertionError, match="no CPU path"):
        ops.orthogonalize(x)
    m = torch.zeros(2, 8, 16)
    with pytest.raises(ValueError, match="momentum must"):
        ops.muon_update(x, x, x, 0.1)
    with pytest.raises(ValueError, match="grad must"):
        ops.muon_update(x, x[:, :4], m, 0.1)
    with pytest.raises(ValueError, match="contiguous"):
        ops.muon_update(x.transpose(1, 2), x.transpose(1, 2), m.transpose(1, 2), 0.1)
    with pytest.raises(ValueError, match="finite"):
        ops.muon_update(x, x, m, float("inf"))
    with pytest.raises(AssertionError, match="no CPU path"):
        ops.muon_update(x, x, m, 0.1)


def test_shapes_under_tracing():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 16, 8, dtype=torch.float16, device="cuda").transpose(1, 2)
        out = torch.ops.moe.orthogonalize(x, 5, 3.0, -4.0, 2.0, 1e-7)
        assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous()
