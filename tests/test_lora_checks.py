"""CPU: what the adapter entry points refuse before anything touches a GPU, at the C ABI and in Python."""
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


def test_c_abi_forward(p):
    good = dict(x=p, w=p, a=p, b=p, ids=p, i64=0, scales=None, out=p, h=None, M=4, N=64, K=128, R=8, L=2, dt=0, ws=p, bytes=1 << 40, s=None)
    call = lambda word, **change: refused(word, "tgg_lora_linear", *{**good, **change}.values())
    for name in ("x", "w", "a", "b", "ids", "out", "ws"):
        call("null", **{name: None})
    call("multiples of 8", N=60)
    call("multiples of 8", K=0)
    call("at most 65536", K=65544)
    call("rank", R=4)
    call("rank", R=136)
    call("rank", R=0)
    call("L=0", L=0)
    call("L=1025", L=1025)
    call("M=-1", M=-1)
    call("M=2147483648", M=1 << 31)
    call("M=134217728", M=1 << 27)  # 512 threads for 16 rows, and fewer than 2^32 in a launch
    call("not supported", dt=2)
    call("16-byte aligned", x=p + 8)
    call("16-byte aligned", h=p + 8)
    call("aligned to their type", ids=p + 2)
    call("aligned to their type", i64=1, ids=p + 4)
    call("aligned to their type", scales=p + 2)
    call("256-byte", ws=p + 16)
    call("too small", bytes=100)
    good["M"] = 0
    assert _native.load().tgg_lora_linear(*good.values()) == 0


def test_c_abi_backward(p):
    good = dict(g=p, x=p, w=p, a=p, b=p, ids=p, i64=0, scales=None, h=p, dx=p, da=p, db=p, M=4, N=64, K=128, R=8, L=2, dt=0, ws=p, bytes=1 << 40, s=None)
    call = lambda word, **change: refused(word, "tgg_lora_linear_bwd", *{**good, **change}.values())
    for name in ("g", "x", "w", "a", "b", "ids", "h", "ws"):
        call("null", **{name: None})
    call("16-byte aligned", da=p + 8)
    call("rank", R=12)
    call("too small", bytes=100)
    good["M"] = 0
    assert _native.load().tgg_lora_linear_bwd(*good.values()) == 0


def test_workspace_bytes(p):
    need = ctypes.c_int64(-1)
    at = ctypes.addressof(need)
    refused("null", "tgg_lora_workspace_bytes", 0, 4, 64, 128, 8, 2, None)
    refused("rank", "tgg_lora_workspace_bytes", 0, 4, 64, 128, 9, 2, at)
    _native.call("tgg_lora_workspace_bytes", 0, 0, 64, 128, 8, 2, at)
    assert need.value == 0
    _native.call("tgg_lora_workspace_bytes", 0, 4, 64, 128, 8, 2, at)
    forward = need.value
    _native.call("tgg_lora_workspace_bytes", 1, 4, 64, 128, 8, 2, at)
    assert need.value > 0 and forward > 0


def test_python_refusals():
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(24, 16, dtype=torch.bfloat16)
    a, b = torch.zeros(3, 8, 16, dtype=torch.bfloat16), torch.zeros(3, 24, 8, dtype=torch.bfloat16)
    ids = torch.zeros(4, dtype=torch.int32)

    def call(match, kind=ValueError, **change):
        args = {**dict(x=x, weight=w, lora_a=a, lora_b=b, adapters=ids, scales=None), **change}
        with pytest.raises(kind, match=match):
            ops.lora_linear(**args)

    call("x must be", x=x[0])
    call("x must be", weight=w[:, :8])
    call("x must be", lora_b=b[:, :16])
    call("x must be", lora_b=b[:2])
    call("not supported", x=x.float(), weight=w.float(), lora_a=a.float(), lora_b=b.float())
    call("share one data type", lora_a=a.half())
    call("multiples of 8", weight=w[:20], lora_b=b[:, :20])
    call("rank", lora_a=a[:, :4], lora_b=b[:, :, :4])
    call("number of adapters", lora_a=a[:0], lora_b=b[:0])
    call("adapters must", adapters=ids[:3])
    call("adapters must", adapters=ids.float())
    call("scales must", scales=torch.ones(2))
    call("scales must", scales=torch.ones(3, dtype=torch.float64))
    call("not differentiable", scales=torch.ones(3, requires_grad=True))
    call("no CPU path", AssertionError)


def test_shapes_under_tracing():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(4, 16, dtype=torch.float16, device="cuda"), torch.empty(24, 16, dtype=torch.float16, device="cuda")
        a, b = torch.empty(3, 8, 16, dtype=torch.float16, device="cuda"), torch.empty(3, 24, 8, dtype=torch.float16, device="cuda")
        ids = torch.empty(4, dtype=torch.int32, device="cuda")
        out, h = torch.ops.moe.lora_linear_hidden(x, w, a, b, ids, None)
        assert out.shape == (4, 24) and out.dtype == x.dtype and h.shape == (4, 8) and h.dtype == torch.float32
        dx, da, db = torch.ops.moe.lora_linear_backward(out, x, w, a, b, ids, None, h, True, False, True)
        assert dx.shape == x.shape and da.numel() == 0 and db.shape == b.shape
