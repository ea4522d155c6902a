"""CPU: what the gated, router and 4-bit entry points refuse before anything touches a GPU, at the C ABI and in Python."""
import ctypes

import pytest
import torch

import triton_grouped_gemm_amd as tgg
from triton_grouped_gemm_amd import _native, ops
from triton_grouped_gemm_amd.gemm.gated import gated_backward, m_grouped_gated_gemm, m_grouped_gated_gemm_projections


@pytest.fixture
def p():
    buf = ctypes.create_string_buffer(4096)
    at = ctypes.addressof(buf)
    yield at + (-at) % 16
    del buf


def refused(word, name, *args):
    assert getattr(_native.load(), name)(*args) == 1
    assert word in _native.last_error(), _native.last_error()


def test_gated_block_c_abi(p):
    good = dict(A=p, B=p, C=p, H=None, sizes=p, i64=0, G=4, M=128, F=64, K=128, tb=1, act=0, dt=0, cu=-1, s=None)
    call = lambda word, **change: refused(word, "tgg_m_grouped_gated_gemm", *{**good, **change}.values())
    call("null", A=None)
    call("null", sizes=None)
    call("G=0", G=0)
    call("G=1025", G=1025)
    call("multiples of 8", F=60)
    call("multiples of 8", K=100)
    call("N=0", F=0)
    call("too large", F=1 << 30)
    call("activation code 2", act=2)
    call("activation code -1", act=-1)
    call("not supported", dt=2)
    call("aligned", C=p + 4)
    call("aligned", H=p + 8)
    call("negative", M=-1)
    good["M"] = 0
    assert _native.load().tgg_m_grouped_gated_gemm(*good.values()) == 0


def test_gated_backward_c_abi(p):
    good = dict(d=p, h=p, dh=p, M=4, F=64, act=1, dt=1, s=None)
    call = lambda word, **change: refused(word, "tgg_gated_backward", *{**good, **change}.values())
    call("null", h=None)
    call("aligned", dh=p + 8)
    call("multiple of 8", F=12)
    call("multiple of 8", F=0)
    call("multiple of 8", M=-1)
    call("not supported", dt=4)
    call("activation code 3", act=3)
    good["M"] = 0
    assert _native.load().tgg_gated_backward(*good.values()) == 0


def test_int4_c_abi(p):
    good = dict(A=p, codes=p, scales=p, zeros=None, C=p, sizes=p, i64=0, G=2, M=8, N=64, K=128, gs=128, act=-1, dt=0, cu=-1, s=None)
    call = lambda word, **change: refused(word, "tgg_m_grouped_gemm_int4", *{**good, **change}.values())
    call("null", codes=None)
    call("null scale", scales=None)
    call("aligned", scales=p + 4)
    call("aligned", A=p + 2)
    call("G=2000", G=2000)
    for gs in (0, 16, 96, 100, -128):
        call("group_size", gs=gs)
    call("multiples of 8", N=60)
    call("multiples of 8", K=60)
    call("multiples of 16", N=48, act=0)
    call("activation code 5", act=5)
    call("not supported", dt=3)
    call("too large", N=1 << 20, K=1 << 14)
    call("does not fit 32 bits", M=1 << 31)
    call("negative", M=-1)
    good["M"] = 0
    assert _native.load().tgg_m_grouped_gemm_int4(*good.values()) == 0


def test_router_c_abi(p):
    forward = dict(l=p, stride=64, T=4, E=64, k=4, scoring=0, renorm=1, dt=0, probs=p, idx=p, s=None)
    call = lambda word, **change: refused(word, "tgg_moe_router", *{**forward, **change}.values())
    call("null", l=None)
    call("null", probs=None)
    call("num_experts=0", E=0)
    call("num_experts=1025", E=1025)
    call("topk=0", k=0)
    call("topk=65", k=65, E=128)
    call("topk=9", k=9, E=8)
    call("scoring code 2", scoring=2)
    call("type code 3", dt=3)
    call("aligned", l=p + 1)
    call("aligned", l=p + 2, dt=2)
    call("negative", T=-1)
    backward = dict(l=p, stride=64, probs=p, idx=p, grad=p, T=4, E=64, k=4, scoring=0, renorm=1, dt=0, out=p, s=None)
    for name in ("probs", "idx", "grad", "out"):
        refused("null", "tgg_moe_router_bwd", *{**backward, name: None}.values())
    forward["T"] = backward["T"] = 0
    assert _native.load().tgg_moe_router(*forward.values()) == 0
    assert _native.load().tgg_moe_router_bwd(*backward.values()) == 0


def test_python_entry_points_want_gpu_tensors_and_known_names():
    a, b, sizes = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(2, 32, 64, dtype=torch.bfloat16), torch.tensor([2, 2])
    for call in (m_grouped_gated_gemm, m_grouped_gated_gemm_projections):
        with pytest.raises(AssertionError, match="GPU"):
            call(a, b, sizes, True)
        with pytest.raises(ValueError, match="activation"):
            call(a, b, sizes, True, "swish")
    with pytest.raises(AssertionError, match="GPU"):
        gated_backward(torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(4, 32))
    with pytest.raises(AssertionError, match="not supported"):
        gated_backward(torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.bfloat16))
    with pytest.raises(AssertionError, match="GPU"):
        ops.gated_gmm(a, b, sizes, trans_b=True)
    with pytest.raises(AssertionError, match="GPU"):
        ops.topk_router(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="scoring"):
        ops.topk_router(torch.zeros(4, 8), 2, scoring="tanh")


def test_aliases():
    tgg.install_aliases()
    import gemm.gated
    import gemm.INT4.m_grouped_gemm_int4 as int4
    from quant.int4_cast import pack_int4
    assert gemm.gated.m_grouped_gated_gemm is m_grouped_gated_gemm
    assert int4.m_grouped_gemm_int4 is tgg.gemm.INT4.m_grouped_gemm_int4.m_grouped_gemm_int4 and callable(pack_int4)
