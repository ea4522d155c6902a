"""The 4-bit weight layout and its quantizer (no GPU needed)."""
import pytest
import torch

from triton_grouped_gemm_amd.gemm.INT4.m_grouped_gemm_int4 import m_grouped_gemm_int4
from triton_grouped_gemm_amd.quant.int4_cast import pack_int4, per_group_cast_to_int4, unpack_int4


@pytest.mark.parametrize("g,n,k", [(1, 8, 8), (2, 16, 128), (3, 40, 200), (1, 72, 640)])
def test_round_trip_and_layout(g, n, k):
    v = torch.randint(0, 16, (g, n, k), generator=torch.Generator().manual_seed(n))
    codes = pack_int4(v)
    assert codes.shape == (g, -(-n // 16), -(-k // 128), 64, 16) and codes.dtype == torch.uint8
    assert torch.equal(unpack_int4(codes, n, k).long(), v)
    # the layout as the header states it, value by value
    for _ in range(50):
        e, c, i = (int(torch.randint(0, hi, (1,))) for hi in (g, n, k))
        s, lg, m = i % 128 // 32, i % 32 // 8, i % 8
        byte, high = {0: (0, 0), 2: (0, 1), 4: (1, 0), 6: (1, 1), 1: (2, 0), 3: (2, 1), 5: (3, 0), 7: (3, 1)}[m]
        b = int(codes[e, c // 16, i // 128, 16 * lg + c % 16, 4 * s + byte])
        assert (b >> 4 if high else b & 15) == v[e, c, i]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("gs,k", [(32, 96), (64, 200), (128, 128), (256, 520)])
def test_quantised_values_are_within_a_step(gs, k, dtype, zeros):
    w = torch.randn(2, 24, k, generator=torch.Generator().manual_seed(k)).to(dtype)
    w[0, 3] = 0
    codes, scales, points = per_group_cast_to_int4(w, gs, zeros)
    assert scales.dtype == (torch.bfloat16 if dtype == torch.float32 else dtype) and (points is not None) == zeros
    spread = lambda t: t.float().repeat_interleave(gs, 1)[:, :k].transpose(1, 2)
    back = (unpack_int4(codes, 24, k).float() - (spread(points) if zeros else 8)) * spread(scales)
    # Half a step of rounding; the scale's own rounding (2^-9 of up to 15 steps, 0.03) and the zero point's (half a step) can push a value past the last
    # code, where it is cut off.
    assert ((back - w.float()).abs() <= spread(scales) * (1.04 if zeros else 0.54)).all()
    assert (back[0, 3] == 0).all()


def test_refusals():
    v = torch.zeros(1, 8, 8, dtype=torch.int32)
    for bad in (v[0], v.float(), v + 16, v - 1, v[:, :0]):
        with pytest.raises(ValueError):
            pack_int4(bad)
    with pytest.raises(ValueError):
        unpack_int4(pack_int4(v), 24, 8)
    w = torch.zeros(1, 8, 64)
    for bad in (lambda: per_group_cast_to_int4(w, 48), lambda: per_group_cast_to_int4(w.double()), lambda: per_group_cast_to_int4(w[0])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("change", ["group", "activation", "codes", "scales", "dtype", "zeros", "sizes", "k", "gated", "cpu"])
def test_the_product_refuses(change):
    n, k, gs = 64, 64, 32
    x = torch.zeros(4, k, dtype=torch.bfloat16)
    codes, scales, zeros = per_group_cast_to_int4(torch.zeros(2, n, k, dtype=torch.bfloat16), gs, True)
    sizes, activation, error = torch.tensor([2, 2]), None, AssertionError
    if change == "group":
        gs, error = 48, ValueError
    elif change == "activation":
        activation, error = "relu", ValueError
    elif change == "codes":
        codes = codes[:, :3]
    elif change == "scales":
        scales = scales[:, :1]
    elif change == "dtype":
        x = x.half()
    elif change == "zeros":
        zeros = zeros.float()
    elif change == "sizes":
        sizes = sizes[:1]
    elif change == "k":
        x = x[:, :60]
    elif change == "gated":
        codes, scales, zeros = per_group_cast_to_int4(torch.zeros(2, 48, k, dtype=torch.bfloat16), gs, True)
        activation = "silu"
    with pytest.raises(error):
        m_grouped_gemm_int4(x, codes, scales, sizes, gs, zeros, activation)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_that_are_trained_give_operands_without_a_graph(dtype, zeros):
    w = torch.randn(2, 24, 96, generator=torch.Generator().manual_seed(1)).to(dtype)
    want = per_group_cast_to_int4(w, 32, zeros)
    got = per_group_cast_to_int4(torch.nn.Parameter(w.clone()), 32, zeros)
    for x, y in zip(got, want):
        assert (x is None) == (y is None)
        assert x is None or (not x.requires_grad and torch.equal(x, y))
