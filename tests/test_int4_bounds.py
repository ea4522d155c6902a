"""``m_grouped_gemm_int4`` under bounds that a wrong tail of K, scale or zero point does not pass (first the bounds themselves, on the CPU)."""
import pytest
import torch

from _int4 import check, make, reference
from triton_grouped_gemm_amd.gemm.INT4.m_grouped_gemm_int4 import m_grouped_gemm_int4
from triton_grouped_gemm_amd.quant.int4_cast import pack_int4

KINDS = [(torch.bfloat16, 128, False), (torch.bfloat16, 128, True), (torch.bfloat16, 64, True), (torch.bfloat16, 32, False), (torch.float16, 128, False),
         (torch.float16, 32, True)]
IDS = ["bf16_128", "bf16_128z", "bf16_64z", "bf16_32", "fp16_128", "fp16_32z"]


def rounded(x, q, scales, points, sizes, gs, kind=None):
    return reference(x, q, scales, points, sizes, gs, kind)[0].to(x.dtype)


@pytest.mark.parametrize("dtype,gs,zeros", KINDS, ids=IDS)
@pytest.mark.parametrize("k", [264, 1032, 3088, 4112])
def test_the_bounds_reject_what_is_wrong(k, dtype, gs, zeros):
    sizes, n = [16, 40], 72
    x, q, scales, points = make(sizes, n, k, gs, zeros, dtype, k)
    want, slack = reference(x, q, scales, points, sizes, gs, None)
    check(want.to(dtype), want, slack)
    tail = x.clone()
    tail[:, -8:] = 0
    wrong = {"the last eight values of K left out": rounded(tail, q, scales, points, sizes, gs)}
    lost = scales.clone()
    lost[:, -1] = 0
    wrong["the last scale group left out"] = rounded(x, q, lost, points, sizes, gs)
    if zeros:
        moved = points.clone()
        moved[:, -1] = torch.where(moved[:, -1] < 15, moved[:, -1] + 1, moved[:, -1] - 1)
        wrong["the last zero points off by one"] = rounded(x, q, scales, moved, sizes, gs)
    shifted = torch.cat([scales[:, 1:], scales[:, :1]], 1)
    wrong["scales one group off"] = rounded(x, q, shifted, points, sizes, gs)
    noise = torch.randn(want.shape, generator=torch.Generator().manual_seed(1)).double()
    wrong["a hundredth of noise"] = (want + 0.01 * noise * want.norm() / want.numel() ** 0.5).to(dtype)
    one = want.to(dtype)
    one[3, 5] += want.std().to(dtype)
    wrong["one output off by a standard deviation"] = one
    wrong["nothing"] = torch.zeros_like(one)
    for what, got in wrong.items():
        with pytest.raises(AssertionError, match="off by"):
            check(got, want, slack)
            pytest.fail(what + " passes")


CASES = [
    # sizes, n, k, gs, zeros, dtype, activation
    ([1], 32, 32, 32, True, torch.float16, "silu"),
    ([3, 17, 0, 16], 64, 264, 32, False, torch.float16, "gelu_tanh"),
    ([33, 1, 65], 96, 256, 128, False, torch.bfloat16, "silu"),
    ([64, 0, 130], 72, 520, 64, False, torch.bfloat16, None),
    ([31, 48], 1544, 96, 32, True, torch.bfloat16, None),
    ([5], 200, 1000, 256, True, torch.float16, None),
    ([5, 60], 200, 1000, 384, True, torch.bfloat16, None),
    ([200, 2], 64, 640, 128, True, torch.bfloat16, "gelu_tanh"),
    ([1] * 8, 1536, 2048, 128, False, torch.bfloat16, "silu"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[f"{len(c[0])}g{sum(c[0])}r_n{c[1]}_k{c[2]}_gs{c[3]}{'z' if c[4] else ''}{c[6] or ''}" for c in CASES])
def test_cases(dev, case):
    sizes, n, k, gs, zeros, dtype, kind = case
    x, q, scales, points = make(sizes, n, k, gs, zeros, dtype, n + k)
    want, slack = reference(x, q, scales, points, sizes, gs, kind)
    z = None if points is None else points.to(dev)
    for cap in (-1, 3):
        check(m_grouped_gemm_int4(x.to(dev), pack_int4(q.to(dev)), scales.to(dev), torch.tensor(sizes, device=dev), gs, z, kind, numSM=cap), want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gs,zeros", KINDS, ids=IDS)
@pytest.mark.parametrize("k", [256, 264, 768, 1024, 1032, 1544, 2176, 3088, 4112])
def test_lengths_around_the_chunks_of_activations(dev, k, dtype, gs, zeros):
    """Tiles of up to 16, 32, 48 and 64 rows, whose activations pass through shared memory 1024, 512 and 256 values at a time, in each width of tile: 7 row
    tiles are split along K on a whole GPU, take 128 columns a tile on 16 workgroups, 256 on 8 and fewer."""
    sizes, n = [16, 64, 2, 32, 48, 77], 264
    x, q, scales, points = make(sizes, n, k, gs, zeros, dtype, k)
    want, slack = reference(x, q, scales, points, sizes, gs, None)
    args = (x.to(dev), pack_int4(q.to(dev)), scales.to(dev), torch.tensor(sizes, dtype=torch.int32, device=dev), gs, None if points is None else points.to(dev))
    for cap in (-1, 16, 8, 3):
        check(m_grouped_gemm_int4(*args, numSM=cap), want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gs,zeros,kind", [(torch.bfloat16, 128, False, "silu"), (torch.bfloat16, 32, True, "gelu_tanh"), (torch.float16, 64, True, "silu"),
                                                 (torch.float16, 128, False, "gelu_tanh")], ids=["bf16_128", "bf16_32z", "fp16_64z", "fp16_128"])
@pytest.mark.parametrize("n", [288, 416])
@pytest.mark.parametrize("k", [256, 264, 1032])
def test_gated_tiles_of_many_rows_and_columns(dev, k, n, dtype, gs, zeros, kind):
    """Gate and up columns of every width of tile, several tiles of columns, the last one cut: 144 and 208 outputs are no whole tile of 32, 64 or 128.  Tiles
    of more than 32 rows are worked on as two half tiles of 64 outputs where they are 256 columns wide (14 of them: up to 14 workgroups), as two halves of
    their rows where they are split along K (a whole GPU)."""
    sizes = [16, 64, 2, 32, 48, 77]
    x, q, scales, points = make(sizes, n, k, gs, zeros, dtype, k + n)
    want, slack = reference(x, q, scales, points, sizes, gs, kind)
    args = (x.to(dev), pack_int4(q.to(dev)), scales.to(dev), torch.tensor(sizes, dtype=torch.int32, device=dev), gs, None if points is None else points.to(dev), kind)
    for cap in (-1, 20, 14, 3):
        check(m_grouped_gemm_int4(*args, numSM=cap), want, slack)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gs", [32, 64, 128])
def test_every_code_with_every_zero_point(dev, gs, dtype):
    """q - z for all q and z in 0..15 in every place of a block, exact: rows of the identity, scales of one."""
    k, n = 128, 256
    q = torch.arange(n)[:, None].expand(n, k) % 16
    points = (torch.arange(n) // 16).to(torch.uint8)
    args = (torch.eye(k, dtype=dtype, device=dev), pack_int4(q[None].to(dev)), torch.ones(1, k // gs, n, dtype=dtype, device=dev), torch.tensor([k], device=dev), gs)
    got = m_grouped_gemm_int4(*args, points.expand(1, k // gs, n).contiguous().to(dev))
    assert torch.equal(got.float().cpu(), (q.t() - points.float()))
    assert torch.equal(m_grouped_gemm_int4(*args).float().cpu(), q.t() - 8.0)
