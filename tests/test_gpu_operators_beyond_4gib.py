"""Offsets past 32 bits: the gated block, its backward pass, the 4-bit product and the router on operands and results of more than
4 GiB, looked at in sampled rows at both ends and beyond the 4 GiB line.  Bounds as in the operators' own tests."""
import pytest
import torch

from triton_grouped_gemm_amd import ops
from triton_grouped_gemm_amd.gemm.INT4.m_grouped_gemm_int4 import m_grouped_gemm_int4
from triton_grouped_gemm_amd.gemm.gated import gated_backward, m_grouped_gated_gemm, m_grouped_gated_gemm_projections
from triton_grouped_gemm_amd.quant.int4_cast import pack_int4

pytestmark = pytest.mark.gpu

ROWS, F, K = 1_500_003, 1536, 64
SAMPLE = [0, 1, 699_050, 699_051, 1_000_000, 1_398_101, ROWS - 2, ROWS - 1]
SIZES = [700_000, 3, 800_000]


def group_of(row):
    return 0 if row < SIZES[0] else 1 if row < SIZES[0] + SIZES[1] else 2


@pytest.fixture(autouse=True)
def room(dev):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of GPU memory")
    yield
    torch.cuda.empty_cache()


def test_gated_block_and_its_backward_pass(dev):
    gen = torch.Generator(device=dev).manual_seed(1)
    a = torch.randn(ROWS, K, generator=gen, device=dev).to(torch.bfloat16)
    b = (torch.randn(3, 2 * F, K, generator=gen, device=dev) * K ** -0.5).to(torch.bfloat16)
    counts = torch.tensor(SIZES, device=dev)
    out, h = m_grouped_gated_gemm_projections(a, b, counts, True)
    assert torch.equal(out[SAMPLE], m_grouped_gated_gemm(a, b, counts, True)[SAMPLE])
    want_h = torch.stack([b[group_of(r)].double() @ a[r].double() for r in SAMPLE])
    size = torch.stack([b[group_of(r)].double().abs() @ a[r].double().abs() for r in SAMPLE]) * (K + 8) * 2.0 ** -24
    assert ((h[SAMPLE].double() - want_h).abs() <= size + want_h.abs() * 2.0 ** -24).all()
    g, u = want_h[:, :F], want_h[:, F:]
    want = g * torch.sigmoid(g) * u
    slack = 1.13 * (u.abs() + size[:, F:]) * size[:, :F] + g.abs() * size[:, F:] + want.abs() * (2.0 ** -19 + 2.0 ** -8 * (1 + 2.0 ** -6)) + 1e-30
    assert ((out[SAMPLE].double() - want).abs() <= slack).all()
    dh = gated_backward(out, h)
    hs, d = h[SAMPLE].double().requires_grad_(True), out[SAMPLE].double()
    (hs[:, :F] * torch.sigmoid(hs[:, :F]) * hs[:, F:] * d).sum().backward()
    parts = torch.cat([d.abs() * u.abs() * (1 + 2 * g.abs()), d.abs() * g.abs()], 1)
    assert ((dh[SAMPLE].double() - hs.grad).abs() <= parts * 2.0 ** -19 + hs.grad.abs() * 2.0 ** -8 * (1 + 2.0 ** -6) + 1e-30).all()


def test_four_bit_product(dev):
    gen = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(ROWS, K, generator=gen, device=dev).to(torch.bfloat16)
    q = torch.randint(0, 16, (3, F, K), generator=gen, device=dev)
    scales = (torch.rand(3, 2, F, generator=gen, device=dev) * K ** -0.5).to(torch.bfloat16)
    out = m_grouped_gemm_int4(x, pack_int4(q), scales, torch.tensor(SIZES, device=dev), 32)
    for r in SAMPLE:
        s = scales[group_of(r)].double().repeat_interleave(32, 0).t()
        want = ((q[group_of(r)].double() - 8) * s) @ x[r].double()
        slack = (s * 303) @ x[r].double().abs() * (K + 32) * 2.0 ** -24
        assert ((out[r].double() - want).abs() <= slack * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -6) + 1e-38).all()


def test_router(dev):
    tokens, experts = 18_000_001, 128
    x = torch.empty(tokens, experts, dtype=torch.bfloat16, device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(3))
    x.requires_grad_(True)
    probs, idx = ops.topk_router(x, 4, renormalize=False)
    (g,) = torch.autograd.grad(probs, x, torch.ones_like(probs))
    at = [0, 16_777_215, 16_777_216, 16_777_217, tokens - 1]
    leaf = x.detach()[at].double().cpu().requires_grad_(True)
    order = torch.sort(leaf.detach(), dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(idx[at].cpu().long(), order)
    p = torch.gather(torch.softmax(leaf, 1), 1, order)
    assert ((probs.detach()[at].cpu().double() - p.detach()).abs() <= 2.0 ** -18 * p.detach()).all()
    p.sum().backward()
    size = torch.softmax(leaf.detach(), 1) * 2
    assert ((g[at].cpu().double() - leaf.grad).abs() <= 2.0 ** -17 * size + leaf.grad.abs() * 2.0 ** -8).all()
