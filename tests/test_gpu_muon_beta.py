"""``ops.muon_update`` with a momentum that forgets slowly: the gradient's share 1 - beta is rounded once, from beta as it is given."""
import pytest
import torch

from triton_grouped_gemm_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beta", [0.95, 0.999, 0.9999, 1 - 2.0 ** -20])
@pytest.mark.parametrize("shape", [(2, 40, 64), (1, 33, 17)])
def test_momentum_from_zero(dev, beta, shape):
    gen = torch.Generator().manual_seed(3)
    grad = torch.randn(shape, generator=gen).to(dev)
    weight, momentum = torch.zeros(shape, device=dev), torch.zeros(shape, device=dev)
    ops.muon_update(weight, grad, momentum, lr=0.1, beta=beta, steps=1)
    want = (1.0 - beta) * grad.double()
    # the share's rounding and the product's, 2^-24 each
    assert ((momentum.double() - want).abs() <= 2.0 ** -23 * 1.001 * want.abs()).all()


def test_momentum_of_several_steps(dev):
    """beta and 1 - beta add up to 1 but for their roundings: the momentum of a constant gradient approaches it as it should."""
    beta, grad = 0.999, torch.full((1, 16, 24), 3.0, device=dev)
    weight, momentum = torch.zeros_like(grad), torch.zeros_like(grad)
    for k in range(1, 21):
        ops.muon_update(weight, grad, momentum, lr=0.0, beta=beta, steps=1)
        want = 3.0 * (1.0 - beta ** k)
        # per step: two coefficients' roundings and that of the fused sum, each at most 2^-24 of a term of want's size at most
        assert ((momentum.double() - want).abs() <= k * 3 * 2.0 ** -24 * 1.01 * want).all()
