"""Directions in bfloat16 of matrices whose weak directions lie far below their strong ones: the error in front of the last rounding.

With |X| = 1 (Frobenius) at the start.  Two planes leave out at most 2^-23 of a value, fp32 sums round to 2^-24 with signs of their own; a step's three products multiply by coefficients whose
magnitudes add up to 3.4445 + 4.7750 + 2.0315 < 10.3, and what is left out of a weak direction grows with it, by at most 3.4445 a step, 485 in five; later steps' errors grow less, 1 / (1 - 1 / 3.4445) < 1.41 of
the first one's in all.  So the error in front of the rounding has a norm of at most 10.3 * 2^-23 * 485 * 1.41 = 8.4e-4 < 2^-10.  The rounding itself adds at most half a step of each value; what an entry is off beyond
that belongs to the error in front of it.
"""
import pytest
import torch

from triton_grouped_gemm_amd import ops
from triton_grouped_gemm_amd.newton_schulz import COEFFICIENTS

pytestmark = pytest.mark.gpu

LIMIT = 2.0 ** -10

CASES = [  # rows, columns, kind
    (8, 4096, "rank", 4, 0.003),
    (16, 4096, "rank", 8, 0.01),
    (64, 2048, "rank", 32, 0.003),
    (128, 4096, "rank", 64, 0.01),
    (256, 1024, "rank", 128, 0.003),
    (7, 21, "rank", 3, 7e-4),
    (16, 512, "decay", 3, 0),
    (2, 129, "decay", 4.3, 0),
    (512, 2048, "rows", 4, 0),
]


def make(rows, cols, kind, p, noise):
    gen = torch.Generator().manual_seed(rows + cols)
    normal = lambda *shape: torch.randn(*shape, generator=gen, dtype=torch.float64)
    if kind == "rank":  # strong directions over a floor of noise
        x = normal(rows, p) @ normal(p, cols) / p ** 0.5 + noise * normal(rows, cols)
    elif kind == "decay":  # singular values from 1 to 10^-p
        right, left = torch.linalg.qr(normal(cols, rows))[0].t(), torch.linalg.qr(normal(rows, rows))[0]
        x = left @ (torch.logspace(0, -p, rows, dtype=torch.float64)[:, None] * right)
    else:  # all rows but a few are zero
        x = torch.zeros(rows, cols, dtype=torch.float64)
        x[:p] = normal(p, cols)
    return x


def exact(x):
    a, b, c = COEFFICIENTS
    y = x.double()
    y = y / (y.norm() + 1e-7)
    for _ in range(5):
        g = y @ y.t()
        y = a * y + (b * g + c * (g @ g)) @ y
    return y


def beyond_rounding(got, want):
    """The norm of what entries in bfloat16 are off by beyond half a step of theirs."""
    half = torch.ldexp(torch.ones_like(want), torch.frexp(want.abs())[1] - 9)
    return ((got.double() - want).abs() - half).clamp_min(0).norm().item()


@pytest.mark.parametrize("rows,cols,kind,p,noise", CASES)
@pytest.mark.parametrize("tall", [False, True])
def test_directions(dev, rows, cols, kind, p, noise, tall):
    x = make(rows, cols, kind, p, noise).to(torch.bfloat16).to(dev)
    want = exact(x)
    got = ops.orthogonalize(x.t().contiguous()).t() if tall else ops.orthogonalize(x)
    assert beyond_rounding(got, want) <= LIMIT


@pytest.mark.parametrize("rows,cols,kind,p,noise", CASES)
@pytest.mark.parametrize("tall", [False, True])
def test_steps_of_weights(dev, rows, cols, kind, p, noise, tall):
    """Weights of zeros take the direction itself; the gradient in fp32."""
    x = make(rows, cols, kind, p, noise).float().to(dev)
    want = -exact(x)
    grad = x.t().contiguous() if tall else x
    weight, momentum = torch.zeros_like(grad, dtype=torch.bfloat16), torch.zeros_like(grad)
    ops.muon_update(weight, grad, momentum, lr=1.0, beta=0.0, nesterov=False, scale=1.0)
    assert beyond_rounding(weight.t() if tall else weight, want) <= LIMIT


def test_stacks_in_every_tile(dev):
    """Matrices of a stack that is large enough for tiles of 128 and of 256."""
    for count, rows, cols in ((70, 300, 520), (40, 1000, 1304)):
        x = torch.stack([make(rows, cols + i, "rank", rows // 2, 0.003)[:, :cols] for i in range(3)]).to(torch.bfloat16).to(dev)
        got = ops.orthogonalize(x.repeat(count // 3 + 1, 1, 1)[:count])
        for i in (0, 1, count - 1):
            assert beyond_rounding(got[i], exact(x[i % 3])) <= LIMIT
