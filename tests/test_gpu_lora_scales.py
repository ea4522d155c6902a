"""Half precision: gradients of an adapter of which one hidden value is infinite.  The rows of one adapter share a power of two in the sums of its gradients; an infinity must not set it."""
import pytest
import torch

from _lora import check, make, reference
from triton_grouped_gemm_amd import ops

pytestmark = pytest.mark.gpu


def _gradients(x, w, a, b, g, adapters, s):
    leaves = [t.clone().requires_grad_(True) for t in (a, b)]
    return torch.autograd.grad(ops.lora_linear(x, w, *leaves, adapters, s), leaves, g)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("where", ["all rows", "late rows"])
def test_small_gradients_beside_an_infinite_one(dev, sign, where):
    x, w, a, b, g, adapters, s = make(500, 72, 64, 16, 2, torch.float16, 1, dev, "mixed", False)
    x = x * 64
    g = (g.float() * 2e-6).to(torch.float16)
    g[:, 5] = 2e-6 if where == "all rows" else 0.0
    if where == "late rows":
        g[400:, 5] = 2e-6
    b[1, 5] = 0  # what is infinite below counts for nothing elsewhere
    value, bound = reference(x, w, a, b, g, adapters, s, torch.float16)["da"]
    bad = b.clone()
    bad[1, 5, 3] = sign * float("inf")
    da, _ = _gradients(x, w, a, bad, g, adapters, s)
    rest = torch.arange(16, device=dev) != 3
    check("da", da[:, rest], value[:, rest], bound[:, rest])
    check("da of the other adapter", da[0], value[0], bound[0])
    assert not torch.isfinite(da[1, 3]).any()


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_small_hidden_values_beside_an_infinite_one(dev, sign):
    x, w, a, b, g, adapters, s = make(500, 72, 64, 16, 2, torch.float16, 2, dev, "mixed", False)
    x = (x.float() * 2.0 ** -9).to(torch.float16)
    a = (a.float() * 2.0 ** -9).to(torch.float16)
    g = g * 64
    x[:, 7] = 2.0 ** -9
    a[1, :, 7] = 0
    value, bound = reference(x, w, a, b, g, adapters, s, torch.float16)["db"]
    bad = a.clone()
    bad[1, 3, 7] = sign * float("inf")
    _, db = _gradients(x, w, bad, b, g, adapters, s)
    rest = torch.arange(16, device=dev) != 3
    check("db", db[:, :, rest], value[:, :, rest], bound[:, :, rest])
    check("db of the other adapter", db[0], value[0], bound[0])
    assert not torch.isfinite(db[1, :, 3]).any()
