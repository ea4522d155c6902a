"""``ops.lora_linear`` on contiguous operands that do not begin at a multiple of 16 bytes: slices of a flat buffer, and gradients that autograd hands back as such."""
import pytest
import torch

from _lora import make
from triton_grouped_gemm_amd import ops

pytestmark = pytest.mark.gpu


def moved(t, by=1):
    """The same values, contiguous, ``by`` elements into a buffer."""
    flat = t.new_zeros(t.numel() + 8)
    out = flat[by:by + t.numel()].view(t.shape)
    out.copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16 != 0
    return out


@pytest.mark.parametrize("m", [5, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_operands(dev, m, dtype):
    x, w, a, b, g, adapters, s = make(m, 72, 64, 16, 4, dtype, 1, dev)
    want = ops.lora_linear(x, w, a, b, adapters, s)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, a, b)]
    grads = torch.autograd.grad(ops.lora_linear(*leaves, adapters, s), leaves, g)
    for i in range(4):
        args = [moved(t, 1 + i) if j == i else t for j, t in enumerate((x, w, a, b))]
        assert torch.equal(ops.lora_linear(*args, adapters, s), want)
        assert torch.equal(torch.ops.moe.lora_linear(*args, adapters, s), want)
        odd = [t.requires_grad_(True) for t in args]
        out = ops.lora_linear(*odd, adapters, s)
        got = torch.autograd.grad(out, odd, g)
        assert all(torch.equal(p, q) for p, q in zip(got, grads))
        for t in odd:
            t.requires_grad_(False)
    assert torch.equal(ops.lora_linear(x, w, a, b, moved(adapters), moved(s)), want)


@pytest.mark.parametrize("m", [5, 200])
def test_a_gradient_from_autograd(dev, m):
    """A row of a concatenation: its gradient is a view two bytes into the concatenation's."""
    x, w, a, b, g, adapters, s = make(m, 72, 64, 16, 4, torch.bfloat16, 2, dev)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, a, b)]
    want = torch.autograd.grad(ops.lora_linear(*leaves, adapters, s), leaves, g)
    out = ops.lora_linear(*leaves, adapters, s)
    both = torch.cat((torch.zeros(1, dtype=out.dtype, device=dev), out.flatten()))
    got = torch.autograd.grad(both, leaves, torch.cat((torch.ones(1, dtype=out.dtype, device=dev), g.flatten())))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    odd = moved(g)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(ops.lora_linear(*leaves, adapters, s), leaves, odd), want))
    _, h = torch.ops.moe.lora_linear_hidden(x, w, a, b, adapters, s)
    for args in ((odd, x, h), (g, moved(x), h), (g, x, moved(h))):
        got = torch.ops.moe.lora_linear_backward(args[0], args[1], w, a, b, adapters, s, args[2], True, True, True)
        assert all(torch.equal(p, q) for p, q in zip(got, (want[0], want[2], want[3])))


def test_adapters_of_a_flat_buffer(dev):
    """Parameters that are slices of one buffer, as optimisers keep them."""
    x, w, a, b, g, adapters, s = make(150, 72, 64, 16, 4, torch.bfloat16, 3, dev)
    want = ops.lora_linear(x, w, a, b, adapters, s)
    flat = torch.zeros(3 + a.numel() + b.numel(), dtype=a.dtype, device=dev)
    flat[3:3 + a.numel()], flat[3 + a.numel():] = a.flatten(), b.flatten()
    flat.requires_grad_(True)
    out = ops.lora_linear(x, w, flat[3:3 + a.numel()].view(a.shape), flat[3 + a.numel():].view(b.shape), adapters, s)
    assert torch.equal(out, want)
    grad, = torch.autograd.grad(out, flat, g)
    leaves = [t.clone().requires_grad_(True) for t in (a, b)]
    da, db = torch.autograd.grad(ops.lora_linear(x, w, *leaves, adapters, s), leaves, g)
    assert (grad[:3] == 0).all() and torch.equal(grad[3:3 + a.numel()], da.flatten()) and torch.equal(grad[3 + a.numel():], db.flatten())
