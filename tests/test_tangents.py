"""Forward-mode derivatives of the adapter and orthogonalisation operators, which have none: a tangent is refused, not dropped.  The kernels are stood in for on the CPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from triton_grouped_gemm_amd import lora, ops

REFUSED = "jvp|forward"


def _standin(x, weight, lora_a, lora_b, adapters, scales, keep_h):
    lora._check(x, weight, lora_a, lora_b, adapters, scales)
    s = torch.ones(lora_a.shape[0]) if scales is None else scales
    mine = adapters.long()
    h = s[mine, None] * (lora_a.float()[mine] * x.float()[:, None]).sum(-1)
    out = x.float() @ weight.float().t() + (lora_b.float()[mine] * h[:, None]).sum(-1)
    return out.to(x.dtype), h if keep_h else None


@pytest.fixture
def cpu(monkeypatch):
    monkeypatch.setattr(lora, "require_gpu", lambda *tensors: None)
    monkeypatch.setattr(lora, "_launch", _standin)


def _operands():
    gen = torch.Generator().manual_seed(0)
    t = lambda *shape: torch.randn(*shape, generator=gen).to(torch.bfloat16)
    return [t(4, 16), t(24, 16), t(3, 8, 16), t(3, 24, 8), torch.tensor([0, 2, 1, 1], dtype=torch.int32), torch.rand(3, generator=gen)]


def _lora_tangents(args):
    for i in (0, 1, 2, 3, 5):
        with fwd.dual_level():
            dual = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match=REFUSED):
                ops.lora_linear(*dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match=REFUSED):
                ops.lora_linear(*dual)
        with pytest.raises(RuntimeError, match=REFUSED):
            torch.func.jvp(lambda t: ops.lora_linear(*args[:i], t, *args[i + 1:]), (args[i],), (torch.ones_like(args[i]),))


def _lora_gradient_tangents(args):
    """The gradient of a loss whose other factor has a tangent: the backward pass refuses it."""
    for wanted in (0, 1, 2):
        leaves = [t.clone().requires_grad_(j == wanted) if t.is_floating_point() else t for j, t in enumerate(args)]
        with fwd.dual_level():
            out = ops.lora_linear(*leaves)
            factor = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match=REFUSED):
                torch.autograd.grad((out * factor).sum(), leaves[wanted])


def _orthogonalize_tangents(x):
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match=REFUSED):
            ops.orthogonalize(fwd.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match=REFUSED):
        torch.func.jvp(ops.orthogonalize, (x,), (torch.ones_like(x),))
    for i in range(3):
        args = [x.clone(), x.clone(), torch.zeros_like(x)]
        with fwd.dual_level():
            args[i] = fwd.make_dual(args[i], torch.ones_like(x))
            with pytest.raises(RuntimeError, match=REFUSED):
                ops.muon_update(*args, 0.1)


def test_lora_linear(cpu):
    args = _operands()
    want = ops.lora_linear(*args)
    _lora_tangents(args)
    with fwd.dual_level():  # nothing here has a tangent
        assert torch.equal(ops.lora_linear(*args), want)


def test_lora_linear_gradients(cpu):
    _lora_gradient_tangents(_operands())


def test_orthogonalize_and_muon_update():
    _orthogonalize_tangents(torch.randn(2, 8, 16, generator=torch.Generator().manual_seed(1)))


@pytest.mark.gpu
def test_on_the_gpu(dev):
    args = [t.to(dev) for t in _operands()]
    want = ops.lora_linear(*args)
    _lora_tangents(args)
    _lora_gradient_tangents(args)
    with fwd.dual_level():
        assert torch.equal(ops.lora_linear(*args), want)
    x = torch.randn(2, 8, 16, generator=torch.Generator().manual_seed(1)).to(dev)
    want = ops.orthogonalize(x)
    _orthogonalize_tangents(x)
    with fwd.dual_level():
        assert torch.equal(ops.orthogonalize(x), want)
