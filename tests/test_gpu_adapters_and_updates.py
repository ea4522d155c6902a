"""The adapter and orthogonalisation operators together and beside the library's others, as a trainer calls them."""
import gc

import pytest
import torch

from triton_grouped_gemm_amd import ops

pytestmark = pytest.mark.gpu


def _layer(dev, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t = lambda *shape, scale=1.0: (torch.randn(*shape, generator=gen) * scale).to(torch.bfloat16).to(dev)
    return t(300, 64), t(96, 64, scale=64 ** -0.5), t(4, 8, 64, scale=64 ** -0.5), t(4, 96, 8, scale=8 ** -0.5), t(6, 128, 96, scale=96 ** -0.5), \
        torch.randint(-1, 4, (300,), generator=gen).to(torch.int32).to(dev), t(300, 16)


def _forward(x, weight, a, b, experts, adapters, logits):
    """A projection with adapters, then experts: routed, multiplied, brought back."""
    h = ops.lora_linear(x, weight, a, b, adapters)
    probs, index = ops.topk_router(logits[:, :6].contiguous(), 2)
    rows, row_map = ops.permute(h, index, num_experts=6)
    _, sizes = ops.permute_map(index, num_experts=6)
    return ops.unpermute(ops.gmm(rows, experts, sizes, trans_b=True), row_map, probs)


def test_a_layer_runs_and_its_gradients_are_those_of_the_formulas(dev):
    x, weight, a, b, experts, adapters, logits = _layer(dev)
    leaves = [t.clone().requires_grad_(True) for t in (x, a, b, experts)]
    out = _forward(leaves[0], weight, leaves[1], leaves[2], leaves[3], adapters, logits)
    grad = torch.randn(out.shape, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    got = torch.autograd.grad(out, leaves, grad)

    # the same in 64 bits, dense
    refs = [t.double().clone().requires_grad_(True) for t in (x, a, b, experts)]
    rx, ra, rb, re = refs
    merged = weight.double()[None] + torch.bmm(rb, ra.contiguous())
    each = torch.einsum("mk,lnk->lmn", rx, merged)
    plain = rx @ weight.double().t()
    h = torch.where((adapters >= 0)[:, None], each[adapters.clamp_min(0).long(), torch.arange(300, device=dev)], plain)
    probs, index = ops.topk_router(logits[:, :6].contiguous(), 2)
    want = torch.zeros(300, 128, dtype=torch.float64, device=dev)
    for k in range(2):
        every = torch.einsum("mn,enf->emf", h, re.transpose(1, 2))
        want = want + probs[:, k, None].double() * every[index[:, k].long(), torch.arange(300, device=dev)]
    want_grads = torch.autograd.grad(want, refs, grad.double())
    # bf16 roundings between the operators: h, the experts' rows, their gradients and the results, at most eight half steps of 2^-8 of the magnitudes' norm, of which sums keep less
    u = 8 * 2.0 ** -8
    assert (out.double() - want).norm() <= u * want.norm()
    for g, w in zip(got, want_grads):
        assert (g.double() - w).norm() <= u * w.norm()


def test_a_step_of_every_kind_of_weight(dev):
    """Experts' and adapters' gradients go into muon_update in the stacks that backward gives; the update is the documented one of that very gradient."""
    x, weight, a, b, experts, adapters, logits = _layer(dev, 3)
    leaves = [t.clone().requires_grad_(True) for t in (a, b, experts)]
    out = _forward(x, weight, *leaves, adapters, logits)
    out.float().square().mean().backward()
    for leaf in leaves:
        before, grad = leaf.detach().clone(), leaf.grad
        momentum = torch.zeros(leaf.shape, dtype=torch.float32, device=dev)
        ops.muon_update(leaf, grad, momentum, lr=0.1, beta=0.0, nesterov=False)
        assert leaf.dtype == torch.bfloat16 and torch.isfinite(leaf.float()).all()
        assert torch.equal(momentum, grad.float())
        rows, cols = leaf.shape[-2:]
        step = 0.1 * max(1.0, rows / cols) ** 0.5 * ops.orthogonalize(grad.float()).double()
        # the direction's two forms: in bf16 1.1e-3 of its norm and more exact (half precision products); then the weights' rounding
        off = (leaf.detach().double() - (before.double() - step)).norm()
        assert off <= 2.0 ** -8 * step.norm() + 2.0 ** -8 * before.double().norm()
    # several steps in a row keep running on updated leaves
    for _ in range(2):
        for leaf in leaves:
            leaf.grad = None
        _forward(x, weight, *leaves, adapters, logits).float().square().mean().backward()
        for leaf in leaves:
            ops.muon_update(leaf, leaf.grad, torch.zeros(leaf.shape, dtype=torch.float32, device=dev), lr=0.01)
    assert all(torch.isfinite(leaf.float()).all() for leaf in leaves)


def test_muon_update_is_seen_by_autograd(dev):
    """A leaf that is updated in place after a forward call makes that call's backward pass fail, as torch's own in-place operators do."""
    x, weight, a, b, _, adapters, _ = _layer(dev, 4)
    leaf = a.clone().requires_grad_(True)
    out = ops.lora_linear(x, weight, leaf, b, adapters)
    ops.muon_update(leaf, torch.ones_like(a), torch.zeros(a.shape, device=dev), lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_two_graphs_with_a_common_leaf(dev):
    """A backward pass captured while an eager graph of the same leaves lives."""
    x, weight, a, b, _, adapters, _ = _layer(dev, 5)
    leaves = [t.clone().requires_grad_(True) for t in (x, a, b)]
    eager = ops.lora_linear(leaves[0], weight, leaves[1], leaves[2], adapters)
    grad = torch.ones_like(eager)
    want = torch.autograd.grad(eager, leaves, grad, retain_graph=True)
    torch.cuda.synchronize()
    # what may be captured: leaves of the graph's own over the same memory (autograd waits for the stream that a leaf's gradient was last made on)
    own = [t.detach().requires_grad_(True) for t in leaves]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.lora_linear(own[0], weight, own[1], own[2], adapters)
        got = torch.autograd.grad(out, own, grad)
    for _ in range(3):
        again = torch.autograd.grad(eager, leaves, grad, retain_graph=True)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, got, again))


def test_workspaces_of_calls_on_two_streams_are_their_own(dev):
    x, weight, a, b, _, adapters, _ = _layer(dev, 6)
    want = ops.lora_linear(x, weight, a, b, adapters)
    stack = torch.randn(3, 200, 140, generator=torch.Generator().manual_seed(7)).to(dev)
    want_o = ops.orthogonalize(stack)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(side):
            o = ops.orthogonalize(stack)
        y = ops.lora_linear(x, weight, a, b, adapters)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(o, want_o)


@pytest.fixture
def memory_given_back():
    """What a large test leaves in the allocator goes back to the device: a library's lasting workspace would otherwise settle in it and keep it."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_operators_beyond_two_to_the_31_values(dev, memory_given_back):
    """Element numbers past 31 bits: the last matrix of a stack, and the last rows of a batch."""
    if torch.cuda.get_device_properties(dev).total_memory < 200 << 30:
        pytest.skip("needs 200 GiB")
    count = 8200  # x 512 x 520 values: 2.18e9
    stack = torch.empty(count, 512, 520, dtype=torch.bfloat16, device=dev)
    for i in range(0, count, 1025):
        stack[i:i + 1025] = torch.randn(1025, 512, 520, generator=torch.Generator(device=dev).manual_seed(i), device=dev)
    got = ops.orthogonalize(stack, steps=1)
    for i in (0, 4123, count - 1):
        alone = ops.orthogonalize(stack[i], steps=1).double()  # (in other tiles: sums in another order, under the type's rounding)
        assert (got[i].double() - alone).norm() <= 2.0 ** -8 * alone.norm()
    del got, stack
    torch.cuda.empty_cache()
    m, k, n = 70000, 32768, 64
    x = torch.empty(m, k, dtype=torch.bfloat16, device=dev)
    for i in range(0, m, 10000):
        x[i:i + 10000] = torch.randn(10000, k, generator=torch.Generator(device=dev).manual_seed(i), device=dev)
    gen = torch.Generator(device=dev).manual_seed(1)
    w = torch.randn(n, k, generator=gen, device=dev).to(torch.bfloat16)
    a, b = torch.randn(2, 8, k, generator=gen, device=dev).to(torch.bfloat16), (torch.randn(2, n, 8, generator=gen, device=dev)).to(torch.bfloat16)
    adapters = (torch.arange(m, device=dev) % 3 - 1).to(torch.int32)
    xl, al = x.requires_grad_(True), a.clone().requires_grad_(True)
    out = ops.lora_linear(xl, w, al, b, adapters)
    rows = torch.tensor([0, 1, 2, 65535, 65536, 69998, 69999], device=dev)
    want = ops.lora_linear(x.detach()[rows], w, a, b, adapters[rows])
    # another route (few rows): sums in another order
    magnitude = x.detach()[rows].double().abs() @ w.double().abs().t()
    assert ((out.detach()[rows].double() - want.double()).abs() <= 2 * 2.0 ** -8 * want.double().abs() + 2.0 ** -16 * magnitude * 64).all()
    dx, da = torch.autograd.grad(out, (xl, al), torch.ones_like(out))
    small = x.detach()[rows].requires_grad_(True)
    dxr = torch.autograd.grad(ops.lora_linear(small, w, a, b, adapters[rows]), small, torch.ones(7, n, dtype=torch.bfloat16, device=dev))[0]
    assert ((dx[rows].double() - dxr.double()).norm() <= 2.0 ** -7 * dxr.double().norm())
    dh = torch.ones(1, n, dtype=torch.float64, device=dev) @ b[0].double()  # the same for every row of the adapter
    want_da = dh.t() @ x.detach()[adapters == 0].sum(0, keepdim=True, dtype=torch.float64)
    assert (da[0].double() - want_da).norm() <= 2.0 ** -7 * want_da.norm()


def test_weights_beyond_four_gigabytes(dev, memory_given_back):
    """The last rows and columns of shared weights and adapters at the sides' limit, in both directions."""
    if torch.cuda.get_device_properties(dev).total_memory < 200 << 30:
        pytest.skip("needs 200 GiB")
    n, k, r = 65536, 65536, 16
    gen = torch.Generator(device=dev).manual_seed(3)
    w = torch.empty(n, k, dtype=torch.bfloat16, device=dev)
    for i in range(0, n, 8192):
        w[i:i + 8192] = torch.randn(8192, k, generator=gen, device=dev)
    t = lambda *shape: torch.randn(*shape, generator=gen, device=dev).to(torch.bfloat16)
    a, b = t(2, r, k) * 2.0 ** -4, t(2, n, r)
    for m in (5, 150):
        x, g = t(m, k), t(m, n)
        adapters = (torch.arange(m, device=dev) % 3 - 1).to(torch.int32)
        xl = x.clone().requires_grad_(True)
        out = ops.lora_linear(xl, w, a, b, adapters)
        dx, = torch.autograd.grad(out, xl, g)
        has = (adapters >= 0)[:, None]
        mine = adapters.clamp_min(0).long()
        h = torch.stack([x[i].double() @ a[mine[i]].double().t() for i in range(m)]) * has
        dh = torch.stack([g[i].double() @ b[mine[i]].double() for i in range(m)]) * has
        for part in (slice(0, 64), slice(n - 64, n)):
            want = x.double() @ w[part].double().t() + (b[:, part].double()[mine] * h[:, None, :]).sum(-1)
            want_dx = g.double() @ w[:, part].double() + (a[:, :, part].double()[mine] * dh[:, :, None]).sum(1)
            # one rounding to bf16, half a step of 2^-8, and sums in fp32: 65536 terms of like size give 2^-24 * 65536 = 2^-8 at the very most
            assert (out[:, part].double() - want).norm() <= 2.0 ** -7 * want.norm()
            assert (dx[:, part].double() - want_dx).norm() <= 2.0 ** -7 * want_dx.norm()
