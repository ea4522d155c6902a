"""``ops.topk_router`` against the definition in 64 bits: the order is exact (equal logits by index), probabilities and gradients
are fp32.

Bounds: an exponential's argument l - max is one rounding off (2^-24 of it, |l - max| up to 40 here), expf two steps, sums of
up to 1024 terms and a quotient a few more, all relative to the value: 2^-24 (40 + 16) < 2^-18.  A gradient is a difference of such
products, so its bound goes by their magnitudes; in 16-bit logits' type it is rounded once more.
"""
import pytest
import torch

from triton_grouped_gemm_amd import ops

pytestmark = pytest.mark.gpu

FP32 = 2.0 ** -18


def order64(logits, k):
    """Indices by descending logit, ties by index, NaN first; -1 in the place of masked ones."""
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, 1e300), torch.where(torch.isposinf(x), torch.full_like(x, 1e299), x))
    idx = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    return torch.where(torch.isneginf(torch.gather(x, 1, idx)), torch.full_like(idx, -1), idx)


def reference(logits, k, scoring, renorm, grad=None):
    idx = order64(logits, k)
    leaf = logits.double().clone()
    masked = torch.isneginf(leaf)
    leaf[masked] = -1e6
    leaf.requires_grad_(True)
    # (renormalised softmax depends on the chosen logits alone: through log_softmax the others would get the 64-bit sum's own rounding as a gradient)
    if scoring == "softmax":
        logp = leaf if renorm else torch.log_softmax(leaf, 1)
    else:
        logp = torch.nn.functional.logsigmoid(leaf)
    real = idx >= 0
    picked = torch.where(real, torch.gather(logp, 1, idx.clamp_min(0)), torch.full((), -2e6, dtype=torch.float64))
    probs = torch.softmax(picked, 1) if renorm else torch.exp(picked)
    probs = torch.where(real, probs, torch.zeros_like(probs))
    if grad is None:
        return probs.detach(), idx
    (g,) = torch.autograd.grad((probs * grad.double()).sum(), leaf)
    g = torch.where(masked, torch.zeros_like(g), g)
    # magnitudes of what the gradient is a difference of
    size = torch.zeros_like(g)
    pd = (probs.detach() * grad.double()).abs()
    size.scatter_add_(1, idx.clamp_min(0), torch.where(real, pd + (probs.detach() * pd.sum(1, keepdim=True) if renorm else 0), torch.zeros_like(pd)))
    if scoring == "softmax" and not renorm:
        size = size + torch.softmax(leaf.detach(), 1) * pd.sum(1, keepdim=True)
    return probs.detach(), idx, g, size


def draw(tokens, experts, dtype, seed, masked=0.0, scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(tokens, experts, generator=gen) * scale).to(dtype)
    if masked:
        x[torch.rand(tokens, experts, generator=gen) < masked] = float("-inf")
        x[0] = float("-inf")
        x[-1, 1:] = float("-inf")
    return x, torch.randn(tokens, min(experts, 64), generator=gen)


SHAPES = [(1, 1, 1), (3, 4, 4), (5, 8, 2), (17, 33, 16), (64, 128, 8), (33, 127, 7), (9, 129, 17), (40, 256, 6), (7, 257, 33),
          (5, 512, 64), (6, 1000, 10), (4, 1024, 64), (21, 16, 16), (1000, 60, 4)]


@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,experts,k", SHAPES)
def test_forward_and_gradient(dev, tokens, experts, k, dtype, scoring, renorm):
    masked = 0.3 if (tokens + experts) % 2 else 0.0
    logits, d = draw(tokens, experts, dtype, tokens * experts, masked)
    d = d[:, :k]
    want_p, want_i, want_g, size = reference(logits, k, scoring, renorm, d)
    leaf = logits.to(dev).requires_grad_(True)
    probs, idx = ops.topk_router(leaf, k, scoring=scoring, renormalize=renorm)
    assert probs.dtype == torch.float32 and idx.dtype == torch.int32 and probs.is_contiguous() and not idx.requires_grad
    assert torch.equal(idx.cpu().long(), want_i)
    p = probs.detach().cpu().double()
    assert ((p - want_p).abs() <= FP32 * want_p + 1e-38).all()
    assert (p[want_i < 0] == 0).all()
    no_grad = ops.topk_router(leaf.detach(), k, scoring=scoring, renormalize=renorm)
    assert torch.equal(no_grad[0], probs.detach()) and torch.equal(no_grad[1], idx)
    (g,) = torch.autograd.grad(probs, leaf, d.to(dev))
    assert g.dtype == dtype
    u = 0 if dtype is torch.float32 else torch.finfo(dtype).eps / 2
    slack = 2 * FP32 * size + u * want_g.abs() * (1 + 2 ** -6) + ((torch.finfo(dtype).tiny * torch.finfo(dtype).eps) if u else 1e-38)
    over = (g.cpu().double() - want_g).abs() - slack
    assert (over <= 0).all(), f"gradient off by {over.max().item():.2e} more than allowed"


def test_ties_and_zeros_go_to_the_lowest_index(dev):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.zeros(3, 200, dtype=dtype)
        x[0, ::2] = -0.0
        x[1] = torch.arange(200) % 3 == 1
        x[2, 150:] = 1
        probs, idx = ops.topk_router(x.to(dev), 5)
        assert idx.tolist() == [[0, 1, 2, 3, 4], [1, 4, 7, 10, 13], [150, 151, 152, 153, 154]]
        assert torch.equal(probs.cpu(), torch.full((3, 5), 0.2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masks_of_the_lowest_value_are_numbers(dev, scoring, dtype):
    low = torch.finfo(dtype).min
    x = torch.full((3, 40), low, dtype=dtype)
    x[1, 7] = 3.0
    x[2, :20] = float("-inf")
    probs, idx = ops.topk_router(x.to(dev), 4, scoring=scoring)
    assert idx.tolist() == [[0, 1, 2, 3], [7, 0, 1, 2], [20, 21, 22, 23]]
    assert torch.equal(probs.cpu(), torch.tensor([[0.25] * 4, [1.0, 0, 0, 0], [0.25] * 4]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_nan_and_infinity_show_in_their_rows_alone(dev, dtype):
    x, _ = draw(8, 100, dtype, 3)
    clean = ops.topk_router(x.to(dev), 6, renormalize=False)
    x[2, 40] = float("nan")
    x[3, 41] = -float("nan")
    x[5, 9] = float("inf")
    probs, idx = ops.topk_router(x.to(dev), 6, renormalize=False)
    assert torch.equal(idx.cpu().long(), order64(x, 6)) and idx[2, 0] == 40 and idx[3, 0] == 41 and idx[5, 0] == 9
    assert torch.isnan(probs[[2, 3, 5]]).all()
    keep = [0, 1, 4, 6, 7]
    assert torch.equal(probs[keep], clean[0][keep])


def test_rows_without_any_expert_have_no_gradient(dev):
    for scoring in ("softmax", "sigmoid"):
        for renorm in (True, False):
            x = torch.full((4, 50), float("-inf"), device=dev, requires_grad=True)
            probs, idx = ops.topk_router(x, 3, scoring=scoring, renormalize=renorm)
            assert (idx == -1).all() and (probs == 0).all()
            (g,) = torch.autograd.grad(probs, x, torch.ones_like(probs))
            assert torch.equal(g, torch.zeros_like(g))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_far_logits_keep_their_proportions(dev, scoring):
    """Chosen scores that vanish in fp32 are normalised all the same."""
    x = torch.tensor([[-200.0, -201.0, -230.0, -500.0]])
    probs, _ = ops.topk_router(x.to(dev), 3, scoring=scoring)
    want, _ = reference(x, 3, scoring, True)
    assert ((probs.cpu().double() - want).abs() <= FP32 * want).all()


@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_gradient_against_differences(dev, scoring, renorm):
    x, d = draw(6, 48, torch.float32, 12, scale=1.0)
    d = d[:, :5]
    gen = torch.Generator().manual_seed(3)
    v = torch.randn(x.shape, generator=gen).double()
    at = order64(x, 5)

    def loss(t):  # the choice held, as in the gradient
        y = x.double() + t * v
        s = torch.softmax(y, 1) if scoring == "softmax" else torch.sigmoid(y)
        p = torch.gather(s, 1, at)
        return ((p / p.sum(1, keepdim=True) if renorm else p) * d.double()).sum()

    slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
    leaf = x.to(dev).requires_grad_(True)
    probs, _ = ops.topk_router(leaf, 5, scoring=scoring, renormalize=renorm)
    (g,) = torch.autograd.grad(probs, leaf, d.to(dev))
    _, _, _, size = reference(x, 5, scoring, renorm, d)
    assert (g.cpu().double() * v).sum().sub(slope).abs() <= 2 * FP32 * (size * v.abs()).sum() + 1e-8


def test_strides_streams_and_odd_bases(dev):
    x, d = draw(50, 128, torch.bfloat16, 5)
    want = ops.topk_router(x.to(dev), 8)
    wide = torch.zeros(50, 200, dtype=torch.bfloat16, device=dev)
    for first in (0, 1, 7, 72):
        wide[:, first:first + 128] = x.to(dev)
        view = wide[:, first:first + 128].detach().requires_grad_(True)
        probs, idx = ops.topk_router(view, 8)
        assert torch.equal(probs.detach(), want[0]) and torch.equal(idx, want[1])
        (g,) = torch.autograd.grad(probs, view, d[:, :8].to(dev))
        leaf = x.to(dev).requires_grad_(True)
        (h,) = torch.autograd.grad(ops.topk_router(leaf, 8)[0], leaf, d[:, :8].to(dev))
        assert torch.equal(g, h)
    assert all(torch.equal(a, b) for a, b in zip(ops.topk_router(x.to(dev).t().contiguous().t(), 8), want))
    side = torch.cuda.Stream()
    y = x.to(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.topk_router(y, 8)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_and_replayed(dev):
    x, d = draw(300, 64, torch.bfloat16, 6, masked=0.2)
    leaf, dd = x.to(dev).requires_grad_(True), d[:, :6].to(dev)

    def step():
        probs, idx = ops.topk_router(leaf, 6, renormalize=False)
        return probs.detach(), idx, torch.autograd.grad(probs, leaf, dd)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        with torch.no_grad():
            leaf.copy_(torch.roll(x, turn, 0).to(dev))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_compiled(dev):
    x, d = draw(30, 48, torch.bfloat16, 4)
    leaf, dd = x.to(dev).requires_grad_(True), d[:, :4].to(dev)
    fn = lambda t: ops.topk_router(t, 4, scoring="sigmoid")
    want, want_idx = fn(leaf)
    got, got_idx = torch.compile(fn, backend="aot_eager")(leaf)
    assert torch.equal(got, want) and torch.equal(got_idx, want_idx)
    assert torch.equal(torch.autograd.grad(got, leaf, dd)[0], torch.autograd.grad(want, leaf, dd)[0])


def test_the_gradient_has_no_gradient(dev):
    x = torch.randn(5, 20, device=dev, requires_grad=True)
    probs, _ = ops.topk_router(x, 3)
    (g,) = torch.autograd.grad(probs[:, 0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


def test_no_tokens(dev):
    x = torch.empty(0, 16, device=dev, requires_grad=True)
    probs, idx = ops.topk_router(x, 4)
    assert probs.shape == idx.shape == (0, 4)
    probs.sum().backward()
    assert x.grad.shape == (0, 16)


def test_refusals(dev):
    x = torch.zeros(4, 16, device=dev)
    for bad in (lambda: ops.topk_router(x, 0), lambda: ops.topk_router(x, 17), lambda: ops.topk_router(x, 4, scoring="tanh"),
                lambda: ops.topk_router(x.double(), 4), lambda: ops.topk_router(x[0], 1), lambda: ops.topk_router(x[:, :0], 1),
                lambda: ops.topk_router(torch.zeros(2, 1025, device=dev), 4), lambda: ops.topk_router(torch.zeros(2, 100, device=dev), 65)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(AssertionError):
        ops.topk_router(x.cpu(), 4)


def test_the_layer_takes_what_the_router_gives(dev):
    """Routing, movement and weighted combination: tokens without experts come out as zeros."""
    tokens, experts, hidden = 40, 16, 64
    logits, _ = draw(tokens, experts, torch.bfloat16, 8, masked=0.4)
    x = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    probs, idx = ops.topk_router(logits.to(dev), 3)
    rows, row_map = ops.permute(x, idx, num_experts=experts)
    back = ops.unpermute(rows, row_map, probs)
    assert torch.equal(back[0], torch.zeros_like(back[0]))
    full = (probs.sum(1) > 0)
    # the probabilities sum to one within three roundings each, the combination rounds once
    assert ((back.float() - x.float()).abs()[full] <= x.float().abs()[full] * (2.0 ** -8 + 2.0 ** -20)).all()
