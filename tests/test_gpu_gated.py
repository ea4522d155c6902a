"""The gated feed-forward block: ``m_grouped_gated_gemm``, ``gated_backward`` and the differentiable ``ops.gated_gmm`` against the
formulas in 64 bits.

Bounds, with u the half step of the operands' type (torch.finfo(t).eps / 2):
  projections  a sum of K products in fp32 is off by at most (K + 8) 2^-24 times the sum of the products' magnitudes; they are
               stored in fp32;
  outputs      act(gate) up: the slopes of both activations stay within 1.13, so the sums' errors arrive as
               1.13 |up| e_gate + |act| e_up; the activation itself (exp2 and reciprocal good to an ulp, its argument rounded) is
               off by at most 2^-19 of its value for |gate| up to 16; then u of the value for the one rounding;
  gradients    dh is rounded to the operands' type before it enters the products, u of each of its values; sums of it are
               bounded with the magnitudes.
"""
import pytest
import torch

from triton_grouped_gemm_amd import _native, ops
from triton_grouped_gemm_amd.gemm.gated import gated_backward, m_grouped_gated_gemm, m_grouped_gated_gemm_projections

pytestmark = pytest.mark.gpu


def act64(x, kind):
    if kind == "silu":
        return x * torch.sigmoid(x)
    return 0.5 * x * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(sizes, k, f, dtype, trans_b, seed, extra=0):
    gen = torch.Generator().manual_seed(seed)
    m = sum(sizes) + extra
    a = torch.randn(m, k, generator=gen).to(dtype)
    shape = (len(sizes), 2 * f, k) if trans_b else (len(sizes), k, 2 * f)
    b = (torch.randn(*shape, generator=gen) * k ** -0.5).to(dtype)
    grad = torch.randn(m, f, generator=gen).to(dtype)
    return a, b, grad


def reference(a, b, sizes, trans_b, kind):
    """out, h in 64 bits and the bounds of their errors before the last rounding, for the rows that groups own."""
    f = (b.shape[1] if trans_b else b.shape[2]) // 2
    outs, hs, eh = [], [], []
    row = 0
    for g, n in enumerate(sizes):
        w = b[g].double().t() if trans_b else b[g].double()
        x = a[row:row + n].double()
        hs.append(x @ w)
        eh.append((x.abs() @ w.abs()) * (a.shape[1] + 8) * 2.0 ** -24)
        row += n
    h, e = torch.cat(hs), torch.cat(eh)
    act = act64(h[:, :f], kind)
    out = act * h[:, f:]
    eo = 1.13 * (h[:, f:].abs() + e[:, f:]) * e[:, :f] + act.abs() * e[:, f:] + out.abs() * 2.0 ** -19 + 1e-30
    return out, h, eo, e


def check(got, want, slack, dtype, what):
    got = got.double().cpu()
    over = (got - want).abs() - (want.abs() * half_step(dtype) * (1 + 2 ** -6) + slack * (1 + half_step(dtype)) + (torch.finfo(dtype).tiny * torch.finfo(dtype).eps))
    assert torch.isfinite(got).all() and (over <= 0).all(), f"{what}: off by {over.max().item():.3e} more than allowed"


CASES = [
    # sizes, k, f, dtype, trans_b, activation
    ([1], 8, 8, torch.bfloat16, True, "silu"),
    ([1], 64, 128, torch.float16, False, "gelu_tanh"),
    ([3, 0, 1, 130], 200, 88, torch.bfloat16, True, "gelu_tanh"),
    ([0, 5, 300, 0, 64], 192, 136, torch.float16, True, "silu"),
    ([257, 31], 72, 344, torch.bfloat16, False, "silu"),
    ([0, 0, 17], 520, 8, torch.float16, False, "silu"),
    ([600, 1, 255], 256, 264, torch.bfloat16, False, "gelu_tanh"),
    ([512, 700], 1000, 520, torch.bfloat16, True, "silu"),
    ([4] * 64, 256, 768, torch.bfloat16, True, "silu"),
    # whole slabs of K and, for [K, 2 F] weights, whole tiles of columns: the four-wave kernel's; half tiles, full ones and both in turn
    ([700, 0, 128, 129, 1], 256, 200, torch.bfloat16, True, "gelu_tanh"),
    ([300, 513, 20, 256], 384, 256, torch.float16, False, "silu"),
    ([60, 100, 3], 512, 128, torch.bfloat16, False, "gelu_tanh"),
    ([1000], 640, 264, torch.float16, True, "silu"),
    ([520, 40, 700], 256, 384, torch.bfloat16, False, "silu"),
    ([256, 256, 384], 256, 128, torch.float16, False, "gelu_tanh"),
]


# the shape-agnostic kernel, the routes of ordinary calls, the eight-wave kernel alone, the four-wave and the deep-ring kernel wherever they can
PATHS = {"generic": ("force_generic", 1, 0), "routed": ("four_wave", 1, 1), "eight_wave": ("four_wave", 0, 1), "four_wave": ("four_wave", 2, 1),
         "deep": ("deep", 2, 1)}


@pytest.fixture(params=sorted(PATHS))
def path(request):
    key, value, back = PATHS[request.param]
    _native.set_option(key, value)
    yield request.param
    _native.set_option(key, back)


@pytest.mark.parametrize("case", CASES, ids=[f"{len(c[0])}g{sum(c[0])}r_k{c[1]}_f{c[2]}_{'nt' if c[4] else 'nn'}" for c in CASES])
def test_forward(dev, case, path):
    sizes, k, f, dtype, trans_b, kind = case
    a, b, _ = make(sizes, k, f, dtype, trans_b, 7 * k + f)
    want, h64, eo, eh = reference(a, b, sizes, trans_b, kind)
    ad, bd = a.to(dev), b.to(dev)
    counts = torch.tensor(sizes, dtype=torch.int64 if k % 16 else torch.int32, device=dev)
    out = m_grouped_gated_gemm(ad, bd, counts, trans_b, kind)
    both, h = m_grouped_gated_gemm_projections(ad, bd, counts, trans_b, kind)
    check(out, want, eo, dtype, "out")
    assert torch.equal(out, both) and h.dtype == torch.float32
    check(h, h64, eh, torch.float32, "projections")


def _window(rows, cols, dtype, dev, fill):
    """A [rows, cols] view with guarded memory on both sides."""
    base = torch.full((rows * cols + 512,), fill, dtype=dtype, device=dev)
    return base, base[256:256 + rows * cols].view(rows, cols)


@pytest.mark.parametrize("trans_b", [True, False])
@pytest.mark.parametrize("rows,f,k", [(5, 24, 136), (700, 136, 136), (90, 128, 256), (900, 256, 384)])
def test_rows_behind_the_last_group_and_neighbours_are_left_alone(dev, path, trans_b, rows, f, k):
    extra = 9
    sizes = [rows // 3, 0, rows - rows // 3]
    a, b, _ = make(sizes, k, f, torch.bfloat16, trans_b, 3, extra)
    a[rows:] = float("nan")
    out_base, out = _window(rows + extra, f, torch.bfloat16, dev, 7.0)
    h_base, h = _window(rows + extra, 2 * f, torch.float32, dev, 9.0)
    ad, bd, counts = a.to(dev), b.to(dev), torch.tensor(sizes, dtype=torch.int32, device=dev)
    _native.call("tgg_m_grouped_gated_gemm", ad.data_ptr(), bd.data_ptr(), out.data_ptr(), h.data_ptr(), counts.data_ptr(), 0,
                 3, rows + extra, f, k, int(trans_b), 0, _native.BF16, -1, _native.stream_of(ad))
    want, h64, eo, eh = reference(a, b, sizes, trans_b, "silu")
    check(out[:rows], want, eo, torch.bfloat16, "out")
    check(h[:rows], h64, eh, torch.float32, "projections")
    assert (out[rows:] == 7.0).all() and (h[rows:] == 9.0).all()
    assert (out_base[:256] == 7.0).all() and (out_base[-256:] == 7.0).all() and (h_base[:256] == 9.0).all() and (h_base[-256:] == 9.0).all()


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,f", [(1, 8), (3, 344), (129, 768), (1000, 40)])
def test_gradient_of_the_projections(dev, rows, f, dtype, kind):
    gen = torch.Generator().manual_seed(rows + f)
    h = (torch.randn(rows, 2 * f, generator=gen) * 3).clamp(-16, 16)
    h[0, :8] = torch.tensor([0.0, -0.0, 16.0, -16.0, 1e-3, -1e-3, 5.0, -5.0])
    d = torch.randn(rows, f, generator=gen).to(dtype)
    leaf = h.double().requires_grad_(True)
    (act64(leaf[:, :f], kind) * leaf[:, f:] * d.double()).sum().backward()
    got = gated_backward(d.to(dev), h.to(dev), kind).double().cpu()
    # slope = sigma + act (1 - sigma) z': each part is good to 2^-19 of its magnitude up to |gate| = 16, where z' stays below 56
    x = h[:, :f].double().abs()
    parts = torch.cat([d.double().abs() * h[:, f:].double().abs() * (1 + x * (1.6 + 0.22 * x * x) * torch.exp(-x)), (d.double() * x).abs()], 1)
    slack = parts * 2.0 ** -19
    if dtype is torch.float16:
        slack = slack + 2.0 ** -25  # subnormal steps of the result
    check(got, leaf.grad, slack, dtype, "dh")


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
def test_gradient_far_out(dev, kind):
    """Beyond |gate| = 100 the activations are x or 0 and their slopes 1 or 0, up to the largest numbers."""
    x = torch.tensor([1e2, 1e10, 1e25, 3e38, -1e2, -1e10, -1e25, -3e38])
    h = torch.cat([x, torch.ones(8)])[None].to(dev)
    d = torch.ones(1, 8, dtype=torch.bfloat16, device=dev)
    got = gated_backward(d, h, kind).float().cpu()[0]
    assert torch.equal(got[:8], torch.tensor([1.0] * 4 + [0.0] * 4))
    assert torch.equal(got[8:12], x[:4].bfloat16().float()) and (got[12:].abs() <= 1e-30).all()


def _gradients64(a, b, grad, sizes, trans_b, kind):
    """Gradients in 64 bits and bounds for those made from fp32 projections and a rounded dh."""
    f, u = grad.shape[1], half_step(a.dtype)
    das, ea, dbs, eb = [], [], [], []
    row = 0
    for g, n in enumerate(sizes):
        x = a[row:row + n].double().requires_grad_(True)
        w = b[g].double().requires_grad_(True)
        wt = w.t() if trans_b else w
        h = x @ wt
        h.retain_grad()
        d = grad[row:row + n].double()
        (act64(h[:, :f], kind) * h[:, f:] * d).sum().backward()
        das.append(x.grad)
        dbs.append(w.grad)
        gate, up = h[:, :f].detach().abs(), h[:, f:].detach().abs()
        # u of dh itself; |second derivative| <= 1.2 for both activations, each projection off by (K + 8) 2^-24 of its products' magnitudes, the slopes
        # good to 2^-19 of theirs
        eh = (x.detach().abs() @ wt.detach().abs()) * (a.shape[1] + 8) * 2.0 ** -24
        e = torch.cat([d.abs() * (1.13 * eh[:, f:] + 1.2 * up * eh[:, :f] + 3 * up * 2.0 ** -19), d.abs() * (1.13 * eh[:, :f] + gate * 2.0 ** -19)], 1)
        e = (e + u * h.grad.abs()) * (1 + 2 ** -6)
        wa, xa, dha = wt.detach().abs(), x.detach().abs(), h.grad.abs()
        ea.append(e @ wa.t() + (dha @ wa.t()) * (2 * f + 8) * 2.0 ** -24)
        ew = xa.t() @ e + (xa.t() @ dha) * (n + 8) * 2.0 ** -24
        eb.append(ew.t() if trans_b else ew)
        row += n
    return torch.cat(das), torch.stack(dbs), torch.cat(ea), torch.stack(eb)


GRAD_CASES = [
    ([5, 0, 40], 64, 72, torch.bfloat16, True, "silu"),
    ([1, 300], 136, 40, torch.float16, False, "gelu_tanh"),
    ([64, 65, 0, 3], 256, 136, torch.bfloat16, False, "silu"),
    ([513, 30], 192, 264, torch.float16, True, "silu"),
]


@pytest.mark.parametrize("case", GRAD_CASES, ids=[f"{len(c[0])}g{sum(c[0])}r_{'nt' if c[4] else 'nn'}" for c in GRAD_CASES])
def test_gradients(dev, case):
    sizes, k, f, dtype, trans_b, kind = case
    a, b, grad = make(sizes, k, f, dtype, trans_b, 11 * f)
    want_a, want_b, ea, eb = _gradients64(a, b, grad, sizes, trans_b, kind)
    ad, bd = a.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True)
    counts = torch.tensor(sizes, device=dev)
    out = ops.gated_gmm(ad, bd, counts, activation=kind, trans_b=trans_b)
    out.backward(grad.to(dev))
    check(ad.grad, want_a, ea, dtype, "da")
    check(bd.grad, want_b, eb, dtype, "db")
    empty = [g for g, n in enumerate(sizes) if n == 0]
    assert torch.count_nonzero(bd.grad[empty]) == 0
    # only one of the two asked for
    only_a = torch.autograd.grad(ops.gated_gmm(ad, bd.detach(), counts, kind, trans_b), ad, grad.to(dev))[0]
    only_b = torch.autograd.grad(ops.gated_gmm(ad.detach(), bd, counts, kind, trans_b), bd, grad.to(dev))[0]
    assert torch.equal(only_a, ad.grad) and torch.equal(only_b, bd.grad)


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
def test_gradients_against_differences(dev, kind):
    """The loss's difference along random directions, in 64 bits, against the kernels' gradients: the step's third-order term is
    below 1e-6 of the difference, so what is left is the gradients' own error, bounded with their magnitudes."""
    sizes, k, f = [7, 0, 33], 64, 48
    a, b, grad = make(sizes, k, f, torch.bfloat16, True, 5)
    gen = torch.Generator().manual_seed(1)
    va, vb = torch.randn(a.shape, generator=gen).double(), torch.randn(b.shape, generator=gen).double()
    loss = lambda t: (reference(a.double() + t * va, b.double() + t * k ** -0.5 * vb, sizes, True, kind)[0] * grad.double()).sum()
    step = 1e-4
    slope = (loss(step) - loss(-step)) / (2 * step)
    ad, bd = a.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True)
    ops.gated_gmm(ad, bd, torch.tensor(sizes, device=dev), kind, True).backward(grad.to(dev))
    _, _, ea, eb = _gradients64(a, b, grad, sizes, True, kind)
    got = (ad.grad.double().cpu() * va).sum() + (bd.grad.double().cpu() * vb * k ** -0.5).sum()
    u = half_step(torch.bfloat16)
    allowed = ((ea + u * ad.grad.double().cpu().abs()) * va.abs()).sum() + ((eb + u * bd.grad.double().cpu().abs()) * vb.abs() * k ** -0.5).sum()
    assert (got - slope).abs() <= allowed + 1e-5 * slope.abs()
    # errors of independent roundings add up like their squares: the signed sum stays far below the bound
    assert (got - slope).abs() <= 0.1 * allowed


def test_infinities_and_nan_stay_in_their_rows(dev):
    sizes, k, f = [4, 4], 64, 32
    a, b, _ = make(sizes, k, f, torch.bfloat16, True, 2)
    clean = m_grouped_gated_gemm(a.to(dev), b.to(dev), torch.tensor(sizes, device=dev), True)
    a[1, 3] = float("nan")
    a[6, 0] = float("inf")
    out = m_grouped_gated_gemm(a.to(dev), b.to(dev), torch.tensor(sizes, device=dev), True)
    assert torch.isnan(out[1]).all() and not torch.isfinite(out[6]).any()
    keep = [0, 2, 3, 4, 5, 7]
    assert torch.equal(out[keep], clean[keep])


def test_no_rows_and_all_groups_empty(dev):
    b = torch.randn(2, 32, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    a = torch.empty(0, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    out = ops.gated_gmm(a, b, torch.zeros(2, dtype=torch.int32, device=dev), trans_b=True)
    assert out.shape == (0, 16)
    out.sum().backward()
    assert a.grad.shape == a.shape and torch.count_nonzero(b.grad) == 0
    a = torch.randn(5, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    out = ops.gated_gmm(a, b, torch.zeros(2, dtype=torch.int32, device=dev), trans_b=True)
    assert out.shape == (5, 16)


def test_strided_operands_other_streams_and_sizes_on_the_host(dev):
    sizes, k, f = [9, 70], 128, 64
    a, b, grad = make(sizes, k, f, torch.bfloat16, True, 4)
    want = m_grouped_gated_gemm(a.to(dev), b.to(dev), torch.tensor(sizes, device=dev), True)
    wide = torch.zeros(79, 2 * k, dtype=torch.bfloat16, device=dev)
    wide[:, :k] = a.to(dev)
    assert torch.equal(ops.gated_gmm(wide[:, :k], b.to(dev), torch.tensor(sizes), trans_b=True), want)
    flipped = b.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.gated_gmm(a.to(dev), flipped, torch.tensor(sizes, device=dev), trans_b=True), want)
    side = torch.cuda.Stream()
    ad, bd, counts = a.to(dev), b.to(dev), torch.tensor(sizes, device=dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.gated_gmm(ad, bd, counts, trans_b=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


def test_captured_and_replayed(dev):
    sizes, k, f = [33, 0, 200], 256, 128
    a, b, grad = make(sizes, k, f, torch.bfloat16, True, 6)
    ad, bd, gd, counts = a.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True), grad.to(dev), torch.tensor(sizes, dtype=torch.int32, device=dev)

    def step():
        out = ops.gated_gmm(ad, bd, counts, trans_b=True)
        return (out.detach(), *torch.autograd.grad(out, (ad, bd), gd))

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
        split = [[33, 0, 200], [0, 233, 0], [100, 100, 33], [1, 2, 230]][turn]
        with torch.no_grad():
            ad.copy_(torch.roll(a, turn, 0).to(dev))
            counts.copy_(torch.tensor(split, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_compiled(dev):
    sizes, k, f = [12, 50], 64, 40
    a, b, grad = make(sizes, k, f, torch.bfloat16, True, 8)
    counts = torch.tensor(sizes, device=dev)
    ad, bd = a.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True)
    fn = lambda x, w: ops.gated_gmm(x, w, counts, "gelu_tanh", True)
    want = fn(ad, bd)
    want_grads = torch.autograd.grad(want, (ad, bd), grad.to(dev))
    got = torch.compile(fn, backend="aot_eager")(ad, bd)
    got_grads = torch.autograd.grad(got, (ad, bd), grad.to(dev))
    assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(got_grads, want_grads))


def test_more_than_512_groups(dev):
    sizes = [(i * 7) % 3 for i in range(700)]
    a, b, _ = make(sizes, 32, 16, torch.bfloat16, True, 9)
    want, _, eo, _ = reference(a, b, sizes, True, "silu")
    out = m_grouped_gated_gemm(a.to(dev), b.to(dev), torch.tensor(sizes, device=dev), True)
    check(out, want, eo, torch.bfloat16, "out")


@pytest.mark.parametrize("change", ["dtype", "k", "f", "activation", "sizes", "cpu"])
def test_refusals(dev, change):
    a, b = torch.zeros(4, 64, dtype=torch.bfloat16, device=dev), torch.zeros(2, 32, 64, dtype=torch.bfloat16, device=dev)
    sizes, kind = torch.tensor([2, 2], device=dev), "silu"
    error = AssertionError
    if change == "dtype":
        b = b.half()
    elif change == "k":
        a, b = a[:, :60], b[:, :, :60]
    elif change == "f":
        b = b[:, :24]
    elif change == "activation":
        kind, error = "relu", ValueError
    elif change == "sizes":
        sizes = sizes[:1]
    else:
        b = b.cpu()
    for call in (lambda: m_grouped_gated_gemm(a, b, sizes, True, kind), lambda: ops.gated_gmm(a, b, sizes, kind, True),
                 lambda: ops.gated_gmm(a.clone().requires_grad_(True), b, sizes, kind, True)):
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("tokens,hidden,ffn,experts,topk,scoring", [(300, 256, 128, 8, 2, "softmax"), (77, 128, 64, 16, 4, "sigmoid")])
def test_a_training_layer(dev, tokens, hidden, ffn, experts, topk, scoring):
    """Router, movement, gated block, down projection and combination with all gradients, against the layer in 64 bits with the same
    choice of experts.  Rows are rounded to bfloat16 after the block, after the down projection and at the end, gradients after every
    product: at most five roundings on a way, each 2^-9.2 of the norm, which add like squares to 0.0038; the bound leaves as much again
    for sums that cancel."""
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=gen).to(torch.bfloat16)
    wr = (torch.randn(hidden, experts, generator=gen) * hidden ** -0.5).to(torch.bfloat16)
    w1 = (torch.randn(experts, 2 * ffn, hidden, generator=gen) * hidden ** -0.5).to(torch.bfloat16)
    w2 = (torch.randn(experts, hidden, ffn, generator=gen) * ffn ** -0.5).to(torch.bfloat16)
    logits = (x.float() @ wr.float())
    logits[:, 3] = float("-inf")  # an expert without tokens
    grad = torch.randn(tokens, hidden, generator=gen).to(torch.bfloat16)

    leaves = [t.to(dev).requires_grad_(True) for t in (x, logits, w1, w2)]
    xd, ld, w1d, w2d = leaves
    probs, idx = ops.topk_router(ld, topk, scoring=scoring)
    rows, row_map = ops.permute(xd, idx, num_experts=experts)
    _, counts = ops.permute_map(idx, num_experts=experts)
    y = ops.gmm(ops.gated_gmm(rows, w1d, counts, trans_b=True), w2d, counts, trans_b=True)
    out = ops.unpermute(y, row_map, probs)
    got = torch.autograd.grad(out, leaves, grad.to(dev))

    exact = [t.double().requires_grad_(True) for t in (x, logits.clamp_min(-1e9), w1, w2)]
    xe, le, w1e, w2e = exact
    chosen = torch.gather(le, 1, idx.cpu().long())
    if scoring == "softmax":
        p = torch.softmax(chosen, 1)
    else:
        p = torch.sigmoid(chosen)
        p = p / p.sum(1, keepdim=True)
    want = 0
    for j in range(topk):
        e = idx[:, j].cpu().long()
        h = torch.stack([w1e[e[t]] @ xe[t] for t in range(tokens)])
        a = act64(h[:, :ffn], "silu") * h[:, ffn:]
        want = want + p[:, j:j + 1] * torch.stack([w2e[e[t]] @ a[t] for t in range(tokens)])
    grads = torch.autograd.grad(want, exact, grad.double())
    for name, a, b in (("out", out, want), *zip(("dx", "dlogits", "dw1", "dw2"), got, grads)):
        a, b = a.detach().double().cpu(), b.detach()
        assert (a - b).norm() <= 7.6e-3 * b.norm(), f"{name}: {((a - b).norm() / b.norm()).item():.2e}"
    assert torch.count_nonzero(got[2][3]) == 0 and torch.count_nonzero(got[1][:, 3]) == 0
