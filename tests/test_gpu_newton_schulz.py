"""``ops.orthogonalize`` and ``ops.muon_update`` against the formulas in 64 bits.

One step, entry by entry.  With ``|.|`` taken of every entry, a matrix held in two planes of half precision is off by 2^-22 |X|, the
normalisation by 2^-22 |X| more, and a sum of n products in fp32 by at most n 2^-24 of the sum of their magnitudes (three products for one where both planes are
multiplied, whose left-out part is 2^-22 of it).  Where only high planes are multiplied, each operand is off by 2^-11 of itself, and 2^-11 of what is left on the
diagonal after its mean is taken out, which is at most twice the diagonal's largest value.  These carry over as

    e_G = (2 h + n 2^-24) |X||X|^T,    e_P = |b| e_G + |c| ((2 h + m 2^-24) |G'||G'| + 2 |G| e_G),    e_X' = |a| e_X + (2 h + m 2^-24) |P'||X| + e_P |X| + |P| e_X,

with h = 2^-21 or 2^-11 and G', P' the matrices with magnitudes enlarged by the shift.  To this comes the last rounding, and the absolute error of a
plane's smallest steps (2^-25 / 1024 in every entry, from the scale of the planes).

Several steps, in the Frobenius norm.  The step's map of singular values has a slope of at most L = max |a + 3 b s^2 + 5 c s^4| over [0, s_max], and the
Frobenius norm of an error grows by at most L a step (the step is an odd function of the singular values); each step adds the norm of the bound above.
"""
import pytest
import torch

from triton_grouped_gemm_amd import ops
from triton_grouped_gemm_amd.newton_schulz import COEFFICIENTS

pytestmark = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def wide(x):
    return x.transpose(-2, -1) if x.shape[-2] > x.shape[-1] else x


def one_step(x, ex, precise, coefficients):
    """The step of one matrix in 64 bits and the bound of its error, for an error of at most ex in x."""
    a, b, c = coefficients
    m, n = x.shape
    h, reps = (2.0 ** -21, 3) if precise else (2.0 ** -11, 1)
    gn, gm = 2 * h + reps * (n + 8) * 2.0 ** -24, 2 * h + reps * (m + 8) * 2.0 ** -24
    eye = torch.eye(m, dtype=torch.float64, device=x.device)
    ax = x.abs()
    g = x @ x.t()
    eg = gn * (ax @ ax.t()) + ex @ ax.t() + ax @ ex.t()
    shift = g.diagonal().abs().max()
    gs = g.abs() + shift * eye
    p = b * g + c * (g @ g)
    ep = abs(b) * eg + abs(c) * (gm * (gs @ gs) + 2 * g.abs() @ eg) + h * (abs(b) + 2 * abs(c) * shift) * gs  # (the linear term takes A as the products do)
    ps = p.abs() + p.diagonal().abs().max() * eye
    out = a * x + p @ x
    eo = abs(a) * ex + gm * (ps @ ax) + ep @ ax + ps @ ex + 2.0 ** -21 * out.abs() + 2.0 ** -30
    return out, eo


def reference(x, steps, precise, coefficients=COEFFICIENTS, eps=1e-7):
    """What a matrix becomes, the bound of the entries' errors (steps <= 1) and of the error's Frobenius norm."""
    w = wide(x.double())
    y = w / (w.norm() + eps)
    ey = 2.0 ** -21 * y.abs() + 2.0 ** -34
    total = ey.norm()
    a, b, c = coefficients
    for k in range(steps):
        top = torch.linalg.matrix_norm(y, 2)
        s = torch.linspace(0, 1, 1001, dtype=torch.float64, device=x.device) * top
        slope = (a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max()
        _, local = one_step(y, torch.zeros_like(y), precise, coefficients)
        total = slope * total + local.norm()
        y, ey = one_step(y, ey, precise, coefficients)
    if x.shape[-2] > x.shape[-1]:
        y, ey = y.t(), ey.t()
    return y, ey, total


def make(shape, kind, dtype, seed, dev):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=gen)
    if kind == "few":  # a few strong directions
        r = max(1, min(shape[-2:]) // 16)
        x = 0.1 * x + torch.randn(*shape[:-1], r, generator=gen) @ torch.randn(*shape[:-2], r, shape[-1], generator=gen)
    elif kind == "large":
        x = x * 1e4
    elif kind == "small":
        x = x * 1e-4
    return x.to(dtype).to(dev)


def check_entries(got, x, dtype, steps=1, coefficients=COEFFICIENTS, eps=1e-7):
    precise = dtype != torch.bfloat16
    for i in range(x.reshape(-1, *x.shape[-2:]).shape[0]):
        g, xi = got.reshape(-1, *x.shape[-2:])[i], x.reshape(-1, *x.shape[-2:])[i]
        want, err, _ = reference(xi, steps, precise, coefficients, eps)
        over = (g.double() - want).abs() - (want.abs() * half_step(dtype) + err * (1 + half_step(dtype)) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps)
        assert torch.isfinite(g.float()).all() and (over <= 0).all(), f"matrix {i}: off by {over.max().item():.3e} more than allowed"


SHAPES = [(1, 1, 1), (3, 1, 7), (2, 9, 1), (2, 16, 24), (1, 63, 65), (3, 64, 64), (2, 130, 129), (1, 128, 256), (1, 257, 400), (2, 520, 136), (1, 384, 1000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_one_step(dev, shape, dtype):
    for seed, kind in enumerate(("random", "few")):
        x = make(shape, kind, dtype, seed, dev)
        check_entries(ops.orthogonalize(x, steps=1), x, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_step_of_wide_tiles(dev, dtype):
    """Stacks large enough for tiles of 128 and of 256, below and beside the diagonal, with tails."""
    for shape in ((70, 300, 520), (40, 700, 264), (40, 1000, 1304), (24, 1800, 1100)):
        x = make(shape, "random", dtype, 5, dev)
        got = ops.orthogonalize(x, steps=1)
        pick = [0, shape[0] // 2, shape[0] - 1]
        check_entries(got[pick], x[pick], dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 40, 33), (1, 256, 256), (2, 300, 700), (1, 900, 130)])
def test_five_steps(dev, shape, dtype):
    for seed, kind in enumerate(("random", "few", "large", "small")):
        if kind == "large" and dtype == torch.float16:
            continue  # beyond the type
        x = make(shape, kind, dtype, 10 + seed, dev)
        got = ops.orthogonalize(x)
        for i in range(shape[0]):
            want, _, total = reference(x[i], 5, dtype != torch.bfloat16)
            off = (got[i].double() - want).norm()
            assert off <= total + half_step(dtype) * want.norm() + 1e-30, (kind, off / want.norm(), total / want.norm())


def test_no_steps_other_coefficients_and_leading_dimensions(dev):
    x = make((2, 3, 20, 50), "random", torch.float32, 3, dev)
    got = ops.orthogonalize(x, steps=0, eps=0.5)
    check_entries(got, x, torch.float32, steps=0, eps=0.5)
    other = (1.5, -0.5, 0.0)
    check_entries(ops.orthogonalize(x, steps=1, coefficients=other), x, torch.float32, coefficients=other)
    assert ops.orthogonalize(x[0, 0]).shape == (20, 50)
    assert torch.equal(ops.orthogonalize(x[0, 0]), ops.orthogonalize(x)[0, 0])
    assert ops.orthogonalize(x[:0]).shape == (0, 3, 20, 50)


def test_strided_input(dev):
    x = make((3, 60, 100), "random", torch.bfloat16, 4, dev)
    assert torch.equal(ops.orthogonalize(x[:, ::2, 5:90]), ops.orthogonalize(x[:, ::2, 5:90].contiguous()))
    assert torch.equal(ops.orthogonalize(x.transpose(1, 2)), ops.orthogonalize(x.transpose(1, 2).contiguous()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_matrices_that_begin_anywhere(dev, dtype):
    """Contiguous stacks that are not aligned to 16 bytes, as slices of a flat buffer are."""
    for shape in ((2, 24, 40), (3, 40, 24), (2, 33, 17)):
        flat = torch.zeros(shape[0] * shape[1] * shape[2] + 8, dtype=dtype, device=dev)
        x = make(shape, "random", dtype, 8, dev)
        part = flat[1:1 + x.numel()].view(shape)
        part.copy_(x)
        assert part.data_ptr() % 16 != 0
        assert torch.equal(ops.orthogonalize(part), ops.orthogonalize(x))
        whole, mom = x.clone(), torch.zeros(shape, device=dev)
        ops.muon_update(whole, x, mom, 0.1)
        odd = torch.zeros(x.numel() + 8, device=dev)[1:1 + x.numel()].view(shape)
        w = flat.clone()[1:1 + x.numel()].view(shape)
        ops.muon_update(w, part, odd, 0.1)
        assert torch.equal(w, whole) and torch.equal(odd, mom)
        assert (flat[0] == 0) and (flat[1 + x.numel():] == 0).all()


def test_shared_memory_is_refused(dev):
    w = make((2, 16, 16), "random", torch.float32, 9, dev)
    m = torch.zeros_like(w)
    for args in ((w, m, m), (w, w, m), (m, w, m)):
        with pytest.raises(ValueError, match="share memory"):
            ops.muon_update(*args, 0.1)
    both = torch.zeros(3, 16, 16, device=dev)
    with pytest.raises(ValueError, match="share memory"):
        ops.muon_update(both[:2], w, both[1:], 0.1)


def test_zeros_nan_and_infinity_stay_in_their_matrix(dev):
    x = make((5, 70, 90), "random", torch.float32, 6, dev)
    plain = ops.orthogonalize(x)
    y = x.clone()
    y[1] = 0
    y[2, 3, 4] = float("nan")
    y[4, 69, 89] = float("inf")
    got = ops.orthogonalize(y)
    assert (got[1] == 0).all()
    assert torch.isnan(got[2]).all() and torch.isnan(got[4]).all()
    assert torch.equal(got[0], plain[0]) and torch.equal(got[3], plain[3])


def test_same_bits_every_time(dev):
    x = make((3, 333, 777), "few", torch.bfloat16, 7, dev)
    first = ops.orthogonalize(x)
    for _ in range(3):
        assert torch.equal(ops.orthogonalize(x), first)


@pytest.mark.parametrize("weight_dtype,grad_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.float16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_update(dev, weight_dtype, grad_dtype, nesterov):
    lr, beta, decay = 0.02, 0.9, 0.1
    for shape in ((2, 100, 72), (1, 33, 264)):
        w, g = make(shape, "random", weight_dtype, 20, dev), make(shape, "few", grad_dtype, 21, dev)
        mom = make(shape, "few", torch.float32, 22, dev)
        w0, m0 = w.double(), mom.double()
        ops.muon_update(w, g, mom, lr, beta=beta, nesterov=nesterov, weight_decay=decay, steps=1)
        want_m = beta * m0 + (1 - beta) * g.double()
        # two products and a sum in fp32, and the coefficients' own rounding
        assert ((mom.double() - want_m).abs() <= 2.0 ** -22 * (m0.abs() + g.double().abs())).all()
        u = beta * want_m + (1 - beta) * g.double() if nesterov else want_m
        scale = max(1.0, shape[1] / shape[2]) ** 0.5
        for i in range(shape[0]):
            # u's rounding errors, relative to the magnitudes that it is the sum of, pass the step as an error of x does
            y, _, _ = reference(u[i], 0, True)
            eu = 2.0 ** -20 * (m0[i].abs() + g[i].double().abs()) / u[i].norm() + 2.0 ** -20 * y.abs() + 2.0 ** -34
            y, eu = wide(y), (eu.t() if shape[1] > shape[2] else eu)
            out, err = one_step(y, eu, weight_dtype != torch.bfloat16, COEFFICIENTS)
            if shape[1] > shape[2]:
                out, err = out.t(), err.t()
            want = (1 - lr * decay) * w0[i] - lr * scale * out
            bound = lr * scale * err + 2.0 ** -22 * (w0[i].abs() + lr * scale * out.abs())
            over = (w[i].double() - want).abs() - (want.abs() * half_step(weight_dtype) + bound * 1.01 + torch.finfo(weight_dtype).tiny)
            assert (over <= 0).all(), over.max().item()


def test_muon_update_gives_what_its_parts_give(dev):
    """The step's direction is orthogonalize's of the momentum (in fp32, whose products are the precise ones)."""
    w, g = make((2, 200, 88), "random", torch.float32, 30, dev), make((2, 200, 88), "few", torch.bfloat16, 31, dev)
    mom = torch.zeros_like(w)
    w0 = w.clone()
    ops.muon_update(w, g, mom, 0.5, beta=0.0, nesterov=False, scale=1.0)
    assert torch.equal(mom, g.float())
    want = w0.double() - 0.5 * ops.orthogonalize(g.float()).double()
    assert ((w.double() - want).abs() <= 2.0 ** -22 * (w0.abs() + want.abs() + 1)).all()


def test_scale_defaults_to_the_shape(dev):
    g = make((1, 64, 16), "random", torch.float32, 32, dev)
    ws = []
    for kw in ({}, {"scale": 2.0}):
        w = torch.zeros(1, 64, 16, device=dev)
        ops.muon_update(w, g, torch.zeros_like(w), 0.1, **kw)
        ws.append(w)
    assert torch.equal(*ws)


def test_captured_and_replayed(dev):
    """A graph of both operators replays on new values, with eager calls of other sizes in between."""
    x = make((2, 120, 300), "random", torch.bfloat16, 40, dev)
    w, mom = make((2, 120, 300), "random", torch.float32, 41, dev), torch.zeros(2, 120, 300, device=dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.orthogonalize(x)
        ops.muon_update(w.clone(), x, mom.clone(), 0.1)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.orthogonalize(x)
        ops.muon_update(w, x, mom, 0.1)
    for seed in range(4):
        x.copy_(make((2, 120, 300), "few", torch.bfloat16, 50 + seed, dev))
        ew, em = w.clone(), mom.clone()
        eager = ops.orthogonalize(x)
        ops.muon_update(ew, x, em, 0.1)
        ops.orthogonalize(make((1, 50, 60), "random", torch.float32, seed, dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(w, ew) and torch.equal(mom, em)


def test_two_streams_at_once(dev):
    xs = [make((2, 300, 400), "random", torch.bfloat16, 60 + i, dev) for i in range(2)]
    want = [ops.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.orthogonalize(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
