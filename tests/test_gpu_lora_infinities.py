"""``ops.lora_linear``: infinities in operands come out as the formulas say, whatever stands beside a row.  Hidden values enter the second product in two parts, and half-precision adapters in two as well;
a part that is zero, or of the other sign, must not make a NaN of an infinity."""
import pytest
import torch

from _lora import make
from triton_grouped_gemm_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
INF = float("inf")
# few rows; tiles of one adapter; of requests one after another; of mixed rows; adapters with more than one step of depth a plane
BATCHES = [(40, "each", 16), (300, "1", 16), (300, "1", 40), (300, "runs", 24), (300, "each", 8), (300, "each", 72)]


def same_kind(got, want):
    """NaN where there is one, infinities of the same sign, everything else finite."""
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN elsewhere"
    assert torch.equal(got == INF, want == INF) and torch.equal(got == -INF, want == -INF), "infinities elsewhere"


def formulas(x, w, a, b, g, adapters, s):
    """out, dx, da, db in 64 bits, row by row."""
    x, w, a, b, g = (t.double() for t in (x, w, a, b, g))
    has = (adapters >= 0) & (adapters < a.shape[0])
    mine = torch.where(has, adapters, 0).long()
    scale = (torch.ones(a.shape[0], device=x.device) if s is None else s).double()[mine][:, None]
    none = torch.zeros((), dtype=torch.float64, device=x.device)
    h = torch.where(has[:, None], scale * (x[:, None] * a[mine]).sum(-1), none)
    dh = torch.where(has[:, None], scale * (g[:, :, None] * b[mine]).sum(1), none)
    out = (x[:, None] * w).sum(-1) + torch.where(has[:, None], (b[mine] * h[:, None]).sum(-1), none)
    dx = (g[:, :, None] * w).sum(1) + torch.where(has[:, None], (a[mine] * dh[:, :, None]).sum(1), none)
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for l in range(a.shape[0]):
        at = torch.nonzero(adapters == l).flatten()
        da[l] = (dh[at][:, :, None] * x[at][:, None]).sum(0)
        db[l] = (g[at][:, :, None] * h[at][:, None]).sum(0)
    return out, dx, da, db


def run(x, w, a, b, g, adapters, s):
    leaves = [t.clone().requires_grad_(True) for t in (x, a, b)]
    out = ops.lora_linear(leaves[0], w, leaves[1], leaves[2], adapters, s)
    plain = ops.lora_linear(x, w, a, b, adapters, s)
    assert torch.equal(torch.isnan(plain), torch.isnan(out)) and torch.equal(plain == INF, out == INF)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


def operands(m, ids, r, dtype, seed, dev):
    x, w, a, b, g, adapters, s = make(m, 40, 48, r, 4, dtype, seed, dev, ids, True)
    adapters[:2] = 1  # whatever the order, someone has the adapter that is tampered with
    return x, w, a, b, g, adapters, s


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,ids,r", BATCHES)
def test_infinite_adapters(dev, m, ids, r, dtype):
    x, w, a, b, g, adapters, s = operands(m, ids, r, dtype, 1, dev)
    bad = b.clone()
    bad[1, 5, 3], bad[1, 9, 2], bad[1, 20, r - 1] = INF, -INF, INF
    bad[1, 7, 0] = bad[1, 7, 1] = INF  # two that agree or cancel, by the row's signs
    got, want = run(x, w, a, bad, g, adapters, s), formulas(x, w, a, bad, g, adapters, s)
    same_kind(got[0], want[0])
    assert (got[0][:2, 5].double().abs() == INF).all()
    bad = a.clone()
    bad[1, 3, 5], bad[1, 2, 9], bad[1, r - 1, 20] = INF, -INF, INF
    bad[1, 0, 7] = bad[1, 1, 7] = INF
    # dx alone: h has NaN now (zero times infinity has not: x is nowhere zero), and out with it
    got, want = run(x, w, bad, b, g, adapters, s), formulas(x, w, bad, b, g, adapters, s)
    same_kind(got[1], want[1])
    assert (got[1][:2, 5].double().abs() == INF).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,ids,r", BATCHES)
def test_infinite_rows(dev, m, ids, r, dtype):
    """All weights positive: a row with an infinity is infinite everywhere, also where an infinite adapter meets it."""
    x, w, a, b, g, adapters, s = operands(m, ids, r, dtype, 2, dev)
    w, a, b = w.abs() + 0.01, a.abs() + 0.01, b.abs() + 0.01
    x, g = x.clone(), g.clone()
    x[0, 4] = g[0, 4] = INF
    got = run(x, w, a, b, g, adapters, s)
    assert (got[0][0] == INF).all() and (got[1][0] == INF).all()
    assert torch.isfinite(got[0][1:]).all() and torch.isfinite(got[1][1:]).all()
    x[0, 4] = g[0, 4] = -INF
    got = run(x, w, a, b, g, adapters, s)
    assert (got[0][0] == -INF).all() and (got[1][0] == -INF).all()
    b = b.clone()
    b[1, 6, 2] = INF
    got = run(x, w, a, b, g, adapters, s)
    assert (got[0][0] == -INF).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,ids,r", BATCHES + [(6001, "mixed", 16)])
def test_gradients_of_infinite_rows(dev, m, ids, r, dtype):
    x, w, a, b, g, adapters, s = operands(m, ids, r, dtype, 3, dev)
    odd = x.clone()
    odd[1, 4], odd[1, 30] = INF, -INF
    odd[0, 11] = INF
    got, want = run(odd, w, a, b, g, adapters, s), formulas(odd, w, a, b, g, adapters, s)
    same_kind(got[2], want[2])
    assert (got[2][1, :, 4].double().abs() == INF).all()
    odd = g.clone()
    odd[1, 4], odd[0, 30] = INF, -INF
    got, want = run(x, w, a, b, odd, adapters, s), formulas(x, w, a, b, odd, adapters, s)
    same_kind(got[3], want[3])
    same_kind(got[2], want[2])
    assert (got[3][1, 4].double().abs() == INF).all()


def test_an_infinity_times_a_value_far_below_the_others(dev):
    """Half precision: a hidden value 2^-40 of the largest that it shares a scale with is not zero."""
    x, w, a, b, g, adapters, s = make(200, 40, 48, 16, 1, F16, 4, dev, "0", False)
    x = (x.float().sign() * 4e4).to(F16)
    x[7] = 0
    x[7, 3] = 2.0 ** -24
    g = g.clone()
    g[7, 4] = INF
    got, want = run(x, w, a, b, g, adapters, s), formulas(x, w, a, b, g, adapters, s)
    assert (want[3][0, 4].abs() == INF).all()
    same_kind(got[3][0, 4], want[3][0, 4])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("ids,r", [("runs", 24), ("mixed", 16), ("1", 8)])
def test_wide_tiles(dev, ids, r, dtype):
    """Products large enough for tiles of 256 rows in both directions: an infinite entry of B (of A) reaches one column of its adapter's rows, with the sign of their hidden value."""
    x, w, a, b, g, adapters, s = make(4096, 4096, 4096, r, 4, dtype, 5, dev, ids, True)
    rows = adapters == 1
    bad_a, bad_b = a.clone(), b.clone()
    places = [(700, 3, INF), (1299, 0, -INF), (4095, r - 1, INF)]
    for at, q, value in places:
        bad_a[1, q, at] = bad_b[1, at, q] = value
    leaf = x.clone().requires_grad_(True)
    out = ops.lora_linear(x, w, a, bad_b, adapters, s)
    dx, = torch.autograd.grad(ops.lora_linear(leaf, w, bad_a, b, adapters, s), leaf, g)
    h, dh = x.double() @ a[1].double().t(), g.double() @ b[1].double()
    for got, hidden in ((out, h), (dx, dh)):
        want = torch.zeros(4096, 4096, dtype=torch.float64, device=dev)
        for at, q, value in places:
            want[rows, at] = hidden[rows, q].sign() * value
        same_kind(got, want)
