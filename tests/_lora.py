"""The adapter operators' oracle: the formulas in 64 bits, and the bounds of the kernels' errors.

A sum of n products in fp32 is off by at most (n + 16) 2^-24 of the sum of their magnitudes.  The hidden values h and dh are such sums; they enter the second
product in two planes: of bfloat16 in out and dx (whatever the operands' type), which leave out at most 2^-8 of 2^-8 of a value, 2^-16; of the operands' type in dA and
dB, in fp16 2^-21 and 2^-34 of the largest value that they share a scale with.  With |.| taken of every entry, e_h = c_K s |x||A|^T and e_dh = c_N s |g||B|, the results are off by at most

    out  c_K |x||W|^T + (2^-16 + c_4R) |h||B|^T + e_h |B|^T
    dx   c_N |g||W|   + (2^-16 + c_4R) |dh||A|  + e_dh |A|
    dA   ((2^-16 + c_M) |dh| + e_dh)^T |x|          dB   |g|^T ((2^-16 + c_M) |h| + e_h)      (fp16: 2^-21)

before their one rounding, which adds half a step.
"""
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(m, n, k, r, count, dtype, seed, dev, ids="mixed", scales=True, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen)
    w = torch.randn(n, k, generator=gen) * k ** -0.5
    a = torch.randn(count, r, k, generator=gen) * k ** -0.5 * spread
    b = torch.randn(count, n, r, generator=gen) * r ** -0.5 / spread
    g = torch.randn(m, n, generator=gen)
    if ids == "mixed":
        adapters = torch.randint(-1, count, (m,), generator=gen)
    elif ids == "runs":
        adapters = torch.sort(torch.randint(0, 4, (m,), generator=gen)).values
        adapters = torch.randint(-1, count, (4,), generator=gen)[adapters]
    elif ids == "none":
        adapters = torch.full((m,), -1)
    elif ids == "outside":  # beyond the adapters on either side
        adapters = torch.randint(-5, count + 5, (m,), generator=gen)
    elif ids == "each":
        adapters = torch.arange(m) % count
    else:
        adapters = torch.full((m,), int(ids))
    s = torch.rand(count, generator=gen) + 0.5 if scales else None
    out = [t.to(dtype).to(dev) for t in (x, w, a, b, g)]
    return (*out, adapters.to(torch.int32).to(dev), None if s is None else s.to(dev))


def reference(x, w, a, b, g, adapters, s, dtype):
    """{name: (value, bound)} in 64 bits, on the operands' device."""
    x, w, a, b, g = (t.detach().double() for t in (x, w, a, b, g))
    m, k = x.shape
    n, (count, r) = w.shape[0], a.shape[:2]
    plane = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -21
    c = lambda length: (length + 16) * 2.0 ** -24
    out, e_out = x @ w.t(), c(k) * (x.abs() @ w.abs().t())
    dx, e_dx = g @ w, c(n) * (g.abs() @ w.abs())
    h, e_hid = torch.zeros(m, r, dtype=torch.float64, device=x.device), torch.zeros(m, r, dtype=torch.float64, device=x.device)
    da, e_da, db, e_db = torch.zeros_like(a), torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(b)
    for l in range(count):
        at = torch.nonzero(adapters == l).flatten()
        if not len(at):
            continue
        sl = 1.0 if s is None else s[l].double()
        xl, gl = x[at], g[at]
        hl, dhl = sl * (xl @ a[l].t()), sl * (gl @ b[l])
        e_h, e_dh = c(k) * sl * (xl.abs() @ a[l].abs().t()), c(n) * sl * (gl.abs() @ b[l].abs())
        h[at], e_hid[at] = hl, e_h + 2.0 ** -23 * hl.abs()
        shared = lambda v: 0.0 if dtype == torch.bfloat16 else 2.0 ** -34 * v.abs().max()
        out[at] += hl @ b[l].t()
        e_out[at] += ((2.0 ** -16 + c(4 * r)) * hl.abs() + e_h) @ b[l].abs().t()
        dx[at] += dhl @ a[l]
        e_dx[at] += ((2.0 ** -16 + c(4 * r)) * dhl.abs() + e_dh) @ a[l].abs()
        rows = 2 * len(at)
        da[l], e_da[l] = dhl.t() @ xl, ((plane + c(rows)) * dhl.abs() + shared(dhl) + e_dh).t() @ xl.abs()
        db[l], e_db[l] = gl.t() @ hl, gl.abs().t() @ ((plane + c(rows)) * hl.abs() + shared(hl) + e_h)
    # the two products' sums meet in one accumulator
    e_out += 2.0 ** -23 * out.abs()
    e_dx += 2.0 ** -23 * dx.abs()
    return {"out": (out, e_out), "h": (h, e_hid), "dx": (dx, e_dx), "da": (da, e_da), "db": (db, e_db)}


def check(name, got, want, bound):
    u = half_step(got.dtype)
    smallest = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    over = (got.double() - want).abs() - (want.abs() * u + bound * (1 + u) + smallest)
    assert torch.isfinite(got.float()).all(), f"{name}: not finite"
    assert (over <= 0).all(), f"{name}: off by {over.max().item():.3e} more than allowed"
