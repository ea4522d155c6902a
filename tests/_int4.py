"""The 4-bit product in 64 bits with the bounds of what the kernel adds, as it adds it."""
import torch


def act64(x, kind):
    if kind == "silu":
        return x * torch.sigmoid(x)
    return 0.5 * x * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(sizes, n, k, gs, zeros, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(sum(sizes), k, generator=gen).to(dtype)
    q = torch.randint(0, 16, (len(sizes), n, k), generator=gen)
    scales = ((torch.rand(len(sizes), -(-k // gs), n, generator=gen) + 0.1) * k ** -0.5 / 4).to(dtype)
    scales = torch.where(torch.rand(scales.shape, generator=gen) < 0.2, -scales, scales)
    points = torch.randint(0, 16, scales.shape, generator=gen, dtype=torch.uint8) if zeros else None
    return x, q, scales, points


def reference(x, q, scales, points, sizes, gs, kind):
    """The outputs in 64 bits and the bounds of their errors before the one rounding.

    The kernel sums L = min(gs, 128) values of K at a time in fp32 and adds each sum, times its scale, to the output's.  In half precision a partial
    sum has L products x (q - z); in bfloat16 it has 2 L: L of x times minus the bias (136, or 144 with zero points) and L of x times the code
    plus 128 (plus 144 less the zero point).  Summed in whatever order, n terms are off by at most (n + 8) 2^-24 of the sum of their magnitudes.
    So are the ceil(K / L) scaled partial sums, with those sums' own magnitudes and (with K cut in four) the four waves' joined."""
    n, k = q.shape[1:]
    part = min(gs, 128)
    blocks = -(-k // part)
    biased = x.dtype is torch.bfloat16
    bias, base = (144.0, 144.0) if points is not None else (136.0, 128.0)
    pad = blocks * part - k
    cut = lambda t: torch.nn.functional.pad(t, (0, pad)).unflatten(-1, (blocks, part))
    outs, errs, row = [], [], 0
    for g, m in enumerate(sizes):
        spread = lambda t: t.double().t().repeat_interleave(gs, 1)[:, :k]  # [N, K]
        s = spread(scales[g])
        z = spread(points[g]) if points is not None else torch.full_like(s, 8.0)
        code = q[g].double()
        xs = cut(x[row:row + m].double()).transpose(0, 1)  # [block, row, value]
        weights = lambda w: cut(w).permute(1, 2, 0)  # [block, value, column]
        scale = weights(s)[:, 0]  # [block, column]
        sums = xs @ weights(code - z) * scale[:, None]
        y = sums.sum(0)
        if biased:
            term = bias + (code + base - (z if points is not None else 0)).abs()
            terms = 2 * part
        else:
            term, terms = (code - z).abs(), part
        e = (xs.abs() @ weights(term) * scale.abs()[:, None]).sum(0) * (terms + 8) * 2.0 ** -24
        e = e + sums.abs().sum(0) * (blocks + 8) * 2.0 ** -24
        if kind:
            f = n // 2
            a = act64(y[:, :f], kind)
            e = 1.13 * (y[:, f:].abs() + e[:, f:]) * e[:, :f] + a.abs() * e[:, f:] + (a * y[:, f:]).abs() * 2.0 ** -19
            y = a * y[:, f:]
        outs.append(y)
        errs.append(e)
        row += m
    return torch.cat(outs), torch.cat(errs)


def check(got, want, slack):
    """Every output within its bound, and all of them together within the rounding's: rounding moves an output by at most half a step of
    its own, so all outputs by at most half a step of their norm.  On average it is less than half of that (errors spread evenly over
    the step and values over the binade: (1 / 7) ^ 0.5 of it), which leaves more than the sums' errors need: those go by the bounds above only if all of
    their roundings agree, while n independent ones grow like n ^ 0.5."""
    u = half_step(got.dtype)
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all()
    over = (got - want).abs() - (want.abs() * u * (1 + 2 ** -6) + slack * (1 + u) + tiny)
    assert (over <= 0).all(), f"off by {over.max().item():.3e} more than allowed"
    off = (got - want).norm() / want.norm()
    assert off <= u, f"off by {(off / u).item():.3f} half steps of the outputs' norm"
