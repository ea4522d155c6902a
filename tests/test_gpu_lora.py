"""``ops.lora_linear`` and its gradients against the formulas in 64 bits (bounds in _lora.py)."""
import pytest
import torch

from _lora import check, make, reference
from triton_grouped_gemm_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16

CASES = [
    # m, n, k, r, adapters, dtype, ids, scales
    (1, 8, 8, 8, 1, BF16, "0", False),
    (1, 264, 520, 16, 3, F16, "2", True),
    (3, 72, 2056, 24, 5, BF16, "mixed", True),
    (16, 128, 128, 128, 4, F16, "each", False),
    (17, 200, 328, 40, 30, BF16, "each", True),
    (31, 520, 64, 8, 2, F16, "runs", True),
    (64, 1000, 1032, 64, 64, BF16, "each", True),
    (64, 136, 72, 72, 7, F16, "none", True),
    (65, 64, 64, 16, 4, BF16, "mixed", True),
    (130, 264, 200, 32, 3, F16, "runs", True),
    (128, 256, 256, 8, 1, BF16, "0", False),
    (300, 392, 1000, 120, 9, BF16, "mixed", True),
    (257, 8, 4096, 64, 2, F16, "outside", True),
    (513, 1544, 8, 16, 200, BF16, "each", False),
    (1000, 136, 136, 24, 1024, F16, "each", True),
    (700, 128, 392, 72, 6, BF16, "none", False),
    (127, 520, 264, 16, 100, BF16, "each", True),
    (129, 520, 264, 16, 100, BF16, "each", True),
    (140, 72, 64, 16, 4, F16, "mixed", True),
    (8200, 136, 264, 40, 3, BF16, "mixed", True),
    (8193, 72, 136, 64, 2, F16, "runs", False),
]


def run(x, w, a, b, g, adapters, s):
    leaves = [t.clone().requires_grad_(True) for t in (x, a, b)]
    out = ops.lora_linear(leaves[0], w, leaves[1], leaves[2], adapters, s)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


@pytest.mark.parametrize("m,n,k,r,count,dtype,ids,scales", CASES)
def test_forward_and_gradients(dev, m, n, k, r, count, dtype, ids, scales):
    t = make(m, n, k, r, count, dtype, 1, dev, ids, scales)
    want = reference(*t, dtype)
    x, w, a, b, g, adapters, s = t
    check("out", ops.lora_linear(x, w, a, b, adapters, s), *want["out"])
    check("out, 64-bit ids", ops.lora_linear(x, w, a, b, adapters.long(), s), *want["out"])
    for name, got in zip(("out", "dx", "da", "db"), run(*t)):
        check(name, got, *want[name])


@pytest.mark.parametrize("dtype,ids", [(BF16, "mixed"), (F16, "runs")])
def test_wide_tiles_and_parts_of_the_rows(dev, dtype, ids):
    """Enough tiles for the wide ones in both directions; the adapters' gradients are summed in parts."""
    t = make(6001, 2568, 4104, 16, 5, dtype, 2, dev, ids)
    want = reference(*t, dtype)
    for name, got in zip(("out", "dx", "da", "db"), run(*t)):
        check(name, got, *want[name])


@pytest.mark.parametrize("m,dtype,ids", [(6001, BF16, "mixed"), (6001, F16, "runs"), (2050, BF16, "runs"), (1025, BF16, "runs"), (513, F16, "0")])
def test_gradients_in_parts_of_the_rows(dev, m, dtype, ids):
    """Few columns: the rows are shared out over many workgroups, of which some have no row of an adapter."""
    t = make(m, 264, 392, 24, 2, dtype, 5, dev, ids)
    want = reference(*t, dtype)
    for name, got in zip(("out", "dx", "da", "db"), run(*t)):
        check(name, got, *want[name])


def test_hidden_values(dev):
    for m in (5, 200):
        x, w, a, b, g, adapters, s = make(m, 64, 256, 24, 3, BF16, 3, dev)
        _, h = torch.ops.moe.lora_linear_hidden(x, w, a, b, adapters, s)
        value, bound = reference(x, w, a, b, g, adapters, s, BF16)["h"]
        assert ((h.double() - value).abs() <= bound).all()
        assert (h[adapters < 0] == 0).all()


@pytest.mark.parametrize("spread", [2.0 ** -14, 2.0 ** 13])
def test_half_precision_keeps_hidden_values_beyond_its_range(dev, spread):
    """Adapters whose hidden values are far below (above) half precision's range while the outputs are ordinary."""
    for m in (20, 150):
        t = make(m, 72, 64, 16, 2, F16, 4, dev, "mixed", False, spread)
        x, w, a, b, g, adapters, s = t
        a = (a.float() * (0.5 if spread > 1 else 1)).to(F16)
        x = x * (8 if spread > 1 else 0.125)
        t = (x, w, a, b, g, adapters, s)
        want = reference(*t, F16)
        got = run(*t)
        check("out", got[0], *want["out"])
        # the gradient of a far-away factor may itself leave the type's range
        for name, value in zip(("dx", "da", "db"), got[1:]):
            if want[name][0].abs().max() < 60000:
                check(name, value, *want[name])


def test_small_gradients_in_half_precision(dev):
    x, w, a, b, g, adapters, s = make(300, 72, 64, 16, 2, F16, 5, dev, "mixed", False)
    g = (g.float() * 2e-6).to(F16)
    g[:150] = 0  # the first rows bring no scale along
    x = x * 64
    want = reference(x, w, a, b, g, adapters, s, F16)
    for name, got in zip(("out", "dx", "da", "db"), run(x, w, a, b, g, adapters, s)):
        check(name, got, *want[name])


def test_gradients_against_differences(dev):
    """The directional derivative of sum(g out) in every operand, from outputs that are exact to half a step."""
    x, w, a, b, g, adapters, s = make(90, 64, 48, 8, 3, F16, 6, dev)
    _, dx, da, db = run(x, w, a, b, g, adapters, s)
    gd = g.double()
    for name, t, grad in (("x", x, dx), ("a", a, da), ("b", b, db)):
        d = torch.randn(t.shape, generator=torch.Generator().manual_seed(7)).to(dev).half()
        step = 0.25
        lo, hi = (t.double() - step * d.double()).half(), (t.double() + step * d.double()).half()
        move = hi.double() - lo.double()  # what the operand really moved
        args = lambda v: {"x": (v, w, a, b), "a": (x, w, v, b), "b": (x, w, a, v)}[name]
        up, down = ops.lora_linear(*args(hi), adapters, s).double(), ops.lora_linear(*args(lo), adapters, s).double()
        measured, told = ((up - down) * gd).sum(), (grad.double() * move).sum()
        # out is linear in each operand: what is left is the outputs' and the gradients' rounding (2^-11 each), whose signs are independent (four deviations)
        noise = (((up.abs() + down.abs()) * gd.abs()).square().sum() + (grad.double() * move).square().sum()).sqrt() * 2.0 ** -11
        middle = ((grad.double().abs() * 2.0 ** -11) * (lo.double() + hi.double() - 2 * t.double()).abs()).sum()
        assert (measured - told).abs() <= 4 * noise + middle, name


def test_shared_weights_gradient(dev):
    x, w, a, b, g, adapters, s = make(333, 136, 200, 16, 4, BF16, 8, dev)
    wl = w.clone().requires_grad_(True)
    out = ops.lora_linear(x, wl, a, b, adapters, s)
    (dw,) = torch.autograd.grad(out, wl, g)
    want = g.double().t() @ x.double()
    check("dw", dw, want, (333 + 16) * 2.0 ** -24 * (g.double().abs().t() @ x.double().abs()))


@pytest.mark.parametrize("wanted", [(True, False, False), (False, True, False), (False, False, True), (True, True, False)])
def test_some_gradients_only(dev, wanted):
    t = make(150, 72, 136, 16, 4, BF16, 9, dev)
    x, w, a, b, g, adapters, s = t
    _, *all_three = run(*t)
    leaves = [v.clone().requires_grad_(on) for v, on in zip((x, a, b), wanted)]
    out = ops.lora_linear(leaves[0], w, leaves[1], leaves[2], adapters, s)
    got = torch.autograd.grad(out, [v for v in leaves if v.requires_grad], g)
    for value, want in zip(got, [v for v, on in zip(all_three, wanted) if on]):
        assert torch.equal(value, want)


def test_empty_batch_and_empty_adapters(dev):
    x, w, a, b, g, adapters, s = make(0, 72, 64, 8, 3, BF16, 10, dev)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, a, b)]
    out = ops.lora_linear(*leaves, adapters, s)
    assert out.shape == (0, 72)
    grads = torch.autograd.grad(out, leaves, torch.zeros_like(out))
    assert all((g == 0).all() for g in grads)
    t = make(100, 72, 64, 8, 3, BF16, 11, dev, "1")
    _, _, da, db = run(*t)
    assert (da[0] == 0).all() and (da[2] == 0).all() and (db[0] == 0).all() and (db[2] == 0).all() and (da[1] != 0).any()


@pytest.mark.parametrize("m,dtype", [(40, BF16), (300, BF16), (300, F16)])
def test_rows_do_not_touch_each_other(dev, m, dtype):
    """NaN in a row, or in another adapter, stays there; a row's bits do not depend on what stands beside it."""
    x, w, a, b, g, adapters, s = make(m, 136, 72, 16, 5, dtype, 12, dev, "each")
    plain = ops.lora_linear(x, w, a, b, adapters, s)
    y = x.clone()
    y[7] = float("nan")
    got = ops.lora_linear(y, w, a, b, adapters, s)
    rest = torch.arange(m, device=dev) != 7
    assert torch.isnan(got[7]).all() and torch.equal(got[rest], plain[rest])
    bad = a.clone()
    bad[3] = float("inf")
    got = ops.lora_linear(x, w, bad, b, adapters, s)
    rest = adapters != 3
    assert torch.equal(got[rest], plain[rest]) and not torch.isfinite(got[~rest]).any()
    bad = b.clone()
    bad[2] = float("nan")
    got = ops.lora_linear(x, w, a, bad, adapters, s)
    rest = adapters != 2
    assert torch.equal(got[rest], plain[rest]) and torch.isnan(got[~rest]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_broken_adapter_in_the_backward_pass(dev, dtype):
    """Its own gradients, and those of its rows, are what the formulas say; nobody else's change."""
    t = make(200, 136, 72, 16, 5, dtype, 18, dev, "each")
    x, w, a, b, g, adapters, s = t
    _, dx, da, db = run(*t)
    bad = a.clone()
    bad[1, 3, 5] = float("nan")
    _, dx2, da2, db2 = run(x, w, bad, b, g, adapters, s)
    others, rest = torch.arange(5, device=dev) != 1, adapters != 1
    assert torch.equal(dx2[rest], dx[rest]) and torch.isnan(dx2[~rest][:, 5]).all()
    assert torch.equal(da2, da)  # (dA reads B, x and the gradient)
    assert torch.equal(db2[others], db[others]) and torch.isnan(db2[1][:, 3]).all()
    bad = b.clone()
    bad[4] = float("inf")
    _, dx2, da2, db2 = run(x, w, a, bad, g, adapters, s)
    others, rest = torch.arange(5, device=dev) != 4, adapters != 4
    assert torch.equal(dx2[rest], dx[rest]) and not torch.isfinite(dx2[~rest]).any()
    assert torch.equal(da2[others], da[others]) and torch.equal(db2, db)


def test_another_stream_and_a_side_effect_free_call(dev):
    x, w, a, b, g, adapters, s = make(120, 64, 64, 16, 3, BF16, 19, dev)
    want = ops.lora_linear(x, w, a, b, adapters, s)
    kept = [t.clone() for t in (x, w, a, b, adapters, s)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.lora_linear(x, w, a, b, adapters, s)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(p, q) for p, q in zip(kept, (x, w, a, b, adapters, s)))


def test_compiled(dev):
    x, w, a, b, g, adapters, s = make(90, 64, 72, 16, 3, BF16, 21, dev)
    want = run(x, w, a, b, g, adapters, s)
    call = torch.compile(lambda x, a, b: ops.lora_linear(x, w, a, b, adapters, s) * 1.0, fullgraph=True, backend="aot_eager")
    leaves = [t.clone().requires_grad_(True) for t in (x, a, b)]
    out = call(*leaves)
    got = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(p, q) for p, q in zip((out.detach(), *got), want))
    with torch.no_grad():
        assert torch.equal(call(x, a, b), want[0])


def test_the_native_path_and_the_operator_agree(dev):
    for m in (3, 200):
        x, w, a, b, g, adapters, s = make(m, 64, 72, 16, 3, F16, 22, dev)
        assert torch.equal(ops.lora_linear(x, w, a, b, adapters, s), torch.ops.moe.lora_linear(x, w, a, b, adapters, s))
        _, h = torch.ops.moe.lora_linear_hidden(x, w, a, b, adapters, s)
        assert all(torch.equal(p, q) for p, q in zip(run(x, w, a, b, g, adapters, s)[1:], torch.ops.moe.lora_linear_backward(g, x, w, a, b, adapters, s, h, True, True, True)))


def test_strided_operands(dev):
    x, w, a, b, g, adapters, s = make(90, 64, 72, 16, 5, BF16, 13, dev)
    want = ops.lora_linear(x, w, a, b, adapters, s)
    assert torch.equal(ops.lora_linear(x.t().contiguous().t(), w.t().contiguous().t(), a.transpose(1, 2).contiguous().transpose(1, 2),
                                       b.transpose(1, 2).contiguous().transpose(1, 2), adapters.repeat_interleave(2)[::2], s.repeat_interleave(2)[::2]), want)


def test_same_bits_every_time(dev):
    t = make(3000, 264, 520, 32, 7, BF16, 14, dev)
    first = run(*t)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(run(*t), first))


def test_leaves_shared_by_two_calls(dev):
    """One adapter set used twice: its gradients add up."""
    x, w, a, b, g, adapters, s = make(120, 64, 64, 16, 3, BF16, 15, dev)
    al = a.clone().requires_grad_(True)
    (ops.lora_linear(x, w, al, b, adapters, s) + ops.lora_linear(x, w, al, b, adapters, s)).backward(g)
    _, _, da, _ = run(x, w, a, b, g, adapters, s)
    assert torch.equal(al.grad, (da.float() * 2).to(BF16))


def test_captured_and_replayed(dev):
    """Forward of a decode batch and of a long one, and a backward pass, in one graph; new values and adapters at every replay, eager work in between."""
    small, large = make(20, 136, 200, 16, 6, BF16, 16, dev), make(400, 136, 200, 16, 6, BF16, 17, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.lora_linear(small[0], *small[1:4], *small[5:])
        run(*large)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    leaves = [t.clone().requires_grad_(True) for t in (large[0], large[2], large[3])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out_small = ops.lora_linear(small[0], *small[1:4], *small[5:])
        out = ops.lora_linear(leaves[0], large[1], leaves[1], leaves[2], large[5], large[6])
        grads = torch.autograd.grad(out, leaves, large[4])
    for seed in range(4):
        new_small, new_large = make(20, 136, 200, 16, 6, BF16, 20 + seed, dev), make(400, 136, 200, 16, 6, BF16, 30 + seed, dev, "runs")
        with torch.no_grad():
            for old, new in zip(small, new_small):
                old.copy_(new)
            for old, new in zip((leaves[0], large[1], leaves[1], leaves[2], large[4], large[5], large[6]), new_large):
                old.copy_(new)
        want_small = ops.lora_linear(new_small[0], *new_small[1:4], *new_small[5:])
        want = run(*new_large)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out_small, want_small)
        assert all(torch.equal(p, q) for p, q in zip((out.detach(), *grads), want))


def test_two_streams_at_once(dev):
    ts = [make(300, 264, 200, 32, 6, BF16, 40 + i, dev) for i in range(2)]
    want = [run(*t) for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*ts[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(p, q) for each in got[i] for p, q in zip(each, want[i]))


def test_operators_pass_opcheck(dev):
    x, w, a, b, g, adapters, s = make(70, 64, 72, 16, 3, BF16, 50, dev)
    torch.library.opcheck(torch.ops.moe.lora_linear, (x, w, a, b, adapters, s), test_utils=("test_schema", "test_faketensor"))
    _, h = torch.ops.moe.lora_linear_hidden(x, w, a, b, adapters, None)
    torch.library.opcheck(torch.ops.moe.lora_linear_backward, (g, x, w, a, b, adapters, None, h, True, False, True), test_utils=("test_schema", "test_faketensor"))
