"""``m_grouped_gemm_int4`` against the definition in 64 bits.

Bound before the one rounding: sums of K products in fp32 are off by at most (K + 32) 2^-24 of the sum of the summed terms' magnitudes.
In half precision those terms are x (q - z) s; in bfloat16 the operands are q + 128 (up to 159 with zero points) and the sum starts from
-(128 + 8) or -144 times the activations, so the magnitudes are up to 303 |x| s.  A gated block passes the sums' errors on with the
activation's slope (at most 1.13) and adds 2^-19 of its value.
"""
import pytest
import torch

from triton_grouped_gemm_amd import _native, ops
from triton_grouped_gemm_amd.gemm.INT4.m_grouped_gemm_int4 import m_grouped_gemm_int4
from triton_grouped_gemm_amd.quant.int4_cast import pack_int4, per_group_cast_to_int4, unpack_int4

pytestmark = pytest.mark.gpu


def act64(x, kind):
    if kind == "silu":
        return x * torch.sigmoid(x)
    return 0.5 * x * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)))


def make(sizes, n, k, gs, zeros, dtype, seed, extra=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(sum(sizes) + extra, k, generator=gen).to(dtype)
    q = torch.randint(0, 16, (len(sizes), n, k), generator=gen)
    scales = ((torch.rand(len(sizes), -(-k // gs), n, generator=gen) + 0.1) * k ** -0.5 / 4).to(dtype)
    scales = torch.where(torch.rand(scales.shape, generator=gen) < 0.2, -scales, scales)
    points = torch.randint(0, 16, scales.shape, generator=gen, dtype=torch.uint8) if zeros else None
    return x, q, scales, points


def reference(x, q, scales, points, sizes, gs, kind):
    n, k = q.shape[1:]
    outs, errs, row = [], [], 0
    for g, m in enumerate(sizes):
        spread = lambda t: t.double().repeat_interleave(gs, 0)[:k].t()
        s = spread(scales[g])
        z = spread(points[g]) if points is not None else 8.0
        xs = x[row:row + m].double()
        y = xs @ ((q[g].double() - z) * s).t()
        terms = s.abs() * 303 if x.dtype is torch.bfloat16 else ((q[g].double() - z) * s).abs()
        e = (xs.abs() @ terms.t()) * (k + 32) * 2.0 ** -24
        if kind:
            f = n // 2
            a = act64(y[:, :f], kind)
            e = 1.13 * (y[:, f:].abs() + e[:, f:]) * e[:, :f] + a.abs() * e[:, f:] + (a * y[:, f:]).abs() * 2.0 ** -19
            y = a * y[:, f:]
        outs.append(y)
        errs.append(e)
        row += m
    return torch.cat(outs), torch.cat(errs)


def check(got, want, slack, dtype):
    got, u = got.double().cpu(), torch.finfo(dtype).eps / 2
    over = (got - want).abs() - (want.abs() * u * (1 + 2 ** -6) + slack * (1 + u) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps)
    assert torch.isfinite(got).all() and (over <= 0).all(), f"off by {over.max().item():.3e} more than allowed"


CASES = [
    # sizes, n, k, gs, zeros, dtype, activation
    ([1], 8, 8, 32, False, torch.bfloat16, None),
    ([1], 32, 32, 32, True, torch.float16, "silu"),
    ([0, 1, 0], 40, 136, 64, True, torch.bfloat16, None),
    ([3, 17, 0, 16], 64, 264, 32, False, torch.float16, "gelu_tanh"),
    ([33, 1, 65], 96, 256, 128, False, torch.bfloat16, "silu"),
    ([64, 0, 130], 72, 520, 64, False, torch.bfloat16, None),
    ([31, 48], 1544, 96, 32, True, torch.bfloat16, None),
    ([5], 200, 1000, 256, True, torch.float16, None),
    ([200, 2], 64, 640, 128, True, torch.bfloat16, "gelu_tanh"),
    ([2] * 100, 352, 384, 128, False, torch.float16, None),
    ([0] * 300 + [4, 0, 1] * 100, 32, 128, 64, False, torch.bfloat16, None),
    ([7, 0, 20] * 20, 2048, 256, 128, False, torch.bfloat16, "silu"),
    ([1] * 8, 1536, 2048, 128, False, torch.bfloat16, "silu"),
]


@pytest.mark.parametrize("case", CASES, ids=[f"{len(c[0])}g{sum(c[0])}r_n{c[1]}_k{c[2]}_gs{c[3]}{'z' if c[4] else ''}{c[6] or ''}" for c in CASES])
def test_forward(dev, case):
    sizes, n, k, gs, zeros, dtype, kind = case
    x, q, scales, points = make(sizes, n, k, gs, zeros, dtype, n + k)
    want, slack = reference(x, q, scales, points, sizes, gs, kind)
    codes = pack_int4(q.to(dev))
    assert torch.equal(codes.cpu(), pack_int4(q))
    counts = torch.tensor(sizes, dtype=torch.int64 if n % 16 else torch.int32, device=dev)
    z = None if points is None else points.to(dev)
    got = m_grouped_gemm_int4(x.to(dev), codes, scales.to(dev), counts, gs, z, kind)
    check(got, want, slack, dtype)
    capped = m_grouped_gemm_int4(x.to(dev), codes, scales.to(dev), counts, gs, z, kind, numSM=3)
    check(capped, want, slack, dtype)


@pytest.mark.parametrize("dtype,gs,zeros", [(torch.bfloat16, 128, False), (torch.float16, 32, True), (torch.bfloat16, 64, True)], ids=["bf16_128", "fp16_32z", "bf16_64z"])
@pytest.mark.parametrize("k", [256, 264, 768, 1024, 1032, 1544, 2176, 3088, 4112])
def test_lengths_around_the_chunks_of_activations(dev, k, dtype, gs, zeros):
    """Tiles of up to 16, 32, 48 and 64 rows, whose activations pass through shared memory 1024, 512 and 256 values at a time, side by side and split along K."""
    sizes, n = [16, 64, 2, 32, 48, 77], 264
    x, q, scales, points = make(sizes, n, k, gs, zeros, dtype, k)
    want, slack = reference(x, q, scales, points, sizes, gs, None)
    args = (x.to(dev), pack_int4(q.to(dev)), scales.to(dev), torch.tensor(sizes, dtype=torch.int32, device=dev), gs, None if points is None else points.to(dev))
    for cap in (None, 16, 8, 3):  # 7 row tiles: split along K, 128 columns a tile, 256, and several tiles a workgroup
        got = m_grouped_gemm_int4(*args) if cap is None else m_grouped_gemm_int4(*args, numSM=cap)
        check(got, want, slack, dtype)


@pytest.mark.parametrize("kind", [None, "silu"])
@pytest.mark.parametrize("rows", [5, 90])
def test_rows_behind_the_last_group_and_neighbours_are_left_alone(dev, rows, kind):
    n, k, gs, extra = 96, 200, 64, 7
    sizes = [rows // 2, 0, rows - rows // 2]
    x, q, scales, points = make(sizes, n, k, gs, True, torch.bfloat16, 3, extra)
    x[rows:] = float("nan")
    f = n // 2 if kind else n
    base = torch.full(((rows + extra) * f + 512,), 7.0, dtype=torch.bfloat16, device=dev)
    out = base[256:256 + (rows + extra) * f].view(rows + extra, f)
    xd, cd, sd, zd, counts = x.to(dev), pack_int4(q.to(dev)), scales.to(dev), points.to(dev), torch.tensor(sizes, dtype=torch.int32, device=dev)
    _native.call("tgg_m_grouped_gemm_int4", xd.data_ptr(), cd.data_ptr(), sd.data_ptr(), zd.data_ptr(), out.data_ptr(), counts.data_ptr(), 0, 3,
                 rows + extra, n, k, gs, 0 if kind else -1, _native.BF16, -1, _native.stream_of(xd))
    want, slack = reference(x[:rows], q, scales, points, sizes, gs, kind)
    check(out[:rows], want, slack, torch.bfloat16)
    assert (out[rows:] == 7.0).all() and (base[:256] == 7.0).all() and (base[-256:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_that_are_not_finite_stay_in_their_rows(dev, dtype):
    sizes, n, k, gs = [4, 30], 64, 256, 128
    x, q, scales, _ = make(sizes, n, k, gs, False, dtype, 2)
    args = (pack_int4(q.to(dev)), scales.to(dev), torch.tensor(sizes, device=dev), gs)
    clean = m_grouped_gemm_int4(x.to(dev), *args)
    x[1, 3] = float("nan")
    x[20, 0] = float("inf")
    out = m_grouped_gemm_int4(x.to(dev), *args)
    assert torch.isnan(out[1]).all() and not torch.isfinite(out[20]).any()
    keep = [r for r in range(34) if r not in (1, 20)]
    assert torch.equal(out[keep], clean[keep])


def test_equal_calls_give_equal_bits(dev):
    sizes, n, k = [3, 0, 40, 1], 512, 2048
    x, q, scales, _ = make(sizes, n, k, 128, False, torch.bfloat16, 9)
    args = (x.to(dev), pack_int4(q.to(dev)), scales.to(dev), torch.tensor(sizes, device=dev))
    first = m_grouped_gemm_int4(*args)
    for _ in range(5):
        assert torch.equal(m_grouped_gemm_int4(*args), first)


def test_strided_operands_other_streams_and_no_rows(dev):
    sizes, n, k = [9, 20], 64, 128
    x, q, scales, _ = make(sizes, n, k, 64, False, torch.bfloat16, 4)
    codes, sd, counts = pack_int4(q.to(dev)), scales.to(dev), torch.tensor(sizes, device=dev)
    want = m_grouped_gemm_int4(x.to(dev), codes, sd, counts, 64)
    wide = torch.zeros(29, 2 * k, dtype=torch.bfloat16, device=dev)
    wide[:, :k] = x.to(dev)
    flipped = sd.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(m_grouped_gemm_int4(wide[:, :k], codes, flipped, torch.tensor(sizes), 64), want)
    side = torch.cuda.Stream()
    xd = x.to(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m_grouped_gemm_int4(xd, codes, sd, counts, 64)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert m_grouped_gemm_int4(xd[:0], codes, sd, counts * 0, 64).shape == (0, n)


def test_captured_replayed_and_compiled(dev):
    sizes, n, k = [9, 0, 60], 128, 384
    x, q, scales, points = make(sizes, n, k, 32, True, torch.bfloat16, 6)
    xd, codes, sd, zd = x.to(dev), pack_int4(q.to(dev)), scales.to(dev), points.to(dev)
    counts = torch.tensor(sizes, dtype=torch.int32, device=dev)
    call = lambda: m_grouped_gemm_int4(xd, codes, sd, counts, 32, zd, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for turn, split in enumerate([[9, 0, 60], [69, 0, 0], [1, 2, 66], [23, 23, 23]]):
        xd.copy_(torch.roll(x, turn, 0).to(dev))
        counts.copy_(torch.tensor(split, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        assert torch.equal(got, call())
    assert torch.equal(torch.compile(lambda t: m_grouped_gemm_int4(t, codes, sd, counts, 32, zd, "silu"), backend="aot_eager")(xd), call())


def test_a_decode_layer_of_four_bit_experts(dev):
    """Router, movement, gated block, down projection and combination of a decode step, against the same layer in 64 bits over the dequantised
    weights: the layer rounds its rows to bfloat16 after the block, after the down projection and at the end (2^-8 each, the first two
    through sums whose terms may cancel), so the error goes by the magnitudes."""
    tokens, hidden, ffn, experts, topk, gs = 7, 256, 128, 16, 4, 64
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(tokens, hidden, generator=gen).to(torch.bfloat16)
    logits = torch.randn(tokens, experts, generator=gen).to(torch.bfloat16)
    w1 = (torch.randn(experts, 2 * ffn, hidden, generator=gen) * hidden ** -0.5).to(torch.bfloat16)
    w2 = (torch.randn(experts, hidden, ffn, generator=gen) * ffn ** -0.5).to(torch.bfloat16)
    c1, s1, _ = per_group_cast_to_int4(w1.to(dev), gs)
    c2, s2, z2 = per_group_cast_to_int4(w2.to(dev), gs, zeros=True)
    probs, idx = ops.topk_router(logits.to(dev), topk)
    rows, row_map = ops.permute(x.to(dev), idx, num_experts=experts)
    _, counts = ops.permute_map(idx, num_experts=experts)
    y = m_grouped_gemm_int4(m_grouped_gemm_int4(rows, c1, s1, counts, gs, activation="silu"), c2, s2, counts, gs, z2)
    out = ops.unpermute(y, row_map, probs)

    spread = lambda t, k: t.double().cpu().repeat_interleave(gs, 1)[:, :k].transpose(1, 2)
    d1 = (unpack_int4(c1, 2 * ffn, hidden).double().cpu() - 8) * spread(s1, hidden)
    d2 = (unpack_int4(c2, hidden, ffn).double().cpu() - spread(z2, ffn)) * spread(s2, ffn)
    p, top = torch.softmax(logits.double(), 1).topk(topk)
    p = p / p.sum(1, keepdim=True)
    u = 2.0 ** -8
    for t in range(tokens):
        want, slack = 0, 0
        for j in range(topk):
            h = d1[top[t, j]] @ x[t].double()
            a = act64(h[:ffn], "silu") * h[ffn:]
            want = want + p[t, j] * (d2[top[t, j]] @ a)
            slack = slack + p[t, j] * (d2[top[t, j]].abs() @ a.abs()) * 2 * u
        assert ((out[t].double().cpu() - want).abs() <= slack + want.abs() * u * 1.02).all()
