"""What the adapter and orthogonalisation operators of the library are measured on.

Three operators over stacks of matrices:

  lora   ``ops.lora_linear``: a shared projection with low-rank adapters beside it, another one for every row, forward or
         with the gradients of activations and adapters (the shared weights are frozen)
  ortho  ``ops.orthogonalize``: Newton-Schulz orthogonalisation of every matrix of a stack
  muon   ``ops.muon_update``: a stack's momentum, its orthogonalised direction and the weights' step, in place

Shapes are those of the repository's benchmark and tests (weights of 1536 x 2048, 2048 x 768, 4096 x 1536 and 1304 x 1000,
decode batches of 64 sequences, training batches of 16384 rows) and generic ones between and beside them.  ``run`` computes an
operator from elementary torch operations, or, where ``own`` is set, calls the library.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7

# No drawn case costs more than the largest listed one.
MOST_FLOPS = 6e12
MOST_BYTES = 9e8


def listed():
    return [
        # One token of one request through a small projection.  Launch and host time.
        {"name": "lora_token", "op": "lora", "rows": 1, "k": 2048, "n": 768, "rank": 8, "adapters": 4, "requests": 1,
         "mixed": False, "none": 0.0, "scales": False, "dtype": "bf16", "train": False},
        # A decode step of 64 sequences, every one with an adapter of its own choice out of 128.
        {"name": "lora_decode", "op": "lora", "rows": 64, "k": 4096, "n": 4096, "rank": 16, "adapters": 128, "requests": 64,
         "mixed": True, "none": 0.1, "scales": True, "dtype": "bf16", "train": False},
        # Half precision, odd sizes: 37 rows, K and N no multiples of a tile, rank 24.
        {"name": "lora_odd", "op": "lora", "rows": 37, "k": 1000, "n": 1544, "rank": 24, "adapters": 5, "requests": 37,
         "mixed": True, "none": 0.2, "scales": True, "dtype": "fp16", "train": False},
        # Prefill of 24 requests of unequal lengths, rank 64.
        {"name": "lora_prefill", "op": "lora", "rows": 8192, "k": 2048, "n": 4096, "rank": 64, "adapters": 16, "requests": 24,
         "mixed": False, "none": 0.1, "scales": True, "dtype": "bf16", "train": False},
        # A training batch: forward, activation gradient, gradients of eight adapters.
        {"name": "lora_train", "op": "lora", "rows": 16384, "k": 4096, "n": 4096, "rank": 16, "adapters": 8, "requests": 32,
         "mixed": False, "none": 0.0, "scales": True, "dtype": "bf16", "train": True},
        # The same pass on a small ragged batch whose rows come in any order, some without an adapter.
        {"name": "lora_train_mixed", "op": "lora", "rows": 2047, "k": 1536, "n": 2048, "rank": 32, "adapters": 16,
         "requests": 2047, "mixed": True, "none": 0.2, "scales": False, "dtype": "fp16", "train": True},
        # One small square matrix: a chain of short products.
        {"name": "ortho_one", "op": "ortho", "count": 1, "rows": 512, "cols": 512, "dtype": "bf16", "steps": 5},
        # The down projections' gradients of eight experts, tall matrices.
        {"name": "ortho_tall", "op": "ortho", "count": 8, "rows": 2048, "cols": 768, "dtype": "bf16", "steps": 5},
        # Odd sizes in 32 bits.
        {"name": "ortho_fp32", "op": "ortho", "count": 3, "rows": 1001, "cols": 1303, "dtype": "fp32", "steps": 5},
        # The gate/up projections' gradients of a layer of 64 experts.
        {"name": "ortho_experts", "op": "ortho", "count": 64, "rows": 1536, "cols": 2048, "dtype": "bf16", "steps": 5},
        # The optimiser's step for sixteen experts' down projections held in 16 bits.
        {"name": "muon_experts", "op": "muon", "count": 16, "rows": 2048, "cols": 768, "dtype": "bf16", "steps": 5,
         "nesterov": True, "weight_decay": 0.1},
        # The step for one matrix of 32-bit weights, plain momentum.
        {"name": "muon_fp32", "op": "muon", "count": 1, "rows": 1304, "cols": 1000, "dtype": "fp32", "steps": 5,
         "nesterov": False, "weight_decay": 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["lora", "lora", "ortho", "muon"])
        if op == "lora":
            rank = rng.choice([8, 16, 24, 32, 40, 64, 128])
            rows, mixed = _log_int(rng, 1, 16384), rng.random() < 0.5
            case = {"op": op, "rows": rows, "k": 8 * _log_int(rng, 8, 512), "n": 8 * _log_int(rng, 4, 512), "rank": rank,
                    "adapters": _log_int(rng, 1, 2048 // rank), "requests": rows if mixed else min(rows, _log_int(rng, 1, 64)),
                    "mixed": mixed, "none": rng.choice([0.0, 0.1, 0.5]), "scales": rng.random() < 0.5,
                    "dtype": rng.choice(["bf16", "fp16"]), "train": rng.random() < 0.4}
        else:
            case = {"op": op, "count": _log_int(rng, 1, 64), "rows": _log_int(rng, 8, 2048), "cols": _log_int(rng, 8, 2048),
                    "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "steps": 5}
            if op == "muon":
                case["dtype"] = rng.choice(["bf16", "fp32"])
                case["nesterov"], case["weight_decay"] = rng.random() < 0.5, rng.choice([0.0, 0.1])
        cost = work(case)
        if cost["flops"] <= MOST_FLOPS and cost["bytes"] <= MOST_BYTES:
            return case


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "lora":
        m, k, n, r = case["rows"], case["k"], case["n"], case["rank"]
        picks = case["requests"] * (1.0 - case["none"])
        used = case["adapters"] * (1.0 - (1.0 - 1.0 / case["adapters"]) ** picks)  # adapters that some row has, on average
        pair = r * (k + n)
        moved = (m * (k + n) + n * k + used * pair) * size + 4 * m
        low = 2 * m * (1.0 - case["none"]) * pair
        if not case["train"]:
            return {"bytes": moved, "flops": 2 * m * n * k + low}
        # the output's gradient in, the activations' and every adapter's out
        return {"bytes": moved + (m * (k + n) + case["adapters"] * pair) * size, "flops": 4 * m * n * k + 3 * low}
    count, few, many = case["count"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # a step: X X^T and (X X^T)^2 are symmetric, half of each says all; then the product with X
    flops = count * case["steps"] * (few * few * many + few ** 3 + 2 * few * few * many)
    values = count * few * many
    if case["op"] == "ortho":
        return {"bytes": 2 * values * size, "flops": flops}
    return {"bytes": values * (3 * size + 8), "flops": flops}  # weights and momentum in and out, the gradient in


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=DTYPES[case["dtype"]]):
        return (torch.randn(shape, generator=generator, device="cuda") * scale).to(dtype)

    def whole(hi, *shape):
        return torch.randint(0, hi, shape, generator=generator, device="cuda")

    state = dict(case)
    if case["op"] == "lora":
        m, k, n, r, adapters = (case[x] for x in ("rows", "k", "n", "rank", "adapters"))
        state["x"] = normal(m, k).requires_grad_(case["train"])
        state["weight"] = normal(n, k, scale=k ** -0.5)
        state["a"] = normal(adapters, r, k, scale=k ** -0.5).requires_grad_(case["train"])
        state["b"] = normal(adapters, n, r, scale=0.5 * r ** -0.5).requires_grad_(case["train"])
        # each request's adapter; a request's rows follow one another unless the batch is mixed
        chosen = whole(adapters, case["requests"])
        chosen[torch.rand(case["requests"], generator=generator, device="cuda") < case["none"]] = -1
        if case["mixed"]:
            ids = chosen[:m]
        else:
            cuts = torch.sort(whole(m, case["requests"] - 1)).values
            ids = chosen[torch.searchsorted(cuts, torch.arange(m, device="cuda"), right=True)]
        state["ids"] = ids.to(torch.int32)
        state["s"] = torch.rand(adapters, generator=generator, device="cuda") + 0.5 if case["scales"] else None
        if case["train"]:
            state["grad"] = normal(m, n)
        return state
    # a gradient's spectrum: a few strong directions over a floor of noise
    count, rows, cols = case["count"], case["rows"], case["cols"]
    inner = max(1, min(rows, cols) // 8)

    def gradient(dtype):
        left = torch.randn(count, rows, inner, generator=generator, device="cuda")
        right = torch.randn(count, inner, cols, generator=generator, device="cuda")
        strong = torch.matmul(left, right.mul_((inner * rows * cols) ** -0.5))
        return strong.add_(torch.randn(strong.shape, generator=generator, device="cuda"), alpha=0.3 * (rows * cols) ** -0.5).to(dtype)

    if case["op"] == "ortho":
        state["x"] = gradient(DTYPES[case["dtype"]])
        return state
    state["grad"] = gradient(DTYPES[case["dtype"]])
    state["momentum"] = gradient(torch.float32)
    state["weight"] = normal(count, rows, cols, scale=cols ** -0.5)
    return state


LR, BETA = 0.02, 0.95


# ---- the library's operators -----------------------------------------------------------------------------------------

def _run_own(s):
    from triton_grouped_gemm_amd import ops
    if s["op"] == "lora":
        out = ops.lora_linear(s["x"], s["weight"], s["a"], s["b"], s["ids"], scales=s["s"])
        if not s["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["x"], s["a"], s["b"]), s["grad"]))
    if s["op"] == "ortho":
        return ops.orthogonalize(s["x"], steps=s["steps"])
    ops.muon_update(s["weight"], s["grad"], s["momentum"], lr=LR, beta=BETA, nesterov=s["nesterov"],
                    weight_decay=s["weight_decay"], steps=s["steps"])
    return s["weight"], s["momentum"]


# ---- the plain forms: 32 bits, one rounding at the end ------------------------------------------------------------------

def _lora_plain(s):
    """All adapters side by side, [L R, K] and [L R, N]; a row keeps the part of its own."""
    x, w = s["x"].detach().float(), s["weight"].float()
    count, r, k = s["a"].shape
    a = s["a"].detach().float().reshape(count * r, k)
    b = s["b"].detach().float().transpose(1, 2).reshape(count * r, s["n"])
    keep = (s["ids"][:, None] == torch.arange(count, device=x.device)).float()
    if s["s"] is not None:
        keep = keep * s["s"]
    keep = keep.repeat_interleave(r, dim=1)
    h = (x @ a.t()) * keep
    out = (x @ w.t() + h @ b).to(s["x"].dtype)
    if not s["train"]:
        return out
    g = s["grad"].float()
    dh = (g @ b.t()) * keep
    dx = (g @ w + dh @ a).to(s["x"].dtype)
    da = (dh.t() @ x).to(s["x"].dtype).view(count, r, k)
    db = (h.t() @ g).to(s["x"].dtype).view(count, r, s["n"]).transpose(1, 2).contiguous()
    return out, dx, da, db


def _newton_schulz_plain(x, steps):
    """x in 32 bits -> the iterated matrices, in 32 bits."""
    a, b, c = COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1).contiguous() if tall else x
    x = (x / (x.double().square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)).float()  # (a long sum, and its error grows with every step)
    for _ in range(steps):
        gram = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-2, -1).contiguous() if tall else x


def _muon_plain(s):
    w, m = s["weight"], s["momentum"]
    g = s["grad"].float()
    m.mul_(BETA).add_(g, alpha=1.0 - BETA)
    u = BETA * m + (1.0 - BETA) * g if s["nesterov"] else m
    scale = max(1.0, s["rows"] / s["cols"]) ** 0.5
    w.copy_((w.float() * (1.0 - LR * s["weight_decay"]) - LR * scale * _newton_schulz_plain(u, s["steps"])).to(w.dtype))
    return w, m


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "lora":
        return _lora_plain(state)
    if state["op"] == "ortho":
        return _newton_schulz_plain(state["x"].float(), state["steps"]).to(state["x"].dtype)
    return _muon_plain(state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _exact_lora(s):
    """Each adapter merged into a matrix of its own: y = x (W + s B A)^T."""
    x, w = s["x"].detach().double(), s["weight"].double()
    out, train = torch.empty(s["rows"], s["n"], dtype=torch.float64, device="cuda"), s["train"]
    dx = torch.empty_like(x)
    da = torch.zeros(s["a"].shape, dtype=torch.float64, device="cuda")
    db = torch.zeros(s["b"].shape, dtype=torch.float64, device="cuda")
    for l in range(-1, s["adapters"]):
        at = torch.nonzero(s["ids"] == l).flatten()
        if not len(at):
            continue
        merged = w
        if l >= 0:
            scale = 1.0 if s["s"] is None else s["s"][l].double()
            a, b = s["a"].detach()[l].double(), s["b"].detach()[l].double()
            merged = w + scale * torch.mm(b, a)
        out[at] = torch.mm(x[at], merged.t())
        if train:
            g = s["grad"][at].double()
            dx[at] = torch.mm(g, merged)
            if l >= 0:
                full = torch.mm(g.t(), x[at]) * scale  # of the merged matrix
                da[l] = torch.mm(b.t(), full)
                db[l] = torch.mm(full, a.t())
    return (out, dx, da, db) if train else out


def _exact_directions(x, steps):
    """One matrix after another, the smaller side's products on the side where they belong."""
    found = torch.empty_like(x)
    for i in range(x.shape[0]):
        y = x[i] / (torch.linalg.vector_norm(x[i]) + EPS)
        for _ in range(steps):
            if y.shape[0] <= y.shape[1]:
                z = torch.mm(y, y.t())
                once = torch.mm(z, y)
                y = COEFFICIENTS[0] * y + COEFFICIENTS[1] * once + COEFFICIENTS[2] * torch.mm(z, once)
            else:
                z = torch.mm(y.t(), y)
                once = torch.mm(y, z)
                y = COEFFICIENTS[0] * y + COEFFICIENTS[1] * once + COEFFICIENTS[2] * torch.mm(once, z)
        found[i] = y
    return found


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lora":
        return _exact_lora(s)
    if case["op"] == "ortho":
        return _exact_directions(s["x"].double(), case["steps"])
    grad = s["grad"].double()
    momentum = s["momentum"].double() * BETA + grad * (1.0 - BETA)
    u = momentum * BETA + grad * (1.0 - BETA) if case["nesterov"] else momentum
    scale = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return s["weight"].double() * (1.0 - LR * case["weight_decay"]) - LR * scale * _exact_directions(u, case["steps"]), momentum
