"""What the routing, gated and 4-bit operators of the library are measured on.

Three operators of a mixture-of-experts feed-forward layer:

  router  ``ops.topk_router``: expert ids and probabilities from the router's logits, forward or with the gradient
  gated   ``ops.gated_gmm``: both projections of a gated feed-forward block, the activation and the product in one grouped
          kernel, forward or with the gradients of activations and weights
  int4    ``m_grouped_gemm_int4``: grouped products with 4-bit weights and group scales, plain or gated

Shapes are those of the repository's benchmark and tests (128 experts, top-8, N x K of 1536 x 2048, 2048 x 768 and
4096 x 1536, up to 81920 tokens) and generic ones between and beside them.  ``run`` computes an operator from elementary
torch operations in 32 bits, or, where ``own`` is set, calls the library.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# No drawn case costs more than the largest listed one.
MOST_FLOPS = 8.3e11
MOST_BYTES = 1.1e9
# The most multiplications that the 64-bit form is asked for.
MOST_EXACT = 9e11


def listed():
    return [
        # Routing of one decode step: 64 sequences, normalised sigmoid scores.  Launch and host time.
        {"name": "router_decode", "op": "router", "tokens": 64, "experts": 128, "topk": 8, "dtype": "bf16",
         "scoring": "sigmoid", "renormalize": True, "masked": 0.0, "train": False},
        # Routing of a training batch of the benchmark's size, with its gradient.
        {"name": "router_train", "op": "router", "tokens": 81920, "experts": 128, "topk": 8, "dtype": "bf16",
         "scoring": "softmax", "renormalize": True, "masked": 0.0, "train": True},
        # Odd sizes, 32-bit logits, a tenth of them masked (and some rows wholly), probabilities over all experts: every
        # logit of a row gets a gradient.
        {"name": "router_masked", "op": "router", "tokens": 16383, "experts": 161, "topk": 6, "dtype": "fp32",
         "scoring": "softmax", "renormalize": False, "masked": 0.1, "train": True},
        # A small model's block on a handful of tokens, [K, 2F] weights in half precision.  Launch and host time.
        {"name": "gated_small", "op": "gated", "groups": 8, "rows": 96, "k": 512, "f": 344, "dtype": "fp16",
         "trans_b": False, "activation": "gelu_tanh", "train": False},
        # A decode step of 64 sequences, top-8 of 128 experts: four rows per expert, the launch streams weights.
        {"name": "gated_decode", "op": "gated", "groups": 128, "rows": 512, "k": 2048, "f": 768, "dtype": "bf16",
         "trans_b": True, "activation": "silu", "train": False},
        # A moderate ragged batch, no size a multiple of a tile, K with a tail.
        {"name": "gated_ragged", "op": "gated", "groups": 16, "rows": 8191, "k": 1000, "f": 1304, "dtype": "bf16",
         "trans_b": False, "activation": "silu", "train": False},
        # Prefill of 16384 tokens, top-8: the forward pass alone.
        {"name": "gated_prefill", "op": "gated", "groups": 128, "rows": 131072, "k": 2048, "f": 768, "dtype": "bf16",
         "trans_b": True, "activation": "silu", "train": False},
        # A training micro-batch: forward, activation gradient and weight gradient.
        {"name": "gated_train", "op": "gated", "groups": 128, "rows": 32768, "k": 2048, "f": 768, "dtype": "bf16",
         "trans_b": True, "activation": "silu", "train": True},
        # One token through its eight experts' gate/up projections, activation fused.
        {"name": "int4_token", "op": "int4", "groups": 128, "rows": 8, "n": 1536, "k": 2048, "group_size": 128,
         "zeros": False, "activation": "silu", "dtype": "bf16"},
        # The down projection of a decode step of 64 sequences.
        {"name": "int4_decode", "op": "int4", "groups": 128, "rows": 512, "n": 2048, "k": 768, "group_size": 128,
         "zeros": False, "activation": "none", "dtype": "bf16"},
        # Half precision, small scale groups with zero points, K no multiple of 128, tens of rows per expert.
        {"name": "int4_zeros", "op": "int4", "groups": 64, "rows": 2047, "n": 1544, "k": 2080, "group_size": 32,
         "zeros": True, "activation": "none", "dtype": "fp16"},
        # A large decode batch: 64 rows per expert on average, gate/up projection of the repository's decode sizes.
        {"name": "int4_batch", "op": "int4", "groups": 128, "rows": 8192, "n": 4096, "k": 1536, "group_size": 128,
         "zeros": False, "activation": "silu", "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["router", "gated", "int4"])
        if op == "router":
            experts = _log_int(rng, 4, 512)
            case = {"op": op, "tokens": _log_int(rng, 1, 81920), "experts": experts,
                    "topk": rng.randint(1, min(16, experts)), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                    "scoring": rng.choice(["softmax", "sigmoid"]), "renormalize": rng.random() < 0.5,
                    "masked": rng.choice([0.0, 0.1, 0.5]), "train": rng.random() < 0.5}
        elif op == "gated":
            case = {"op": op, "groups": _log_int(rng, 1, 128), "rows": _log_int(rng, 1, 131072),
                    "k": 8 * _log_int(rng, 8, 512), "f": 8 * _log_int(rng, 4, 256), "dtype": rng.choice(["bf16", "fp16"]),
                    "trans_b": rng.random() < 0.6, "activation": rng.choice(["silu", "gelu_tanh"]),
                    "train": rng.random() < 0.4}
        else:
            groups = _log_int(rng, 1, 128)
            activation = rng.choice(["none", "none", "silu", "gelu_tanh"])
            n = 8 * _log_int(rng, 4, 512) if activation == "none" else 32 * _log_int(rng, 2, 128)
            case = {"op": op, "groups": groups, "rows": _log_int(rng, 1, 64 * groups), "n": n,
                    "k": 32 * _log_int(rng, 2, 128), "group_size": rng.choice([32, 64, 128]),
                    "zeros": rng.random() < 0.5, "activation": activation, "dtype": rng.choice(["bf16", "fp16"])}
        cost = work(case)
        if cost["flops"] <= MOST_FLOPS and cost["bytes"] <= MOST_BYTES:
            return case


def _filled(case):
    """Groups that have rows, on average: rows choose their experts evenly."""
    return case["groups"] * (1.0 - (1.0 - 1.0 / case["groups"]) ** case["rows"])


def work(case):
    if case["op"] == "router":
        t, e, k, size = case["tokens"], case["experts"], case["topk"], BYTES[case["dtype"]]
        moved = t * e * size + 8 * t * k
        if case["train"]:
            moved += 4 * t * k + t * e * size
        return {"bytes": moved, "flops": 4 * t * e}
    if case["op"] == "gated":
        m, k, f, size = case["rows"], case["k"], case["f"], BYTES[case["dtype"]]
        weights = 2 * f * k * size
        moved = m * k * size + int(_filled(case) * weights) + m * f * size
        products = 1
        if case["train"]:  # the output's gradient in, the activations' and every group's weights' out
            moved += m * f * size + m * k * size + case["groups"] * weights
            products = 3
        return {"bytes": moved, "flops": products * 2 * m * 2 * f * k}
    m, n, k, size = case["rows"], case["n"], case["k"], BYTES[case["dtype"]]
    scale_groups = -(-k // case["group_size"])
    per_expert = n * k // 2 + n * scale_groups * (size + (1 if case["zeros"] else 0))
    outputs = n if case["activation"] == "none" else n // 2
    return {"bytes": int(_filled(case) * per_expert) + m * (k + outputs) * size, "flops": 2 * m * n * k}


def _sizes(case, generator):
    """Rows of every group: each row picks its expert, evenly."""
    picks = torch.randint(0, case["groups"], (case["rows"],), generator=generator, device="cuda")
    return torch.bincount(picks, minlength=case["groups"]).to(torch.int32)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=DTYPES[case["dtype"]]):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        flat = out.view(-1)
        for start in range(0, flat.numel(), 1 << 27):  # in pieces: the 32-bit values of all of it need not be in memory at once
            part = flat[start:start + (1 << 27)]
            part.copy_(torch.randn(part.numel(), generator=generator, device="cuda") * scale)
        return out

    state = dict(case)
    if case["op"] == "router":
        logits = normal(case["tokens"], case["experts"], scale=2.0)
        if case["masked"]:
            drop = torch.rand(logits.shape, generator=generator, device="cuda") < case["masked"]
            drop |= (torch.rand(case["tokens"], 1, generator=generator, device="cuda") < 0.01)  # rows without any expert
            logits = logits.masked_fill(drop, float("-inf"))
        state["logits"] = logits.requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = normal(case["tokens"], case["topk"], dtype=torch.float32)
        return state
    state["sizes"] = _sizes(case, generator)
    state["bounds"] = [0] + torch.cumsum(state["sizes"], 0).tolist()
    if case["op"] == "gated":
        g, m, k, f = case["groups"], case["rows"], case["k"], case["f"]
        state["a"] = normal(m, k).requires_grad_(case["train"])
        shape = (g, 2 * f, k) if case["trans_b"] else (g, k, 2 * f)
        state["b"] = normal(*shape, scale=k ** -0.5).requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = normal(m, f)
        return state
    g, m, n, k = case["groups"], case["rows"], case["n"], case["k"]
    state["x"] = normal(m, k)
    state["codes"] = torch.randint(0, 256, (g, -(-n // 16), -(-k // 128), 64, 16), generator=generator, device="cuda", dtype=torch.uint8)
    scales = torch.rand((g, -(-k // case["group_size"]), n), generator=generator, device="cuda") * 0.2 + 0.1
    state["scales"] = (scales * k ** -0.5).to(DTYPES[case["dtype"]])
    state["zero_points"] = torch.randint(4, 12, scales.shape, generator=generator, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    return state


# ---- the library's operators -----------------------------------------------------------------------------------------

def _run_own(s):
    if s["op"] == "router":
        from triton_grouped_gemm_amd import ops
        probs, indices = ops.topk_router(s["logits"], s["topk"], scoring=s["scoring"], renormalize=s["renormalize"])
        if not s["train"]:
            return probs, indices
        return probs.detach(), indices, torch.autograd.grad(probs, s["logits"], s["grad"])[0]
    if s["op"] == "gated":
        from triton_grouped_gemm_amd import ops
        out = ops.gated_gmm(s["a"], s["b"], s["sizes"], activation=s["activation"], trans_b=s["trans_b"])
        if not s["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["a"], s["b"]), s["grad"]))
    from triton_grouped_gemm_amd.gemm.INT4.m_grouped_gemm_int4 import m_grouped_gemm_int4
    activation = None if s["activation"] == "none" else s["activation"]
    return m_grouped_gemm_int4(s["x"], s["codes"], s["scales"], s["sizes"], group_size=s["group_size"],
                               zeros=s["zero_points"], activation=activation)


# ---- the plain forms: 32 bits, one rounding at the end ------------------------------------------------------------------

def _act(x, kind):
    z = x if kind == "silu" else 1.5957691216057308 * (x + 0.044715 * x * x * x)
    return x / (1.0 + torch.exp(-z))


def _act_slope(x, kind):
    if kind == "silu":
        z, dz = x, 1.0
    else:
        z, dz = 1.5957691216057308 * (x + 0.044715 * x * x * x), 1.5957691216057308 * (1.0 + 0.134145 * x * x)
    sig = 1.0 / (1.0 + torch.exp(-z))
    return sig + x * sig * (1.0 - sig) * dz


def _router_plain(s):
    k, logits = s["topk"], s["logits"].detach().float()
    indices = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = torch.gather(logits, 1, indices)
    none = chosen == float("-inf")
    top = logits.max(dim=1, keepdim=True).values
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    if s["scoring"] == "softmax":
        scores = torch.exp(logits - top)
        if not s["renormalize"]:
            scores = scores / scores.sum(dim=1, keepdim=True).clamp_min(1e-30)
    else:
        scores = 1.0 / (1.0 + torch.exp(-logits))
    probs = torch.where(none, torch.zeros_like(chosen), torch.gather(scores, 1, indices))
    if s["renormalize"]:
        probs = probs / probs.sum(dim=1, keepdim=True).clamp_min(1e-30)
    ids = torch.where(none, torch.full_like(indices, -1), indices).to(torch.int32)
    if not s["train"]:
        return probs, ids
    grad = torch.where(none, torch.zeros_like(probs), s["grad"])
    if s["renormalize"] or s["scoring"] == "softmax":
        part = probs * (grad - (grad * probs).sum(dim=1, keepdim=True)) if s["renormalize"] else probs * grad
    else:
        part = probs * grad
    if s["scoring"] == "sigmoid":
        part = part * torch.where(none, torch.zeros_like(probs), 1.0 / (1.0 + torch.exp(chosen)))
    out = torch.zeros_like(logits).scatter_add_(1, indices, part)
    if s["scoring"] == "softmax" and not s["renormalize"]:
        out = out - scores * (grad * probs).sum(dim=1, keepdim=True)
    return probs, ids, out.to(s["logits"].dtype)


def _gated_plain(s):
    a, b, bounds, f = s["a"].detach(), s["b"].detach(), s["bounds"], s["f"]
    out = torch.empty(a.shape[0], f, dtype=a.dtype, device=a.device)
    if s["train"]:
        da, db = torch.empty_like(a), torch.zeros_like(b)
    for g in range(s["groups"]):
        rows = slice(bounds[g], bounds[g + 1])
        if rows.start == rows.stop:
            continue
        x, w = a[rows].float(), b[g].float()
        w = w.t() if s["trans_b"] else w  # [K, 2F]
        h = x @ w
        gate, up = h[:, :f], h[:, f:]
        act = _act(gate, s["activation"])
        out[rows] = (act * up).to(a.dtype)
        if s["train"]:
            d = s["grad"][rows].float()
            dh = torch.cat([d * up * _act_slope(gate, s["activation"]), d * act], dim=1)
            da[rows] = (dh @ w.t()).to(a.dtype)
            dw = x.t() @ dh
            db[g] = (dw.t() if s["trans_b"] else dw).to(b.dtype)
    return (out, da, db) if s["train"] else out


def _unpack(codes, n, k):
    """[N/16, K/128, lane, 16 bytes] of one group -> the 4-bit values [N, K] in 32 bits."""
    blocks_n, blocks_k = codes.shape[:2]
    c = codes.view(blocks_n, blocks_k, 4, 16, 4, 4)  # 8-value chunk of the step, column, step of 32 values, byte
    nibbles = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2)  # position p holds value 2 (p mod 4) + p / 4 of the chunk
    values = nibbles.view(blocks_n, blocks_k, 4, 16, 4, 2, 4).transpose(-1, -2).reshape(blocks_n, blocks_k, 4, 16, 4, 8)
    return values.permute(0, 3, 1, 4, 2, 5).reshape(blocks_n * 16, blocks_k * 128)[:n, :k].float()


def _int4_plain(s):
    x, bounds, n, k, size = s["x"], s["bounds"], s["n"], s["k"], s["group_size"]
    outputs = n if s["activation"] == "none" else n // 2
    out = torch.empty(x.shape[0], outputs, dtype=x.dtype, device=x.device)
    for g in range(s["groups"]):
        rows = slice(bounds[g], bounds[g + 1])
        if rows.start == rows.stop:
            continue
        zero = s["zero_points"][g].float() if s["zero_points"] is not None else torch.full_like(s["scales"][g], 8.0, dtype=torch.float32)
        spread = lambda t: t.repeat_interleave(size, dim=0)[:k].t()
        w = (_unpack(s["codes"][g], n, k) - spread(zero)) * spread(s["scales"][g].float())
        y = x[rows].float() @ w.t()
        if s["activation"] != "none":
            y = _act(y[:, :outputs], s["activation"]) * y[:, outputs:]
        out[rows] = y.to(x.dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"router": _router_plain, "gated": _gated_plain, "int4": _int4_plain}[state["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _exact_router(s):
    logits = s["logits"].detach().double()
    t, e = logits.shape
    k = s["topk"]
    # position of every expert in its row's order: how many come before it
    left = logits.clone()
    ids = []
    for _ in range(k):
        best = left.max(dim=1, keepdim=True).values
        at = torch.where(left == best, torch.arange(e, device=logits.device), e).min(dim=1).values
        at = torch.where(best[:, 0] == float("-inf"), -1, at)
        ids.append(at)
        left = torch.where(torch.arange(e, device=logits.device) == at[:, None], float("-inf"), left)
    ids = torch.stack(ids, dim=1)
    real = ids >= 0
    leaf = torch.where(logits == float("-inf"), torch.full_like(logits, -1e6), logits).requires_grad_(True)
    with torch.enable_grad():
        weights = torch.log_softmax(leaf, dim=1) if s["scoring"] == "softmax" else torch.nn.functional.logsigmoid(leaf)
        picked = torch.gather(weights, 1, ids.clamp_min(0))
        picked = torch.where(real, picked, torch.full_like(picked, -2e6))
        if s["renormalize"]:
            probs = torch.softmax(picked, dim=1)
        else:
            probs = torch.exp(picked)
        probs = torch.where(real, probs, torch.zeros_like(probs))
        if not s["train"]:
            return probs.detach(), ids.to(torch.int32)
        (grad,) = torch.autograd.grad((probs * s["grad"].double()).sum(), leaf)
    grad = torch.where(logits == float("-inf"), torch.zeros_like(grad), grad)
    return probs.detach(), ids.to(torch.int32), grad


def _exact_gated(s):
    f, bounds = s["f"], s["bounds"]
    outs, das = [], []
    dbs = torch.zeros(s["b"].shape, dtype=torch.float64, device="cuda") if s["train"] else None
    for g in range(s["groups"]):
        lo, hi = bounds[g], bounds[g + 1]
        x = s["a"].detach()[lo:hi].double().requires_grad_(s["train"])
        w = s["b"].detach()[g].double().requires_grad_(s["train"])
        with torch.set_grad_enabled(s["train"]):
            gate_w, up_w = (w[:f].t(), w[f:].t()) if s["trans_b"] else (w[:, :f], w[:, f:])
            gate, up = torch.mm(x, gate_w), torch.mm(x, up_w)
            if s["activation"] == "silu":
                y = gate * torch.sigmoid(gate) * up
            else:
                y = 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3))) * up
            if s["train"]:
                dx, dw = torch.autograd.grad(y, (x, w), s["grad"][lo:hi].double())
                das.append(dx)
                dbs[g] = dw
        outs.append(y.detach())
    return (torch.cat(outs), torch.cat(das), dbs) if s["train"] else torch.cat(outs)


def _exact_int4(s):
    n, k, size = s["n"], s["k"], s["group_size"]
    row, col = torch.arange(n, device="cuda")[:, None], torch.arange(k, device="cuda")[None, :]
    tile = (row // 16) * (-(-k // 128)) + col // 128
    lane = (col % 32) // 8 * 16 + row % 16
    place = (col % 2) * 4 + col % 8 // 2  # among the eight nibbles of the chunk's four bytes
    at = (tile * 64 + lane) * 16 + col % 128 // 32 * 4 + place // 2
    shift = place % 2 * 4
    outs = []
    for g in range(s["groups"]):
        lo, hi = s["bounds"][g], s["bounds"][g + 1]
        q = (s["codes"][g].reshape(-1)[at].to(torch.int64) >> shift) & 15
        zero = 8 if s["zero_points"] is None else s["zero_points"][g].double().t()[:, (col // size)[0]]
        w = (q.double() - zero) * s["scales"][g].double().t()[:, (col // size)[0]]
        y = torch.mm(s["x"][lo:hi].double(), w.t())
        if s["activation"] == "silu":
            y = y[:, :n // 2] * torch.sigmoid(y[:, :n // 2]) * y[:, n // 2:]
        elif s["activation"] == "gelu_tanh":
            gate = y[:, :n // 2]
            y = 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3))) * y[:, n // 2:]
        outs.append(y)
    return torch.cat(outs)


def exact(case, seed):
    if work(case)["flops"] > MOST_EXACT:
        return None
    state = prepare(case, seed)
    return {"router": _exact_router, "gated": _exact_gated, "int4": _exact_int4}[case["op"]](state)
