"""Cases that measure the tensor operators: 8-bit rows and their scores, and the softmax loss over a base.

`run` computes one pass, in plain torch operations (own = False) or through proxima_b200 (own = True), on what
`prepare` made. `work` counts the bytes and operations a pass cannot do without; `exact` is the same pass in 64 bits.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100


def listed():
    return [
        # One embedding arriving from a model, cut to 8 bits before it is scored.
        {"name": "quantize_query_768_f32", "op": "quantize", "n": 1, "d": 768, "type": "f32"},
        # A base of 1M x 128 cut to 8 bits when an index is built, and read back.
        {"name": "quantize_base_1m_128_f32", "op": "quantize", "n": 1_000_000, "d": 128, "type": "f32"},
        # One query against a base of 1M x 128: the base's read is the cost.
        {"name": "scores_1_1m_128_f32", "op": "scores", "m": 1, "n": 1_000_000, "d": 128, "type": "f32", "bias": False},
        # A small batch against the same base.
        {"name": "scores_64_1m_128_f32", "op": "scores", "m": 64, "n": 1_000_000, "d": 128, "type": "f32", "bias": False},
        # A batch of 1000 sentence embeddings against 100k: the whole score matrix, for fusion with another ranker.
        {"name": "scores_1000_100k_384_f32", "op": "scores", "m": 1000, "n": 100_000, "d": 384, "type": "f32", "bias": False},
        # The largest: 10k queries against 100k rows of 768, scores in 16 bits.
        {"name": "scores_10k_100k_768_bf16", "op": "scores", "m": 10_000, "n": 100_000, "d": 768, "type": "bf16", "bias": False},
        # Odd sizes with a term per row (L2 order: minus half the row's squared norm).
        {"name": "scores_37_99991_100_f16", "op": "scores", "m": 37, "n": 99_991, "d": 100, "type": "f16", "bias": True},
        # Log-likelihood of one query's row under a softmax over 100k rows (evaluation, no gradient).
        {"name": "softmax_1_100k_384_bf16", "op": "softmax", "t": 1, "v": 100_000, "d": 384, "type": "bf16",
         "grad": False, "bias": False, "ignored": 0.0},
        # A training step of 1000 queries against a whole base of 100k x 384.
        {"name": "softmax_1000_100k_384_bf16_train", "op": "softmax", "t": 1000, "v": 100_000, "d": 384, "type": "bf16",
         "grad": True, "bias": False, "ignored": 0.0},
        # In-batch training: every query's own row against the batch's other rows, some queries ignored.
        {"name": "softmax_8192_8192_768_f16_train", "op": "softmax", "t": 8192, "v": 8192, "d": 768, "type": "f16",
         "grad": True, "bias": False, "ignored": 0.1},
        # Odd sizes; a term per row that corrects for how rows were sampled, and leaves some rows out.
        {"name": "softmax_333_50021_100_bf16_train", "op": "softmax", "t": 333, "v": 50_021, "d": 100, "type": "bf16",
         "grad": True, "bias": True, "ignored": 0.05},
        # A base of 1M x 128 as the classes of 1000 queries, evaluated.
        {"name": "softmax_1000_1m_128_bf16", "op": "softmax", "t": 1000, "v": 1_000_000, "d": 128, "type": "bf16",
         "grad": False, "bias": False, "ignored": 0.0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _dim(rng):
    # Embedding sizes are mostly multiples of 8, with odd ones among them.
    d = _log_int(rng, 16, 1024)
    return d if rng.random() < 0.25 else (d + 7) // 8 * 8


def draw(rng):
    op = rng.choice(["quantize", "scores", "scores", "softmax", "softmax"])
    d = _dim(rng)
    if op == "quantize":
        n = _log_int(rng, 1, 128_000_000 // d)
        return {"op": op, "n": n, "d": d, "type": rng.choice(["f32", "f16", "bf16"])}
    if op == "scores":
        n = _log_int(rng, 1000, 1_000_000)
        m = _log_int(rng, 1, min(10_000, 1_000_000_000 // n))
        return {"op": op, "m": m, "n": n, "d": d, "type": rng.choice(["f32", "f16", "bf16"]), "bias": rng.random() < 0.5}
    v = _log_int(rng, 256, 1_000_000)
    t = _log_int(rng, 1, max(1, min(8192, 200_000_000 // v, 38_000_000_000 // (v * d))))
    return {"op": op, "t": t, "v": v, "d": d, "type": rng.choice(["f16", "bf16"]), "grad": rng.random() < 0.7,
            "bias": rng.random() < 0.5, "ignored": rng.choice([0.0, 0.1])}


def _embeddings(n, d, gen):
    x = torch.randn(n, d, device="cuda", generator=gen)
    return x / x.square().sum(1, keepdim=True).sqrt()


def _pitched(n, d, unit, dtype):
    """An n x d array whose rows start on 16-byte boundaries, as an index stores them."""
    return torch.empty(n, (d + unit - 1) // unit * unit, dtype=dtype, device="cuda")[:, :d]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    d, dtype = case["d"], _TYPES[case["type"]]
    if case["op"] == "quantize":
        s["x"] = _embeddings(case["n"], d, gen).to(dtype)
    elif case["op"] == "scores":
        s["queries"] = _embeddings(case["m"], d, gen)
        rows = _embeddings(case["n"], d, gen)
        s["scales"] = rows.abs().amax(1) / 127
        s["codes"] = _pitched(case["n"], d, 16, torch.int8)
        s["codes"].copy_((rows / s["scales"][:, None]).round().clamp(-127, 127))
        # Rows of several lengths, as an L2 base has.
        s["scales"] *= torch.rand(case["n"], device="cuda", generator=gen) + 0.5
        s["bias"] = None
        if case["bias"]:
            s["bias"] = -0.5 * (s["codes"].float() * s["scales"][:, None]).square().sum(1)
    else:
        t, v = case["t"], case["v"]
        rows = _embeddings(v, d, gen)
        targets = torch.randint(0, v, (t,), device="cuda", generator=gen)
        # A query is its row, moved by noise of the same length.
        q = rows[targets] + _embeddings(t, d, gen)
        q = q / q.square().sum(1, keepdim=True).sqrt()
        s["bias"] = None
        if case["bias"]:
            b = torch.randn(v, device="cuda", generator=gen)
            left_out = torch.rand(v, device="cuda", generator=gen) < 0.1
            left_out[targets] = False
            s["bias"] = b.masked_fill(left_out, -math.inf)
        if case["ignored"]:
            targets = targets.masked_fill(torch.rand(t, device="cuda", generator=gen) < case["ignored"], IGNORE)
            targets[0] = targets[0].clamp(min=0)
        s["targets"] = targets
        s["scale"] = 20.0  # a temperature of 0.05
        # Gradients of a mean over many queries underflow in fp16, where programs scale the loss: the sum does it here.
        s["reduction"] = ("sum" if dtype == torch.float16 else "mean") if case["grad"] else "none"
        s["queries"], s["rows"] = _pitched(t, d, 8, dtype), _pitched(v, d, 8, dtype)
        s["queries"].copy_(q)
        s["rows"].copy_(rows)
        if case["grad"]:
            s["queries"].requires_grad_()
            s["rows"].requires_grad_()
    return s


def run(state):
    with torch.set_grad_enabled(bool(state.get("grad"))):
        return _own(state) if own else _plain(state)


def _own(s):
    import proxima_b200 as px

    if s["op"] == "quantize":
        codes, scales = px.quantize_rows(s["x"])
        return px.dequantize_rows(codes, scales), scales
    if s["op"] == "scores":
        codes, scales = px.quantize_rows(s["queries"])
        return px.int8_scores(codes, scales, s["codes"], s["scales"], bias=s["bias"], dtype=_TYPES[s["type"]])
    loss = px.softmax_cross_entropy(s["queries"], s["rows"], s["targets"], scale=s["scale"], bias=s["bias"],
                                    ignore_index=IGNORE, reduction=s["reduction"])
    if not s["grad"]:
        return loss
    return (loss.detach(), *torch.autograd.grad(loss, (s["queries"], s["rows"])))


def _plain_quantize(x):
    x = x.float()
    # The quotients in 64 bits: in 32 some land on the other side of a half.
    scales = (x.abs().amax(1).double() / 127).float()
    return (x.double() / scales.double()[:, None]).round().clamp(-127, 127).float(), scales


@torch.no_grad()
def _plain(s):
    if s["op"] == "quantize":
        codes, scales = _plain_quantize(s["x"])
        return codes.to(torch.int8).float() * scales[:, None], scales
    if s["op"] == "scores":
        codes, scales = _plain_quantize(s["queries"])
        out = (codes @ s["codes"].float().T) * scales[:, None] * s["scales"]
        if s["bias"] is not None:
            out += s["bias"]
        return out.to(_TYPES[s["type"]])
    q, rows, targets = s["queries"].float(), s["rows"].float(), s["targets"]
    z = (q @ rows.T) * s["scale"]
    if s["bias"] is not None:
        z += s["bias"]
    used = targets != IGNORE
    at = torch.where(used, targets, 0)[:, None]
    target = z.gather(1, at)
    # The loss is softplus(log of the other rows' sum - target): no cancellation where the target's own share is near 1.
    z.scatter_(1, at, -math.inf)
    top = z.amax(1, keepdim=True)
    p = (z - top).exp()
    total = p.sum(1, keepdim=True)
    a = top + total.log() - target
    loss = torch.where(used, (a.clamp(min=0) + torch.log1p((-a.abs()).exp()))[:, 0], 0.0)
    if not s["grad"]:
        return loss
    share = 1 / (1 + (-a).exp())  # of the other rows; the target's gradient is minus it
    p *= share / total
    p.scatter_(1, at, -share)
    parts = used.sum() if s["reduction"] == "mean" else 1
    p *= used[:, None] * (s["scale"] / parts)
    return loss.sum() / parts, (p @ rows).to(s["queries"].dtype), (p.T @ q).to(s["rows"].dtype)


def work(case):
    d, size = case["d"], _TYPES[case["type"]].itemsize
    if case["op"] == "quantize":
        n = case["n"]
        # x read, codes and scales written and read, the values they stand for written (fp32).
        return {"bytes": n * d * (size + 2 + 4) + 8 * n, "flops": 3 * n * d}
    if case["op"] == "scores":
        m, n = case["m"], case["n"]
        return {"bytes": 4 * m * d + n * d + 4 * n * (2 if case["bias"] else 1) + m * n * size, "flops": 2 * m * n * d}
    t, v = case["t"], case["v"]
    inputs = (t + v) * d * size + 8 * t + (4 * v if case["bias"] else 0)
    if not case["grad"]:
        return {"bytes": inputs + 4 * t, "flops": 2 * t * v * d}
    # The logits once, and the two gradients.
    return {"bytes": inputs + (t + v) * d * size + 4, "flops": 6 * t * v * d}


def _exact_quantize(x):
    x = x.double()
    peak = torch.linalg.vector_norm(x, math.inf, dim=1)
    # The scale is kept as an fp32 number, and the codes are whole multiples of that number.
    scales = peak.div(127).to(torch.float32).double()
    return torch.div(x, scales.unsqueeze(1)).round().clamp(-127, 127), scales


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        codes, scales = _exact_quantize(s["x"])
        return torch.einsum("nd,n->nd", codes, scales), scales
    if case["op"] == "scores":
        codes, scales = _exact_quantize(s["queries"])
        # In slices of the base: a score matrix in 64 bits may be 8 GB.
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for lo in range(0, case["n"], 65_536):
            part = slice(lo, lo + 65_536)
            rows = s["codes"][part].double() * s["scales"][part].double().unsqueeze(1)
            out[:, part] = torch.matmul(codes * scales.unsqueeze(1), rows.T)
            if s["bias"] is not None:
                out[:, part].add_(s["bias"][part].double())
        return out
    q, rows, targets = s["queries"].detach().double(), s["rows"].detach().double(), s["targets"]
    used = targets.ne(IGNORE)
    count = int(used.sum()) if s["reduction"] == "mean" else 1
    losses, dq, drows = [], [], torch.zeros_like(rows)
    step = max(1, 400_000_000 // case["v"])
    for lo in range(0, case["t"], step):
        part = slice(lo, lo + step)
        logits = torch.matmul(q[part] * s["scale"], rows.T)
        if s["bias"] is not None:
            logits += s["bias"].double()
        norm = torch.logsumexp(logits, 1)
        pick = torch.arange(logits.shape[0], device="cuda")
        label = targets[part].clamp(min=0)
        losses.append((norm - logits[pick, label]) * used[part])
        if case["grad"]:
            g = torch.exp(logits.sub_(norm.unsqueeze(1)))
            g[pick, label] -= 1.0
            g.mul_((used[part].double() * (s["scale"] / count)).unsqueeze(1))
            dq.append(torch.matmul(g, rows))
            drows.addmm_(g.T, q[part])
    loss = torch.cat(losses)
    if not case["grad"]:
        return loss
    return loss.sum() / count, torch.cat(dq), drows
