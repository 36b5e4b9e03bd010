"""Cases of the 8-bit item scores and of the softmax loss over an item table.

`own` chooses between the operators' plain form in torch and the framework's kernels.  Four passes:

  quantize  rows of a table to int8 with a scale per row, and the values that the codes stand for
  scores    queries quantised, then scored against a table that is kept in int8 (products of int8, int32 sums)
  loss      softmax cross entropy of queries over every row of a table (evaluation: the loss of each query)
  step      the same with the mean over the queries and both gradients (training); targets < 0 take no part
"""
import math

import torch

own = False

MANY = 131072      # a table of 2^17 rows, where the framework's kNN starts to take its largest path
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}


def listed():
    return [
        # one search request against the 1M-row table: how fast 768 MB of codes are read
        {"name": "scores one of 1M", "op": "scores", "m": 1, "n": 1_000_000, "d": 768, "out": "f32"},
        # requests gathered for a moment, a table of 100k rows
        {"name": "scores batch of 32", "op": "scores", "m": 32, "n": 100_000, "d": 768, "out": "f32"},
        # offline: a block of the table against a large part of it
        {"name": "scores block", "op": "scores", "m": 4096, "n": MANY, "d": 768, "out": "bf16"},
        # a small table with odd sizes: latency
        {"name": "scores odd", "op": "scores", "m": 37, "n": 1500, "d": 33, "out": "f32"},
        # a table on its way into the index
        {"name": "quantize table", "op": "quantize", "n": 262_144, "d": 768, "type": "f32"},
        # the centroids of a clustering stage
        {"name": "quantize odd", "op": "quantize", "n": 5000, "d": 33, "type": "bf16"},
        # evaluation of a few queries on all 1M rows
        {"name": "loss of 16 on 1M", "op": "loss", "t": 16, "v": 1_000_000, "d": 768, "type": "bf16"},
        # evaluation of a validation set, odd sizes
        {"name": "loss odd", "op": "loss", "t": 1000, "v": 30_001, "d": 96, "type": "f32"},
        # training: the largest step
        {"name": "step large", "op": "step", "t": 4096, "v": MANY, "d": 768, "type": "bf16"},
        # training in full precision
        {"name": "step f32", "op": "step", "t": 1024, "v": 100_000, "d": 768, "type": "f32"},
        # training on clusters: few classes, odd sizes
        {"name": "step odd", "op": "step", "t": 700, "v": 1500, "d": 33, "type": "bf16"},
        # training of the small configuration, 10k x 64
        {"name": "step 10k x 64", "op": "step", "t": 256, "v": 10_000, "d": 64, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scores", "quantize", "loss", "step"])
    d = rng.choice([_log(rng, 16, 1024), 64, 96, 128, 256, 384, 768])
    if op == "quantize":
        return {"op": op, "n": _log(rng, 1000, 200_000), "d": d, "type": rng.choice(["f32", "bf16"])}
    n = _log(rng, 1000, 1_000_000 if op == "scores" else 300_000)
    rows = _log(rng, 1, 4096) if op != "step" else _log(rng, 32, 4096)
    most = 4096 * MANY // (1 if op == "scores" else 2)  # keeps every draw below the largest listed case
    rows = max(1, min(rows, most // n, most * 768 // (n * d)))
    if op == "scores":
        return {"op": op, "m": rows, "n": n, "d": d, "out": rng.choice(["f32", "bf16"]) if rows * n < 2**28 else "bf16"}
    kind = rng.choice(["f32", "bf16"])
    if kind == "f32":
        rows = max(1, min(rows, most * 96 // (n * d)))
    return {"op": op, "t": rows, "v": n, "d": d, "type": kind}


def _rows_of(d):
    """Bytes from one row of codes to the next: whole pieces of 16."""
    return (d + 15) // 16 * 16


def _unit(x):
    return x / x.norm(dim=1, keepdim=True)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, d = case["op"], case["d"]

    def normal(n):
        return torch.randn(n, d, device="cuda", generator=g)

    if op == "quantize":
        # rows of different lengths, as embeddings that nobody normalised
        x = normal(case["n"])
        x *= torch.rand(case["n"], 1, device="cuda", generator=g) + 0.5
        return {"case": case, "x": x.to(TYPES[case["type"]])}
    if op == "scores":
        codes = torch.zeros(case["n"], _rows_of(d), device="cuda", dtype=torch.int8)
        codes[:, :d] = torch.randint(-127, 128, (case["n"], d), device="cuda", generator=g, dtype=torch.int8)
        scale = (torch.rand(case["n"], device="cuda", generator=g) + 0.5) / 1000
        return {"case": case, "q": normal(case["m"]), "codes": codes, "scale": scale}
    # unit rows; a query points towards its target with as much of something else; every 16th has no target
    c = _unit(normal(case["v"]))
    t = torch.randint(0, case["v"], (case["t"],), device="cuda", generator=g)
    q = _unit(c[t] + _unit(normal(case["t"])))
    if op == "step":
        t[3::16] = -1
    kind = TYPES[case["type"]]
    return {"case": case, "q": q.to(kind), "c": c.to(kind), "t": t, "s": 20.0}


def _quantized(x):
    """Codes (as f32) and scales: scale = max|x| / 127, code = rint(x (127 / max|x|))."""
    most = x.abs().amax(1, keepdim=True)
    code = torch.round(x * (127.0 / most)).clamp(-127, 127)
    return code, (most / 127.0)[:, 0]


def _plain(state):
    case = state["case"]
    op, d = case["op"], case["d"]
    if op == "quantize":
        code, scale = _quantized(state["x"].float())
        return {"values": code * scale[:, None], "scale": scale}
    if op == "scores":
        code, scale = _quantized(state["q"])
        table = state["codes"][:, :d].float()
        # products of codes are below 2^14: sums of 1024 of them are whole in 32 bits
        total = code[:, :1024] @ table[:, :1024].T
        y = total * scale[:, None] * state["scale"]
        return y.to(TYPES[case["out"]])
    q, c, t, s = state["q"].float(), state["c"].float(), state["t"], state["s"]
    has = t >= 0
    at = t.clamp(min=0)[:, None]
    z = q @ c.T
    z *= s
    # the sum over the others apart from the target's logit: a loss near 0 is their share, and not a difference of two
    own_z = z.gather(1, at)
    z.scatter_(1, at, torch.where(has[:, None], -math.inf, own_z))
    most = z.amax(1, keepdim=True).clamp(min=-3e38)
    rest = (z - most).exp_().sum(1, keepdim=True).log() + most
    x = rest - own_z
    soft = x.clamp(min=0) + (-x.abs()).exp().log1p()
    loss = torch.where(has, soft[:, 0], 0.0)
    if op == "loss":
        return loss
    count = has.sum().clamp(min=1)
    lse = own_z + soft
    z = z.sub_(lse).exp_()
    z.scatter_(1, at, -(rest - lse).exp())
    z *= (has / count)[:, None]
    return {"loss": loss.sum() / count, "dq": ((z @ c) * s).to(state["q"].dtype), "dc": ((z.T @ q) * s).to(state["c"].dtype)}


def _framework(state):
    import sys

    if "matternet-rs_amd" not in sys.path:
        sys.path.insert(0, "matternet-rs_amd")
    import surfface_hip as S

    case = state["case"]
    if case["op"] == "quantize":
        rows = S.quantize_rows(state["x"])
        return {"values": S.dequantize_rows(rows), "scale": rows.scale}
    if case["op"] == "scores":
        table = S.Int8Rows(state["codes"], state["scale"], case["d"])
        return S.scores_i8(S.quantize_rows(state["q"]), table, dtype=TYPES[case["out"]])
    if case["op"] == "loss":
        return S.softmax_loss(state["q"], state["c"], state["t"], scale=state["s"], reduction="none")
    q, c = state["q"].detach().requires_grad_(), state["c"].detach().requires_grad_()
    loss = S.softmax_loss(q, c, state["t"], scale=state["s"])
    dq, dc = torch.autograd.grad(loss, (q, c))
    return {"loss": loss.detach(), "dq": dq, "dc": dc}


def run(state):
    return _framework(state) if own else _plain(state)


def work(case):
    d = case["d"]
    if case["op"] == "quantize":
        n = case["n"]
        return {"bytes": n * d * (BYTES[case["type"]] + 1 + 4) + 4 * n, "flops": 3 * n * d}
    if case["op"] == "scores":
        m, n = case["m"], case["n"]
        return {"bytes": 4 * m * d + n * (d + 4) + m * n * BYTES[case["out"]], "flops": 2 * m * n * d}
    t, v, size = case["t"], case["v"], BYTES[case["type"]]
    if case["op"] == "loss":
        return {"bytes": (t + v) * d * size + 12 * t, "flops": 2 * t * v * d}
    # the logits once for the loss and, as they are not kept, once more for the gradients; dQ and dC
    return {"bytes": 2 * (t + v) * d * size + 8 * t, "flops": 8 * t * v * d}


def exact(case, seed):
    state = prepare(case, seed)
    d = case["d"]
    if case["op"] == "quantize":
        # which of two codes a value next to a border gets is a matter of the 32-bit formula
        return {"values": None, "scale": state["x"].double().abs().max(dim=1).values / 127}
    if case["op"] == "scores":
        x = state["q"]
        top = x.abs().max(dim=1).values
        codes = torch.round(x * (127.0 / top)[:, None]).double()
        step = top.double() / 127
        y = torch.empty(case["m"], case["n"], device="cuda", dtype=torch.float64)
        for k in range(0, case["n"], 65536):
            part = slice(k, k + 65536)
            y[:, part] = step[:, None] * state["scale"][part].double() * torch.mm(codes, state["codes"][part, :d].double().t().contiguous())
        return y
    q, c, t = state["q"].double(), state["c"].double(), state["t"]
    valid = (t >= 0).nonzero()[:, 0]
    loss = torch.zeros(case["t"], device="cuda", dtype=torch.float64)
    dq, dc = torch.zeros_like(q), torch.zeros_like(c)
    some = max(1, 2**26 // case["v"])
    for k in range(0, len(valid), some):
        rows = valid[k:k + some]
        z = torch.mm(q[rows], c.t().contiguous()) * state["s"]
        p = torch.softmax(z, dim=1)
        at = (torch.arange(len(rows), device="cuda"), t[rows])
        loss[rows] = torch.logsumexp(z, dim=1) - z[at]
        if case["op"] == "step":
            p[at] -= 1.0
            p *= state["s"] / len(valid)
            dq[rows] = torch.mm(p, c)
            dc += torch.mm(p.t().contiguous(), q[rows])
    if case["op"] == "loss":
        return loss
    return {"loss": loss.sum() / max(1, len(valid)), "dq": dq, "dc": dc}
