"""What is measured of the 8-bit and grouped operators: the cases, their inputs, their plain form in elementary torch
operations and what each has to move and compute.

Four operators, as one block of tokens (or of a frame's feature pixels) goes through them:
  norm     rms_norm_fp8: residual addition, root-mean-square norm, output in e4m3 with a scale per row and 128 columns
  gate     silu_mul_fp8: silu(gate) * up, output in e4m3 with a scale per row and 128 columns
  product  matmul_fp8: e4m3 rows times e4m3 weights, a scale per (row, 128 of K) and per (128 of N, 128 of K)
  grouped  grouped_matmul_fp8 / grouped_matmul: the same with one weight matrix per expert and ragged row groups
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
LEAST = 2.0 ** -100          # a block's largest magnitude counts as at least this, so that its scale is a normal number
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through a block's norm: latency
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 2048, "type": "bf16", "residual": True},
        # a 1024 x 512 frame's feature grid (65 x 129 pixels of 2048 channels): bandwidth
        {"name": "norm a frame's pixels", "op": "norm", "rows": 8385, "cols": 2048, "type": "bf16", "residual": True},
        # a first norm without residual, in 32 bits, of a width that ends inside a block of 128
        {"name": "norm odd width fp32", "op": "norm", "rows": 4099, "cols": 1000, "type": "fp32", "residual": False},
        # a decode batch between the two products of a gated block
        {"name": "gate decode batch", "op": "gate", "rows": 16, "cols": 4096, "type": "bf16"},
        # a frame's pixels between the two products
        {"name": "gate a frame's pixels", "op": "gate", "rows": 8385, "cols": 4096, "type": "bf16"},
        # one token times one weight matrix: the weights' bytes
        {"name": "product one token", "op": "product", "rows": 1, "cols": 4096, "inner": 2048, "out": "bf16"},
        # a small odd batch against a long inner size
        {"name": "product small batch", "op": "product", "rows": 33, "cols": 2048, "inner": 8192, "out": "bf16"},
        # nothing is a multiple of a tile: rows, columns and an inner size that ends inside a block of 128; 32-bit output
        {"name": "product ragged fp32 out", "op": "product", "rows": 517, "cols": 1001, "inner": 2056, "out": "fp32"},
        # a prompt of 8192 tokens, wide layer: matrix rate
        {"name": "product long prompt", "op": "product", "rows": 8192, "cols": 8192, "inner": 8192, "out": "bf16"},
        # one token's 8 experts of 64: the chosen experts' weights once
        {"name": "grouped one token", "op": "grouped", "tokens": 1, "topk": 8, "experts": 64, "cols": 2048, "inner": 2048, "type": "fp8", "gather": True, "skew": 1.0},
        # a prompt routed unevenly over 32 experts, rows gathered by token
        {"name": "grouped long prompt", "op": "grouped", "tokens": 8192, "topk": 2, "experts": 32, "cols": 4096, "inner": 2048, "type": "fp8", "gather": True, "skew": 1.0},
        # the same kind of work on 16-bit weights, odd counts, rows already in order
        {"name": "grouped odd bf16", "op": "grouped", "tokens": 2741, "topk": 2, "experts": 16, "cols": 1000, "inner": 2048, "type": "bf16", "gather": False, "skew": 0.5},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size over its logarithm: one in three as it falls (odd ones among them), the others multiples of 64."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 1 / 3 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(["norm", "gate", "product", "product", "grouped", "grouped"])
    if op in ("norm", "gate"):
        case = {"op": op, "rows": _log(rng, 1, 16384), "cols": _size(rng, 64, 8192), "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
        if op == "norm":
            case["residual"] = rng.random() < 2 / 3
        case["rows"] = min(case["rows"], (1 << 26) // case["cols"])
        return case
    if op == "product":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _size(rng, 64, 8192), "inner": _size(rng, 64, 8192),
                "out": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    experts = _log(rng, 2, 64)
    case = {"op": op, "tokens": _log(rng, 1, 8192), "topk": rng.randint(1, min(8, experts)), "experts": experts,
            "cols": _size(rng, 64, 4096), "inner": _size(rng, 64, 4096) // 8 * 8, "type": rng.choice(["fp8", "fp8", "bf16", "fp16"]),
            "gather": rng.random() < 0.5, "skew": rng.choice([0.0, 0.5, 1.0])}
    case["tokens"] = min(case["tokens"], max(1, 16384 // case["topk"]))
    return case


# --------------------------------------------------------------------------------------------------------------- inputs
def _pad16(n):
    return -(-n // 16) * 16


def _activations(g, rows, cols):
    """Rows of normal values whose channels differ in size, a few of them by much, as a model's do."""
    size = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    size = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, 20 * size, size)
    return torch.randn(rows, cols, generator=g, device="cuda") * size


def _e4m3(v):
    """e4m3 values in rows whose stride is a multiple of 16 bytes (the columns behind the last are zero)."""
    q = torch.zeros(*v.shape[:-1], _pad16(v.shape[-1]), dtype=torch.float8_e4m3fn, device=v.device)
    q[..., : v.shape[-1]] = v.to(torch.float8_e4m3fn)
    return q[..., : v.shape[-1]]


def _held_rows(v):
    """Rows held in 8 bits with a scale per row and 128 columns; the scales of one block of columns lie side by side."""
    rows, cols = v.shape
    nb = -(-cols // BLOCK)
    s = torch.nn.functional.pad(v, (0, nb * BLOCK - cols)).view(rows, nb, BLOCK).abs().amax(2).clamp_min(LEAST) / E4M3_MAX
    q = _e4m3(v / s.repeat_interleave(BLOCK, 1)[:, :cols])
    return q, s.t().contiguous().t()


def _held_weights(v):
    """Weight matrices [..., N, K] held in 8 bits with a scale per 128 x 128 block."""
    n, k = v.shape[-2:]
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    p = torch.nn.functional.pad(v, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(*v.shape[:-2], nb, BLOCK, kb, BLOCK)
    s = p.abs().amax((-3, -1)).clamp_min(LEAST) / E4M3_MAX
    q = (p / s[..., :, None, :, None]).reshape(*v.shape[:-2], nb * BLOCK, kb * BLOCK)[..., :n, :k]
    return _e4m3(q), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = {"op": op, "case": case}
    if op == "norm":
        t = TYPES[case["type"]]
        state["x"] = _activations(g, case["rows"], case["cols"]).to(t)
        state["residual"] = (4 * _activations(g, case["rows"], case["cols"])).to(t) if case["residual"] else None
        state["weight"] = (1 + 0.2 * torch.randn(case["cols"], generator=g, device="cuda")).to(t)
    elif op == "gate":
        state["x"] = _activations(g, case["rows"], 2 * case["cols"]).to(TYPES[case["type"]])
    elif op == "product":
        state["xq"], state["xs"] = _held_rows(_activations(g, case["rows"], case["inner"]))
        state["wq"], state["ws"] = _held_weights(torch.randn(case["cols"], case["inner"], generator=g, device="cuda") / math.sqrt(case["inner"]))
        state["out_dtype"] = TYPES[case["out"]]
    else:
        experts, tokens, topk = case["experts"], case["tokens"], case["topk"]
        liked = case["skew"] * torch.randn(experts, generator=g, device="cuda")
        chosen = (torch.randn(tokens, experts, generator=g, device="cuda") + liked).topk(topk, 1).indices.reshape(-1)
        order = torch.sort(chosen, stable=True).indices
        counts = torch.bincount(chosen, minlength=experts)
        state["offsets"] = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
        state["rows"] = (order // topk).to(torch.int32) if case["gather"] else None
        state["longest"] = int(counts.max())
        x = _activations(g, tokens if case["gather"] else tokens * topk, case["inner"])
        w = torch.randn(experts, case["cols"], case["inner"], generator=g, device="cuda") / math.sqrt(case["inner"])
        if case["type"] == "fp8":
            state["xq"], state["xs"] = _held_rows(x)
            state["wq"], state["ws"] = _held_weights(w)
        else:
            state["x"], state["w"] = x.to(TYPES[case["type"]]), w.to(TYPES[case["type"]])
    return state


# ----------------------------------------------------------------------------------------------------------- plain form
def _quantised(y):
    rows, cols = y.shape
    nb = -(-cols // BLOCK)
    s = torch.nn.functional.pad(y, (0, nb * BLOCK - cols)).view(rows, nb, BLOCK).abs().amax(2).clamp_min(LEAST) / E4M3_MAX
    return (y / s.repeat_interleave(BLOCK, 1)[:, :cols]).to(torch.float8_e4m3fn), s


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].float()
    q, scale = _quantised(y)
    return [q, scale] if s["residual"] is None else [q, scale, h.to(s["x"].dtype)]


def _plain_gate(s):
    gate, up = s["x"].float().chunk(2, 1)
    return list(_quantised(gate / (1 + torch.exp(-gate)) * up))


def _values_of_rows(q, s):
    return q.float() * s.repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _values_of_weights(q, s):
    n, k = q.shape[-2:]
    return q.float() * s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _plain_product(s):
    return [(_values_of_rows(s["xq"], s["xs"]) @ _values_of_weights(s["wq"], s["ws"]).t()).to(s["out_dtype"])]


def _plain_grouped(s):
    off = s["offsets"].long()
    row = torch.arange(s["case"]["tokens"] * s["case"]["topk"], device=off.device)
    expert = torch.searchsorted(off, row, right=True) - 1
    few = len(row) <= s["case"]["experts"]      # then each row takes a copy of its expert's matrix
    if "xq" in s:
        wq, ws = (s["wq"].view(torch.uint8)[expert].view(torch.float8_e4m3fn), s["ws"][expert]) if few else (s["wq"], s["ws"])
        x, w, out = _values_of_rows(s["xq"], s["xs"]), _values_of_weights(wq, ws), torch.bfloat16
    else:
        x, w, out = s["x"].float(), (s["w"][expert] if few else s["w"]).float(), s["x"].dtype
    if s["rows"] is not None:
        x = x[s["rows"].long()]
    if few:
        return [torch.bmm(x[:, None], w.transpose(1, 2).contiguous())[:, 0].to(out)]
    # every expert's rows side by side, as many places as the longest group needs, one batched product
    place = row - off[expert]
    held = x.new_zeros(w.shape[0], s["longest"], x.shape[1])
    held[expert, place] = x
    return [torch.bmm(held, w.transpose(1, 2).contiguous())[expert, place].to(out)]


def run(state):
    if own:
        from diga_amd import matmul as M
        op = state["op"]
        if op == "norm":
            q, scale, h = M.rms_norm_fp8(state["x"], state["weight"], state["residual"], EPS)
            return [q, scale] if h is None else [q, scale, h]
        if op == "gate":
            return list(M.silu_mul_fp8(state["x"]))
        if op == "product":
            return [M.matmul_fp8(state["xq"], state["xs"], state["wq"], state["ws"], state["out_dtype"])]
        if "xq" in state:
            return [M.grouped_matmul_fp8(state["xq"], state["xs"], state["wq"], state["ws"], state["offsets"], state["rows"])]
        return [M.grouped_matmul(state["x"], state["w"], state["offsets"], state["rows"])]
    return {"norm": _plain_norm, "gate": _plain_gate, "product": _plain_product, "grouped": _plain_grouped}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_blocks(y):
    """y over its blocks' scales, unrounded, and the scales."""
    scale = torch.stack([b.abs().max(1).values.clamp(min=LEAST) / E4M3_MAX for b in y.split(BLOCK, 1)], 1)
    return torch.cat([b / scale[:, i : i + 1] for i, b in enumerate(y.split(BLOCK, 1))], 1), scale


def _exact_product(x, xs, w, ws):
    """Block by block of the inner size: the sum of products, then its two scales."""
    total = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    row = torch.arange(w.shape[0], device=x.device) // BLOCK
    for b in range(xs.shape[1]):
        part = x[:, b * BLOCK : (b + 1) * BLOCK].double() @ w[:, b * BLOCK : (b + 1) * BLOCK].double().t()
        total += part * xs[:, b : b + 1].double() * ws[row, b].double()
    return total


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        y = s["weight"].double() * (h / (h.square().sum(1, keepdim=True) / h.shape[1] + EPS).sqrt())
        return list(_exact_blocks(y)) + ([] if s["residual"] is None else [h])
    if s["op"] == "gate":
        n = case["cols"]
        x = s["x"].double()
        return list(_exact_blocks(x[:, :n] * torch.sigmoid(x[:, :n]) * x[:, n:]))
    if s["op"] == "product":
        return [_exact_product(s["xq"], s["xs"], s["wq"], s["ws"])]
    off = s["offsets"].tolist()
    of = s["rows"].long() if s["rows"] is not None else torch.arange(off[-1], device="cuda")
    parts = []
    for e in range(case["experts"]):
        i = of[off[e] : off[e + 1]]
        if "xq" in s:
            parts.append(_exact_product(s["xq"].view(torch.uint8)[i].view(torch.float8_e4m3fn), s["xs"][i], s["wq"][e], s["ws"][e]))
        else:
            parts.append(s["x"][i].double() @ s["w"][e].double().t())
    return [torch.cat(parts)]


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("norm", "gate"):
        n, c = case["rows"], case["cols"]
        size = TYPES[case["type"]].itemsize
        out = n * c + 4 * n * -(-c // BLOCK)
        if op == "gate":
            return {"bytes": 2 * n * c * size + out, "flops": 8 * n * c}
        return {"bytes": n * c * size * (3 if case["residual"] else 1) + c * size + out, "flops": 8 * n * c}
    if op == "product":
        m, n, k = case["rows"], case["cols"], case["inner"]
        kb = -(-k // BLOCK)
        return {"bytes": m * k + n * k + 4 * kb * (m + -(-n // BLOCK)) + m * n * TYPES[case["out"]].itemsize, "flops": 2 * m * n * k}
    t, n, k = case["tokens"] * case["topk"], case["cols"], case["inner"]
    size = 1 if case["type"] == "fp8" else 2
    used = min(case["experts"], t)        # experts that get a row
    read = (case["tokens"] if case["gather"] else t) * k * size + used * n * k * size
    if size == 1:
        read += 4 * -(-k // BLOCK) * ((case["tokens"] if case["gather"] else t) + used * -(-n // BLOCK))
    return {"bytes": read + t * n * 2 + 4 * (case["experts"] + 1) + (4 * t if case["gather"] else 0), "flops": 2 * t * n * k}
